// Attention of a batch whose sequences share long prefixes (sm_100a).
//
//   out = sum_j p_j v_j,  p = softmax_j(scale * q . k_j)
//
// over a sequence's prefix and its own keys, one pass over the keys with the running
// maximum m and sum l of the softmax:
//   m' = max(m, max s),  p = 2^(s - m'),  l' = l 2^(m - m') + sum p,  O' = O 2^(m - m') + p V
// (s in units of log2).  Parts of the keys computed apart are joined by the same rule.
//
// A work item is a tile of 128 query rows (or 2 of 128, where head size and rows allow) of
// one key/value head, and a range of keys, 64 at a time.  There are three ways to make tiles:
//   * by sequence: the rows (token, query head of the group) of one sequence against its
//     prefix and then its own keys.
//   * stacked: for the prefix, the rows of all sequences that share it are stacked, so a
//     prefix is read once for the batch and not once per sequence; each sequence's own
//     keys are a further item, and the parts are joined by a second kernel.  For few
//     query rows, whose own keys need the tiles' rows for little: 32 single tokens behind
//     4 x 4096, 8 heads on one of 256: 50 us, 148 us by sequence.
//   * mixed: stacked tiles that go through the prefix and then through the own keys of
//     each of their sequences, the product with V writing that sequence's rows alone.
//     For tiles of few sequences, when there are tiles enough: no parts to join.  16
//     prefixes of 304 x 8 sequences of 50 tokens: 39 us, 46 us by sequence.
// In the first two the key range is split over more items when tiles are few.  No value
// of one request enters another's sums, not even multiplied by zero.
//
// One item per CTA:
//   softmax warps   8 per 128 rows, two threads a row (32 keys of a block each): scores from
//                   tensor memory to registers, mask, maximum, exponentials, sum; p (16
//                   bit) back to tensor memory
//   one warp        TMA producer: a ring of 128-byte-swizzled tiles, a stage holding K of
//                   one block and V of the one two before it, the two used together
//   one warp a tile tcgen05.mma issuer: S = Q K^T (both operands in shared memory),
//                   O += P V (P in tensor memory, V as the MN-major operand)
// S of the next block is computed while this block's softmax runs (two score buffers a
// row tile).  O is rescaled only when the maximum has grown by more than 2^8 since the
// last time: until then p stays below 2^8, and l and O carry the same factor.  fp16 has 5
// exponent bits: its p, l and O carry a further 2^7 (p below 2^15), so that a long tail of
// keys far below the maximum is weighed down to 2^-32 of it, not to 2^-25.
//
// p is rounded to the operands' 16 bits for the product with V (l sums the unrounded
// ones), which adds about as much error as the rounding of the output itself: 2.2-2.3e-3
// of its norm in bf16 where that alone is 1.7e-3, 2.6e-4 and 2.1e-4 in fp16.  p as two
// 16-bit parts, in the place of the fp32 scores, brings that down to the output's rounding
// for a second product and the splitting: 4 x 50 tokens 13.2 us for 11.8, 16 x 8 x 50 48.8
// for 44.1, 32 single tokens behind 32768 57 for 50, 16 x 56 behind 2 histories 233 for
// 159.  Not taken: it costs more than the bits that the output can hold are worth.
//
// Bounds: at head sizes up to 128 a block of 64 keys asks 128 rows x 64 exponentials of
// each tile, as long as its products; with the softmax's latency between the two products
// the main loop holds 76% of the measured matrix rate at a head size of 256 (0.99 us a
// block of keys for 128 rows), 64% at 128 (1.17 us for 256 rows), 44% at 64 (0.86 us);
// launch, start and end of a CTA are 8 us beside that (148 tiles behind one prefix of 2048
// to 8192).  16 x 56 tokens, 32 heads of 128 behind 2 histories of up to 8192: 159 us where
// the tiles fit one wave, up to 214 us where unevenly shared histories leave a second one;
// their products alone 41-55 us.  Small calls are launch, prologue and join: one sequence
// of 50 tokens 11 us.
#include "serving.cuh"

namespace actune {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.f;  // growth of the maximum (log2) that O is rescaled for
constexpr int kSiteAttn = 300;
template <typename T>
constexpr float kRoom = std::is_same<T, __half>::value ? 7.f : 0.f;  // log2 of what p, l and O carry

// Tiles by sequence; stacked tiles for the prefix and tiles by sequence for the own keys;
// stacked tiles for both.
enum : int { kBySequence = 0, kStacked = 1, kMixed = 2 };
constexpr int kMixedSeqs = 16;  // sequences that a mixed tile may touch

// n / d for 0 <= n < 2^31 by multiplication: an item's place in the grid and a row's
// place in its sequence are several divisions deep before the first load can start.
struct Divisor {
  uint32_t d, mul, shift;
  void set(int64_t by) {
    d = (uint32_t)by, shift = 0;
    while (((uint64_t)1 << shift) < d) ++shift;
    mul = (uint32_t)((((uint64_t)1 << 32) * (((uint64_t)1 << shift) - d)) / d + 1);
  }
  __device__ __forceinline__ int div(int n) const { return (int)((__umulhi((uint32_t)n, mul) + (uint32_t)n) >> shift); }
  // n -> n / d, the remainder returned.
  __device__ __forceinline__ int split(int& n) const {
    const int q = div(n), r = n - q * (int)d;
    n = q;
    return r;
  }
};

struct AttnParams {
  const void *q, *pk, *pv, *k, *v;
  const int32_t *starts, *prefix_lens, *lens;
  void* out;
  float* o_part;  // [splits, rows, D]
  float2* ml;     // [splits, rows]: m (log2 units), l
  int64_t q_b, q_t, q_h, pk_g, pk_p, pk_h, pv_g, pv_p, pv_h, k_b, k_s, k_h, v_b, v_s, v_h;
  int B, T, H, KV, D, G, P, S;
  int rep;          // query heads per key/value head
  int causal;
  float scale;      // scale * log2(e)
  int tiles_per_seq;
  int kind;         // how tiles are made: kBySequence, kStacked or kMixed
  int prefix_tiles; // upper bound on the stacked tiles of a key/value head
  int prefix_splits, own_splits;  // by sequence: prefix_splits of both together
  int splits;       // parts per row; 1: write out directly
  int q_boxes;      // query tiles come by tensor map (tokens evenly spaced, rep a divisor of 128)
  Divisor by_full_tiles, by_prefixes, by_kv, by_own_tiles, by_tiles_per_seq, by_per_seq, by_rep, by_prefix_splits, by_own_splits;
};

__device__ __forceinline__ int clamp_len(const int32_t* lens, int i, int most) {
  return lens == nullptr ? most : max(0, min(lens[i], most));
}

// ------------------------------------------------------------------ any layout
// One CTA per query row; a warp takes every fourth key, a lane every 32nd element.
template <typename T>
__global__ void __launch_bounds__(128) prefix_attention_any_kernel(const AttnParams p) {
  __shared__ float part_o[4][256];
  __shared__ float2 part_ml[4];
  griddep_enter();
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t row = blockIdx.x;
  const int h = (int)(row % p.H), t = (int)(row / p.H % p.T), b = (int)(row / p.H / p.T);
  const int kv = h / p.rep;
  int g = (int)((int64_t)b * p.G / p.B);
  if (p.starts != nullptr) {
    g = 0;
    for (int i = 1; i < p.G; ++i) g += p.starts[i] <= b;
  }
  const int plen = clamp_len(p.prefix_lens, g, p.P), slen = clamp_len(p.lens, b, p.S);
  const int own = p.causal ? max(0, min(slen, slen - p.T + t + 1)) : slen;
  const T* q = reinterpret_cast<const T*>(p.q) + b * p.q_b + t * p.q_t + h * p.q_h;
  float qv[8], o[8] = {};
#pragma unroll
  for (int i = 0; i < 8; ++i) qv[i] = lane + 32 * i < p.D ? widen<T>(q[lane + 32 * i]) : 0.f;
  float m = -INFINITY, l = 0.f;
  const int64_t keys = (int64_t)plen + own;
  for (int64_t j = warp; j < keys; j += 4) {
    const T *key, *value;
    if (j < plen) {
      key = reinterpret_cast<const T*>(p.pk) + g * p.pk_g + j * p.pk_p + kv * p.pk_h;
      value = reinterpret_cast<const T*>(p.pv) + g * p.pv_g + j * p.pv_p + kv * p.pv_h;
    } else {
      key = reinterpret_cast<const T*>(p.k) + b * p.k_b + (j - plen) * p.k_s + kv * p.k_h;
      value = reinterpret_cast<const T*>(p.v) + b * p.v_b + (j - plen) * p.v_s + kv * p.v_h;
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < p.D) s = fmaf(qv[i], widen<T>(key[lane + 32 * i]), s);
#pragma unroll
    for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
    s *= p.scale;
    const float top = fmaxf(m, s), ref = top == -INFINITY ? 0.f : top;
    const float grow = exp2f(m - ref), e = exp2f(s - ref);
    l = fmaf(l, grow, e);
#pragma unroll
    for (int i = 0; i < 8; ++i)
      if (lane + 32 * i < p.D) o[i] = fmaf(o[i], grow, e * widen<T>(value[lane + 32 * i]));
    m = top;
  }
#pragma unroll
  for (int i = 0; i < 8; ++i) part_o[warp][lane + 32 * i] = o[i];
  if (lane == 0) part_ml[warp] = make_float2(m, l);
  __syncthreads();
  float top = -INFINITY, total = 0.f;
#pragma unroll
  for (int w = 0; w < 4; ++w) top = fmaxf(top, part_ml[w].x);
  float weight[4];
#pragma unroll
  for (int w = 0; w < 4; ++w) {
    weight[w] = part_ml[w].y == 0.f ? 0.f : exp2f(part_ml[w].x - top);
    total += weight[w] * part_ml[w].y;
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  for (int d = threadIdx.x; d < p.D; d += 128) {
    float a = 0.f;
#pragma unroll
    for (int w = 0; w < 4; ++w)
      if (weight[w] != 0.f) a = fmaf(weight[w], part_o[w][d], a);
    reinterpret_cast<T*>(p.out)[row * p.D + d] = narrow<T>(a * inv);
  }
}

// ------------------------------------------------------------------ tensor cores
__device__ __forceinline__ void mma16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}

// The same, leaving the accumulator's rows whose bit of `off` is set as they are.
__device__ __forceinline__ void mma16_ts_rows(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc,
                                              const uint32_t (&off)[4]) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %6, %7, %8}, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc), "r"(off[0]), "r"(off[1]), "r"(off[2]), "r"(off[3])
      : "memory");
}

// MN-major operand in 128-byte-swizzled tiles of 64 columns x `rows` rows (128 bytes a
// row, 8-row atoms of 1024 bytes): LBO = the next 64 columns, SBO = the next 8 rows.
__device__ __forceinline__ uint64_t smem_desc_mn_sw128(uint32_t saddr, uint32_t rows) {
  return (uint64_t)((saddr >> 4) & 0x3FFFu) | ((uint64_t)(rows * 128u >> 4) << 16) | ((uint64_t)(1024u >> 4) << 32) |
         ((uint64_t)1u << 46) | ((uint64_t)2u << 61);
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]),
      "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]),
      "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}

__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
      "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

__device__ __forceinline__ void tmem_wait_ld16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// DP: the head size rounded up to 64, 128 or 256 (the rest of a row is zeros).
// NT: row tiles of 128 per CTA.
template <int DP, int NT>
struct AttnCfg {
  static constexpr int BN = 64;  // keys per block
  static constexpr int NB = 2;   // score buffers per tile: the next block's are computed ahead
  static constexpr int ROWS = 128 * NT;
  static constexpr int Q_BYTES = ROWS * DP * 2;
  static constexpr int SLOT_BYTES = BN * DP * 2;        // one K or V block
  static constexpr int STAGE_BYTES = 2 * SLOT_BYTES;    // K of a block and V of the one NB before it
  static constexpr int FIT = (226 * 1024 - 512 - NT * 1024 - Q_BYTES) / STAGE_BYTES;  // beside the static arrays
  static constexpr int RING = FIT > 6 ? 6 : FIT;
  static constexpr int SMEM = 1024 + Q_BYTES + RING * STAGE_BYTES;
  static constexpr int O_COL = 0, S_COL = NT * DP;      // tensor memory columns: O, then the score buffers
  static constexpr int TMEM_COLS = 512;
  static constexpr int WARPS = 8 * NT + 1 + NT;         // softmax, producer, issuers
  static_assert(S_COL + NT * NB * BN <= TMEM_COLS && RING >= 2 && SMEM + NT * 1024 + 512 <= 227 * 1024, "fits");
};

// A mixed tile's sequences seq0 .. seq0 + count - 1 (those with rows in it), by index.
struct TileSeqs {
  int count;
  int row[kMixedSeqs + 1];    // first row in the tile; the last entry is the end
  int block[kMixedSeqs + 1];  // first of the sequence's own blocks, counted over the tile's
  int len[kMixedSeqs];        // own keys
};

struct AttnItem {
  int nrows;         // rows of the tile; 0: nothing to do
  int row0;          // first row, counted from sequence seq0: ((b - seq0) * T + t) * rep + r
  int seq0, g, b;    // b: the sequence of the own-key blocks
  int kv, split;
  int plen, slen;
  int pb0, pb1, sb0, sb1;  // blocks of the prefix and of the sequence's own keys
};

// What the CTA works on; by one warp.
template <int BN, int ROWS, bool MIXED>
__device__ AttnItem attn_item(const AttnParams& p, int lane, TileSeqs& seqs) {
  AttnItem it = {};
  const int per_seq = p.T * p.rep;
  int x = blockIdx.x;
  // Full tiles first: the last one of each prefix may have few rows, and fills the gaps.
  const int full_items = p.kind != kBySequence ? (p.prefix_tiles - p.G) * p.KV * p.prefix_splits : 0;
  const int prefix_items = p.kind != kBySequence ? p.prefix_tiles * p.KV * p.prefix_splits : 0;
  // Part `i` of `blocks` blocks dealt to d.d parts: [begin, end).
  const auto deal = [](int blocks, const Divisor& d, int i, int& begin, int& end) {
    int each = blocks;
    const int more = d.split(each);  // that many parts get one more
    begin = i * each + min(i, more);
    end = begin + each + (i < more);
  };
  if (x < prefix_items) {
    const bool full = x < full_items;
    if (!full) x -= full_items;
    const int tile = full ? p.by_full_tiles.split(x) : p.by_prefixes.split(x);
    it.kv = p.by_kv.split(x), it.split = x;
    // The prefix whose stacked rows hold this tile: running count of tiles, 32 prefixes a step.
    int before = 0;
    bool found = false;
    for (int base = 0; base < p.G && !found; base += 32) {
      const int g = base + lane;
      int s0 = 0, s1 = 0;
      if (g < p.G) {
        if (p.starts != nullptr) {
          s0 = g == 0 ? 0 : max(0, min(p.starts[g], p.B));
          s1 = g == p.G - 1 ? p.B : max(s0, min(p.starts[g + 1], p.B));
        } else {  // sequences b with b * G / B == g
          s0 = (int)(((int64_t)g * p.B + p.G - 1) / p.G);
          s1 = (int)(((int64_t)(g + 1) * p.B + p.G - 1) / p.G);
        }
      }
      const int rows = (s1 - s0) * per_seq, mine = full ? rows / ROWS : rows % ROWS != 0;
      int upto = mine;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += a;
      }
      const unsigned hit = __ballot_sync(0xffffffffu, before + upto > tile);
      if (hit != 0) {
        const int src = __ffs(hit) - 1;
        const int first = before + upto - mine;
        it.g = base + src;
        it.seq0 = __shfl_sync(0xffffffffu, s0, src);
        const int all = __shfl_sync(0xffffffffu, rows, src);
        it.row0 = full ? (tile - __shfl_sync(0xffffffffu, first, src)) * ROWS : all / ROWS * ROWS;
        it.nrows = min(ROWS, all - it.row0);
        found = true;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (!found) return it;
    it.b = it.seq0;
    it.plen = clamp_len(p.prefix_lens, it.g, p.P);
    if constexpr (MIXED) {
      // The tile's first sequence becomes seq0, and a lane works out each sequence's share.
      const int skip = p.by_per_seq.div(it.row0);
      it.seq0 += skip, it.b = it.seq0, it.row0 -= skip * per_seq;
      const int count = p.by_per_seq.div(it.row0 + it.nrows - 1) + 1;
      int blocks = 0, len = 0, begin = it.nrows;
      if (lane < count) {
        len = clamp_len(p.lens, it.seq0 + lane, p.S);
        begin = max(0, lane * per_seq - it.row0);
        int seen = len;  // by the sequence's last row in the tile
        if (p.causal) {
          const int last = min((lane + 1) * per_seq, it.row0 + it.nrows) - 1 - lane * per_seq;
          seen = max(0, min(len, len - p.T + p.by_rep.div(last) + 1));
        }
        blocks = (seen + BN - 1) / BN;
      }
      int upto = blocks;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += a;
      }
      if (lane == 0) seqs.count = count;
      if (lane <= count && lane <= kMixedSeqs) seqs.row[lane] = begin, seqs.block[lane] = upto - blocks;
      if (lane < count && lane < kMixedSeqs) seqs.len[lane] = len;
      it.pb1 = (it.plen + BN - 1) / BN;
      it.sb1 = __shfl_sync(0xffffffffu, upto, 31);
      return it;
    }
    deal((it.plen + BN - 1) / BN, p.by_prefix_splits, it.split, it.pb0, it.pb1);
    return it;
  }
  x -= prefix_items;
  int tile = p.by_own_tiles.split(x);
  it.kv = p.by_kv.split(x);
  const int part = x;
  it.row0 = p.by_tiles_per_seq.split(tile) * ROWS;
  it.b = it.seq0 = tile;
  it.nrows = min(ROWS, per_seq - it.row0);
  it.slen = clamp_len(p.lens, it.b, p.S);
  int seen = it.slen;  // own keys that the tile's last row sees
  if (p.causal) seen = max(0, min(seen, it.slen - p.T + p.by_rep.div(it.row0 + it.nrows - 1) + 1));
  const int own = (seen + BN - 1) / BN;
  if (p.kind == kStacked) {
    it.split = p.prefix_splits + part;
    deal(own, p.by_own_splits, part, it.sb0, it.sb1);
    return it;
  }
  it.split = part;
  int g = 0;
  if (p.starts != nullptr) {
    for (int i = 1 + lane; i < p.G; i += 32) g += p.starts[i] <= it.b;
    g = __reduce_add_sync(0xffffffffu, g);
  } else if (p.G > 1) {
    g = (int)((int64_t)it.b * p.G / p.B);
  }
  it.g = g;
  it.plen = clamp_len(p.prefix_lens, g, p.P);
  const int prefix = (it.plen + BN - 1) / BN;
  int c0, c1;  // of the prefix's blocks and then the own ones
  deal(prefix + own, p.by_prefix_splits, part, c0, c1);
  it.pb0 = min(c0, prefix), it.pb1 = min(c1, prefix);
  it.sb0 = max(0, c0 - prefix), it.sb1 = max(0, c1 - prefix);
  return it;
}

// (MIXED a parameter of the kernel: carried along, its tests cost the others 2-4%.)
template <typename T, int DP, int NT, bool MIXED>
__global__ void __launch_bounds__(AttnCfg<DP, NT>::WARPS * 32, 1)
    prefix_attention_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_pk, const __grid_constant__ CUtensorMap tm_pv,
                            const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                            const AttnParams p) {
  using C = AttnCfg<DP, NT>;
  constexpr int BN = C::BN, NB = C::NB, RING = C::RING;
  extern __shared__ uint8_t smem_raw[];
  // step[t][i % NB], completed once per block i: the scores of block i are there, and O
  // holds the blocks up to i - NB.  NB further steps follow the last block's.
  __shared__ __align__(8) uint64_t full[RING], empty[RING], step[NT][NB], p_ready[NT][NB], drained[NT], q_full[NT];
  __shared__ uint32_t tmem_holder;
  __shared__ AttnItem item_sh;
  __shared__ TileSeqs seqs;
  __shared__ float pair_sh[2][C::ROWS];  // a row's two threads: maxima, at the end sums
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr int kProducer = 8 * NT, kIssuer = 8 * NT + 1;

  // What needs no input comes before the wait for the kernel before.
  if (warp == kIssuer) {
    tmem_alloc(&tmem_holder, C::TMEM_COLS);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < RING; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], NT);
    }
    for (int i = 0; i < NB * NT; ++i) {
      mbar_init(&step[0][0] + i, 1);
      mbar_init(&p_ready[0][0] + i, 8);
    }
    for (int i = 0; i < NT; ++i) {
      mbar_init(&drained[i], 1);
      mbar_init(&q_full[i], p.q_boxes ? 1 : 8);
    }
    fence_barrier_init();
  }
  if (warp == kProducer && lane == 0) {
    prefetch_tensormap(&tm_q);
    prefetch_tensormap(&tm_pk);
    prefetch_tensormap(&tm_pv);
    prefetch_tensormap(&tm_k);
    prefetch_tensormap(&tm_v);
  }
  griddep_wait();
  if (warp == kProducer) {
    const AttnItem it = attn_item<BN, C::ROWS, MIXED>(p, lane, seqs);
    if (lane == 0) item_sh = it;
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  // Behind the allocation: a dependent that took the tensor memory first would wait for this
  // launch to end, and this one for the memory.
  griddep_launch_dependents();
  const uint32_t tmem = tmem_holder;
  const AttnItem it = item_sh;
  const int per_seq = p.T * p.rep;
  const int np = it.pb1 - it.pb0, nblk = np + it.sb1 - it.sb0;
  // Stage j of the ring holds K(j) and V(j - NB): what the issuers need at one point.
  const int stages = nblk > 0 ? nblk + NB : 0;
  uint8_t* ring = smem + C::Q_BYTES;
  bool ok = true;

  if (warp == kProducer) {
    if (lane == 0) {
      if (p.q_boxes && nblk > 0) {
        // Rows (token, head of the group) of a tile are a box of whole tokens; what lies
        // behind the last row is another sequence's or nothing's, and no row that counts.
        const int token = it.seq0 * p.T + p.by_rep.div(it.row0);
        for (int t = 0; t < NT; ++t) {
          mbar_arrive_expect_tx(&q_full[t], 128 * DP * 2);
          for (int c = 0; c < DP / 64; ++c)
            tma_load_4d(smem_u32(smem) + t * (128 * DP * 2) + c * (128 * 128), &tm_q, 64 * c, it.kv * p.rep,
                        token + t * p.by_rep.div(128), 0, smem_u32(&q_full[t]));
        }
      }
      int issued = 0;
      int of[2] = {0, 0};  // mixed tiles: the sequence K and V are at
      for (int j = 0; j < stages; ++j) {
        const int slot = j % RING;
        if (j >= RING && !mbar_wait(&empty[slot], (j / RING - 1) & 1, kSiteAttn)) break;
        mbar_arrive_expect_tx(&full[slot], ((j < nblk) + (j >= NB)) * C::SLOT_BYTES);
        for (int is_v = 0; is_v < 2; ++is_v) {
          const int i = is_v ? j - NB : j;
          if (i < 0 || i >= nblk) continue;
          const bool prefix = i < np;
          const CUtensorMap* map = prefix ? (is_v ? &tm_pv : &tm_pk) : (is_v ? &tm_v : &tm_k);
          int key = (prefix ? it.pb0 + i : it.sb0 + i - np) * BN, who = prefix ? it.g : it.b;
          if (MIXED && !prefix) {
            while (i - np >= seqs.block[of[is_v] + 1]) ++of[is_v];
            key = (i - np - seqs.block[of[is_v]]) * BN, who = it.seq0 + of[is_v];
          }
          const uint32_t at = smem_u32(ring) + slot * C::STAGE_BYTES + is_v * C::SLOT_BYTES;
#pragma unroll
          for (int c = 0; c < DP / 64; ++c) tma_load_4d(at + c * BN * 128, map, 64 * c, it.kv, key, who, smem_u32(&full[slot]));
        }
        ++issued;
      }
      // Never leave the CTA with copies still landing in shared memory.
      for (int j = issued > RING ? issued - RING : 0; j < issued; ++j)
        mbar_wait(&full[j % RING], (j / RING) & 1, kSiteAttn + 1);
      for (int t = 0; p.q_boxes && nblk > 0 && t < NT; ++t) mbar_wait(&q_full[t], 0, kSiteAttn + 1);
    }
  } else if (warp >= kIssuer) {
    // One issuing thread per row tile: it is held while its MMAs and commits go out, which
    // the other tile's overlap.  The ring is walked in order and every operand is an
    // increment of the one before: address arithmetic between two MMAs is time the tensor
    // core waits.
    const int t = warp - kIssuer;
    const bool used = t * 128 < it.nrows;  // a tile without rows goes through the steps alone
    if (nblk > 0 && lane == 0) {
      const uint64_t q_desc = smem_desc_sw128(smem_u32(smem) + t * (128 * DP * 2));
      const uint64_t k_desc0 = smem_desc_sw128(smem_u32(ring)), v_desc0 = smem_desc_mn_sw128(smem_u32(ring) + C::SLOT_BYTES, BN);
      constexpr uint32_t kStageStep = C::STAGE_BYTES >> 4;
      const uint32_t o_col = tmem + C::O_COL + t * DP, s_col = tmem + C::S_COL + t * NB * BN;
      int slot = 0;
      uint32_t lap = 0;
      auto next = [&] {
        if (++slot == RING) slot = 0, lap ^= 1;
      };
      auto scores = [&](uint32_t s_at) {  // S = Q K^T
        const uint64_t k_desc = k_desc0 + (uint32_t)slot * kStageStep;
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
          mma16_ss(s_at, q_desc + (k / 4) * (128 * 128 / 16) + (k % 4) * 2,
                   k_desc + (k / 4) * (BN * 128 / 16) + (k % 4) * 2, idesc_16<T>(BN, false), k > 0);
      };
      ok = mbar_wait(&q_full[t], 0, kSiteAttn + 2);
      int buffer = 0;
      uint32_t turn = 0;  // p_ready's phase
      int of = 0;         // mixed tiles: the sequence V is at
      for (int i = -NB; i < nblk && ok; ++i) {
        // O += P(i) V(i), then S(i + NB) = Q K^T over the p just taken.
        const uint32_t s_at = s_col + buffer * BN;
        ok = mbar_wait(&full[slot], lap, kSiteAttn + 2) &&
             (i < 0 || mbar_wait(&p_ready[t][buffer], turn, kSiteAttn + 3));
        if (!ok) break;
        tc_fence_after();
        if (i >= 0 && used) {
          const uint64_t v_desc = v_desc0 + (uint32_t)slot * kStageStep;
          // Each half of the keys has its p over its own scores.
          const auto p_at = [&](int k) { return s_at + (k / (BN / 32)) * (BN / 2) + (k % (BN / 32)) * 8; };
          if (MIXED && i >= np) {
            // Own keys of one sequence: rows of the others keep their O, whatever p and V hold.
            while (i - np >= seqs.block[of + 1]) ++of;
            const bool add = np > 0 || i - np > seqs.block[of];
            uint32_t off[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) {
              const int lo = seqs.row[of] - t * 128 - 32 * w, hi = seqs.row[of + 1] - t * 128 - 32 * w;
              const uint32_t below = lo <= 0 ? 0u : lo >= 32 ? ~0u : (1u << lo) - 1u;
              const uint32_t upto = hi <= 0 ? 0u : hi >= 32 ? ~0u : (1u << hi) - 1u;
              off[w] = ~(upto & ~below);
            }
            const bool any = (off[0] & off[1] & off[2] & off[3]) != ~0u;
#pragma unroll
            for (int k = 0; k < BN / 16 && any; ++k)
              mma16_ts_rows(o_col, p_at(k), v_desc + k * (2048 / 16), idesc_16<T>(DP, true), add || k > 0, off);
          } else {
#pragma unroll
            for (int k = 0; k < BN / 16; ++k)
              mma16_ts(o_col, p_at(k), v_desc + k * (2048 / 16), idesc_16<T>(DP, true), i > 0 || k > 0);
          }
        }
        if (i + NB < nblk && used) scores(s_at);
        mma_commit(&step[t][buffer]);
        mma_commit(&empty[slot]);
        next();
        if (++buffer == NB) buffer = 0, turn ^= i >= 0;
      }
      if (ok) {
        const int last = nblk - 1 + NB;
        mbar_wait(&step[t][last % NB], (last / NB) & 1, kSiteAttn + 4);
      } else {
        // A wait ran out: the outputs are void, but nothing may read shared memory after the CTA.
        mma_commit(&drained[t]);
        mbar_wait(&drained[t], 0, kSiteAttn + 4);
      }
    }
  } else {
    // Two threads share a row, each with half the keys of a block: two warps a tile on each
    // SM sub-core hide one another's latencies.
    const int t = warp >> 3, half = (warp >> 2) & 1;
    const int my = t * 128 + (warp & 3) * 32 + lane;  // row of the CTA
    const int pair_bar = 1 + t * 4 + (warp & 3);      // the two warps of these 32 rows
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 tensor-memory lanes
    int b = it.row0 + my;
    int head = p.by_per_seq.split(b);  // row of its sequence: token * rep + head of the group
    int tok = head;
    head = it.kv * p.rep + p.by_rep.split(tok);
    const int my_seq = b;  // among the tile's
    b += it.seq0;
    const bool live = my < it.nrows;
    if (nblk > 0 && !p.q_boxes) {
      // Q as the boxes would bring it: K-major, 128-byte swizzled, in column tiles of 64; a
      // warp brings half of each of its 32 rows; rows and columns past the end are zeros.
      constexpr int CH = DP / 8;  // 16-byte pieces of a row
      const T* q = reinterpret_cast<const T*>(p.q);
      const int64_t mine = live ? b * p.q_b + tok * p.q_t + head * p.q_h : -1;
      for (int c = half * 32 + lane; c < 32 * CH; c += 64) {
        const int rr = c / CH, x = c % CH;
        const int64_t at = __shfl_sync(0xffffffffu, mine, rr);
        const bool there = at >= 0 && 8 * x < p.D;
        const int row = (warp & 3) * 32 + rr;
        copy16_or_zero(smem_u32(smem) + t * (128 * DP * 2) + (x >> 3) * (128 * 128) + row * 128 + (((x & 7) ^ (row & 7)) << 4),
                       q + (there ? at + 8 * x : 0), there);
      }
      copy16_wait();
      fence_proxy_async_smem();
      __syncwarp();
      if (lane == 0) mbar_arrive(&q_full[t]);
    }
    const int my_len = MIXED ? (live ? seqs.len[my_seq] : 0) : it.slen;
    int own_end = my_len;  // own keys this row sees
    if (p.causal) own_end = max(0, min(my_len, my_len - p.T + tok + 1));
    const bool idle = t * 128 + (warp & 3) * 32 >= it.nrows;
    float m = -INFINITY, l = 0.f;
    const uint32_t o_addr = tmem + lanes + C::O_COL + t * DP;
    constexpr int HALF = BN / 2;  // keys of a block that are this thread's
    static_assert(HALF == 32, "a thread's scores are one load");
    const uint32_t s_addr0 = tmem + lanes + C::S_COL + t * NB * BN + half * HALF;
    // Blocks that hold keys some row of the warp does not see: the prefix's last if it is
    // not full, and the own ones from own_mask on.
    const int mask_prefix = np > 0 && (int64_t)it.pb1 * BN > it.plen ? np - 1 : -1;
    const int own_mask =
        MIXED ? np : np + max(0, (int)__reduce_min_sync(0xffffffffu, own_end) / BN - it.sb0);
    int of = 0;  // mixed tiles: the sequence the block belongs to
    int buffer = 0;
    uint32_t turn = 0;
    for (int i = 0; i < nblk; ++i) {
      ok = ok && mbar_wait(&step[t][buffer], turn, kSiteAttn + 6);
      ok = __all_sync(0xffffffffu, ok);
      const bool masked = i == mask_prefix || i >= own_mask;
      int end = BN;  // keys of this half that the row sees
      bool idle_here = idle;
      if (masked) {
        const bool prefix = i < np;
        int key = (prefix ? it.pb0 + i : it.sb0 + i - np) * BN;
        int len = prefix ? it.plen : my_len, sees = prefix ? it.plen : own_end;
        if (MIXED && !prefix) {
          while (i - np >= seqs.block[of + 1]) ++of;
          key = (i - np - seqs.block[of]) * BN, len = seqs.len[of];
          const bool its = live && my_seq == of;
          if (!its) sees = 0;
          // No row of this warp is the sequence's: its p are for nobody.  (One that is, but
          // sees none of the block, needs zeros.)
          idle_here = idle || !__any_sync(0xffffffffu, its);
        }
        end = sees - key - half * HALF;
        // Cache rows past the length may hold anything, and p = 0 would not hide a NaN.
        // (Each tile clears them before its own product; the second time changes nothing.
        // The step above says that this stage's last use is over, so that its next phase is
        // the one waited for.)
        const int filled = len - key;
        if (filled < BN && key + filled < (prefix ? p.P : p.S)) {
          const int j = i + NB;
          ok = ok && mbar_wait(&full[j % RING], (j / RING) & 1, kSiteAttn + 5);
          uint8_t* v = ring + (j % RING) * C::STAGE_BYTES + C::SLOT_BYTES;
          const int gone = BN - filled;
          for (int c = threadIdx.x & 255; c < gone * (DP / 8); c += 256) {
            const int rr = filled + c % gone, col = c / gone;
            *reinterpret_cast<uint4*>(v + (col >> 3) * (BN * 128) + rr * 128 + (col & 7) * 16) = make_uint4(0, 0, 0, 0);
          }
          fence_proxy_async_smem();
        }
      }
      const uint32_t s_addr = s_addr0 + buffer * BN;
      uint32_t x[32], pk[16];
      if (!idle_here) {
        tc_fence_after();
        tmem_ld32(s_addr, x);
      }
      if (!idle_here) {  // else: whatever these rows' p hold stays in them
        tmem_wait_ld32(x);
        if (masked) {
#pragma unroll
          for (int j = 0; j < 32; ++j) x[j] = j < end ? x[j] : 0xff800000u;
        }
        // The exponentials are taken against the maximum so far while the block's own is
        // found beside them.  Only where that is more than 2^8 above (or there is none yet)
        // O and l are brought to the new maximum and the exponentials taken again.
        for (bool again = false;; again = true) {
          const float ref = m == -INFINITY ? 0.f : m - kRoom<T>;
          const float2 c2 = make_float2(p.scale, p.scale), r2 = make_float2(-ref, -ref);
          float top[2] = {-INFINITY, -INFINITY};
          float2 add[2] = {};
#pragma unroll
          for (int j = 0; j < 16; ++j) {
            const float2 v = make_float2(__uint_as_float(x[2 * j]), __uint_as_float(x[2 * j + 1]));
            top[j & 1] = fmaxf(top[j & 1], fmaxf(v.x, v.y));
            float2 e = ffma2(v, c2, r2);
            e.x = exp2_approx(e.x), e.y = exp2_approx(e.y);
            add[j & 1] = fadd2(add[j & 1], e);
            pk[j] = pack16<T>(e.x, e.y);
          }
          const float mx = fmaxf(top[0], top[1]) * p.scale;
          // (A warp whose wait ran out goes on without data, so that no barrier lacks it.)
          if (again || named_barrier_and(pair_bar, 64, !(mx - m > kRescale))) {
            add[0] = fadd2(add[0], add[1]);
            l += add[0].x + add[0].y;
            break;
          }
          pair_sh[half][my] = mx;
          named_barrier_sync(pair_bar, 64);
          const float both = fmaxf(mx, pair_sh[half ^ 1][my]);
          const bool grown = both - m > kRescale;
          if (i > 0 && __any_sync(0xffffffffu, grown && m != -INFINITY)) {  // m = -inf: O and l are zero
            const float f = grown && m != -INFINITY ? exp2_approx(m - both) : 1.f;
            // The step that tells that O holds the block before this one.
            const int s = i - 1 + NB;
            ok = ok && mbar_wait(&step[t][s % NB], (s / NB) & 1, kSiteAttn + 7);
            ok = __all_sync(0xffffffffu, ok);
            tc_fence_after();
#pragma unroll 1
            for (int d = half * (DP / 2); d < (half + 1) * (DP / 2); d += 32) {
              uint32_t o[32];
              tmem_ld32(o_addr + d, o);
              tmem_wait_ld32(o);
#pragma unroll
              for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
              tmem_st32(o_addr + d, o);
            }
            l *= f;
          }
          if (grown) m = both;
        }
      }
      if (!idle_here) {
        tmem_st16(s_addr, pk);  // two to a column, over this half's scores
        tmem_wait_st();
        tc_fence_before();
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[t][buffer]);
      if (++buffer == NB) buffer = 0, turn ^= 1;
    }
    if (nblk > 0 && ok) {
      const int last = nblk - 1 + NB;
      ok = mbar_wait(&step[t][last % NB], (last / NB) & 1, kSiteAttn + 8);
    }
    ok = __all_sync(0xffffffffu, ok);
    pair_sh[half][my] = l;
    named_barrier_sync(pair_bar, 64);
    l += pair_sh[half ^ 1][my];
    if (ok && !idle) {
      // O from tensor memory by rows (a thread each), to global memory by lines: through
      // this warp's share of the tile's Q, which nothing reads any more.  Straight from a
      // thread per row, every 16 bytes of a store would be a memory sector of their own.
      tc_fence_after();
      constexpr int CH = DP / 16;  // 16-byte pieces that a row has in the warp's share
      uint8_t* stage = smem + t * (128 * DP * 2) + (warp & 7) * (32 * DP);
      const auto piece = [&](int r, int j) {
        return reinterpret_cast<uint4*>(stage + r * DP + ((j ^ (DP > 64 ? r & 7 : r >> 1 & 3)) << 4));
      };
      const int row = (b * p.T + tok) * p.H + head;
      const int64_t rows = (int64_t)p.B * p.T * p.H;
      const float inv = l == 0.f ? 0.f : 1.f / l;
      if (p.splits > 1 && live && half == 0) p.ml[it.split * rows + row] = make_float2(m, nblk > 0 ? l : 0.f);
      // fp32 parts take two rounds of DP / 4 columns, finished rows one of DP / 2.
      for (int round = 0; round < (p.splits == 1 ? 1 : nblk > 0 ? 2 : 0); ++round) {
        const int col = half * (DP / 2) + round * (DP / 4);
        if (p.splits == 1) {
#pragma unroll
          for (int c = 0; c < DP / 2; c += 32) {
            uint32_t o[32], w[16];
            if (nblk > 0) tmem_ld32(o_addr + col + c, o);
            tmem_wait_ld32(o);
#pragma unroll
            for (int e = 0; e < 16; ++e)
              w[e] = l == 0.f ? 0u : pack16<T>(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
#pragma unroll
            for (int e = 0; e < 4; ++e) *piece(lane, c / 8 + e) = make_uint4(w[4 * e], w[4 * e + 1], w[4 * e + 2], w[4 * e + 3]);
          }
        } else {
#pragma unroll
          for (int c = 0; c < DP / 4; c += 16) {
            uint32_t o[16];
            tmem_ld16(o_addr + col + c, o);
            tmem_wait_ld16(o);
#pragma unroll
            for (int e = 0; e < 4; ++e) *piece(lane, c / 4 + e) = make_uint4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
          }
        }
        __syncwarp();
        const int per = p.splits == 1 ? 8 : 4;  // columns of a piece
#pragma unroll 4
        for (int c = lane; c < 32 * CH; c += 32) {
          const int r = c / CH, j = c % CH;
          const int at = __shfl_sync(0xffffffffu, live ? row : -1, r), d = col + j * per;
          if (at < 0 || d >= p.D) continue;
          const uint4 u = *piece(r, j);
          if (p.splits == 1)
            *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + (int64_t)at * p.D + d) = u;
          else
            *reinterpret_cast<uint4*>(p.o_part + (it.split * rows + at) * p.D + d) = u;
        }
        __syncwarp();
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kIssuer) tmem_dealloc(tmem, C::TMEM_COLS);
}

constexpr int kMostSplits = 96;  // parts of a row

// Joins the parts of a row: one warp per row, D a multiple of 8.
template <typename T>
__global__ void __launch_bounds__(128) prefix_attention_join_kernel(const AttnParams p) {
  griddep_enter();
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)p.B * p.T * p.H, row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  // Weights first, a part per lane (kMostSplits of them): the loads of O then depend on
  // nothing and go out together.  A part that saw no key has l = 0 and no O.
  float2 ml[kMostSplits / 32];
  float top = -INFINITY, total = 0.f;
#pragma unroll
  for (int i = 0; i < kMostSplits / 32; ++i) {
    const int s = lane + 32 * i;
    ml[i] = s < p.splits ? p.ml[s * rows + row] : make_float2(-INFINITY, 0.f);
    top = fmaxf(top, ml[i].x);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  float weight[kMostSplits / 32];
#pragma unroll
  for (int i = 0; i < kMostSplits / 32; ++i) {
    weight[i] = ml[i].y == 0.f ? 0.f : exp2_approx(ml[i].x - top);
    total = fmaf(weight[i], ml[i].y, total);
  }
#pragma unroll
  for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
  float2 o[4] = {};
#pragma unroll
  for (int i = 0; i < kMostSplits / 32; ++i) {
    const int count = min(32, p.splits - 32 * i);
#pragma unroll 4
    for (int s = 0; s < count; ++s) {
      const float w = __shfl_sync(0xffffffffu, weight[i], s);
      const bool some = __shfl_sync(0xffffffffu, ml[i].y, s) != 0.f;
      const float* src = p.o_part + ((32 * i + s) * rows + row) * p.D;
#pragma unroll
      for (int c = 0; c < 4; ++c) {
        const int d = 64 * c + 2 * lane;
        const float2 a = some && d < p.D ? *reinterpret_cast<const float2*>(src + d) : make_float2(0.f, 0.f);
        o[c] = ffma2(make_float2(w, w), a, o[c]);
      }
    }
  }
  const float inv = total == 0.f ? 0.f : 1.f / total;
  T* dst = reinterpret_cast<T*>(p.out) + row * p.D;
#pragma unroll
  for (int c = 0; c < 4; ++c) {
    const int d = 64 * c + 2 * lane;
    if (d < p.D) *reinterpret_cast<uint32_t*>(dst + d) = pack16<T>(o[c].x * inv, o[c].y * inv);
  }
}

// ------------------------------------------------------------------ host
struct AttnPlan {
  int dp, nt, bn;
  int kind, tiles_per_seq, prefix_tiles, prefix_splits, own_splits, splits;
  int64_t items;
};

constexpr int kSmsPlanned = 148;  // B200; the workspace is sized before a device is known

// How a call is cut into items, from its sizes alone: the ways of making tiles are priced
// in key blocks on the busiest SM, and the cheapest one is taken.
AttnPlan attn_plan(int64_t B, int64_t T, int64_t H, int64_t KV, int64_t D, int64_t G, int64_t P, int64_t S,
                   bool ragged) {
  AttnPlan best = {};
  int64_t best_cost = INT64_MAX;
  const int64_t rep = H / KV, per_seq = T * rep;
  const int dp = D <= 64 ? 64 : D <= 128 ? 128 : 256;
  const int bn = 64;  // AttnCfg::BN
  const int64_t pb = ceil_div(P, bn), ob = ceil_div(S, bn);
  // Eighths of a microsecond, as measured: a block of 64 keys for two row tiles of 128, for
  // one (head size 256, smaller), and a CTA's prologue and epilogue; the second kernel, and
  // the parts written and read at the copy rate.
  constexpr int64_t kStart = 24, kMost = 64;
  const auto join = [&](int64_t splits) { return splits > 1 ? 24 + splits * B * T * H * D * 8 / 800000 : 0; };
  for (int kind = kBySequence; kind <= kMixed; ++kind) {
    if (kind != kBySequence && (P == 0 || B == G)) continue;  // nothing to stack
    const int64_t rows = kind != kBySequence ? ceil_div(B, G) * per_seq : per_seq;
    const int nt = dp <= 128 && rows > 128 ? 2 : 1;
    const int64_t tile = 128 * nt, block = nt == 2 ? 9 : dp == 256 ? 8 : 6;
    AttnPlan c = {};
    c.dp = dp, c.nt = nt, c.bn = bn, c.kind = kind;
    c.tiles_per_seq = (int)ceil_div(per_seq, tile);
    c.prefix_tiles = kind != kBySequence ? (int)(B * per_seq / tile + G) : 0;
    const int64_t own_tiles = B * c.tiles_per_seq * KV;
    // Full tiles of a stack, and the last ones of the prefixes, which uneven groups leave
    // with any number of rows: of two row tiles the second is often empty, and skipped.
    const int64_t stack = ceil_div(B, G) * per_seq;
    const int64_t full = ragged ? B * per_seq / tile : G * (stack / tile);
    const int64_t last = ragged ? G : stack % tile > 0 ? G : 0;
    const int64_t last_block = nt == 1 ? block : ragged ? 7 : stack % tile > 128 ? 9 : 6;
    const auto waves = [&](int64_t items, int64_t blocks) {
      return ceil_div(items, kSmsPlanned) * (blocks * block + kStart);
    };
    int64_t cost = INT64_MAX;
    if (kind == kBySequence) {
      const int64_t all = pb + ob > 0 ? pb + ob : 1;
      for (int64_t n = 1; n <= kMost && n <= (all + 1) / 2; ++n) {
        const int64_t t = waves(own_tiles * n, ceil_div(all, n)) + join(n);
        if (t < cost) cost = t, c.prefix_splits = c.splits = (int)n;
      }
      c.items = own_tiles * c.splits;
    } else if (kind == kStacked) {
      // Blocks per item that fill one wave, prefix and own keys together.  (More parts than
      // that measured slower: 8 single tokens behind 4096, 22 us with 10 + 2 parts, 30 us
      // with 18 + 1.)
      int64_t each = ceil_div(ceil_div(B * per_seq, tile) * KV * pb + own_tiles * ob, kSmsPlanned);
      each = each < 2 ? 2 : each;
      int64_t n = ceil_div(pb, each), os = S > 0 ? ceil_div(ob, each) : 0;
      n = n > kMost ? kMost : n, os = os > 16 ? 16 : os;
      c.prefix_splits = (int)n;
      const int64_t part = ceil_div(pb, n);
      cost = (KV * n * (full * (part * block + kStart) + last * (part * last_block + kStart)) +
              (os > 0 ? own_tiles * os * (ceil_div(ob, os) * block + kStart) : 0)) / kSmsPlanned +
             (part * block + kStart) / 2 + join(n + os);
      c.own_splits = (int)os;
      c.splits = (int)(c.prefix_splits + os);
      c.items = (int64_t)c.prefix_tiles * KV * c.prefix_splits + own_tiles * os;
    } else {
      const int64_t touched = (tile - 1) / per_seq + 2;  // sequences a tile may touch
      if (touched > kMixedSeqs) continue;
      c.prefix_splits = c.splits = 1;
      c.items = (int64_t)c.prefix_tiles * KV;
      // The full tiles come first, and the last of each prefix fill what they leave free.
      const int64_t own = (tile / per_seq + 1) * ob;
      const int64_t t = (pb + own) * block + kStart, t_last = (pb + own) * last_block + kStart;
      const int64_t n = full * KV, n_last = last * KV, free = ceil_div(n, kSmsPlanned) * kSmsPlanned - n;
      cost = ceil_div(n, kSmsPlanned) * t;
      if (n_last > free) {
        const int64_t all = (n * t + n_last * t_last) / kSmsPlanned + t_last / 2;
        cost = cost > all ? cost : all;
      }
    }
    if (cost < best_cost) best_cost = cost, best = c;
  }
  return best;
}

size_t attn_workspace(const AttnPlan& c, int64_t rows, int64_t D) {
  return c.splits > 1 ? (size_t)c.splits * (size_t)rows * ((size_t)D * 4 + 8) : 0;
}

bool attn_sizes_ok(int64_t B, int64_t T, int64_t H, int64_t KV, int64_t D, int64_t G, int64_t P, int64_t S) {
  constexpr int64_t kMost = 0x7fffff00;
  return B >= 0 && T >= 0 && H > 0 && KV > 0 && H % KV == 0 && D > 0 && D <= 256 && G > 0 && P >= 0 && S >= 0 &&
         B <= (1 << 20) && G <= (1 << 20) && H <= 65536 && P <= kMost && S <= kMost && T <= (1 << 24) &&
         B * T * H <= kMost;
}

// [n, rows, heads, D] with D contiguous (extents and strides from the inside out) -> boxes
// of 64 columns x box[0] heads x box[1] rows, 128-byte swizzled.
int encode_rows(CUtensorMap* map, int dtype, const void* base, const int64_t (&extent)[4], const int64_t (&stride)[3],
                const int (&box)[3]) {
  cuuint64_t dims[4], strides[3];
  cuuint32_t boxes[4] = {64, (cuuint32_t)box[0], (cuuint32_t)box[1], (cuuint32_t)box[2]};
  for (int i = 0; i < 4; ++i) dims[i] = (cuuint64_t)extent[i];
  for (int i = 0; i < 3; ++i) strides[i] = (cuuint64_t)stride[i] * 2;
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = tensor_map_encoder()(
      map, dtype == ACTUNE_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
      const_cast<void*>(base), dims, strides, boxes, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? ACTUNE_OK : ACTUNE_ERR_CUDA;
}

// A stride the tensor map takes: a positive multiple of 16 bytes below 2^40 bytes.
// Dimensions of one element have none of their own and get one that fits.
bool map_stride(int64_t* stride, int64_t extent) {
  if (extent <= 1) *stride = 256;
  return *stride > 0 && *stride % 8 == 0 && *stride < ((int64_t)1 << 39);
}

template <typename T, int DP, int NT, bool MIXED>
cudaError_t launch_attn_as(const CUtensorMap (&m)[5], const AttnParams& p, int64_t items, cudaStream_t stream) {
  using C = AttnCfg<DP, NT>;
  const cudaError_t e = ensure_smem_limit<prefix_attention_kernel<T, DP, NT, MIXED>>(C::SMEM);
  if (e != cudaSuccess) return e;
  return launch_pdl(prefix_attention_kernel<T, DP, NT, MIXED>, dim3((unsigned)items), C::WARPS * 32, C::SMEM, stream,
                    m[0], m[1], m[2], m[3], m[4], p);
}

template <typename T, int DP, int NT>
cudaError_t launch_attn(const CUtensorMap (&m)[5], const AttnParams& p, int64_t items, cudaStream_t stream) {
  return p.kind == kMixed ? launch_attn_as<T, DP, NT, true>(m, p, items, stream)
                          : launch_attn_as<T, DP, NT, false>(m, p, items, stream);
}

template <typename T>
cudaError_t dispatch_attn(const CUtensorMap (&m)[5], const AttnParams& p, const AttnPlan& c, cudaStream_t stream) {
  cudaError_t e;
  if (c.dp == 256) e = launch_attn<T, 256, 1>(m, p, c.items, stream);
  else if (c.dp == 128) e = c.nt == 2 ? launch_attn<T, 128, 2>(m, p, c.items, stream) : launch_attn<T, 128, 1>(m, p, c.items, stream);
  else e = c.nt == 2 ? launch_attn<T, 64, 2>(m, p, c.items, stream) : launch_attn<T, 64, 1>(m, p, c.items, stream);
  if (e != cudaSuccess || c.splits == 1) return e;
  const int64_t rows = (int64_t)p.B * p.T * p.H;
  return launch_pdl(prefix_attention_join_kernel<T>, dim3((unsigned)ceil_div(rows, 4)), 128, 0, stream, p);
}

}  // namespace
}  // namespace actune

using namespace actune;

extern "C" {

size_t actune_prefix_attention_workspace_size(int64_t B, int64_t T, int64_t H, int64_t KV, int64_t D, int64_t G,
                                              int64_t P, int64_t S, int ragged) {
  if (!attn_sizes_ok(B, T, H, KV, D, G, P, S) || B == 0 || T == 0) return 0;
  return attn_workspace(attn_plan(B, T, H, KV, D, G, P, S, ragged != 0), B * T * H, D);
}

int actune_prefix_attention(const actune_prefix_attention_args* a, void* stream) {
  if (a == nullptr || a->struct_bytes != sizeof(actune_prefix_attention_args)) return ACTUNE_ERR_INVALID_VALUE;
  if (!attn_sizes_ok(a->B, a->T, a->H, a->KV, a->D, a->G, a->P, a->S) || !(a->scale > 0.f) || a->scale > 3e38f ||
      (a->dtype != ACTUNE_DTYPE_F16 && a->dtype != ACTUNE_DTYPE_BF16))
    return ACTUNE_ERR_INVALID_VALUE;
  for (int64_t s : {a->q_b, a->q_t, a->q_h, a->pk_g, a->pk_p, a->pk_h, a->pv_g, a->pv_p, a->pv_h, a->k_b, a->k_s,
                    a->k_h, a->v_b, a->v_s, a->v_h})
    if (s < 0) return ACTUNE_ERR_INVALID_VALUE;
  int num_sms = 0;
  const int rc = serving_device(&num_sms);
  if (rc != ACTUNE_OK || a->B == 0 || a->T == 0) return rc;
  if (a->q == nullptr || a->out == nullptr || (a->P > 0 && (a->prefix_k == nullptr || a->prefix_v == nullptr)) ||
      (a->S > 0 && (a->k == nullptr || a->v == nullptr)))
    return ACTUNE_ERR_INVALID_VALUE;
  for (const void* x : {a->q, a->prefix_k, a->prefix_v, a->k, a->v, (const void*)a->out})
    if (!is_aligned(x, 2)) return ACTUNE_ERR_MISALIGNED;
  for (const void* x : {a->starts, a->prefix_lens, a->lens})
    if (!is_aligned(x, 4)) return ACTUNE_ERR_MISALIGNED;
  const AttnPlan c = attn_plan(a->B, a->T, a->H, a->KV, a->D, a->G, a->P, a->S, a->starts != nullptr);
  const int64_t rows = a->B * a->T * a->H;
  const size_t need = attn_workspace(c, rows, a->D);
  if (need > 0 && (a->workspace == nullptr || a->workspace_bytes < need)) return ACTUNE_ERR_WORKSPACE;
  if (need > 0 && !is_aligned(a->workspace, 16)) return ACTUNE_ERR_MISALIGNED;

  AttnParams p = {};
  p.q = a->q, p.pk = a->prefix_k, p.pv = a->prefix_v, p.k = a->k, p.v = a->v;
  p.starts = a->starts, p.prefix_lens = a->prefix_lens, p.lens = a->lens, p.out = a->out;
  p.q_b = a->q_b, p.q_t = a->q_t, p.q_h = a->q_h;
  p.pk_g = a->pk_g, p.pk_p = a->pk_p, p.pk_h = a->pk_h, p.pv_g = a->pv_g, p.pv_p = a->pv_p, p.pv_h = a->pv_h;
  p.k_b = a->k_b, p.k_s = a->k_s, p.k_h = a->k_h, p.v_b = a->v_b, p.v_s = a->v_s, p.v_h = a->v_h;
  p.B = (int)a->B, p.T = (int)a->T, p.H = (int)a->H, p.KV = (int)a->KV, p.D = (int)a->D, p.G = (int)a->G;
  p.P = (int)a->P, p.S = (int)a->S, p.rep = p.H / p.KV, p.causal = a->causal != 0, p.scale = a->scale * kLog2e;
  auto* cs = reinterpret_cast<cudaStream_t>(stream);

  // The tensor-core form: what the tensor maps and 16-byte loads of q ask for.
  bool fits = p.D % 8 == 0 && c.items <= 0x7fffffff;
  for (const void* x : {a->q, (const void*)a->out}) fits = fits && is_aligned(x, 16);
  for (int64_t s : {a->B > 1 ? a->q_b : 0, a->T > 1 ? a->q_t : 0, a->H > 1 ? a->q_h : 0}) fits = fits && s % 8 == 0;
  int64_t pk_s[3] = {a->pk_h, a->pk_p, a->pk_g}, pv_s[3] = {a->pv_h, a->pv_p, a->pv_g};
  int64_t k_s[3] = {a->k_h, a->k_s, a->k_b}, v_s[3] = {a->v_h, a->v_s, a->v_b};
  const int64_t prefix_extent[3] = {a->KV, a->P, a->G}, own_extent[3] = {a->KV, a->S, a->B};
  for (int i = 0; i < 3; ++i) {
    if (a->P > 0) fits = fits && map_stride(&pk_s[i], prefix_extent[i]) && map_stride(&pv_s[i], prefix_extent[i]);
    if (a->S > 0) fits = fits && map_stride(&k_s[i], own_extent[i]) && map_stride(&v_s[i], own_extent[i]);
  }
  if (a->P > 0) fits = fits && is_aligned(a->prefix_k, 16) && is_aligned(a->prefix_v, 16);
  if (a->S > 0) fits = fits && is_aligned(a->k, 16) && is_aligned(a->v, 16);
  if (!fits) {
    const dim3 grid((unsigned)rows);
    return serving_status(a->dtype == ACTUNE_DTYPE_BF16
                              ? launch_pdl(prefix_attention_any_kernel<__nv_bfloat16>, grid, 128, 0, cs, p)
                              : launch_pdl(prefix_attention_any_kernel<__half>, grid, 128, 0, cs, p));
  }
  p.tiles_per_seq = c.tiles_per_seq, p.kind = c.kind, p.prefix_tiles = c.prefix_tiles;
  p.prefix_splits = c.prefix_splits, p.own_splits = c.own_splits, p.splits = c.splits;
  p.ml = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(a->workspace) + (size_t)c.splits * rows * p.D * 4);
  p.o_part = reinterpret_cast<float*>(a->workspace);
  p.by_full_tiles.set(c.prefix_tiles > p.G ? c.prefix_tiles - p.G : 1), p.by_prefixes.set(p.G), p.by_kv.set(p.KV);
  p.by_own_tiles.set((int64_t)p.B * c.tiles_per_seq), p.by_tiles_per_seq.set(c.tiles_per_seq);
  p.by_per_seq.set((int64_t)p.T * p.rep), p.by_rep.set(p.rep);
  p.by_prefix_splits.set(c.prefix_splits > 0 ? c.prefix_splits : 1), p.by_own_splits.set(c.own_splits > 0 ? c.own_splits : 1);
  CUtensorMap maps[5] = {};
  int st = ACTUNE_OK;
  // Queries as [B * T tokens, H, D], where the tokens are evenly spaced and a tile of 128
  // rows is whole tokens.
  int64_t q_s[3] = {a->q_h, a->T > 1 ? a->q_t : a->q_b, 0};
  if (128 % p.rep == 0 && (a->B == 1 || a->T == 1 || a->q_b == a->T * a->q_t) && map_stride(&q_s[0], a->H) &&
      map_stride(&q_s[1], a->B * a->T)) {
    p.q_boxes = 1;
    st = encode_rows(&maps[0], a->dtype, a->q, {a->D, a->H, a->B * a->T, 1}, {q_s[0], q_s[1], 256}, {p.rep, 128 / p.rep, 1});
  }
  const auto cache = [&](int i, const void* base, int64_t rows, int64_t n, const int64_t (&str)[3]) {
    if (rows > 0 && st == ACTUNE_OK)
      st = encode_rows(&maps[i], a->dtype, base, {a->D, a->KV, rows, n}, {str[0], str[1], str[2]}, {1, c.bn, 1});
  };
  cache(1, a->prefix_k, a->P, a->G, pk_s);
  cache(2, a->prefix_v, a->P, a->G, pv_s);
  cache(3, a->k, a->S, a->B, k_s);
  cache(4, a->v, a->S, a->B, v_s);
  if (st != ACTUNE_OK) return st;
  return serving_status(a->dtype == ACTUNE_DTYPE_BF16 ? dispatch_attn<__nv_bfloat16>(maps, p, c, cs)
                                                      : dispatch_attn<__half>(maps, p, c, cs));
}

}  // extern "C"
