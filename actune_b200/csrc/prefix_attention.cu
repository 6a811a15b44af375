// Attention of a batch whose sequences share long prefixes (sm_100a).
//
//   out = sum_j p_j v_j,  p = softmax_j(scale * q . k_j)
//
// over a sequence's prefix and its own keys, one pass over the keys with the running
// maximum m and sum l of the softmax:
//   m' = max(m, max s),  p = 2^(s - m'),  l' = l 2^(m - m') + sum p,  O' = O 2^(m - m') + p V
// (s in units of log2).  Parts of the keys computed apart are joined by the same rule.
//
// A work item is a tile of 128 (or 2 x 128) query rows of one key/value head and a range
// of 128 keys (64 at head sizes above 128) at a time.  There are two ways to make tiles:
//   * by sequence: the rows (token, query head of the group) of one sequence against its
//     prefix and then its own keys.  One launch when there are tiles enough.
//   * stacked: for the prefix, the rows of all sequences that share it are stacked, so a
//     prefix is read once for the batch and not once per sequence; each sequence's own
//     keys are a further item, and the parts are joined by a second kernel.
// Either way the key range is split over more items when tiles are few.  A tile never
// holds rows of one sequence and keys of another's own, so no value of one request
// enters another's sums, not even multiplied by zero.
//
// One item per CTA:
//   softmax warps   4 per 128 rows, thread = row: scores from tensor memory to registers,
//                   mask, maximum, exponentials, sum; p (16 bit) back to tensor memory
//   one warp        TMA producer: K and V blocks into a ring of 128-byte-swizzled tiles
//   one warp        tcgen05.mma issuer: S = Q K^T (both operands in shared memory),
//                   O += P V (P in tensor memory, V as the MN-major operand)
// S of the next block is computed while this block's softmax runs (two score buffers
// for one row tile, the other row tile's scores for two).  O is rescaled only when the
// maximum has grown by more than 2^8 since the last time: until then p stays below 2^8,
// which the 16-bit types and the fp32 sums hold, and l and O carry the same factor.
#include "serving.cuh"

namespace actune {
namespace {

constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescale = 8.f;  // growth of the maximum (log2) that O is rescaled for
constexpr int kSiteAttn = 300;

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
  int stacked;      // 0: tiles by sequence; 1: stacked prefix tiles, then own-key tiles
  int prefix_tiles; // upper bound on the stacked tiles of a key/value head
  int prefix_splits, own_splits;  // by sequence: prefix_splits of both together
  int splits;       // parts per row; 1: write out directly
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
// Instruction descriptor, kind::f16 with fp32 accumulation: M = 128, N; the A operand and
// (b_mn = false) the B operand K-major.
template <typename T>
constexpr uint32_t idesc_16(int N, bool b_mn) {
  constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (fmt << 7) | (fmt << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) |
         ((uint32_t)(128 >> 4) << 24);
}

__device__ __forceinline__ void mma16_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(acc)
      : "memory");
}
__device__ __forceinline__ void mma16_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, uint32_t acc) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(acc)
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

__device__ __forceinline__ void tma_load_4d(uint32_t dst, const CUtensorMap* map, int x, int y, int z, int w,
                                            uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(y), "r"(z), "r"(w), "r"(bar)
      : "memory");
}

__device__ __forceinline__ float exp2_approx(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

template <typename T>
__device__ __forceinline__ uint32_t pack16(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack16<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack16<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// DP: the head size rounded up to 64, 128 or 256 (the rest of a row is zeros).
// NT: row tiles of 128 per CTA.
template <int DP, int NT>
struct AttnCfg {
  static constexpr int BN = DP > 128 ? 64 : 128;       // keys per block
  static constexpr int ROWS = 128 * NT;
  static constexpr int Q_BYTES = ROWS * DP * 2;
  static constexpr int SLOT_BYTES = BN * DP * 2;        // one K or V block
  static constexpr int RING = (224 * 1024 - Q_BYTES) / SLOT_BYTES > 8 ? 8 : (224 * 1024 - Q_BYTES) / SLOT_BYTES;
  static constexpr int SMEM = 1024 + Q_BYTES + RING * SLOT_BYTES;
  static constexpr int O_COL = 0, S_COL = NT * DP;      // tensor memory columns: O, then two score buffers
  static constexpr int TMEM_COLS = 512;
  static constexpr int WARPS = 4 * NT + 2;
  static_assert(S_COL + 2 * BN <= TMEM_COLS && RING >= 4 && SMEM + 512 <= 227 * 1024, "fits");
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
template <int BN, int ROWS>
__device__ AttnItem attn_item(const AttnParams& p, int lane) {
  AttnItem it = {};
  const int per_seq = p.T * p.rep;
  int x = blockIdx.x;
  const int prefix_items = p.stacked ? p.prefix_tiles * p.KV * p.prefix_splits : 0;
  if (x < prefix_items) {
    const int tile = x % p.prefix_tiles;
    x /= p.prefix_tiles;
    it.kv = x % p.KV, it.split = x / p.KV;
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
      const int rows = (s1 - s0) * per_seq, mine = (rows + ROWS - 1) / ROWS;
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
        it.row0 = (tile - __shfl_sync(0xffffffffu, first, src)) * ROWS;
        it.nrows = min(ROWS, __shfl_sync(0xffffffffu, rows, src) - it.row0);
        found = true;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
    if (!found) return it;
    it.b = it.seq0;
    it.plen = clamp_len(p.prefix_lens, it.g, p.P);
    const int64_t blocks = (it.plen + BN - 1) / BN;
    it.pb0 = (int)(blocks * it.split / p.prefix_splits);
    it.pb1 = (int)(blocks * (it.split + 1) / p.prefix_splits);
    return it;
  }
  x -= prefix_items;
  const int tiles = p.B * p.tiles_per_seq;
  const int tile = x % tiles;
  x /= tiles;
  it.kv = x % p.KV;
  const int part = x / p.KV;
  it.b = it.seq0 = tile / p.tiles_per_seq;
  it.row0 = tile % p.tiles_per_seq * ROWS;
  it.nrows = min(ROWS, per_seq - it.row0);
  it.slen = clamp_len(p.lens, it.b, p.S);
  int seen = it.slen;  // own keys that the tile's last row sees
  if (p.causal) seen = max(0, min(seen, it.slen - p.T + (it.row0 + it.nrows - 1) / p.rep + 1));
  const int64_t own = (seen + BN - 1) / BN;
  if (p.stacked) {
    it.split = p.prefix_splits + part;
    it.sb0 = (int)(own * part / p.own_splits);
    it.sb1 = (int)(own * (part + 1) / p.own_splits);
    return it;
  }
  it.split = part;
  int g = 0;
  if (p.starts != nullptr) {
    for (int i = 1 + lane; i < p.G; i += 32) g += p.starts[i] <= it.b;
    g = __reduce_add_sync(0xffffffffu, g);
  } else {
    g = (int)((int64_t)it.b * p.G / p.B);
  }
  it.g = g;
  it.plen = clamp_len(p.prefix_lens, g, p.P);
  const int64_t prefix = (it.plen + BN - 1) / BN, all = prefix + own;
  const int64_t c0 = all * part / p.prefix_splits, c1 = all * (part + 1) / p.prefix_splits;
  it.pb0 = (int)(c0 < prefix ? c0 : prefix), it.pb1 = (int)(c1 < prefix ? c1 : prefix);
  it.sb0 = (int)(c0 < prefix ? 0 : c0 - prefix), it.sb1 = (int)(c1 < prefix ? 0 : c1 - prefix);
  return it;
}

template <typename T, int DP, int NT>
__global__ void __launch_bounds__(AttnCfg<DP, NT>::WARPS * 32, 1)
    prefix_attention_kernel(const __grid_constant__ CUtensorMap tm_pk, const __grid_constant__ CUtensorMap tm_pv,
                            const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                            const AttnParams p) {
  using C = AttnCfg<DP, NT>;
  constexpr int BN = C::BN, RING = C::RING;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[RING], empty[RING], s_full[2], p_ready[2], pv_done[NT], all_done;
  __shared__ uint32_t tmem_holder;
  __shared__ AttnItem item_sh;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  constexpr int kProducer = 4 * NT, kIssuer = 4 * NT + 1;

  griddep_enter();
  if (warp == kProducer) {
    const AttnItem it = attn_item<BN, C::ROWS>(p, lane);
    if (lane == 0) item_sh = it;
    if (lane == 0) {
      prefetch_tensormap(&tm_pk);
      prefetch_tensormap(&tm_pv);
      prefetch_tensormap(&tm_k);
      prefetch_tensormap(&tm_v);
    }
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < RING; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&s_full[i], 1);
      mbar_init(&p_ready[i], 4);
    }
    for (int i = 0; i < NT; ++i) mbar_init(&pv_done[i], 1);
    mbar_init(&all_done, 1);
    fence_barrier_init();
  }
  __syncthreads();
  const AttnItem it = item_sh;
  if (it.nrows <= 0) return;
  if (warp == kIssuer) {
    tmem_alloc(&tmem_holder, C::TMEM_COLS);
    tmem_relinquish();
  }
  const int per_seq = p.T * p.rep;
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = tmem_holder;
  const int np = it.pb1 - it.pb0, nblk = np + it.sb1 - it.sb0;
  // Ring positions of a block's K and V, in the order the issuer needs them.
  auto k_pos = [&](int i) { return NT == 2 ? 2 * i : i == 0 ? 0 : 2 * i - 1; };
  auto v_pos = [&](int i) { return NT == 2 ? 2 * i + 1 : i + 1 < nblk ? 2 * i + 2 : 2 * i + 1; };
  uint8_t* ring = smem + C::Q_BYTES;
  bool ok = true;

  if (warp == kProducer) {
    if (lane == 0) {
      int issued = 0;
      for (int pos = 0; pos < 2 * nblk && ok; ++pos) {
        // pos -> which block, K or V
        int i, is_v;
        if (NT == 2) {
          i = pos >> 1, is_v = pos & 1;
        } else if (pos == 0) {
          i = 0, is_v = 0;
        } else if (pos == 2 * nblk - 1) {
          i = nblk - 1, is_v = 1;
        } else {
          is_v = (pos & 1) == 0;
          i = is_v ? pos / 2 - 1 : (pos + 1) / 2;
        }
        const int slot = pos % RING;
        if (pos >= RING && !mbar_wait(&empty[slot], (pos / RING - 1) & 1, kSiteAttn)) {
          ok = false;
          break;
        }
        mbar_arrive_expect_tx(&full[slot], C::SLOT_BYTES);
        const bool prefix = i < np;
        const CUtensorMap* map = prefix ? (is_v ? &tm_pv : &tm_pk) : (is_v ? &tm_v : &tm_k);
        const int key = (prefix ? it.pb0 + i : it.sb0 + i - np) * BN, who = prefix ? it.g : it.b;
#pragma unroll
        for (int c = 0; c < DP / 64; ++c)
          tma_load_4d(smem_u32(ring + slot * C::SLOT_BYTES + c * BN * 128), map, 64 * c, it.kv, key, who,
                      smem_u32(&full[slot]));
        ++issued;
      }
      // Never leave the CTA with copies still landing in shared memory.
      for (int pos = issued > RING ? issued - RING : 0; pos < issued; ++pos)
        mbar_wait(&full[pos % RING], (pos / RING) & 1, kSiteAttn + 1);
    }
  } else if (warp == kIssuer) {
    if (nblk > 0) named_barrier_sync(1, (4 * NT + 1) * 32);  // Q is in shared memory
    if (lane == 0 && nblk > 0) {
      const uint32_t q0 = smem_u32(smem), r0 = smem_u32(ring);
      auto wait_slot = [&](int pos) { return mbar_wait(&full[pos % RING], (pos / RING) & 1, kSiteAttn + 2); };
      auto scores = [&](int t, int buffer, int pos) {  // S[buffer] = Q_t K^T
        const uint32_t kb = r0 + (pos % RING) * C::SLOT_BYTES, qb = q0 + t * (128 * DP * 2);
#pragma unroll
        for (int k = 0; k < DP / 16; ++k)
          mma16_ss(tmem + C::S_COL + buffer * BN, smem_desc_sw128(qb + (k / 4) * (128 * 128) + (k % 4) * 32),
                   smem_desc_sw128(kb + (k / 4) * (BN * 128) + (k % 4) * 32), idesc_16<T>(BN, false), k > 0);
      };
      auto values = [&](int t, int buffer, int pos, bool first) {  // O_t += P[buffer] V
        const uint32_t vb = r0 + (pos % RING) * C::SLOT_BYTES;
#pragma unroll
        for (int k = 0; k < BN / 16; ++k)
          mma16_ts(tmem + C::O_COL + t * DP, tmem + C::S_COL + buffer * BN + k * 8,
                   smem_desc_mn_sw128(vb + k * 2048, BN), idesc_16<T>(DP, true), !first || k > 0);
      };
      ok = wait_slot(k_pos(0));
      if (ok) {
        tc_fence_after();
        for (int t = 0; t < NT; ++t) {
          scores(t, t, k_pos(0));
          mma_commit(&s_full[t]);
        }
        mma_commit(&empty[k_pos(0) % RING]);
      }
      for (int i = 0; i < nblk && ok; ++i) {
        if constexpr (NT == 1) {
          if (i + 1 < nblk) {
            // The other score buffer: its P was consumed by the product issued before.
            if (!(ok = wait_slot(k_pos(i + 1)))) break;
            tc_fence_after();
            scores(0, (i + 1) & 1, k_pos(i + 1));
            mma_commit(&s_full[(i + 1) & 1]);
            mma_commit(&empty[k_pos(i + 1) % RING]);
          }
          ok = wait_slot(v_pos(i)) && mbar_wait(&p_ready[i & 1], (i >> 1) & 1, kSiteAttn + 3);
          if (!ok) break;
          tc_fence_after();
          values(0, i & 1, v_pos(i), i == 0);
          mma_commit(&empty[v_pos(i) % RING]);
          mma_commit(&pv_done[0]);
        } else {
          for (int t = 0; t < NT && ok; ++t) {
            ok = (t > 0 || wait_slot(v_pos(i))) && mbar_wait(&p_ready[t], i & 1, kSiteAttn + 3);
            if (!ok) break;
            tc_fence_after();
            values(t, t, v_pos(i), i == 0);
            if (t == NT - 1) mma_commit(&empty[v_pos(i) % RING]);
            mma_commit(&pv_done[t]);
            if (i + 1 < nblk) {
              if (t == 0 && !(ok = wait_slot(k_pos(i + 1)))) break;
              tc_fence_after();
              scores(t, t, k_pos(i + 1));
              mma_commit(&s_full[t]);
              if (t == NT - 1) mma_commit(&empty[k_pos(i + 1) % RING]);
            }
          }
        }
      }
      mma_commit(&all_done);
      mbar_wait(&all_done, 0, kSiteAttn + 4);  // nothing in flight reads shared memory after this
    }
  } else {
    const int t = warp >> 2;                      // row tile
    const int my = threadIdx.x;                   // row of the CTA
    const uint32_t lanes = (uint32_t)(warp & 3) << 21;  // this warp's 32 tensor-memory lanes
    const int idx = it.row0 + my, b = it.seq0 + idx / per_seq, r = idx % per_seq;
    const int tok = r / p.rep, head = it.kv * p.rep + r % p.rep;
    const bool live = my < it.nrows;
    if (nblk > 0) {
      // Q, K-major, 128-byte swizzled, in column tiles of 64; a warp brings its 32 rows,
      // rows and columns past the end are zeros.
      constexpr int CH = DP / 8;  // 16-byte pieces of a row
      const T* q = reinterpret_cast<const T*>(p.q);
      const int64_t mine = live ? b * p.q_b + tok * p.q_t + head * p.q_h : -1;
#pragma unroll 4
      for (int c = lane; c < 32 * CH; c += 32) {
        const int rr = c / CH, x = c % CH;
        const int64_t at = __shfl_sync(0xffffffffu, mine, rr);
        uint4 u = make_uint4(0, 0, 0, 0);
        if (at >= 0 && 8 * x < p.D) u = *reinterpret_cast<const uint4*>(q + at + 8 * x);
        const int row = (warp & 3) * 32 + rr;
        uint8_t* dst = smem + t * (128 * DP * 2) + (x >> 3) * (128 * 128) + row * 128;
        *reinterpret_cast<uint4*>(dst + (((x & 7) ^ (row & 7)) << 4)) = u;
      }
      fence_proxy_async_smem();
      named_barrier_sync(1, (4 * NT + 1) * 32);
    }
    int own_end = it.slen;  // own keys this row sees
    if (p.causal) own_end = max(0, min(it.slen, it.slen - p.T + tok + 1));
    float m = -INFINITY, l = 0.f;
    const uint32_t o_addr = tmem + lanes + C::O_COL + t * DP;
    for (int i = 0; i < nblk && ok; ++i) {
      const int buffer = NT == 1 ? i & 1 : t;
      const bool prefix = i < np;
      const int key = (prefix ? it.pb0 + i : it.sb0 + i - np) * BN;
      const int end = (prefix ? it.plen : own_end) - key;  // keys of the block this row sees
      // Cache rows past the length may hold anything, and p = 0 would not hide a NaN.
      const int filled = (prefix ? it.plen : it.slen) - key;
      if (t == 0 && filled < BN && key + filled < (prefix ? p.P : p.S)) {
        const int pos = v_pos(i);
        ok = mbar_wait(&full[pos % RING], (pos / RING) & 1, kSiteAttn + 5);
        uint8_t* v = ring + (pos % RING) * C::SLOT_BYTES;
        const int gone = BN - filled;
        for (int c = my; c < gone * (DP / 8); c += 128) {
          const int r = filled + c % gone, x = c / gone;
          *reinterpret_cast<uint4*>(v + (x >> 3) * (BN * 128) + r * 128 + (x & 7) * 16) = make_uint4(0, 0, 0, 0);
        }
        fence_proxy_async_smem();
      }
      ok = mbar_wait(&s_full[buffer], NT == 1 ? (i >> 1) & 1 : i & 1, kSiteAttn + 6) && ok;
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc_fence_after();
      const uint32_t s_addr = tmem + lanes + C::S_COL + buffer * BN;
      float s[BN];
#pragma unroll
      for (int c = 0; c < BN / 32; ++c) tmem_ld32(s_addr + 32 * c, reinterpret_cast<uint32_t(&)[32]>(s[32 * c]));
      tmem_wait_ld();
      if (!__all_sync(0xffffffffu, end >= BN)) {
#pragma unroll
        for (int j = 0; j < BN; ++j) s[j] = j < end ? s[j] : -INFINITY;
      }
      float top[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int j = 4; j < BN; ++j) top[j & 3] = fmaxf(top[j & 3], s[j]);
      const float mx = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * p.scale;
      const bool grown = mx - m > kRescale;  // m = -inf: O and l are zero, only m is set
      const bool rescale = __any_sync(0xffffffffu, grown && m != -INFINITY);
      // Every phase of pv_done is waited for, here or below: a parity tells only
      // neighbouring phases apart.
      if (rescale) {
        const float f = grown && m != -INFINITY ? exp2_approx(m - mx) : 1.f;
        ok = mbar_wait(&pv_done[t], (i - 1) & 1, kSiteAttn + 7);
        if (!(ok = __all_sync(0xffffffffu, ok))) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(o_addr + 32 * c, o);
          tmem_wait_ld();
#pragma unroll
          for (int j = 0; j < 32; ++j) o[j] = __float_as_uint(__uint_as_float(o[j]) * f);
          tmem_st32(o_addr + 32 * c, o);
        }
        l *= f;
      }
      if (grown) m = mx;
      const float ref = m == -INFINITY ? 0.f : m;
      const float2 c2 = make_float2(p.scale, p.scale), r2 = make_float2(-ref, -ref);
      float2 sum[2] = {};
      uint32_t pk[BN / 2];
#pragma unroll
      for (int j = 0; j < BN / 2; ++j) {
        float2 e = ffma2(make_float2(s[2 * j], s[2 * j + 1]), c2, r2);
        e.x = exp2_approx(e.x), e.y = exp2_approx(e.y);
        sum[j & 1] = fadd2(sum[j & 1], e);
        pk[j] = pack16<T>(e.x, e.y);
      }
#pragma unroll
      for (int c = 0; c < BN / 64; ++c) tmem_st32(s_addr + 32 * c, pk + 32 * c);
      l += (sum[0].x + sum[0].y) + (sum[1].x + sum[1].y);
      tmem_wait_st();
      if (i > 0 && !rescale) ok = mbar_wait(&pv_done[t], (i - 1) & 1, kSiteAttn + 7);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&p_ready[buffer]);
    }
    if (nblk > 0 && ok) ok = mbar_wait(&pv_done[t], (nblk - 1) & 1, kSiteAttn + 8);
    ok = __all_sync(0xffffffffu, ok);
    if (ok) {
      tc_fence_after();
      const int64_t row = ((int64_t)b * p.T + tok) * p.H + head;
      if (p.splits == 1) {
        const float inv = l == 0.f ? 0.f : 1.f / l;
        T* dst = reinterpret_cast<T*>(p.out) + row * p.D;
#pragma unroll
        for (int c = 0; c < DP / 32; ++c) {
          if (32 * c >= p.D) break;
          uint32_t o[32];
          if (nblk > 0) tmem_ld32(o_addr + 32 * c, o);
          tmem_wait_ld();
          if (!live) continue;
#pragma unroll
          for (int j = 0; j < 32; j += 8) {
            if (32 * c + j >= p.D) break;
            uint32_t w[4];
#pragma unroll
            for (int e = 0; e < 4; ++e)
              w[e] = l == 0.f ? 0u
                              : pack16<T>(__uint_as_float(o[j + 2 * e]) * inv, __uint_as_float(o[j + 2 * e + 1]) * inv);
            *reinterpret_cast<uint4*>(dst + 32 * c + j) = make_uint4(w[0], w[1], w[2], w[3]);
          }
        }
      } else {
        const int64_t rows = (int64_t)p.B * p.T * p.H;
        if (live) p.ml[it.split * rows + row] = make_float2(m, nblk > 0 ? l : 0.f);
        if (nblk > 0) {
          float* dst = p.o_part + (it.split * rows + row) * p.D;
#pragma unroll
          for (int c = 0; c < DP / 32; ++c) {
            if (32 * c >= p.D) break;
            uint32_t o[32];
            tmem_ld32(o_addr + 32 * c, o);
            tmem_wait_ld();
            if (!live || l == 0.f) continue;
#pragma unroll
            for (int j = 0; j < 32; j += 4)
              if (32 * c + j < p.D)
                *reinterpret_cast<uint4*>(dst + 32 * c + j) = make_uint4(o[j], o[j + 1], o[j + 2], o[j + 3]);
          }
        }
      }
    }
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kIssuer) tmem_dealloc(tmem, C::TMEM_COLS);
}

// Joins the parts of a row: one warp per row, D a multiple of 8.
template <typename T>
__global__ void __launch_bounds__(128) prefix_attention_join_kernel(const AttnParams p) {
  griddep_enter();
  const int lane = threadIdx.x & 31;
  const int64_t rows = (int64_t)p.B * p.T * p.H, row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 5);
  if (row >= rows) return;
  float top = -INFINITY;
  for (int s = lane; s < p.splits; s += 32) top = fmaxf(top, p.ml[s * rows + row].x);
#pragma unroll
  for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
  float total = 0.f;
  float2 o[4] = {};
  for (int s = 0; s < p.splits; ++s) {
    const float2 ml = p.ml[s * rows + row];
    if (ml.y == 0.f) continue;  // this part saw no key; its O was not written
    const float w = exp2_approx(ml.x - top);
    total = fmaf(w, ml.y, total);
    const float* src = p.o_part + (s * rows + row) * p.D;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
      const int d = 64 * c + 2 * lane;
      if (d < p.D) {
        const float2 a = *reinterpret_cast<const float2*>(src + d);
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
  int stacked, tiles_per_seq, prefix_tiles, prefix_splits, own_splits, splits;
  int64_t items;
};

constexpr int kSmsPlanned = 148;  // B200; the workspace is sized before a device is known

// How a call is cut into items, from its sizes alone.  Both ways of making tiles are
// priced in key blocks on the busiest SM (plus, where parts have to be joined, the
// second kernel and the parts' traffic, about three blocks), and the cheaper one is taken.
AttnPlan attn_plan(int64_t B, int64_t T, int64_t H, int64_t KV, int64_t D, int64_t G, int64_t P, int64_t S) {
  AttnPlan best = {};
  int64_t best_cost = INT64_MAX;
  const int64_t rep = H / KV, per_seq = T * rep;
  const int dp = D <= 64 ? 64 : D <= 128 ? 128 : 256, bn = dp > 128 ? 64 : 128;
  const int64_t pb = ceil_div(P, bn), ob = ceil_div(S, bn);
  constexpr int64_t kJoin = 3, kStart = 2;  // in blocks: joining parts; a CTA's prologue and epilogue
  for (int stacked = 0; stacked < 2; ++stacked) {
    if (stacked && (P == 0 || B == G)) continue;  // nothing to stack
    const int64_t rows = stacked ? ceil_div(B, G) * per_seq : per_seq;
    const int nt = dp <= 128 && rows > 128 ? 2 : 1;
    const int64_t tile = 128 * nt;
    AttnPlan c = {};
    c.dp = dp, c.nt = nt, c.bn = bn, c.stacked = stacked;
    c.tiles_per_seq = (int)ceil_div(per_seq, tile);
    const int64_t own_tiles = B * c.tiles_per_seq * KV;
    int64_t cost;
    if (!stacked) {
      const int64_t all = pb + ob > 0 ? pb + ob : 1;
      int64_t splits = kSmsPlanned / own_tiles;
      splits = splits > all / 2 ? all / 2 : splits;
      splits = splits > 64 ? 64 : splits < 1 ? 1 : splits;
      c.prefix_splits = c.splits = (int)splits;
      c.items = own_tiles * splits;
      cost = ceil_div(c.items, kSmsPlanned) * (ceil_div(all, splits) + kStart) * nt + (splits > 1 ? kJoin : 0);
    } else {
      c.prefix_tiles = (int)(B * per_seq / tile + G);
      const int64_t tiles = ceil_div(B * per_seq, tile) * KV;
      // Blocks per item that fill one wave.
      const int64_t blocks = tiles * pb + own_tiles * ob;
      int64_t each = ceil_div(blocks, kSmsPlanned);
      each = each < 2 ? 2 : each;
      int64_t ps = ceil_div(pb, each), os = S > 0 ? ceil_div(ob, each) : 0;
      ps = ps > 64 ? 64 : ps, os = os > 16 ? 16 : os;
      c.prefix_splits = (int)ps, c.own_splits = (int)os;
      c.splits = (int)(ps + os);
      c.items = (int64_t)c.prefix_tiles * KV * ps + own_tiles * os;
      cost = (ceil_div(tiles * ps * (ceil_div(pb, ps) + kStart) +
                       (os > 0 ? own_tiles * os * (ceil_div(ob, os) + kStart) : 0), kSmsPlanned)) * nt + kJoin;
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

// [n, rows, heads, D] with D contiguous -> boxes of 64 columns x bn rows of one head.
int encode_cache(CUtensorMap* map, int dtype, const void* base, int64_t D, int64_t heads, int64_t rows, int64_t n,
                 int64_t sh, int64_t sr, int64_t sn, int bn) {
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows, (cuuint64_t)n};
  const cuuint64_t strides[3] = {(cuuint64_t)(sh * 2), (cuuint64_t)(sr * 2), (cuuint64_t)(sn * 2)};
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)bn, 1};
  const cuuint32_t estr[4] = {1, 1, 1, 1};
  const CUresult r = tensor_map_encoder()(
      map, dtype == ACTUNE_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
      const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? ACTUNE_OK : ACTUNE_ERR_CUDA;
}

// A stride the tensor map takes: a positive multiple of 16 bytes below 2^40 bytes.
// Dimensions of one element have none of their own and get one that fits.
bool map_stride(int64_t* stride, int64_t extent) {
  if (extent <= 1) *stride = 256;
  return *stride > 0 && *stride % 8 == 0 && *stride < ((int64_t)1 << 39);
}

template <typename T, int DP, int NT>
cudaError_t launch_attn(const CUtensorMap (&m)[4], const AttnParams& p, int64_t items, cudaStream_t stream) {
  using C = AttnCfg<DP, NT>;
  const cudaError_t e = ensure_smem_limit<prefix_attention_kernel<T, DP, NT>>(C::SMEM);
  if (e != cudaSuccess) return e;
  return launch_pdl(prefix_attention_kernel<T, DP, NT>, dim3((unsigned)items), C::WARPS * 32, C::SMEM, stream, m[0],
                    m[1], m[2], m[3], p);
}

template <typename T>
cudaError_t dispatch_attn(const CUtensorMap (&m)[4], const AttnParams& p, const AttnPlan& c, cudaStream_t stream) {
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
                                              int64_t P, int64_t S) {
  if (!attn_sizes_ok(B, T, H, KV, D, G, P, S) || B == 0 || T == 0) return 0;
  return attn_workspace(attn_plan(B, T, H, KV, D, G, P, S), B * T * H, D);
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
  const AttnPlan c = attn_plan(a->B, a->T, a->H, a->KV, a->D, a->G, a->P, a->S);
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
  p.tiles_per_seq = c.tiles_per_seq, p.stacked = c.stacked, p.prefix_tiles = c.prefix_tiles;
  p.prefix_splits = c.prefix_splits, p.own_splits = c.own_splits, p.splits = c.splits;
  p.ml = reinterpret_cast<float2*>(reinterpret_cast<uint8_t*>(a->workspace) + (size_t)c.splits * rows * p.D * 4);
  p.o_part = reinterpret_cast<float*>(a->workspace);
  CUtensorMap maps[4] = {};
  int st = ACTUNE_OK;
  if (a->P > 0) {
    st = encode_cache(&maps[0], a->dtype, a->prefix_k, a->D, a->KV, a->P, a->G, pk_s[0], pk_s[1], pk_s[2], c.bn);
    if (st == ACTUNE_OK)
      st = encode_cache(&maps[1], a->dtype, a->prefix_v, a->D, a->KV, a->P, a->G, pv_s[0], pv_s[1], pv_s[2], c.bn);
  }
  if (a->S > 0 && st == ACTUNE_OK) {
    st = encode_cache(&maps[2], a->dtype, a->k, a->D, a->KV, a->S, a->B, k_s[0], k_s[1], k_s[2], c.bn);
    if (st == ACTUNE_OK)
      st = encode_cache(&maps[3], a->dtype, a->v, a->D, a->KV, a->S, a->B, v_s[0], v_s[1], v_s[2], c.bn);
  }
  if (st != ACTUNE_OK) return st;
  return serving_status(a->dtype == ACTUNE_DTYPE_BF16 ? dispatch_attn<__nv_bfloat16>(maps, p, c, cs)
                                                      : dispatch_attn<__half>(maps, p, c, cs));
}

}  // extern "C"
