// Low-rank adapters of many requests beside a shared projection (sm_100a):
//   out[m] = y[m] + scale[s] * up[s] (down[s] x[m]),   s = slots[m].
//
// plan    rows sorted by adapter into tiles of 4, 16 or 128 rows with one adapter each.
// shrink  v = down x for a tile and a slice of K; the slices' fp32 sums go to the
//         workspace, so that few rows still occupy the machine, in a fixed order.
// expand  out = y + scale * up v for a tile and a range of columns.
//
// Both products are thin (R <= 128 against K and N of thousands): they are bound by
// reading x, down, up and y and writing out, not by the MMA rate, so operands go from
// global memory straight into mma.sync fragments, 16 bytes per lane: the contraction
// index is permuted alike for both operands, so that a lane's consecutive elements fill
// its fragment registers.  v enters the second product as the sum of two 16-bit parts
// (v = hi + lo, 16 bits of significand or more), so it keeps its 32-bit precision up to
// the accumulator for twice a small number of MMAs.
//
// The expand kernel has three forms: 4-row tiles without the matrix units (their time is
// latency: `up` asked for before v is there), 16 rows by mma.sync, and 128 rows on
// tcgen05 with y and out as boxes by TMA (their time is that traffic; with little of it
// tiles of 128 take the 16-row form in parts).  16 requests of 304
// tokens, 2048 -> 32768, rank 64: 178 us, the floor of its bytes 114 us.
#include "serving.cuh"

namespace actune {
namespace {

constexpr int kMaxSlots = 8191;
constexpr int kMaxRank = 128;
constexpr int64_t kMostColumns = 0x7fff0000;  // of N and K: the indexes of a block's steps behind them are 32-bit
constexpr int kFewRows = 4;
constexpr int kHeader = 4;  // plan: tile count, then three padding words

// Tiles of `tile` rows that M rows of S adapters (and of none) can make at most.
inline int64_t max_tiles(int64_t M, int64_t S, int tile) { return M / tile + (S + 1 < M ? S + 1 : M); }

// plan: [kHeader] count; then per tile {slot, first, rows, 0}; then the sorted rows.
__device__ __forceinline__ const int4* plan_tiles(const int32_t* plan) {
  return reinterpret_cast<const int4*>(plan + kHeader);
}

// One CTA (800 rows 6 us, 6400 24 us, 38911 113 us, once for all the projections that a
// batch passes through).  Stable counting sort: 1024 rows at a time, the warps of a chunk
// one after the other, the lanes of a warp ranked among those of the same slot.
__global__ void __launch_bounds__(1024) adapter_plan_kernel(const int32_t* __restrict__ slots, int M, int S, int tile,
                                                            int tiles_cap, int32_t* __restrict__ plan) {
  extern __shared__ int32_t sh[];  // per slot (S + 1: the last is "none"): count, then next place
  __shared__ int warp_rows[32], warp_tiles[32];
  griddep_enter();
  const int n = S + 1;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  for (int i = tid; i < n; i += 1024) sh[i] = 0;
  __syncthreads();
  for (int m = tid; m < M; m += 1024) {
    const int s = slots[m];
    atomicAdd(&sh[(uint32_t)s < (uint32_t)S ? s : S], 1);
  }
  __syncthreads();
  // Exclusive sums of rows and tiles over the slots, and the tile list.
  int4* tiles = reinterpret_cast<int4*>(plan + kHeader);
  int rows_before = 0, tiles_before = 0;
  for (int base = 0; base < n; base += 1024) {
    const int i = base + tid;
    const int c = i < n ? sh[i] : 0, t = (c + tile - 1) / tile;
    int cr = c, ct = t;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int a = __shfl_up_sync(0xffffffffu, cr, o), b = __shfl_up_sync(0xffffffffu, ct, o);
      if (lane >= o) cr += a, ct += b;
    }
    if (lane == 31) warp_rows[warp] = cr, warp_tiles[warp] = ct;
    __syncthreads();
    int r0 = rows_before + cr - c, t0 = tiles_before + ct - t;
    for (int w = 0; w < 32; ++w) {
      if (w < warp) r0 += warp_rows[w], t0 += warp_tiles[w];
      rows_before += warp_rows[w], tiles_before += warp_tiles[w];
    }
    if (i < n) {
      sh[i] = r0;
      for (int j = 0; j < t; ++j)
        tiles[t0 + j] = make_int4(i < S ? i : -1, r0 + j * tile, min(tile, c - j * tile), 0);
    }
    __syncthreads();
  }
  if (tid == 0) plan[0] = tiles_before;
  int32_t* order = plan + kHeader + 4 * (int64_t)tiles_cap;
  for (int base = 0; base < M; base += 1024) {
    const int m = base + tid;
    int s = -1, rank = 0, count = 0;
    if (m < M) {
      s = slots[m];
      if ((uint32_t)s >= (uint32_t)S) s = S;
    }
    const unsigned same = __match_any_sync(0xffffffffu, s);
    rank = __popc(same & ((1u << lane) - 1u));
    count = __popc(same);
    for (int w = 0; w < 32; ++w) {
      if (w == warp && s >= 0) order[sh[s] + rank] = m;
      __syncwarp();
      if (w == warp && s >= 0 && rank == 0) sh[s] += count;
      __syncthreads();
    }
  }
}

struct AdapterParams {
  const void *x, *y, *down, *up;
  const float* scale;
  const int32_t* plan;
  void* out;
  float* v;       // [slices, M, RP] partial sums of down x, rows in plan order; or, for the tcgen05 form,
  void* split;    // [2, M, RP]: down x as hi and lo parts, and
  float* factor;  // [M]: what a row's product with `up` is multiplied by
  int boxes;      // y and out have tensor maps
  int64_t x_stride, y_stride, out_stride;
  int M, N, K, S, R, tiles_cap;
  int slices, k_slice;  // K elements per slice, a multiple of 128
  int col_steps;        // 64-column steps per warp in the expand kernel
};

__device__ __forceinline__ const int32_t* plan_rows(const AdapterParams& p) {
  return p.plan + kHeader + 4 * (int64_t)p.tiles_cap;
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0,
                                                        uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
               : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
               : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

// COUNT (4 or 8) consecutive 16-bit elements row[k ..], zeros from `end` on.
template <typename T, bool VEC, int COUNT>
__device__ __forceinline__ void load_run(uint32_t (&r)[COUNT / 2], const T* row, int k, int end) {
  if constexpr (VEC) {
    if constexpr (COUNT == 8) {
      const uint4 u = k < end ? *reinterpret_cast<const uint4*>(row + k) : make_uint4(0, 0, 0, 0);
      r[0] = u.x, r[1] = u.y, r[2] = u.z, r[3] = u.w;
    } else {
      const uint2 u = k < end ? *reinterpret_cast<const uint2*>(row + k) : make_uint2(0, 0);
      r[0] = u.x, r[1] = u.y;
    }
  } else {
    const uint16_t* e = reinterpret_cast<const uint16_t*>(row);
#pragma unroll
    for (int i = 0; i < COUNT / 2; ++i) {
      const uint32_t lo = k + 2 * i < end ? e[k + 2 * i] : 0, hi = k + 2 * i + 1 < end ? e[k + 2 * i + 1] : 0;
      r[i] = lo | hi << 16;
    }
  }
}

// fp16 has 5 exponent bits: the power of two that brings a row's largest |v| into [1, 2)
// (`down`), and what undoes it (returned).  1 for rows of zeros and of infinities.
__device__ __forceinline__ float fp16_room(float top, float& down) {
  const bool some = top > 0.f && top < __int_as_float(0x7f800000);
  const int e = some ? max(ilogbf(top), -100) : 0;
  down = scalbnf(1.f, -e);
  return scalbnf(1.f, e);
}

// v = hi + lo in T (lo the rounding error of hi, itself rounded).
template <typename T>
__device__ __forceinline__ void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
  const T ah = narrow<T>(a), bh = narrow<T>(b);
  const float al = a - widen<T>(ah), bl = b - widen<T>(bh);
  // An infinity has no remainder (inf - inf would make a NaN of it).
  const T parts[4] = {ah, bh, narrow<T>(isfinite(a) ? al : 0.f), narrow<T>(isfinite(b) ? bl : 0.f)};
  hi = *reinterpret_cast<const uint32_t*>(&parts[0]);
  lo = *reinterpret_cast<const uint32_t*>(&parts[2]);
}

// v = down x for 16 rows of a tile (a tile of 128 takes eight CTAs, blockIdx.z).  The warps
// share K; a warp's steps are 32 elements: lane (g, t) holds elements 8t .. 8t + 7 of rows g
// and g + 8 of x and of row g of each 8-row block of down, two MMAs per block.  Nothing is
// shared between warps until their sums are added in shared memory.
//
// SPLIT: all of K, 8 warps; the sums are complete, and go out as the two 16-bit parts that
// the tcgen05 form takes.  Else one slice of K, 4 warps; its sums go out in fp32.
constexpr int shrink_warps(bool split) { return split ? 8 : 4; }
constexpr int shrink_shared(int rp, bool split) { return (shrink_warps(split) - 1) * 16 * rp * 4; }

template <typename T, int RP, bool VEC, bool SPLIT>
__global__ void __launch_bounds__(32 * shrink_warps(SPLIT)) adapter_shrink_kernel(const AdapterParams p) {
  constexpr int WK = shrink_warps(SPLIT), NT = RP / 8;
  extern __shared__ float part[];  // [WK - 1, 16 * RP]
  griddep_enter();
  if ((int)blockIdx.x >= p.plan[0]) return;
  int4 tile = plan_tiles(p.plan)[blockIdx.x];
  tile.y += blockIdx.z * 16, tile.z -= blockIdx.z * 16;
  if (tile.x < 0 || tile.z <= 0) return;
  const int lane = threadIdx.x & 31, wk = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int32_t* order = plan_rows(p) + tile.y;
  const T* rows[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = g + 8 * h;
    rows[h] = i < tile.z ? reinterpret_cast<const T*>(p.x) + order[i] * p.x_stride : nullptr;
  }
  const T* down = reinterpret_cast<const T*>(p.down) + (int64_t)tile.x * p.R * p.K;
  const int k0 = SPLIT ? 0 : blockIdx.y * p.k_slice, k1 = SPLIT ? p.K : min(p.K, k0 + p.k_slice);
  float acc[NT][4] = {};
  constexpr int UNROLL = RP <= 64 ? 4 : 2;  // steps whose loads go out together
#pragma unroll UNROLL
  for (int k = k0 + wk * 32; k < k1; k += WK * 32) {
    const int e = k + 8 * t;
    uint32_t xa[2][4], db[NT][4];
#pragma unroll
    for (int h = 0; h < 2; ++h) load_run<T, VEC, 8>(xa[h], rows[h], e, rows[h] ? k1 : 0);
#pragma unroll
    for (int j = 0; j < NT; ++j)
      load_run<T, VEC, 8>(db[j], down + (int64_t)(j * 8 + g) * p.K, e, j * 8 + g < p.R ? k1 : 0);
#pragma unroll
    for (int j = 0; j < NT; ++j) {
      const uint32_t a0[4] = {xa[0][0], xa[1][0], xa[0][1], xa[1][1]};
      const uint32_t a1[4] = {xa[0][2], xa[1][2], xa[0][3], xa[1][3]};
      mma16816<T>(acc[j], a0, db[j][0], db[j][1]);
      mma16816<T>(acc[j], a1, db[j][2], db[j][3]);
    }
  }
  if (wk > 0) {
    float* mine = part + (wk - 1) * 16 * RP;
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) mine[(j * 4 + e) * 32 + lane] = acc[j][e];
  }
  __syncthreads();
  if (wk > 0) return;
#pragma unroll
  for (int w = 0; w < WK - 1; ++w)
#pragma unroll
    for (int j = 0; j < NT; ++j)
#pragma unroll
      for (int e = 0; e < 4; ++e) acc[j][e] += part[w * 16 * RP + (j * 4 + e) * 32 + lane];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = g + 8 * h;
    if constexpr (SPLIT) {
      float down_by = 1.f, factor = p.scale[tile.x];
      if constexpr (std::is_same<T, __half>::value) {
        float top = 0.f;
#pragma unroll
        for (int j = 0; j < NT; ++j) top = fmaxf(top, fmaxf(fabsf(acc[j][2 * h]), fabsf(acc[j][2 * h + 1])));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        factor *= fp16_room(top, down_by);
      }
      if (i >= tile.z) continue;
      if (t == 0) p.factor[tile.y + i] = factor;
      T* dst = reinterpret_cast<T*>(p.split) + (int64_t)(tile.y + i) * RP + 2 * t;
#pragma unroll
      for (int j = 0; j < NT; ++j) {
        uint32_t hi, lo;
        split2<T>(acc[j][2 * h] * down_by, acc[j][2 * h + 1] * down_by, hi, lo);
        *reinterpret_cast<uint32_t*>(dst + j * 8) = hi;
        *reinterpret_cast<uint32_t*>(dst + (int64_t)p.M * RP + j * 8) = lo;
      }
    } else {
      if (i >= tile.z) continue;
      float* dst = p.v + ((int64_t)blockIdx.y * p.M + tile.y + i) * RP + 2 * t;
#pragma unroll
      for (int j = 0; j < NT; ++j) *reinterpret_cast<float2*>(dst + j * 8) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
    }
  }
}

// out = y + scale * up v for tiles of kFewRows rows, the single-token case: a thread has
// pairs of columns, reads their rows of `up` 16 bytes at a time (requested before v is
// there, which nothing but the sum over the slices separates from the kernel's start) and
// adds up the products in fp32.  32 requests of one token, 4096 -> 22016, rank 16: 17 us
// with the matrix instructions of the other form, whose loads depend on one another.
template <typename T, int RP>
__global__ void __launch_bounds__(128) adapter_expand_few_kernel(const AdapterParams p) {
  constexpr int PAIRS = RP == 16 ? 2 : 1, PIECES = RP / 8;
  __shared__ float v[kFewRows * RP];
  griddep_enter();
  if ((int)blockIdx.y >= p.plan[0]) return;
  const int4 tile = plan_tiles(p.plan)[blockIdx.y];
  if (tile.x < 0 && p.out == p.y) return;
  const T* up = reinterpret_cast<const T*>(p.up) + (int64_t)max(tile.x, 0) * p.N * p.R;
  const int32_t* order = plan_rows(p) + tile.y;
  const int begin = blockIdx.x * p.col_steps * 256, end = min(p.N, begin + p.col_steps * 256);
  const int pieces = tile.x >= 0 ? p.R / 8 : 0;
  for (int n0 = begin; n0 < end; n0 += 256 * PAIRS) {
    Raw8<T> w[PAIRS][2][PIECES];
    uint32_t yv[PAIRS][kFewRows];
#pragma unroll
    for (int c = 0; c < PAIRS; ++c) {
      const int n = n0 + 2 * (threadIdx.x + 128 * c);
      if (n >= end) continue;
#pragma unroll
      for (int e = 0; e < 2; ++e)
#pragma unroll
        for (int k = 0; k < PIECES; ++k)
          if (k < pieces) w[c][e][k].load(up + (int64_t)(n + e) * p.R + 8 * k);
#pragma unroll
      for (int r = 0; r < kFewRows; ++r)
        if (r < tile.z) yv[c][r] = *reinterpret_cast<const uint32_t*>(reinterpret_cast<const T*>(p.y) + order[r] * p.y_stride + n);
    }
    if (n0 == begin) {
      for (int i = threadIdx.x; i < tile.z * RP; i += 128) {
        float a = 0.f;
        for (int s = 0; tile.x >= 0 && s < p.slices; s += 8) {  // eight loads at a time, added in order
          float part[8];
#pragma unroll
          for (int u = 0; u < 8; ++u)
            part[u] = s + u < p.slices ? p.v[((int64_t)(s + u) * p.M + tile.y) * RP + i] : 0.f;
#pragma unroll
          for (int u = 0; u < 8; ++u) a += part[u];
        }
        v[i] = tile.x >= 0 ? a * p.scale[tile.x] : 0.f;
      }
      __syncthreads();
    }
#pragma unroll
    for (int c = 0; c < PAIRS; ++c) {
      const int n = n0 + 2 * (threadIdx.x + 128 * c);
      if (n >= end) continue;
#pragma unroll
      for (int r = 0; r < kFewRows; ++r) {
        if (r >= tile.z) break;
        float2 a = make_float2(0.f, 0.f);
#pragma unroll
        for (int k = 0; k < PIECES; ++k) {
          if (k >= pieces) break;
          float f[8], g[8];
          w[c][0][k].get(f);
          w[c][1][k].get(g);
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float x = v[r * RP + 8 * k + i];
            a.x = fmaf(x, f[i], a.x), a.y = fmaf(x, g[i], a.y);
          }
        }
        const float2 y = unpack16<T>(yv[c][r]);
        *reinterpret_cast<uint32_t*>(reinterpret_cast<T*>(p.out) + order[r] * p.out_stride + n) =
            pieces > 0 ? pack16<T>(y.x + a.x, y.y + a.y) : yv[c][r];
      }
    }
  }
}

// out = y + scale * up v.  A warp keeps the split v of 16 rows (a tile of 128 takes eight
// CTAs, blockIdx.z) in registers and walks col_steps steps of 64 columns, four warps side by
// side; the columns of a step are dealt so that lane (g, t) ends up with columns 8t .. 8t +
// 7 and 32 + 8t .. 32 + 8t + 7 of rows g and g + 8: a quad's 16-byte pieces of y and out lie
// side by side.
template <typename T, int RP, bool VEC>
__global__ void __launch_bounds__(128) adapter_expand_kernel(const AdapterParams p) {
  constexpr int KS = RP / 16;
  griddep_enter();
  if ((int)blockIdx.y >= p.plan[0]) return;
  int4 tile = plan_tiles(p.plan)[blockIdx.y];
  tile.y += blockIdx.z * 16, tile.z -= blockIdx.z * 16;
  if (tile.z <= 0 || (tile.x < 0 && p.out == p.y)) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int32_t* order = plan_rows(p) + tile.y;
  int64_t row[2];
  uint32_t hi[KS][4], lo[KS][4];
  float factor[2];
  const float scale = tile.x >= 0 ? p.scale[tile.x] : 0.f;
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = g + 8 * h;
    row[h] = i < tile.z ? order[i] : -1;
    float4 v[KS];
    float top = 0.f;
#pragma unroll
    for (int k = 0; k < KS; ++k) v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
    if (i < tile.z && tile.x >= 0) {
      const float* src = p.v + (int64_t)(tile.y + i) * RP + 4 * t;
      constexpr int U = KS <= 2 ? 4 : 1;  // slices whose loads go out together
      for (int s = 0; s < p.slices; s += U, src += U * (int64_t)p.M * RP) {
        float4 a[U][KS];
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int k = 0; k < KS; ++k)
            a[u][k] = s + u < p.slices ? *reinterpret_cast<const float4*>(src + u * (int64_t)p.M * RP + 16 * k)
                                       : make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
          for (int k = 0; k < KS; ++k) v[k].x += a[u][k].x, v[k].y += a[u][k].y, v[k].z += a[u][k].z, v[k].w += a[u][k].w;
      }
    }
    factor[h] = scale;
    if constexpr (std::is_same<T, __half>::value) {
#pragma unroll
      for (int k = 0; k < KS; ++k)
        top = fmaxf(fmaxf(top, fmaxf(fabsf(v[k].x), fabsf(v[k].y))), fmaxf(fabsf(v[k].z), fabsf(v[k].w)));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      float down;
      factor[h] = scale * fp16_room(top, down);
#pragma unroll
      for (int k = 0; k < KS; ++k) v[k].x *= down, v[k].y *= down, v[k].z *= down, v[k].w *= down;
    }
#pragma unroll
    for (int k = 0; k < KS; ++k) {
      split2<T>(v[k].x, v[k].y, hi[k][h], lo[k][h]);
      split2<T>(v[k].z, v[k].w, hi[k][2 + h], lo[k][2 + h]);
    }
  }
  const T* up = reinterpret_cast<const T*>(p.up) + (int64_t)max(tile.x, 0) * p.N * p.R;
  const int span = 4 * 64;
  for (int step = 0; step < p.col_steps; ++step) {
    const int n0 = (blockIdx.x * p.col_steps + step) * span + warp * 64;
    if (n0 >= p.N) break;
    const int n = n0 + 8 * t;
    uint32_t yv[2][2][4];
#pragma unroll
    for (int h = 0; h < 2; ++h)
#pragma unroll
      for (int c = 0; c < 2; ++c)
        load_run<T, VEC, 8>(yv[h][c], reinterpret_cast<const T*>(p.y) + row[h] * p.y_stride, n + 32 * c,
                            row[h] >= 0 ? p.N : 0);
    float acc[8][4] = {};
    if (tile.x >= 0) {
#pragma unroll
      for (int k = 0; k < KS; ++k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int col = n0 + 32 * (j >> 2) + 8 * (g >> 1) + 2 * (j & 3) + (g & 1);
          uint32_t b[2];
          load_run<T, VEC, 4>(b, up + (int64_t)col * p.R, 16 * k + 4 * t, col < p.N ? p.R : 0);
          mma16816<T>(acc[j], hi[k], b[0], b[1]);
          mma16816<T>(acc[j], lo[k], b[0], b[1]);
        }
      }
    }
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      if (row[h] < 0) continue;
      T* dst = reinterpret_cast<T*>(p.out) + row[h] * p.out_stride;
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        const T* yt = reinterpret_cast<const T*>(yv[h][c]);
        T o[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
          const float d = acc[4 * c + i / 2][2 * h + (i & 1)];
          o[i] = tile.x >= 0 ? narrow<T>(fmaf(factor[h], d, widen<T>(yt[i]))) : yt[i];
        }
        if constexpr (VEC) {
          if (n + 32 * c < p.N) *reinterpret_cast<uint4*>(dst + n + 32 * c) = *reinterpret_cast<const uint4*>(o);
        } else {
#pragma unroll
          for (int i = 0; i < 8; ++i)
            if (n + 32 * c + i < p.N) dst[n + 32 * c + i] = o[i];
        }
      }
    }
  }
}

// The same for tiles of 128 rows on the tcgen05 tensor cores: D[128 rows, 128 columns] =
// V up^T, with V = hi + lo kept in shared memory as two K-major operands and the rows of
// `up` as the other, brought by TMA, two products into one accumulator.
//
// With the products out of the way the kernel is what its traffic makes it: y in, out out.
// Both go through a ring of stages in shared memory, several steps ahead, where the
// accumulator's thread of a row (as tensor memory has it) adds its columns in place.  32
// rows that follow one another, as a request's do, come and go as boxes by TMA; others
// through 16-byte asynchronous copies and coalesced stores.  4864 x 32768, rank 64, y in
// and out alone: 167 us by the warps' own loads and stores, 294 us by a bulk copy of 256
// bytes per row (about 30 cycles each), 99 us for a plain copy of the same bytes.
// 8 epilogue warps, four a step (32 rows each), alternating; a producer warp for y, one for
// V and up, an MMA issuer; two accumulators.
template <int RP>
struct ExpandCfg {
  static constexpr int SUB = RP > 64 ? 2 : 1;          // 64-wide K tiles of 128-byte rows
  static constexpr int TILE_BYTES = SUB * 128 * 128;   // 128 rows
  static constexpr int RING = 2;
  static constexpr int Y_BYTES = 2 * 128 * 128;        // 128 rows of y in two 64-column tiles, swizzled
  static constexpr int FIT = (226 * 1024 - 512 - (2 + RING) * TILE_BYTES) / Y_BYTES;
  static constexpr int Y_RING = FIT > 4 ? 4 : FIT;
  static constexpr int SMEM = 1024 + (2 + RING) * TILE_BYTES + Y_RING * Y_BYTES;
  static constexpr int THREADS = 32 * 11;
  static_assert(Y_RING >= 3, "a step under way for each half of the epilogue and one behind them");
};
constexpr int kSiteAdapter = 310;

template <typename T, int RP>
__global__ void __launch_bounds__(ExpandCfg<RP>::THREADS, 1)
    adapter_expand128_kernel(const __grid_constant__ CUtensorMap tm_up, const __grid_constant__ CUtensorMap tm_v,
                             const __grid_constant__ CUtensorMap tm_y, const __grid_constant__ CUtensorMap tm_out,
                             const AdapterParams p) {
  using C = ExpandCfg<RP>;
  constexpr int RING = C::RING, Y_RING = C::Y_RING;
  extern __shared__ uint8_t smem_raw[];
  __shared__ __align__(8) uint64_t full[RING], empty[RING], d_full[2], d_empty[2], y_full[Y_RING], y_empty[Y_RING];
  __shared__ __align__(8) uint64_t v_ready, drained;
  __shared__ uint32_t tmem_holder;
  uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  uint8_t* ring = smem + 2 * C::TILE_BYTES;
  uint8_t* y_ring = ring + RING * C::TILE_BYTES;
  const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
  constexpr int kYProducer = 8, kProducer = 9, kIssuer = 10;
  if (warp == kIssuer) {
    tmem_alloc(&tmem_holder, 256);
    tmem_relinquish();
  }
  if (threadIdx.x == 0) {
    for (int i = 0; i < RING; ++i) {
      mbar_init(&full[i], 1);
      mbar_init(&empty[i], 1);
    }
    for (int i = 0; i < Y_RING; ++i) {
      mbar_init(&y_full[i], 33);  // the producer's lanes, and its box bytes
      mbar_init(&y_empty[i], 4);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&d_full[i], 1);
      mbar_init(&d_empty[i], 4);
    }
    mbar_init(&v_ready, 1);
    mbar_init(&drained, 1);
    fence_barrier_init();
    prefetch_tensormap(&tm_up);
    prefetch_tensormap(&tm_v);
    prefetch_tensormap(&tm_y);
    prefetch_tensormap(&tm_out);
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  griddep_enter();
  const uint32_t tmem = tmem_holder;
  const bool have = (int)blockIdx.y < p.plan[0];
  const int4 tile = have ? plan_tiles(p.plan)[blockIdx.y] : make_int4(-1, 0, 0, 0);
  const bool adapted = tile.x >= 0;
  const int begin = blockIdx.x * p.col_steps * 128, end = min(p.N, begin + p.col_steps * 128);
  const int steps = have && !(tile.x < 0 && p.out == p.y) ? (end - begin + 127) / 128 : 0;
  const int32_t* order = plan_rows(p) + tile.y;
  bool ok = true;
  // 32 rows of the tile (quarter q) as a box: all there, one after the other.
  const auto boxed = [&](int q) {
    return p.boxes && 32 * q + 32 <= tile.z && order[32 * q + 31] - order[32 * q] == 31;
  };
  if (warp == kYProducer) {
    int at[4];  // a quarter's first row if it is a box; else -1
    const T* rows[4];
    int boxes = 0;
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      // A box may bring rows behind the tile's, which count for nothing, but not many.
      const int n = min(32, tile.z - 32 * q);
      at[q] = steps > 0 && p.boxes && n >= 16 && order[32 * q + n - 1] - order[32 * q] == n - 1 ? order[32 * q] : -1;
      boxes += at[q] >= 0;
      const int r = 32 * q + lane;
      rows[q] = steps > 0 && at[q] < 0 && r < tile.z ? reinterpret_cast<const T*>(p.y) + order[r] * p.y_stride : nullptr;
    }
    int issued = 0;
    for (int i = 0; i < steps; ++i) {
      const int slot = i % Y_RING, col = begin + 128 * i;
      ok = i < Y_RING || mbar_wait(&y_empty[slot], (i / Y_RING - 1) & 1, kSiteAdapter + 7);
      if (!(ok = __all_sync(0xffffffffu, ok))) break;
      uint8_t* stage = y_ring + slot * C::Y_BYTES;
      if (lane == 0) {
        mbar_arrive_expect_tx(&y_full[slot], boxes * 2 * 32 * 128);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          if (at[q] >= 0)
            for (int c = 0; c < 2; ++c)
              tma_load_2d(stage + c * (128 * 128) + q * (32 * 128), &tm_y, col + 64 * c, at[q], &y_full[slot]);
      }
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        if (at[q] >= 0 || 32 * q >= tile.z) continue;
        for (int r = 0; r < min(32, tile.z - 32 * q); r += 2) {  // 16 lanes a row
          const int mine = r + (lane >> 4), piece = lane & 15;
          const T* src = reinterpret_cast<const T*>(__shfl_sync(0xffffffffu, (unsigned long long)rows[q], mine));
          const bool there = src != nullptr && col + 8 * piece < end;
          copy16_or_zero(smem_u32(stage) + (piece >> 3) * (128 * 128) + (32 * q + mine) * 128 + (((piece & 7) ^ (mine & 7)) << 4),
                         there ? src + col + 8 * piece : reinterpret_cast<const T*>(p.y), there);
        }
      }
      copy16_arrive(&y_full[slot]);
      ++issued;
    }
    // Never leave the CTA with copies still landing in shared memory.
    for (int i = issued > Y_RING ? issued - Y_RING : 0; i < issued; ++i)
      mbar_wait(&y_full[i % Y_RING], (i / Y_RING) & 1, kSiteAdapter + 8);
  } else if (warp == kProducer) {
    if (lane == 0 && adapted && steps > 0) {
      // Rows behind the tile's are another's, and nothing reads their products.
      mbar_arrive_expect_tx(&v_ready, 2 * C::TILE_BYTES);
      for (int part = 0; part < 2; ++part)
        for (int c = 0; c < C::SUB; ++c)
          tma_load_3d(smem + part * C::TILE_BYTES + c * (128 * 128), &tm_v, 64 * c, tile.y, part, &v_ready);
      int issued = 0;
      for (int i = 0; i < steps; ++i) {
        const int slot = i % RING;
        if (i >= RING && !mbar_wait(&empty[slot], (i / RING - 1) & 1, kSiteAdapter)) break;
        mbar_arrive_expect_tx(&full[slot], C::TILE_BYTES);
        for (int c = 0; c < C::SUB; ++c)
          tma_load_3d(ring + slot * C::TILE_BYTES + c * (128 * 128), &tm_up, 64 * c, begin + 128 * i, tile.x, &full[slot]);
        ++issued;
      }
      for (int i = issued > RING ? issued - RING : 0; i < issued; ++i)
        mbar_wait(&full[i % RING], (i / RING) & 1, kSiteAdapter + 1);
      mbar_wait(&v_ready, 0, kSiteAdapter + 1);
    }
  } else if (warp == kIssuer) {
    if (lane == 0 && adapted && steps > 0) {
      const uint64_t hi = smem_desc_sw128(smem_u32(smem)), lo = smem_desc_sw128(smem_u32(smem) + C::TILE_BYTES);
      const uint64_t up0 = smem_desc_sw128(smem_u32(ring));
      int slot = 0;
      uint32_t lap = 0;
      ok = mbar_wait(&v_ready, 0, kSiteAdapter + 2);
      for (int i = 0; i < steps && ok; ++i) {
        ok = mbar_wait(&full[slot], lap, kSiteAdapter + 3) &&
             (i < 2 || mbar_wait(&d_empty[i & 1], ((i >> 1) - 1) & 1, kSiteAdapter + 4));
        if (!ok) break;
        tc_fence_after();
        const uint64_t up = up0 + (uint32_t)slot * (C::TILE_BYTES >> 4);
#pragma unroll
        for (int k = 0; k < RP / 16; ++k) {
          const uint32_t at = (k / 4) * (128 * 128 / 16) + (k % 4) * 2;
          mma16_ss(tmem + (i & 1) * 128, hi + at, up + at, idesc_16<T>(128, false), k > 0);
        }
#pragma unroll
        for (int k = 0; k < RP / 16; ++k) {
          const uint32_t at = (k / 4) * (128 * 128 / 16) + (k % 4) * 2;
          mma16_ss(tmem + (i & 1) * 128, lo + at, up + at, idesc_16<T>(128, false), 1);
        }
        mma_commit(&empty[slot]);
        mma_commit(&d_full[i & 1]);
        if (++slot == RING) slot = 0, lap ^= 1;
      }
      mma_commit(&drained);
      mbar_wait(&drained, 0, kSiteAdapter + 5);  // nothing in flight reads shared memory after this
    }
  } else {
    const int turn = warp >> 2, quarter = warp & 3, row = quarter * 32 + lane;
    const bool idle = quarter * 32 >= tile.z, box = steps > 0 && boxed(quarter);
    const float factor = adapted && row < tile.z ? p.factor[tile.y + row] : 0.f;
    const int mine = steps > 0 && row < tile.z ? order[row] : -1;
    int sent = -1;  // the slot whose box may still be on its way out
    for (int i = turn; i < steps; i += 2) {
      const int slot = i % Y_RING, col = begin + 128 * i;
      ok = ok && mbar_wait(&y_full[slot], (i / Y_RING) & 1, kSiteAdapter + 9);
      if (adapted) ok = ok && mbar_wait(&d_full[turn], (i >> 1) & 1, kSiteAdapter + 6);
      ok = __all_sync(0xffffffffu, ok);
      uint8_t* stage = y_ring + slot * C::Y_BYTES;
      if (adapted && !idle) {
        tc_fence_after();
        const uint32_t d_at = tmem + ((uint32_t)quarter << 21) + turn * 128;
        uint32_t d[2][32];
        tmem_ld32(d_at, d[0]);
#pragma unroll
        for (int c = 0; c < 4; ++c) {  // 32 columns: the next accumulators are read under this sum
          T* piece[4];
          Raw8<T> y[4];
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            piece[e] = reinterpret_cast<T*>(stage + (c >> 1) * (128 * 128) + row * 128 + (((4 * (c & 1) + e) ^ (row & 7)) << 4));
            y[e].load(piece[e]);
          }
          tmem_wait_ld32(d[c & 1]);
          if (c < 3) tmem_ld32(d_at + 32 * (c + 1), d[(c + 1) & 1]);
#pragma unroll
          for (int e = 0; e < 4; ++e) {
            float v[8];
            y[e].get(v);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = fmaf(factor, __uint_as_float(d[c & 1][8 * e + k]), v[k]);
            y[e].set(v);
            y[e].store(piece[e]);
          }
        }
        tc_fence_before();
        if (box) fence_proxy_async_smem();
      }
      __syncwarp();
      if (adapted && lane == 0) mbar_arrive(&d_empty[turn]);
      if (box) {
        if (lane == 0) {
          for (int c = 0; c < 2; ++c)
            if (col + 64 * c < end)
              tma_store_2d(&tm_out, smem_u32(stage + c * (128 * 128) + quarter * (32 * 128)), col + 64 * c, order[32 * quarter]);
          bulk_commit_group();
          bulk_wait_group_read_1();  // the box of the step before has been read: its slot is free
          if (sent >= 0) mbar_arrive(&y_empty[sent]);
        }
        sent = slot;
      } else {
        for (int r = 0; !idle && r < min(32, tile.z - 32 * quarter); r += 2) {  // 16 lanes a row
          const int rr = r + (lane >> 4), piece = lane & 15;
          const int to = __shfl_sync(0xffffffffu, mine, rr);
          if (to < 0 || col + 8 * piece >= end) continue;
          *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.out) + to * p.out_stride + col + 8 * piece) =
              *reinterpret_cast<const uint4*>(stage + (piece >> 3) * (128 * 128) + (32 * quarter + rr) * 128 + (((piece & 7) ^ (rr & 7)) << 4));
        }
        // The slot's next rows may come as a box: behind what was read and written here.
        fence_proxy_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&y_empty[slot]);
      }
    }
    if (box && lane == 0) bulk_wait_group_all();
    tc_fence_before();
  }
  __syncthreads();
  if (warp == kIssuer) tmem_dealloc(tmem, 256);
}

int padded_rank(int64_t R) { return R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128; }

// Slices of K of the shrink kernel: enough for two CTAs per SM, none shorter than 128
// elements (one 32-element step of each of four warps), at most 32 (the expand kernel
// adds them up).  A function of the sizes alone, so the workspace can be sized first.
constexpr int kSmsPlanned = 148;
constexpr int part_rows(int tile) { return tile < 16 ? tile : 16; }
int k_slices(int64_t M, int64_t K, int64_t S, int tile, int* k_slice) {
  const int64_t tiles = ceil_div(M, part_rows(tile)) + (S < M ? S : M) / 2;
  int64_t slices = ceil_div(2 * kSmsPlanned, tiles);
  slices = slices > ceil_div(K, 128) ? ceil_div(K, 128) : slices;
  slices = slices > 32 ? 32 : slices < 1 ? 1 : slices;
  *k_slice = (int)(ceil_div(ceil_div(K, slices), 128) * 128);
  return (int)ceil_div(K, *k_slice);
}

// 256-column steps a CTA walks: 8 CTAs per SM and more before they get longer.
int steps_per_cta(int64_t spans, const AdapterParams& p, int tile, int most) {
  const int64_t tiles = ceil_div(p.M, tile) + (p.S < p.M ? p.S : p.M) / 2;
  const int64_t steps = spans * tiles / (kSmsPlanned * 8);
  return (int)(steps < 1 ? 1 : steps > most ? most : steps);
}

// The same where an SM holds one CTA: the steps that end first, a CTA's start and end
// taken for two of them.  Up to 16, so that tiles of few rows and of many even out (40 x
// 150 rows 1024 -> 8192: 82 us, 106 us with 64).
int steps_of_one_per_sm(int64_t spans, const AdapterParams& p, int tile) {
  const int64_t tiles = ceil_div(p.M, tile) + (p.S < p.M ? p.S : p.M) / 2;
  int64_t best = INT64_MAX;
  int steps = 1;
  for (int n = 1; n <= 16; ++n) {
    const int64_t cost = ceil_div(tiles * ceil_div(spans, n), kSmsPlanned) * (n + 2);
    if (cost < best) best = cost, steps = n;
  }
  return steps;
}

template <typename T, int RP, bool VEC>
cudaError_t launch_adapter(AdapterParams p, const CUtensorMap* maps, int tile, cudaStream_t stream) {
  const unsigned parts = tile == 128 ? 8 : 1;  // 16-row parts of a tile
  if constexpr (VEC) {
    if (maps != nullptr) {
      using C = ExpandCfg<RP>;
      cudaError_t e = ensure_smem_limit<adapter_shrink_kernel<T, RP, VEC, true>>(shrink_shared(RP, true));
      if (e != cudaSuccess) return e;
      e = launch_pdl(adapter_shrink_kernel<T, RP, VEC, true>, dim3(p.tiles_cap, 1, parts), 32 * shrink_warps(true),
                     shrink_shared(RP, true), stream, p);
      if (e != cudaSuccess) return e;
      e = ensure_smem_limit<adapter_expand128_kernel<T, RP>>(C::SMEM);
      if (e != cudaSuccess) return e;
      const int64_t spans = ceil_div(p.N, 128);
      p.col_steps = steps_of_one_per_sm(spans, p, tile);
      return launch_pdl(adapter_expand128_kernel<T, RP>, dim3((unsigned)ceil_div(spans, p.col_steps), p.tiles_cap),
                        C::THREADS, C::SMEM, stream, maps[0], maps[1], maps[2], maps[3], p);
    }
  }
  cudaError_t e = launch_pdl(adapter_shrink_kernel<T, RP, VEC, false>, dim3(p.tiles_cap, p.slices, parts),
                             32 * shrink_warps(false), shrink_shared(RP, false), stream, p);
  if (e != cudaSuccess) return e;
  const int64_t spans = ceil_div(p.N, 256);
  if constexpr (RP <= 64 && VEC) {
    if (tile == kFewRows && p.R % 8 == 0) {
      p.col_steps = RP == 16 ? (steps_per_cta(2 * spans, p, tile, 8) + 1) / 2 * 2 : steps_per_cta(spans, p, tile, 8);
      return launch_pdl(adapter_expand_few_kernel<T, RP>, dim3((unsigned)ceil_div(spans, p.col_steps), p.tiles_cap), 128, 0,
                        stream, p);
    }
  }
  p.col_steps = steps_per_cta(spans, p, part_rows(tile), 8);
  return launch_pdl(adapter_expand_kernel<T, RP, VEC>, dim3((unsigned)ceil_div(spans, p.col_steps), p.tiles_cap, parts),
                    128, 0, stream, p);
}

template <typename T, bool VEC>
cudaError_t dispatch(const AdapterParams& p, const CUtensorMap* maps, int tile, int rp, cudaStream_t s) {
  switch (rp) {
    case 16: return launch_adapter<T, 16, VEC>(p, maps, tile, s);
    case 32: return launch_adapter<T, 32, VEC>(p, maps, tile, s);
    case 64: return launch_adapter<T, 64, VEC>(p, maps, tile, s);
    default: return launch_adapter<T, 128, VEC>(p, maps, tile, s);
  }
}

// [n, rows, ranks] -> boxes of 64 ranks x 128 rows, 128-byte swizzled (ranks past the end
// read as zero).
int encode_ranks(CUtensorMap* map, int dtype, const void* base, int64_t ranks, int64_t rows, int64_t n) {
  const cuuint64_t dims[3] = {(cuuint64_t)ranks, (cuuint64_t)rows, (cuuint64_t)n};
  const cuuint64_t strides[2] = {(cuuint64_t)(ranks * 2), (cuuint64_t)(rows * ranks * 2)};
  const cuuint32_t box[3] = {64, 128, 1}, estr[3] = {1, 1, 1};
  const CUresult r = tensor_map_encoder()(
      map, dtype == ACTUNE_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3,
      const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? ACTUNE_OK : ACTUNE_ERR_CUDA;
}

// [rows, N] -> boxes of 64 columns x 32 rows, 128-byte swizzled.
int encode_matrix(CUtensorMap* map, int dtype, const void* base, int64_t rows, int64_t N, int64_t stride) {
  const cuuint64_t dims[2] = {(cuuint64_t)N, (cuuint64_t)rows}, strides[1] = {(cuuint64_t)(stride * 2)};
  const cuuint32_t box[2] = {64, 32}, estr[2] = {1, 1};
  const CUresult r = tensor_map_encoder()(
      map, dtype == ACTUNE_DTYPE_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 2,
      const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  return r == CUDA_SUCCESS ? ACTUNE_OK : ACTUNE_ERR_CUDA;
}

bool valid_plan(int64_t M, int64_t S, int tile) {
  return M >= 0 && M <= (1 << 28) && S > 0 && S <= kMaxSlots && (tile == kFewRows || tile == 16 || tile == 128) &&
         max_tiles(M, S, tile) <= 65535;
}

}  // namespace
}  // namespace actune

using namespace actune;

extern "C" {

size_t actune_adapter_plan_size(int64_t M, int64_t S, int tile) {
  if (!valid_plan(M, S, tile)) return 0;
  return 4 * (size_t)(kHeader + 4 * max_tiles(M, S, tile) + M);
}

int actune_adapter_plan(const int32_t* slots, int64_t M, int64_t S, int tile, int32_t* plan, void* stream) {
  if (!valid_plan(M, S, tile) || plan == nullptr || (M > 0 && slots == nullptr)) return ACTUNE_ERR_INVALID_VALUE;
  int num_sms = 0;
  const int rc = serving_device(&num_sms);
  if (rc != ACTUNE_OK) return rc;
  if (!is_aligned(plan, 16) || !is_aligned(slots, 4)) return ACTUNE_ERR_MISALIGNED;
  return serving_status(launch_pdl(adapter_plan_kernel, dim3(1), 1024, (int)(4 * (S + 1)),
                                   reinterpret_cast<cudaStream_t>(stream), slots, (int)M, (int)S, tile,
                                   (int)max_tiles(M, S, tile), plan));
}

size_t actune_adapter_workspace_size(int64_t M, int64_t K, int64_t S, int64_t R, int tile) {
  if (!valid_plan(M, S, tile) || M == 0 || K <= 0 || K > kMostColumns || R <= 0 || R > kMaxRank) return 0;
  int k_slice = 0;
  const size_t rows = (size_t)M * (size_t)padded_rank(R), slices = (size_t)k_slices(M, K, S, tile, &k_slice);
  // The tcgen05 form keeps one sum, as two 16-bit parts, and a factor per row.
  return 4 * (tile == 128 && slices == 1 ? rows + (size_t)M : slices * rows);
}

int actune_adapter_add(const actune_adapter_args* a, void* stream) {
  if (a == nullptr || a->struct_bytes != sizeof(actune_adapter_args)) return ACTUNE_ERR_INVALID_VALUE;
  if (!valid_plan(a->M, a->S, a->tile) || a->N < 0 || a->N > kMostColumns || a->K <= 0 || a->K > kMostColumns ||
      a->R <= 0 || a->R > kMaxRank || a->x_stride < 0 || a->y_stride < 0 || a->out_stride < a->N ||
      (a->dtype != ACTUNE_DTYPE_F16 && a->dtype != ACTUNE_DTYPE_BF16))
    return ACTUNE_ERR_INVALID_VALUE;
  int num_sms = 0;
  const int rc = serving_device(&num_sms);
  if (rc != ACTUNE_OK || a->M == 0 || a->N == 0) return rc;
  if (a->x == nullptr || a->y == nullptr || a->down == nullptr || a->up == nullptr || a->scale == nullptr ||
      a->plan == nullptr || a->out == nullptr || (a->out == a->y && a->out_stride != a->y_stride))
    return ACTUNE_ERR_INVALID_VALUE;
  if (a->workspace == nullptr || a->workspace_bytes < actune_adapter_workspace_size(a->M, a->K, a->S, a->R, a->tile))
    return ACTUNE_ERR_WORKSPACE;
  bool vec = a->K % 8 == 0 && a->N % 8 == 0 && a->R % 4 == 0 && a->x_stride % 8 == 0 && a->y_stride % 8 == 0 &&
             a->out_stride % 8 == 0;
  for (const void* q : {a->x, a->y, a->down, a->up, (const void*)a->out}) {
    if (!is_aligned(q, 2)) return ACTUNE_ERR_MISALIGNED;
    vec = vec && is_aligned(q, 16);
  }
  if (!is_aligned(a->workspace, 16) || !is_aligned(a->plan, 16) || !is_aligned(a->scale, 4))
    return ACTUNE_ERR_MISALIGNED;
  AdapterParams p = {};
  p.x = a->x, p.y = a->y, p.down = a->down, p.up = a->up, p.scale = a->scale, p.plan = a->plan, p.out = a->out;
  p.v = reinterpret_cast<float*>(a->workspace);
  p.x_stride = a->x_stride, p.y_stride = a->y_stride, p.out_stride = a->out_stride;
  p.M = (int)a->M, p.N = (int)a->N, p.K = (int)a->K, p.S = (int)a->S, p.R = (int)a->R;
  p.tiles_cap = (int)max_tiles(a->M, a->S, a->tile);
  p.slices = k_slices(a->M, a->K, a->S, a->tile, &p.k_slice);
  const int rp = padded_rank(a->R);
  auto* cs = reinterpret_cast<cudaStream_t>(stream);
  CUtensorMap both[4] = {};
  const CUtensorMap* maps = nullptr;
  // Rows of `up` a multiple of 16 bytes, as tensor maps want them.  Low ranks with little to
  // read and write are over as soon in 16-row parts, whose many small CTAs wait side by side:
  // 16 x 50 rows 1024 -> 2560 at rank 16, 10.7 us and 11.2 us by tcgen05 (12 x 66 rows 10.3 and
  // 9.7); 16 x 64 rows 1024 -> 8192, 21.5 and 16.8 us; 9 x 209 rows 312 -> 2560 at rank 64,
  // 33.3 and 13.0 us (operands from memory).
  if (vec && a->tile == 128 && a->R % 8 == 0 && (a->R > 32 || a->M * a->N >= 4 << 20)) {
    p.split = a->workspace;
    p.factor = reinterpret_cast<float*>(a->workspace) + a->M * rp;
    int st = encode_ranks(&both[0], a->dtype, a->up, a->R, a->N, a->S);
    if (st == ACTUNE_OK) st = encode_ranks(&both[1], a->dtype, p.split, rp, a->M, 2);
    if (st != ACTUNE_OK) return st;
    maps = both;
    if (p.y_stride > 0) {
      p.boxes = 1;
      st = encode_matrix(&both[2], a->dtype, a->y, a->M, a->N, a->y_stride);
      if (st == ACTUNE_OK) st = encode_matrix(&both[3], a->dtype, a->out, a->M, a->N, a->out_stride);
      if (st != ACTUNE_OK) return st;
    }
  }
  cudaError_t e;
  if (a->dtype == ACTUNE_DTYPE_BF16)
    e = vec ? dispatch<__nv_bfloat16, true>(p, maps, a->tile, rp, cs) : dispatch<__nv_bfloat16, false>(p, maps, a->tile, rp, cs);
  else
    e = vec ? dispatch<__half, true>(p, maps, a->tile, rp, cs) : dispatch<__half, false>(p, maps, a->tile, rp, cs);
  return serving_status(e);
}

}  // extern "C"
