// Low-rank adapters of many requests beside a shared projection (sm_100a):
//   out[m] = y[m] + scale[s] * up[s] (down[s] x[m]),   s = slots[m].
//
// plan    rows sorted by adapter into tiles of 16, 32 or 64 rows with one adapter each.
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
#include "serving.cuh"

namespace actune {
namespace {

constexpr int kMaxSlots = 8191;
constexpr int kMaxRank = 128;
constexpr int kHeader = 4;  // plan: tile count, then three padding words

// Tiles of `tile` rows that M rows of S adapters (and of none) can make at most.
inline int64_t max_tiles(int64_t M, int64_t S, int tile) { return M / tile + (S + 1 < M ? S + 1 : M); }

// plan: [kHeader] count; then per tile {slot, first, rows, 0}; then the sorted rows.
__device__ __forceinline__ const int4* plan_tiles(const int32_t* plan) {
  return reinterpret_cast<const int4*>(plan + kHeader);
}

// One CTA.  Stable counting sort: 1024 rows at a time, the warps of a chunk one after
// the other, the lanes of a warp ranked among those of the same slot.
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
  float* v;  // [slices, M, RP] partial sums of down x, rows in plan order
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

// v[slice, position, 0 .. RP) for one tile and one slice of K.  WM warps side by side
// along the rows (16 each) and 4 / WM along K; a warp's K steps are 32 elements: lane
// (g, t) holds elements 8t .. 8t + 7 of rows g and g + 8 of x and of row g of each
// 8-row block of down, two MMAs per block.  Nothing is shared between warps until
// their sums are added in shared memory.
template <typename T, int WM, int RP, bool VEC>
__global__ void __launch_bounds__(128) adapter_shrink_kernel(const AdapterParams p) {
  constexpr int WK = 4 / WM, NT = RP / 8;
  __shared__ float part[WK > 1 ? (WK - 1) * WM * 16 * RP : 1];
  griddep_enter();
  if ((int)blockIdx.x >= p.plan[0]) return;
  const int4 tile = plan_tiles(p.plan)[blockIdx.x];
  if (tile.x < 0) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int wm = warp % WM, wk = warp / WM;
  const int32_t* order = plan_rows(p) + tile.y;
  const T* rows[2];
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = wm * 16 + g + 8 * h;
    rows[h] = i < tile.z ? reinterpret_cast<const T*>(p.x) + order[i] * p.x_stride : nullptr;
  }
  const T* down = reinterpret_cast<const T*>(p.down) + (int64_t)tile.x * p.R * p.K;
  const int k0 = blockIdx.y * p.k_slice, k1 = min(p.K, k0 + p.k_slice);
  float acc[NT][4] = {};
  if (wm * 16 < tile.z) {
#pragma unroll 2
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
  }
  if constexpr (WK > 1) {
    if (wk > 0) {
      float* mine = part + ((wk - 1) * WM + wm) * 16 * RP;
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
        for (int e = 0; e < 4; ++e) acc[j][e] += part[(w * WM + wm) * 16 * RP + (j * 4 + e) * 32 + lane];
  }
#pragma unroll
  for (int h = 0; h < 2; ++h) {
    const int i = wm * 16 + g + 8 * h;
    if (i >= tile.z) continue;
    float* dst = p.v + ((int64_t)blockIdx.y * p.M + tile.y + i) * RP + 2 * t;
#pragma unroll
    for (int j = 0; j < NT; ++j) *reinterpret_cast<float2*>(dst + j * 8) = make_float2(acc[j][2 * h], acc[j][2 * h + 1]);
  }
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

// out = y + scale * up v.  A warp keeps the split v of MW * 16 rows in registers and
// walks col_steps steps of 64 columns; the columns of a step are dealt so that lane
// (g, t) ends up with columns 16t .. 16t + 15 of rows g and g + 8: 32 contiguous bytes
// of y and out.
template <typename T, int WM, int MW, int RP, bool VEC>
__global__ void __launch_bounds__(128) adapter_expand_kernel(const AdapterParams p) {
  constexpr int WN = 4 / WM, KS = RP / 16;
  griddep_enter();
  if ((int)blockIdx.y >= p.plan[0]) return;
  const int4 tile = plan_tiles(p.plan)[blockIdx.y];
  if (tile.x < 0 && p.out == p.y) return;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int g = lane >> 2, t = lane & 3;
  const int wm = warp % WM, wn = warp / WM;
  const int first = wm * MW * 16;
  if (first >= tile.z) return;
  const int32_t* order = plan_rows(p) + tile.y;
  int64_t row[MW][2];
  uint32_t hi[MW][KS][4], lo[MW][KS][4];
  float factor[MW][2];
  const float scale = tile.x >= 0 ? p.scale[tile.x] : 0.f;
#pragma unroll
  for (int m = 0; m < MW; ++m) {
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int i = first + m * 16 + g + 8 * h;
      row[m][h] = i < tile.z ? order[i] : -1;
      float4 v[KS];
      float top = 0.f;
#pragma unroll
      for (int k = 0; k < KS; ++k) v[k] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (i < tile.z && tile.x >= 0) {
        const float* src = p.v + (int64_t)(tile.y + i) * RP + 4 * t;
        for (int s = 0; s < p.slices; ++s, src += (int64_t)p.M * RP)
#pragma unroll
          for (int k = 0; k < KS; ++k) {
            const float4 a = *reinterpret_cast<const float4*>(src + 16 * k);
            v[k].x += a.x, v[k].y += a.y, v[k].z += a.z, v[k].w += a.w;
          }
      }
      factor[m][h] = scale;
      if constexpr (sizeof(T) == 2 && !std::is_same<T, __nv_bfloat16>::value) {
        // fp16 has 5 exponent bits: bring the row's largest |v| into [1, 2) first.
#pragma unroll
        for (int k = 0; k < KS; ++k)
          top = fmaxf(fmaxf(top, fmaxf(fabsf(v[k].x), fabsf(v[k].y))), fmaxf(fabsf(v[k].z), fabsf(v[k].w)));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
        top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
        if (top > 0.f && top < __int_as_float(0x7f800000)) {
          const int e = max(ilogbf(top), -100);
          const float down = scalbnf(1.f, -e);
#pragma unroll
          for (int k = 0; k < KS; ++k) v[k].x *= down, v[k].y *= down, v[k].z *= down, v[k].w *= down;
          factor[m][h] = scale * scalbnf(1.f, e);
        }
      }
#pragma unroll
      for (int k = 0; k < KS; ++k) {
        split2<T>(v[k].x, v[k].y, hi[m][k][h], lo[m][k][h]);
        split2<T>(v[k].z, v[k].w, hi[m][k][2 + h], lo[m][k][2 + h]);
      }
    }
  }
  const T* up = reinterpret_cast<const T*>(p.up) + (int64_t)max(tile.x, 0) * p.N * p.R;
  const int span = WN * 64;
  for (int step = 0; step < p.col_steps; ++step) {
    const int n0 = (blockIdx.x * p.col_steps + step) * span + wn * 64;
    if (n0 >= p.N) break;
    const int n = n0 + 16 * t;
    uint32_t yv[MW][2][2][4];
#pragma unroll
    for (int m = 0; m < MW; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h)
#pragma unroll
        for (int c = 0; c < 2; ++c)
          load_run<T, VEC, 8>(yv[m][h][c], reinterpret_cast<const T*>(p.y) + row[m][h] * p.y_stride, n + 8 * c,
                              row[m][h] >= 0 ? p.N : 0);
    float acc[MW][8][4] = {};
    if (tile.x >= 0) {
#pragma unroll
      for (int k = 0; k < KS; ++k) {
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const int col = n0 + 16 * (g >> 1) + 2 * j + (g & 1);
          uint32_t b[2];
          load_run<T, VEC, 4>(b, up + (int64_t)col * p.R, 16 * k + 4 * t, col < p.N ? p.R : 0);
#pragma unroll
          for (int m = 0; m < MW; ++m) {
            mma16816<T>(acc[m][j], hi[m][k], b[0], b[1]);
            mma16816<T>(acc[m][j], lo[m][k], b[0], b[1]);
          }
        }
      }
    }
#pragma unroll
    for (int m = 0; m < MW; ++m)
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        if (row[m][h] < 0) continue;
        T* dst = reinterpret_cast<T*>(p.out) + row[m][h] * p.out_stride;
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          const T* yt = reinterpret_cast<const T*>(yv[m][h][c]);
          T o[8];
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            const float d = acc[m][4 * c + i / 2][2 * h + (i & 1)];
            o[i] = tile.x >= 0 ? narrow<T>(fmaf(factor[m][h], d, widen<T>(yt[i]))) : yt[i];
          }
          if constexpr (VEC) {
            if (n + 8 * c < p.N) *reinterpret_cast<uint4*>(dst + n + 8 * c) = *reinterpret_cast<const uint4*>(o);
          } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
              if (n + 8 * c + i < p.N) dst[n + 8 * c + i] = o[i];
          }
        }
      }
  }
}

int padded_rank(int64_t R) { return R <= 16 ? 16 : R <= 32 ? 32 : R <= 64 ? 64 : 128; }

// Slices of K of the shrink kernel: enough for two CTAs per SM, none shorter than 128
// elements (one 32-element step of each of four warps), at most 32 (the expand kernel
// adds them up).  A function of the sizes alone, so the workspace can be sized first.
constexpr int kSmsPlanned = 148;
int k_slices(int64_t M, int64_t K, int64_t S, int tile, int* k_slice) {
  const int64_t tiles = ceil_div(M, tile) + (S < M ? S : M) / 2;
  int64_t slices = ceil_div(2 * kSmsPlanned, tiles);
  slices = slices > ceil_div(K, 128) ? ceil_div(K, 128) : slices;
  slices = slices > 32 ? 32 : slices < 1 ? 1 : slices;
  *k_slice = (int)(ceil_div(ceil_div(K, slices), 128) * 128);
  return (int)ceil_div(K, *k_slice);
}

template <typename T, int TILE, int RP, bool VEC>
cudaError_t launch_adapter(AdapterParams p, cudaStream_t stream) {
  constexpr int WM = TILE / 16;
  cudaError_t e = launch_pdl(adapter_shrink_kernel<T, WM, RP, VEC>, dim3(p.tiles_cap, p.slices), 128, 0, stream, p);
  if (e != cudaSuccess) return e;
  // Two 16-row blocks per warp halve the reads of `up`; at rank 128 the split v of one
  // block already takes 64 registers.
  constexpr int MW = TILE >= 32 && RP <= 64 ? 2 : 1;
  constexpr int EWM = TILE / (16 * MW);
  const int64_t spans = ceil_div(p.N, 64 * (4 / EWM));
  int64_t steps = spans * ceil_div(p.M, TILE) / (kSmsPlanned * 8);
  p.col_steps = (int)(steps < 1 ? 1 : steps > 8 ? 8 : steps);
  return launch_pdl(adapter_expand_kernel<T, EWM, MW, RP, VEC>, dim3((unsigned)ceil_div(spans, p.col_steps), p.tiles_cap),
                    128, 0, stream, p);
}

template <typename T, bool VEC>
cudaError_t dispatch(const AdapterParams& p, int tile, int rp, cudaStream_t s) {
#define ACTUNE_ADAPTER(TILE)                                            \
  switch (rp) {                                                         \
    case 16: return launch_adapter<T, TILE, 16, VEC>(p, s);             \
    case 32: return launch_adapter<T, TILE, 32, VEC>(p, s);             \
    case 64: return launch_adapter<T, TILE, 64, VEC>(p, s);             \
    default: return launch_adapter<T, TILE, 128, VEC>(p, s);            \
  }
  if (tile == 16) {
    ACTUNE_ADAPTER(16)
  } else if (tile == 32) {
    ACTUNE_ADAPTER(32)
  }
  ACTUNE_ADAPTER(64)
#undef ACTUNE_ADAPTER
}

bool valid_plan(int64_t M, int64_t S, int tile) {
  return M >= 0 && M <= (1 << 28) && S > 0 && S <= kMaxSlots && (tile == 16 || tile == 32 || tile == 64) &&
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
  if (!valid_plan(M, S, tile) || M == 0 || K <= 0 || K > 0x7fffff00 || R <= 0 || R > kMaxRank) return 0;
  int k_slice = 0;
  return 4 * (size_t)k_slices(M, K, S, tile, &k_slice) * (size_t)M * (size_t)padded_rank(R);
}

int actune_adapter_add(const actune_adapter_args* a, void* stream) {
  if (a == nullptr || a->struct_bytes != sizeof(actune_adapter_args)) return ACTUNE_ERR_INVALID_VALUE;
  if (!valid_plan(a->M, a->S, a->tile) || a->N < 0 || a->N > 0x7fffff00 || a->K <= 0 || a->K > 0x7fffff00 ||
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
  cudaError_t e;
  if (a->dtype == ACTUNE_DTYPE_BF16)
    e = vec ? dispatch<__nv_bfloat16, true>(p, a->tile, rp, cs) : dispatch<__nv_bfloat16, false>(p, a->tile, rp, cs);
  else
    e = vec ? dispatch<__half, true>(p, a->tile, rp, cs) : dispatch<__half, false>(p, a->tile, rp, cs);
  return serving_status(e);
}

}  // extern "C"
