// Norm after a block, gate, residual scale and the norm before the next block, in one
// pass (sm_100a):
//   u = N(x; post)   s = alpha * residual + gate * u   h = N(s; pre) + shift
// Bound by HBM: a row is read once (x, residual) and written once (h, s), 4 * D values
// for about 12 flops each, so a row's values stay in registers between the two norms.
// The second mean square needs s, which needs the first: two reductions over the row
// that cannot be merged.
#include "serving.cuh"

namespace actune {
namespace {

constexpr int kSiteNorm = 320;

struct NormParams {
  const void *x, *residual, *post, *pre, *gate, *shift;
  void *out, *residual_out;
  uint8_t* packed;
  float* scales;
  int64_t x_stride, residual_stride;
  int T, D, post_rows, pre_rows, gate_rows, shift_rows;
  float alpha, eps, one;  // one: what the weights are relative to (gemma 1, else 0)
  float per_d;            // 1 / D
  int bits, codes8;
};

// The modulation row of batch row `row`, where `rows` of them share one (0: all).
template <typename T>
__device__ __forceinline__ const T* modulation(const void* base, int rows, int row, int D) {
  return base == nullptr ? nullptr : reinterpret_cast<const T*>(base) + (rows ? row / rows : 0) * (int64_t)D;
}
// The first row after `row` that reads another one.
__device__ __forceinline__ int modulation_end(const void* base, int rows, int row) {
  return base == nullptr || rows == 0 ? 0x7fffffff : row - row % rows + rows;
}

// Sum over the threads of a row (TPR of them, consecutive).
template <int TPR>
__device__ __forceinline__ float row_sum(float v, float* red) {
#pragma unroll
  for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
  if constexpr (TPR > 32) {
    if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = v;
    __syncthreads();
    v = 0.f;
#pragma unroll
    for (int i = 0; i < TPR / 32; ++i) v += red[i];
  }
  return v;
}

// The group-64 codes of a lane's 8 rounded values; all 32 lanes call together.
__device__ __forceinline__ void emit_codes(const NormParams& p, const float (&v)[8], int64_t element, bool live) {
  uint32_t word[2];
  float scale;
  int width = p.bits;
  if (p.bits == 8) {
    scale = quantize_lane8<8>(v, word);
  } else if (p.codes8) {
    width = 8;
    scale = p.bits == 4 ? quantize_lane8<4, 8>(v, word) : quantize_lane8<2, 8>(v, word);
  } else {
    scale = p.bits == 4 ? quantize_lane8<4>(v, word) : quantize_lane8<2>(v, word);
  }
  if (!live) return;
  uint8_t* dst = p.packed + element / 8 * width;
  if (width == 8) store_lane_codes<8>(dst, word);
  else if (width == 4) store_lane_codes<4>(dst, word);
  else store_lane_codes<2>(dst, word);
  if ((threadIdx.x & 7) == 0) p.scales[element / 64] = scale;
}

// Few rows, or short ones: TPR threads hold a row, CPT chunks of 8 values each.
template <typename T, int TPR, int CPT>
__global__ void __launch_bounds__(TPR > 128 ? TPR : 128) gated_norm_kernel(const NormParams p) {
  constexpr int ROWS = TPR > 128 ? 1 : 128 / TPR;
  __shared__ float red[2][32];
  const int lane = threadIdx.x % TPR;
  const int row = blockIdx.x * ROWS + threadIdx.x / TPR;
  griddep_enter();  // dependent launch: x is the previous kernel's output
  if (row >= p.T) return;  // ROWS > 1 only with one warp per row: no barrier follows
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
  const T* res = reinterpret_cast<const T*>(p.residual) + row * p.residual_stride;
  Raw8<T> xr[CPT], rr[CPT];
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    const int i = (c * TPR + lane) * 8;
    if (i < p.D) {
      xr[c].load(x + i);
      rr[c].load(res + i);
    }
  }
  float v[CPT][8];
  float inv = 1.f;
  if (p.post) {
    float ss = 0.f;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      if ((c * TPR + lane) * 8 >= p.D) continue;
      xr[c].get(v[c]);
#pragma unroll
      for (int k = 0; k < 8; ++k) ss = fmaf(v[c][k], v[c][k], ss);
    }
    inv = rsqrtf(row_sum<TPR>(ss, red[0]) * p.per_d + p.eps);
  }
  const T* post = modulation<T>(p.post, p.post_rows, row, p.D);
  const T* gate = modulation<T>(p.gate, p.gate_rows, row, p.D);
  float ss = 0.f;
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    const int i = (c * TPR + lane) * 8;
    if (i >= p.D) continue;
    float w[8];
    xr[c].get(v[c]);
    Raw8<T> m;
    if (post) {
      m.load(post + i);
      m.get(w);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] = v[c][k] * inv * (p.one + w[k]);
    }
    if (gate) {
      m.load(gate + i);
      m.get(w);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] *= w[k];
    }
    rr[c].get(w);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      v[c][k] = fmaf(p.alpha, w[k], v[c][k]);
      ss = fmaf(v[c][k], v[c][k], ss);
    }
    m.set(v[c]);
    m.store(reinterpret_cast<T*>(p.residual_out) + (int64_t)row * p.D + i);
  }
  inv = rsqrtf(row_sum<TPR>(ss, red[1]) * p.per_d + p.eps);
  const T* pre = modulation<T>(p.pre, p.pre_rows, row, p.D);
  const T* shift = modulation<T>(p.shift, p.shift_rows, row, p.D);
#pragma unroll
  for (int c = 0; c < CPT; ++c) {
    const int i = (c * TPR + lane) * 8;
    const bool live = i < p.D;
    float w[8];
    if (live) {
      Raw8<T> m;
      m.load(pre + i);
      m.get(w);
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] = v[c][k] * inv * (p.one + w[k]);
      if (shift) {
        m.load(shift + i);
        m.get(w);
#pragma unroll
        for (int k = 0; k < 8; ++k) v[c][k] += w[k];
      }
      m.set(v[c]);
      m.store(reinterpret_cast<T*>(p.out) + (int64_t)row * p.D + i);
      m.get(v[c]);  // the codes are those of the rounded values
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) v[c][k] = 0.f;
    }
    if (p.bits) emit_codes(p, v[c], (int64_t)row * p.D + i, live);
  }
}

// Many rows: CTAs stay, each with a run of consecutive rows.  Rows of x and residual come
// into a ring in shared memory by bulk copies, several rows ahead, and the modulations
// stay in registers until a row has others: read again for every row they are more
// instructions than the 16-bit row itself.  What a row costs besides its values (two sums
// over the CTA, waits) bounds it next, so a thread has two chunks: 38911 x 2048 bf16
// 131 us with a CTA a row, 136 us with one chunk a thread, 112 us so (5.7 TB/s, 89% of the
// copy rate); 10000 x 4096 107, 82, 58 us.
template <int THREADS, int CPT>
struct Stream {
  static constexpr int CTAS = THREADS == 64 ? 8 : 640 / THREADS;  // per SM
  static constexpr int RING_BYTES = (160 << 10) / CTAS;
  static constexpr int MOST = 16;  // stages
};

template <typename T, int THREADS, int CPT>
__global__ void __launch_bounds__(THREADS, Stream<THREADS, CPT>::CTAS) gated_norm_stream_kernel(const NormParams p, int stages) {
  extern __shared__ __align__(16) uint8_t ring[];
  __shared__ __align__(8) uint64_t full[Stream<THREADS, CPT>::MOST];
  __shared__ float red[2][32];
  const int lane = threadIdx.x;
  const int each = p.T / (int)gridDim.x, more = p.T - each * (int)gridDim.x;
  const int first = blockIdx.x * each + min((int)blockIdx.x, more);
  const int end = first + each + ((int)blockIdx.x < more);
  const uint32_t row_bytes = p.D * (uint32_t)sizeof(T);
  if (threadIdx.x == 0) {
    for (int i = 0; i < stages; ++i) mbar_init(&full[i], 1);
    fence_barrier_init();
  }
  __syncthreads();
  griddep_enter();  // dependent launch: x is the previous kernel's output
  const auto fetch = [&](int row, int stage) {
    mbar_arrive_expect_tx(&full[stage], 2 * row_bytes);
    uint8_t* at = ring + stage * 2 * row_bytes;
    bulk_load(at, reinterpret_cast<const T*>(p.x) + row * p.x_stride, row_bytes, &full[stage]);
    bulk_load(at + row_bytes, reinterpret_cast<const T*>(p.residual) + row * p.residual_stride, row_bytes, &full[stage]);
  };
  if (threadIdx.x == 0)
    for (int i = 0; i < stages && first + i < end; ++i) fetch(first + i, i);
  T* out = reinterpret_cast<T*>(p.out) + (int64_t)first * p.D + lane * 8;
  T* res_out = reinterpret_cast<T*>(p.residual_out) + (int64_t)first * p.D + lane * 8;
  float in[CPT][8], pre[CPT][8];  // what u's norm and h's norm are multiplied by
  Raw8<T> shift[CPT];
  int until = first;  // the first row with other modulations
  int stage = 0;
  uint32_t lap = 0;
  bool ok = true;
  for (int row = first; row < end; ++row) {
    if (row == until) {
      const T* post_row = modulation<T>(p.post, p.post_rows, row, p.D);
      const T* gate_row = modulation<T>(p.gate, p.gate_rows, row, p.D);
      const T* pre_row = modulation<T>(p.pre, p.pre_rows, row, p.D);
      const T* shift_row = modulation<T>(p.shift, p.shift_rows, row, p.D);
      until = min(min(modulation_end(p.post, p.post_rows, row), modulation_end(p.gate, p.gate_rows, row)),
                  min(modulation_end(p.pre, p.pre_rows, row), modulation_end(p.shift, p.shift_rows, row)));
#pragma unroll
      for (int c = 0; c < CPT; ++c) {
        const int i = (c * THREADS + lane) * 8;
        if (i >= p.D) continue;
        Raw8<T> a, b, g;
        b.load(pre_row + i);
        if (post_row) a.load(post_row + i);
        if (gate_row) g.load(gate_row + i);
        if (shift_row) shift[c].load(shift_row + i);
        b.get(pre[c]);
#pragma unroll
        for (int k = 0; k < 8; ++k) pre[c][k] += p.one, in[c][k] = 1.f;
        float t[8];
        if (post_row) {
          a.get(t);
#pragma unroll
          for (int k = 0; k < 8; ++k) in[c][k] = p.one + t[k];
        }
        if (gate_row) {
          g.get(t);
#pragma unroll
          for (int k = 0; k < 8; ++k) in[c][k] *= t[k];
        }
      }
    }
    ok = ok && mbar_wait(&full[stage], lap, kSiteNorm);
    const T* at = reinterpret_cast<const T*>(ring + stage * 2 * row_bytes);
    float v[CPT][8], w[8];
    Raw8<T> r[CPT];
    float ss = 0.f, inv = 1.f;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      const int i = (c * THREADS + lane) * 8;
      if (i >= p.D) continue;
      Raw8<T> x;
      x.load(at + i);
      r[c].load(at + p.D + i);
      x.get(v[c]);
#pragma unroll
      for (int k = 0; k < 8; ++k) ss = fmaf(v[c][k], v[c][k], ss);
    }
    // The sum's barrier also says that every thread has its part of the row: the stage can
    // be filled again.
    ss = row_sum<THREADS>(ss, red[0]);
    if (p.post) inv = rsqrtf(ss * p.per_d + p.eps);
    if (threadIdx.x == 0 && row + stages < end) fetch(row + stages, stage);
    if (++stage == stages) stage = 0, lap ^= 1;
    ss = 0.f;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      if ((c * THREADS + lane) * 8 >= p.D) continue;
      r[c].get(w);
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        v[c][k] = fmaf(p.alpha, w[k], v[c][k] * inv * in[c][k]);
        ss = fmaf(v[c][k], v[c][k], ss);
      }
      r[c].set(v[c]);
      r[c].store(res_out + c * THREADS * 8);
    }
    inv = rsqrtf(row_sum<THREADS>(ss, red[1]) * p.per_d + p.eps);
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      const int i = (c * THREADS + lane) * 8;
      const bool live = i < p.D;
      if (live) {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[c][k] = v[c][k] * inv * pre[c][k];
        if (p.shift) {
          shift[c].get(w);
#pragma unroll
          for (int k = 0; k < 8; ++k) v[c][k] += w[k];
        }
        r[c].set(v[c]);
        r[c].store(out + c * THREADS * 8);
        r[c].get(v[c]);  // the codes are those of the rounded values
      } else {
#pragma unroll
        for (int k = 0; k < 8; ++k) v[c][k] = 0.f;
      }
      if (p.bits) emit_codes(p, v[c], (int64_t)row * p.D + i, live);
    }
    out += p.D, res_out += p.D;
  }
  // A wait that ran out: never leave the CTA with copies still landing in shared memory.
  if (!ok)
    for (int i = 0; i < stages; ++i) mbar_wait(&full[(stage + i) % stages], lap ^ (stage + i >= stages), kSiteNorm);
}

// Any width, alignment and stride: one CTA per row, a value at a time.  Up to 256 * CPT
// values stay in registers; CPT = 0: read again for each pass.
template <typename T, int CPT>
__global__ void __launch_bounds__(256) gated_norm_any_kernel(const NormParams p) {
  __shared__ float red[2][32];
  griddep_enter();
  const int64_t row = blockIdx.x;
  const T* x = reinterpret_cast<const T*>(p.x) + row * p.x_stride;
  const T* res = reinterpret_cast<const T*>(p.residual) + row * p.residual_stride;
  const T* post = modulation<T>(p.post, p.post_rows, (int)row, p.D);
  const T* gate = modulation<T>(p.gate, p.gate_rows, (int)row, p.D);
  const T* pre = modulation<T>(p.pre, p.pre_rows, (int)row, p.D);
  const T* shift = modulation<T>(p.shift, p.shift_rows, (int)row, p.D);
  T* out = reinterpret_cast<T*>(p.out) + row * p.D;
  T* res_out = reinterpret_cast<T*>(p.residual_out) + row * p.D;
  const auto stream_value = [&](int i, float a, float r, float inv) {
    if (post) a = a * inv * (p.one + widen<T>(post[i]));
    if (gate) a *= widen<T>(gate[i]);
    return fmaf(p.alpha, r, a);
  };
  const auto normed = [&](int i, float s, float inv) {
    const float h = s * inv * (p.one + widen<T>(pre[i]));
    return shift ? h + widen<T>(shift[i]) : h;
  };
  float inv = 1.f, ss = 0.f;
  if constexpr (CPT > 0) {
    T xv[CPT], rv[CPT];
    float v[CPT];
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      const int i = threadIdx.x + c * 256;
      if (i < p.D) xv[c] = x[i], rv[c] = res[i];
    }
    if (post) {
#pragma unroll
      for (int c = 0; c < CPT; ++c) {
        const float a = (int)threadIdx.x + c * 256 < p.D ? widen<T>(xv[c]) : 0.f;
        ss = fmaf(a, a, ss);
      }
      inv = rsqrtf(row_sum<256>(ss, red[0]) * p.per_d + p.eps);
    }
    ss = 0.f;
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      const int i = threadIdx.x + c * 256;
      if (i >= p.D) continue;
      v[c] = stream_value(i, widen<T>(xv[c]), widen<T>(rv[c]), inv);
      ss = fmaf(v[c], v[c], ss);
      res_out[i] = narrow<T>(v[c]);
    }
    inv = rsqrtf(row_sum<256>(ss, red[1]) * p.per_d + p.eps);
#pragma unroll
    for (int c = 0; c < CPT; ++c) {
      const int i = threadIdx.x + c * 256;
      if (i < p.D) out[i] = narrow<T>(normed(i, v[c], inv));
    }
  } else {
    if (post) {
      for (int i = threadIdx.x; i < p.D; i += 256) {
        const float a = widen<T>(x[i]);
        ss = fmaf(a, a, ss);
      }
      inv = rsqrtf(row_sum<256>(ss, red[0]) * p.per_d + p.eps);
    }
    ss = 0.f;
    for (int i = threadIdx.x; i < p.D; i += 256) {
      const float s = stream_value(i, widen<T>(x[i]), widen<T>(res[i]), inv);
      ss = fmaf(s, s, ss);
      res_out[i] = narrow<T>(s);
    }
    const float inv2 = rsqrtf(row_sum<256>(ss, red[1]) * p.per_d + p.eps);
    for (int i = threadIdx.x; i < p.D; i += 256)
      out[i] = narrow<T>(normed(i, stream_value(i, widen<T>(x[i]), widen<T>(res[i]), inv), inv2));
  }
}

template <typename T, int TPR, int CPT>
cudaError_t launch_rows(const NormParams& p, cudaStream_t stream) {
  constexpr int THREADS = TPR > 128 ? TPR : 128;
  return launch_pdl(gated_norm_kernel<T, TPR, CPT>, dim3((unsigned)ceil_div(p.T, THREADS / TPR)), THREADS, 0, stream,
                    p);
}

template <typename T, int THREADS, int CPT>
cudaError_t launch_stream(const NormParams& p, int num_sms, cudaStream_t stream) {
  using S = Stream<THREADS, CPT>;
  const cudaError_t e = ensure_smem_limit<gated_norm_stream_kernel<T, THREADS, CPT>>(S::RING_BYTES);
  if (e != cudaSuccess) return e;
  const int row_bytes = 2 * p.D * (int)sizeof(T), fit = S::RING_BYTES / row_bytes;
  const int stages = fit < S::MOST ? fit : S::MOST;
  return launch_pdl(gated_norm_stream_kernel<T, THREADS, CPT>, dim3((unsigned)(num_sms * S::CTAS)), THREADS,
                    stages * row_bytes, stream, p, stages);
}

template <typename T, int CPT>
cudaError_t launch_any(const NormParams& p, cudaStream_t stream) {
  return launch_pdl(gated_norm_any_kernel<T, CPT>, dim3((unsigned)p.T), 256, 0, stream, p);
}

template <typename T>
cudaError_t launch_norm(const NormParams& p, bool vec, int num_sms, cudaStream_t stream) {
  if (!vec) {
    if (p.D <= 256) return launch_any<T, 1>(p, stream);
    if (p.D <= 1024) return launch_any<T, 4>(p, stream);
    if (p.D <= 2560) return launch_any<T, 10>(p, stream);
    if (p.D <= 8192) return launch_any<T, 32>(p, stream);
    return launch_any<T, 0>(p, stream);
  }
  const int chunks = (p.D + 7) / 8;
  if (p.T >= num_sms * 16) {
    if (chunks <= 32) return launch_rows<T, 32, 1>(p, stream);
    if (chunks <= 64) return launch_rows<T, 32, 2>(p, stream);
    // fp32 rows of up to 2048 carry twice the bytes an instruction, and are as fast without
    // the ring (20000 x 2048: 100 us, 116 us with it; 8000 x 4096: 116 us, 93 us with it).
    if constexpr (sizeof(T) == 4) {
      if (chunks <= 128) return launch_rows<T, 32, 4>(p, stream);
      if (chunks <= 256) return launch_rows<T, 128, 2>(p, stream);
    } else {
      if (chunks <= 128) return launch_stream<T, 64, 2>(p, num_sms, stream);
      if (chunks <= 256) return launch_stream<T, 128, 2>(p, num_sms, stream);
    }
    if (chunks <= 512) return launch_stream<T, 256, 2>(p, num_sms, stream);
    if (chunks <= 1024 && sizeof(T) == 2) return launch_stream<T, 512, 2>(p, num_sms, stream);
  }
  if (chunks <= 128) return launch_rows<T, 128, 1>(p, stream);
  if (chunks <= 256) return launch_rows<T, 128, 2>(p, stream);
  if (chunks <= 512) return launch_rows<T, 512, 1>(p, stream);
  if (chunks <= 1024) return launch_rows<T, 512, 2>(p, stream);
  return launch_rows<T, 512, 4>(p, stream);
}

}  // namespace
}  // namespace actune

extern "C" int actune_gated_norm(const actune_gated_norm_args* a, void* stream) {
  using namespace actune;
  if (a == nullptr || a->struct_bytes != sizeof(actune_gated_norm_args)) return ACTUNE_ERR_INVALID_VALUE;
  if (a->T < 0 || a->T > 0x7fffffff || a->D <= 0 || a->D > (1 << 24) || a->post_rows < 0 || a->pre_rows < 0 ||
      a->gate_rows < 0 || a->shift_rows < 0 || a->x_stride < 0 || a->residual_stride < 0 || !(a->eps >= 0.f) ||
      (a->dtype != ACTUNE_DTYPE_F32 && a->dtype != ACTUNE_DTYPE_F16 && a->dtype != ACTUNE_DTYPE_BF16) ||
      (a->quant_bits != 0 && a->quant_bits != 2 && a->quant_bits != 4 && a->quant_bits != 8) ||
      (a->quant_bits != 0 && a->D % 64 != 0))
    return ACTUNE_ERR_INVALID_VALUE;
  if (a->T > 0 && (a->x == nullptr || a->residual == nullptr || a->pre_weight == nullptr || a->out == nullptr ||
                   a->residual_out == nullptr || (a->quant_bits != 0 && (a->packed == nullptr || a->scales == nullptr))))
    return ACTUNE_ERR_INVALID_VALUE;
  int num_sms = 0;
  const int rc = serving_device(&num_sms);
  if (rc != ACTUNE_OK || a->T == 0) return rc;
  const uintptr_t size = a->dtype == ACTUNE_DTYPE_F32 ? 4 : 2;
  for (const void* q : {a->x, a->residual, a->post_weight, a->pre_weight, a->gate, a->shift,
                        (const void*)a->out, (const void*)a->residual_out})
    if (!is_aligned(q, size)) return ACTUNE_ERR_MISALIGNED;
  if (a->quant_bits != 0 && (!is_aligned(a->packed, 8) || !is_aligned(a->scales, 4) || !is_aligned(a->out, 16)))
    return ACTUNE_ERR_MISALIGNED;
  bool vec = a->D % 8 == 0 && a->D <= 512 * 4 * 8 && a->x_stride % 8 == 0 && a->residual_stride % 8 == 0;
  for (const void* q : {a->x, a->residual, a->post_weight, a->pre_weight, a->gate, a->shift,
                        (const void*)a->out, (const void*)a->residual_out})
    vec = vec && is_aligned(q, 16);
  const auto rows_of = [&](int64_t r) { return (int)(r < a->T ? r : 0); };  // T or more: one row for all
  NormParams p = {a->x, a->residual, a->post_weight, a->pre_weight, a->gate, a->shift, a->out, a->residual_out,
                  a->packed, a->scales, a->x_stride, a->residual_stride, (int)a->T, (int)a->D, rows_of(a->post_rows),
                  rows_of(a->pre_rows), rows_of(a->gate_rows), rows_of(a->shift_rows), a->residual_scale, a->eps,
                  a->gemma ? 1.f : 0.f, 1.f / (float)a->D, vec ? a->quant_bits : 0, a->codes8};
  auto* cs = reinterpret_cast<cudaStream_t>(stream);
  cudaError_t e = a->dtype == ACTUNE_DTYPE_F32   ? launch_norm<float>(p, vec, num_sms, cs)
                  : a->dtype == ACTUNE_DTYPE_F16 ? launch_norm<__half>(p, vec, num_sms, cs)
                                                 : launch_norm<__nv_bfloat16>(p, vec, num_sms, cs);
  if (e == cudaSuccess && a->quant_bits != 0 && !vec)
    e = launch_quantize_group64(a->out, a->dtype, a->T * (a->D / 64), a->quant_bits, a->codes8 != 0, a->packed,
                                a->scales, num_sms, cs);
  return serving_status(e);
}
