// The global norm over many gradients, and their clipping.
//
//   norm_2 = sqrt(sum x^2)   norm_1 = sum |x|   norm_inf = max |x|   over all tensors
//   x := round(x * min(1, max_norm / (norm_2 + 1e-6)))
//
// A model's gradients are hundreds of tensors of very different sizes, at any alignment when they
// are views of a bucket.  A launch takes all of them: chunks of 32-byte vectors are numbered across
// the tensors, and a grid that fills the chip takes them in turn, so there is no tail per tensor.
// Bound by memory.  Sums are fp64: a value's square is exact there and neither over- nor
// underflows, and what the order of the sum changes is far below the rounding of the result to fp32.  One
// partial per block in a fixed assignment, joined in a fixed order: the same bits every time for the
// same tensors at the same alignment.
#include <cuda_fp16.h>

#include "clip_ops.h"
#include "common.cuh"

namespace oab {
namespace {

constexpr int kThreads = 256;
constexpr int kBlocks = kNumSMs * 8;

template <int CAP>
struct ClipTable {
  int count;
  uint32_t chunks;
  uint32_t chunk_vecs;
  ClipEntry e[CAP];
};

// log2 of the values of a vector
__host__ __device__ __forceinline__ int vec_shift(uint32_t dtype) { return dtype == kClipF32 ? 3 : 4; }
// values in front of the first whole vector
__host__ __device__ __forceinline__ int64_t head_of(const ClipEntry& e) {
  const int sh = vec_shift(e.dtype);
  const int64_t over = (int64_t)((reinterpret_cast<uintptr_t>(e.p) & 31u) >> (5 - sh)), head = over != 0 ? (int64_t(1) << sh) - over : 0;
  return head < e.n ? head : e.n;
}
__host__ __device__ __forceinline__ int64_t vecs_of(const ClipEntry& e) { return (e.n - head_of(e)) >> vec_shift(e.dtype); }

__device__ __forceinline__ float half_to_f32(uint32_t h) { return __half2float(__ushort_as_half((unsigned short)h)); }
__device__ __forceinline__ float load_one(const ClipEntry& e, int64_t i) {
  if (e.dtype == kClipF32) return reinterpret_cast<const float*>(e.p)[i];
  const uint32_t h = reinterpret_cast<const uint16_t*>(e.p)[i];
  return e.dtype == kClipBF16 ? bf16_bits_to_f32(h) : half_to_f32(h);
}
__device__ __forceinline__ void scale_one(const ClipEntry& e, int64_t i, float c) {
  const float x = __fmul_rn(load_one(e, i), c);
  if (e.dtype == kClipF32) reinterpret_cast<float*>(e.p)[i] = x;
  else if (e.dtype == kClipBF16) reinterpret_cast<uint16_t*>(e.p)[i] = (uint16_t)f32_to_bf16_rne_bits(x);
  else reinterpret_cast<__half*>(e.p)[i] = __float2half_rn(x);
}

// kNormInf keeps the bits of the largest |x|: NaN is above infinity there.
template <int NORM>
struct Sum {
  double a = 0.0, b = 0.0;
  uint32_t top = 0;
  __device__ __forceinline__ void take(float x, bool second) {
    if (NORM == kNormInf) {
      const uint32_t u = __float_as_uint(x) & 0x7fffffffu;
      top = u > top ? u : top;
    } else {
      const double d = (double)x;
      double& s = second ? b : a;
      s = NORM == kNormL2 ? __fma_rn(d, d, s) : __dadd_rn(s, fabs(d));
    }
  }
  __device__ __forceinline__ double value() const {
    return NORM == kNormInf ? (double)__uint_as_float(top) : a + b;
  }
};
template <int NORM>
__device__ __forceinline__ double both(double a, double b) {
  if (NORM != kNormInf) return a + b;
  return isnan(a) || isnan(b) ? (double)NAN : fmax(a, b);
}
// over the block; every thread gets it
template <int NORM>
__device__ __forceinline__ double block_join(double v, double* smem) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) v = both<NORM>(v, __shfl_xor_sync(0xffffffffu, v, o));
  __syncthreads();
  if ((threadIdx.x & 31) == 0) smem[threadIdx.x >> 5] = v;
  __syncthreads();
  double r = smem[0];
#pragma unroll
  for (int w = 1; w < kThreads / 32; ++w) r = both<NORM>(r, smem[w]);
  return r;
}

template <int NORM>
__device__ __forceinline__ void take_vec(Sum<NORM>& s, const V8& v, uint32_t dtype) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (dtype == kClipF32) {
      s.take(__uint_as_float(v.w[j]), j & 1);
    } else if (dtype == kClipBF16) {
      s.take(__uint_as_float(v.w[j] << 16), false);
      s.take(__uint_as_float(v.w[j] & 0xffff0000u), true);
    } else {
      s.take(half_to_f32(v.w[j] & 0xffffu), false);
      s.take(half_to_f32(v.w[j] >> 16), true);
    }
  }
}

template <int CAP>
__device__ __forceinline__ const ClipEntry& entry_of(const ClipTable<CAP>& t, uint32_t chunk) {
  int lo = 0, hi = t.count - 1;  // the last tensor whose first chunk is not after this one
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (t.e[mid].first_chunk <= chunk) lo = mid; else hi = mid - 1;
  }
  return t.e[lo];
}

template <int NORM, int CAP>
__global__ void __launch_bounds__(kThreads)
grad_norm_kernel(const __grid_constant__ ClipTable<CAP> table, double* partials) {
  __shared__ double smem[kThreads / 32];
  Sum<NORM> s;
  for (uint32_t c = blockIdx.x; c < table.chunks; c += gridDim.x) {
    const ClipEntry& e = entry_of(table, c);
    const int sh = vec_shift(e.dtype);
    const int64_t head = head_of(e), vecs = vecs_of(e);
    const int64_t begin = (int64_t)(c - e.first_chunk) * table.chunk_vecs;
    const int64_t end = begin + table.chunk_vecs < vecs ? begin + table.chunk_vecs : vecs;
    const char* base = reinterpret_cast<const char*>(e.p) + (head << (5 - sh));
    const uint32_t dtype = e.dtype;
    for (int64_t v = begin + threadIdx.x; v < end; v += 4 * kThreads) {
      V8 r[4];
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (v + u * kThreads < end) r[u] = ld32(base + (v + u * kThreads) * 32);
#pragma unroll
      for (int u = 0; u < 4; ++u)
        if (v + u * kThreads < end) take_vec<NORM>(s, r[u], dtype);
    }
    if (begin == 0) {  // what is in front of and behind the whole vectors
      const int64_t tail = head + (vecs << sh);
      if (threadIdx.x < 32 && threadIdx.x < head) s.take(load_one(e, threadIdx.x), false);
      if (threadIdx.x >= 32 && threadIdx.x < 64 && tail + threadIdx.x - 32 < e.n) s.take(load_one(e, tail + threadIdx.x - 32), false);
    }
  }
  const double v = block_join<NORM>(s.value(), smem);
  if (threadIdx.x == 0) partials[blockIdx.x] = v;
}

// {coef, norm} from the partials; every block that asks gets the same.
template <int NORM>
__device__ __forceinline__ float2 finish(const double* __restrict__ partials, int n, float max_norm, double* smem) {
  double v = 0.0;
  for (int i = threadIdx.x; i < n; i += kThreads) v = both<NORM>(v, partials[i]);
  v = block_join<NORM>(v, smem);
  const float norm = (float)(NORM == kNormL2 ? sqrt(v) : v);
  const float coef = __fdiv_rn(max_norm, __fadd_rn(norm, 1e-6f));
  return make_float2(coef > 1.f ? 1.f : coef, norm);
}
template <int NORM>
__global__ void __launch_bounds__(kThreads)
grad_norm_finish_kernel(const double* __restrict__ partials, int n, float max_norm, float* out) {
  __shared__ double smem[kThreads / 32];
  const float2 r = finish<NORM>(partials, n, max_norm, smem);
  if (threadIdx.x == 0) {
    out[0] = r.x;
    out[1] = r.y;
  }
}

__device__ __forceinline__ V8 scaled(V8 v, uint32_t dtype, float c) {
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (dtype == kClipF32) {
      v.w[j] = __float_as_uint(__fmul_rn(__uint_as_float(v.w[j]), c));
    } else if (dtype == kClipBF16) {
      v.w[j] = f32x2_to_bf16x2_rne(__fmul_rn(__uint_as_float(v.w[j] << 16), c), __fmul_rn(__uint_as_float(v.w[j] & 0xffff0000u), c));
    } else {
      const float lo = __fmul_rn(half_to_f32(v.w[j] & 0xffffu), c), hi = __fmul_rn(half_to_f32(v.w[j] >> 16), c);
      const __half2 h = __floats2half2_rn(lo, hi);
      v.w[j] = *reinterpret_cast<const uint32_t*>(&h);
    }
  }
  return v;
}

// NORM < 0: the coefficient is out[0]; otherwise it comes from the partials, and block 0 of the
// first launch leaves it there.  Chunks in the reverse order: what the norm read last is still in L2.
template <int NORM, int CAP>
__global__ void __launch_bounds__(kThreads)
grad_scale_kernel(const __grid_constant__ ClipTable<CAP> table, const double* __restrict__ partials, int n, float max_norm,
                  float* out, int write_out) {
  __shared__ double smem[kThreads / 32];
  float c;
  if (NORM < 0) {
    c = *out;
  } else {
    const float2 r = finish < NORM < 0 ? 0 : NORM > (partials, n, max_norm, smem);
    if (write_out && blockIdx.x == 0 && threadIdx.x == 0) {
      out[0] = r.x;
      out[1] = r.y;
    }
    c = r.x;
  }
  if (c == 1.f) return;
  for (uint32_t k = blockIdx.x; k < table.chunks; k += gridDim.x) {
    const uint32_t chunk = table.chunks - 1 - k;
    const ClipEntry& e = entry_of(table, chunk);
    const int sh = vec_shift(e.dtype);
    const int64_t head = head_of(e), vecs = vecs_of(e);
    const int64_t begin = (int64_t)(chunk - e.first_chunk) * table.chunk_vecs;
    const int64_t end = begin + table.chunk_vecs < vecs ? begin + table.chunk_vecs : vecs;
    char* base = reinterpret_cast<char*>(e.p) + (head << (5 - sh));
    const uint32_t dtype = e.dtype;
    for (int64_t v = begin + threadIdx.x; v < end; v += 2 * kThreads) {
      V8 r[2];
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (v + u * kThreads < end) r[u] = ld32(base + (v + u * kThreads) * 32);
#pragma unroll
      for (int u = 0; u < 2; ++u)
        if (v + u * kThreads < end) st32(base + (v + u * kThreads) * 32, scaled(r[u], dtype, c));
    }
    if (begin == 0) {
      const int64_t tail = head + (vecs << sh);
      if (threadIdx.x < 32 && threadIdx.x < head) scale_one(e, threadIdx.x, c);
      if (threadIdx.x >= 32 && threadIdx.x < 64 && tail + threadIdx.x - 32 < e.n) scale_one(e, tail + threadIdx.x - 32, c);
    }
  }
}

// Fills a launch's table; the number of its blocks.
template <int CAP>
unsigned fill(ClipTable<CAP>& t, const ClipEntry* entries, int count) {
  t.count = count;
  int64_t all = 0;
  for (int i = 0; i < count; ++i) {
    t.e[i] = entries[i];
    all += vecs_of(entries[i]);
  }
  // 8 KB a chunk while that gives every block four at most, 64 KB beyond: the norm of 1.27 G bf16 values
  // takes 387 us that way, 404 in chunks of 32 KB and 401 of 128 KB (clipped: 1191, 1201, 1226; one GPU, in
  // turn, each within 2 us)
  const int sh = all <= int64_t(kBlocks) * 1024 ? 8 : 11;
  t.chunk_vecs = 1u << sh;
  int64_t chunks = 0;
  for (int i = 0; i < count; ++i) {
    t.e[i].first_chunk = (uint32_t)chunks;
    const int64_t own = (vecs_of(t.e[i]) + t.chunk_vecs - 1) >> sh;
    chunks += own < 1 ? 1 : own;
  }
  if (chunks >= (int64_t(1) << 31)) return 0;
  t.chunks = (uint32_t)chunks;
  return (unsigned)(chunks < kBlocks ? chunks : kBlocks);
}

template <int CAP>
cudaError_t norm_pass(const ClipTable<CAP>& t, unsigned grid, int norm, double* partials, int& n, cudaStream_t st) {
  count_launch();
  if (norm == kNormL2) grad_norm_kernel<kNormL2, CAP><<<grid, kThreads, 0, st>>>(t, partials + n);
  else if (norm == kNormL1) grad_norm_kernel<kNormL1, CAP><<<grid, kThreads, 0, st>>>(t, partials + n);
  else grad_norm_kernel<kNormInf, CAP><<<grid, kThreads, 0, st>>>(t, partials + n);
  n += (int)grid;
  return cudaGetLastError();
}
template <int CAP>
cudaError_t scale_pass(const ClipTable<CAP>& t, unsigned blocks, int norm, float max_norm, const double* partials, int n, float* out,
                       int write_out, cudaStream_t st) {
  // Two loads a thread, and twice as many blocks as fit at once where each still has eight chunks:
  // 1.27 G bf16 values, norm and scaling, 1198 us (1272 with the blocks that fit; 1240 with four
  // loads); 88 M values of both types 89 us and 84.
  const unsigned grid = t.chunks >= 16u * kBlocks ? 2u * kBlocks : blocks;
  count_launch();
  if (norm == kNormL2) grad_scale_kernel<kNormL2, CAP><<<grid, kThreads, 0, st>>>(t, partials, n, max_norm, out, write_out);
  else if (norm == kNormL1) grad_scale_kernel<kNormL1, CAP><<<grid, kThreads, 0, st>>>(t, partials, n, max_norm, out, write_out);
  else if (norm == kNormInf) grad_scale_kernel<kNormInf, CAP><<<grid, kThreads, 0, st>>>(t, partials, n, max_norm, out, write_out);
  else grad_scale_kernel<-1, CAP><<<grid, kThreads, 0, st>>>(t, partials, n, max_norm, out, write_out);
  return cudaGetLastError();
}

// Calls f(table, blocks, index) for every kClipMany tensors.
template <class F>
cudaError_t each_launch(const ClipEntry* entries, int64_t count, const F& f) {
  for (int64_t at = 0; at < count; at += kClipMany) {
    const int k = (int)(count - at < kClipMany ? count - at : kClipMany);
    cudaError_t e;
    const auto take = [&](auto table) {
      const unsigned grid = fill(table, entries + at, k);
      return grid == 0 ? cudaErrorInvalidValue : f(table, grid, at);
    };
    if (k <= kClipFew) e = take(ClipTable<kClipFew>());
    else if (k <= kClipSome) e = take(ClipTable<kClipSome>());
    else e = take(ClipTable<kClipMany>());
    if (e != cudaSuccess) return e;
  }
  return cudaSuccess;
}

}  // namespace

int64_t clip_partials(int64_t count) { return kBlocks * ((count + kClipMany - 1) / kClipMany); }

cudaError_t launch_grad_norm(const ClipEntry* entries, int64_t count, int norm, float max_norm, bool scale, double* partials,
                             float* out, cudaStream_t st) {
  if (count <= 0 || norm < kNormL2 || norm > kNormInf || count > (int64_t(1) << 30)) return cudaErrorInvalidValue;
  int n = 0;
  const bool one = count <= kClipMany;  // the table serves both launches
  cudaError_t e = each_launch(entries, count, [&](const auto& t, unsigned grid, int64_t) {
    const cudaError_t r = norm_pass(t, grid, norm, partials, n, st);
    return r != cudaSuccess || !one || !scale ? r : scale_pass(t, grid, norm, max_norm, partials, n, out, 1, st);
  });
  if (e != cudaSuccess || (one && scale)) return e;
  if (scale)
    return each_launch(entries, count, [&](const auto& t, unsigned grid, int64_t at) {
      return scale_pass(t, grid, norm, max_norm, partials, n, out, at == 0, st);
    });
  count_launch();
  if (norm == kNormL2) grad_norm_finish_kernel<kNormL2><<<1, kThreads, 0, st>>>(partials, n, max_norm, out);
  else if (norm == kNormL1) grad_norm_finish_kernel<kNormL1><<<1, kThreads, 0, st>>>(partials, n, max_norm, out);
  else grad_norm_finish_kernel<kNormInf><<<1, kThreads, 0, st>>>(partials, n, max_norm, out);
  return cudaGetLastError();
}

cudaError_t launch_grad_scale(const ClipEntry* entries, int64_t count, const float* coef, cudaStream_t st) {
  return each_launch(entries, count, [&](const auto& t, unsigned grid, int64_t) {
    return scale_pass(t, grid, -1, 0.f, nullptr, 0, const_cast<float*>(coef), 0, st);
  });
}

}  // namespace oab
