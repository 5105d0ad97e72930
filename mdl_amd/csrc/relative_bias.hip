// A learned relative position bias made whole, and its gradient.
//
// out[h, i, j] = table[bucket(i + k_len - q_len - j), h]: every value is one
// of few, so the forward is bound by its stores and the gradient (sums of the
// upstream gradient over the places of each bucket) by its loads.  Both work
// on blocks of one head: bias values by distance are staged in LDS, and the
// gradient is first summed along diagonals (one distance each), in registers,
// then by bucket, with one owner for every sum.  16 heads of 2048 x 2048 in
// bf16 (134 MB) take 28 us to write, 4.8 TB/s, and 34 + 4 to sum.
#include "common.cuh"

namespace mdl {

constexpr int kBiasThreads = 256;
constexpr int kBiasRows = 32;       // rows of a block
constexpr int kBiasMaxBuckets = 1024;

struct BiasCall {
  const void* table;       // [buckets, heads]
  const int32_t* starts;   // of one direction: per_side - 1
  int64_t q_len, k_len;
  int32_t heads, buckets, per_side;  // per_side: buckets of one direction
};

// Bucket of a signed distance (query column - key column).
__device__ __forceinline__ int signed_bucket(const int32_t* starts, int per_side, bool two, int64_t d) {
  const int64_t x = d < 0 ? (two ? -d : 0) : d;
  int lo = 0, hi = per_side - 1;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= x) lo = mid + 1;
    else hi = mid;
  }
  return d < 0 && two ? lo + per_side : lo;
}

// The signed distances of a bucket, [*lo, *hi).
__device__ __forceinline__ void bucket_range(const int32_t* starts, int per_side, bool two, int k, int64_t* lo,
                                             int64_t* hi) {
  const int64_t far = int64_t(1) << 40;
  const int s = k < per_side ? k : k - per_side;
  const int64_t from = s == 0 ? 0 : starts[s - 1], to = s == per_side - 1 ? far : starts[s];
  if (k < per_side) {
    *lo = s == 0 && !two ? -far : from;  // causal: keys after the query are at distance 0
    *hi = to;
  } else {
    *lo = -to + 1;
    *hi = -(from == 0 ? 1 : from) + 1;  // the second half starts at distance -1
  }
}

// --------------------------------------------------------------- forward --
//
// A block writes kBiasRows rows of 256 pieces (16 bytes) of one head.  A
// thread keeps the piece's columns and walks down the rows: its values move
// along by one column a row, so a row needs one new value.

template <typename T, bool kVec>
__global__ __launch_bounds__(kBiasThreads) void relative_bias_kernel(BiasCall a, T* out) {
  constexpr int E = 16 / sizeof(T), kCols = kBiasThreads * E;
  __shared__ T lds[kCols + kBiasRows];
  __shared__ int32_t lds_starts[kBiasMaxBuckets];
  const int h = blockIdx.z;
  const int64_t i0 = (int64_t)blockIdx.y * kBiasRows, j0 = (int64_t)blockIdx.x * kCols;
  const bool two = a.buckets != a.per_side;
  for (int i = threadIdx.x; i < a.per_side - 1; i += kBiasThreads) lds_starts[i] = a.starts[i];
  __syncthreads();
  // lds[x]: distance of (row kBiasRows - 1, column 0) - x
  const int64_t top = i0 + kBiasRows - 1 + a.k_len - a.q_len - j0;
  for (int x = threadIdx.x; x < kCols + kBiasRows - 1; x += kBiasThreads)
    lds[x] = static_cast<const T*>(a.table)[(int64_t)signed_bucket(lds_starts, a.per_side, two, top - x) * a.heads + h];
  __syncthreads();
  const int c = threadIdx.x * E;
  if (j0 + c >= a.k_len) return;
  const int64_t rows = a.q_len - i0 < kBiasRows ? a.q_len - i0 : kBiasRows;
  T* p = out + ((int64_t)h * a.q_len + i0) * a.k_len + j0 + c;
  T w[E];  // row i's values: lds[kBiasRows - 1 - i + c ..]
#pragma unroll
  for (int e = 0; e < E; ++e) w[e] = lds[kBiasRows - 1 + c + e];
  for (int64_t i = 0; i < rows; ++i) {
    if (i) {
#pragma unroll
      for (int e = E - 1; e > 0; --e) w[e] = w[e - 1];
      w[0] = lds[kBiasRows - 1 - (int)i + c];
    }
    if constexpr (kVec) {
      u32x4 x;
      if constexpr (sizeof(T) == 2) {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = (uint32_t)w[2 * k] | ((uint32_t)w[2 * k + 1] << 16);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) x[k] = __float_as_uint(w[k]);
      }
      st_policy<kStream>(reinterpret_cast<u32x4*>(p), x);
    } else {
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (j0 + c + e < a.k_len) *to_global(p + e) = w[e];
    }
    p += a.k_len;
  }
}

// -------------------------------------------------------------- gradient --
//
// A wave takes kBiasRows rows of 64 pieces.  Walking down E rows at a time, a
// lane adds its E x E square into 2E - 1 diagonals; the E - 1 upper ones go on
// in the next square, the others are complete for this lane and are added to
// the wave's sums by distance in 16-byte pieces (lanes' distances differ, so
// no addition need be atomic and every sum has a fixed order; LDS atomics
// took 70 us where this takes 34, 16 heads of 2048 x 2048 in bf16: 3.9 TB/s).

template <typename T, bool kVec>
__global__ __launch_bounds__(kBiasThreads) void relative_bias_grad_kernel(BiasCall a, const T* grad, float* partial) {
  constexpr int E = 16 / sizeof(T), kCols = kWave * E, kWaves = kBiasThreads / kWave;
  constexpr int kSums = kCols + kBiasRows;
  __shared__ __align__(16) float lds[kWaves][kSums];
  const int h = blockIdx.z, wave = threadIdx.x / kWave, lane = lane_id();
  const int64_t i0 = (int64_t)blockIdx.y * kBiasRows;
  const int64_t j0 = ((int64_t)blockIdx.x * kWaves + wave) * kCols;  // the wave's columns
  const bool two = a.buckets != a.per_side;
  for (int x = lane; x < kSums; x += kWave) lds[wave][x] = 0.f;
  wave_sync();
  auto add_to = [&](float* at, const float (&v)[2 * E - 1]) {
#pragma unroll
    for (int q = 0; q < E / 4; ++q) {
      f32x4 x = reinterpret_cast<f32x4*>(at)[q];
#pragma unroll
      for (int k = 0; k < 4; ++k) x[k] += v[4 * q + k];
      reinterpret_cast<f32x4*>(at)[q] = x;
    }
    wave_sync();
  };
  // lds[x]: distance x + base
  const int64_t base = i0 + a.k_len - a.q_len - (j0 + kCols - 1);
  const int64_t j = j0 + (int64_t)lane * E;
  const T* p = grad + ((int64_t)h * a.q_len + i0) * a.k_len + j;
  float* sums = lds[wave] + (kCols - 1 - lane * E);  // sums[i - e]: row i, column e of the lane
  float diag[2 * E - 1];                             // diag[r - e + E - 1] of the square
#pragma unroll
  for (int x = 0; x < 2 * E - 1; ++x) diag[x] = 0.f;
#pragma unroll
  for (int i = 0; i < kBiasRows; i += E) {
    float v[E][E];
#pragma unroll
    for (int r = 0; r < E; ++r) {
#pragma unroll
      for (int e = 0; e < E; ++e) v[r][e] = 0.f;
      if (i0 + i + r < a.q_len) {
        if constexpr (kVec) {
          if (j < a.k_len) RowIO<T, E>::template load<kStream>(p, v[r]);
        } else {
#pragma unroll
          for (int e = 0; e < E; ++e)
            if (j + e < a.k_len) {
              if constexpr (sizeof(T) == 2) v[r][e] = bf16_to_f32(*to_global(p + e));
              else v[r][e] = *to_global(p + e);
            }
        }
      }
      p += a.k_len;
    }
#pragma unroll
    for (int r = 0; r < E; ++r)
#pragma unroll
      for (int e = 0; e < E; ++e) diag[r - e + E - 1] += v[r][e];
    // distances -(E - 1) .. 0 of the square's rows are complete: E neighbouring
    // sums a lane, no two lanes the same
    add_to(sums + i - (E - 1), diag);
#pragma unroll
    for (int x = 0; x < E - 1; ++x) diag[x] = diag[x + E];
#pragma unroll
    for (int x = E - 1; x < 2 * E - 1; ++x) diag[x] = 0.f;
  }
  add_to(sums + kBiasRows - (E - 1), diag);  // what the last square left open
  __syncthreads();
  float* part = partial + (((int64_t)h * gridDim.y + blockIdx.y) * gridDim.x + blockIdx.x) * a.buckets;
  for (int k = wave; k < a.buckets; k += kWaves) {
    int64_t lo, hi;
    bucket_range(a.starts, a.per_side, two, k, &lo, &hi);
    float s = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const int64_t wbase = base + (int64_t)(wave - w) * kCols;
      int64_t from = lo - wbase, to = hi - wbase;
      if (from < 0) from = 0;
      if (to > kSums - 1) to = kSums - 1;
      for (int64_t x = from + lane; x < to; x += kWave) s += lds[w][x];
    }
    for (int x = 32; x >= 1; x >>= 1) s += __shfl_xor(s, x);
    if (lane == 0) part[k] = s;
  }
}

// grad_table[bucket, head]: the blocks' parts in order.  A block sums 8
// buckets of one head, 32 threads each.
template <typename TB>
__global__ __launch_bounds__(256) void bias_partial_sum_kernel(const float* partial, int64_t parts, int buckets,
                                                               int heads, TB* grad) {
  __shared__ float smem[256];
  const int head = blockIdx.y, k = blockIdx.x * 8 + (threadIdx.x & 7), part = threadIdx.x >> 3;
  float s = 0.f;
  if (k < buckets) {
    const float* p = partial + (int64_t)head * parts * buckets + k;
#pragma unroll 4
    for (int64_t i = part; i < parts; i += 32) s += p[i * buckets];
  }
  smem[threadIdx.x] = s;
  __syncthreads();
  if (threadIdx.x < 8 && k < buckets) {
    double t = 0.;
    for (int i = 0; i < 32; ++i) t += (double)smem[8 * i + threadIdx.x];
    if constexpr (sizeof(TB) == 2) grad[(int64_t)k * heads + head] = f32_to_bf16((float)t);
    else grad[(int64_t)k * heads + head] = (float)t;
  }
}

int sum_bias_parts(const float* partial, int64_t parts, int32_t buckets, int32_t heads, int32_t dtype, void* grad,
                   hipStream_t s) {
  const dim3 grid((unsigned)((buckets + 7) / 8), (unsigned)heads);
  if (dtype == MDL_F32)
    hipLaunchKernelGGL(bias_partial_sum_kernel<float>, grid, dim3(256), 0, s, partial, parts, buckets, heads,
                       static_cast<float*>(grad));
  else
    hipLaunchKernelGGL(bias_partial_sum_kernel<bf16_t>, grid, dim3(256), 0, s, partial, parts, buckets, heads,
                       static_cast<bf16_t*>(grad));
  MDL_CHECK_LAUNCH("bias_partial_sum_kernel");
  return MDL_OK;
}

int bias_check(const char* what, int64_t heads, int64_t q_len, int64_t k_len, int32_t buckets, int32_t bidirectional,
               const int32_t* starts, int32_t dtype) {
  const std::string w(what);
  if (heads < 1 || q_len < 0 || k_len < q_len)
    return fail(MDL_ERR_INVALID, w + ": needs heads and 0 <= q_len <= k_len");
  if (heads > 65535 || k_len > 0x3fffffff || (q_len + kBiasRows - 1) / kBiasRows > 65535)
    return fail(MDL_ERR_UNSUPPORTED, w + ": too many rows");
  const int per_side = bidirectional ? buckets / 2 : buckets;
  if (per_side < 1 || (bidirectional && buckets % 2) || (per_side > 1 && !starts))
    return fail(MDL_ERR_INVALID, w + ": buckets");
  if (buckets > kBiasMaxBuckets) return fail(MDL_ERR_UNSUPPORTED, w + ": at most 1024 buckets");
  if (dtype != MDL_F32 && dtype != MDL_BF16) return fail(MDL_ERR_INVALID, w + ": dtype");
  return MDL_OK;
}

dim3 bias_grid(int64_t heads, int64_t q_len, int64_t k_len, int64_t cols) {
  return dim3((unsigned)((k_len + cols - 1) / cols), (unsigned)((q_len + kBiasRows - 1) / kBiasRows), (unsigned)heads);
}

int64_t bias_cols(int32_t dtype) { return (int64_t)kBiasThreads * (dtype == MDL_BF16 ? 8 : 4); }

}  // namespace mdl

using namespace mdl;

extern "C" {

int mdl_relative_bias(const void* table, const int32_t* bucket_starts, int32_t num_buckets, int32_t bidirectional,
                      int32_t heads, int64_t q_len, int64_t k_len, int32_t dtype, void* out, void* stream) {
  if (int rc = bias_check("mdl_relative_bias", heads, q_len, k_len, num_buckets, bidirectional, bucket_starts, dtype))
    return rc;
  if (q_len == 0) return MDL_OK;
  if (!table || !out) return fail(MDL_ERR_INVALID, "mdl_relative_bias: null pointer");
  const BiasCall a{table, bucket_starts, q_len, k_len, heads, num_buckets, bidirectional ? num_buckets / 2 : num_buckets};
  const dim3 grid = bias_grid(heads, q_len, k_len, bias_cols(dtype));
  const int64_t e = dtype == MDL_BF16 ? 8 : 4;
  const bool vec = reinterpret_cast<uintptr_t>(out) % 16 == 0 && k_len % e == 0;
  const hipStream_t s = as_stream(stream);
  if (dtype == MDL_BF16)
    hipLaunchKernelGGL((vec ? relative_bias_kernel<bf16_t, true> : relative_bias_kernel<bf16_t, false>), grid,
                       dim3(kBiasThreads), 0, s, a, static_cast<bf16_t*>(out));
  else
    hipLaunchKernelGGL((vec ? relative_bias_kernel<float, true> : relative_bias_kernel<float, false>), grid,
                       dim3(kBiasThreads), 0, s, a, static_cast<float*>(out));
  MDL_CHECK_LAUNCH("relative_bias_kernel");
  return MDL_OK;
}

size_t mdl_relative_bias_grad_workspace_bytes(int32_t num_buckets, int32_t heads, int64_t q_len, int64_t k_len,
                                              int32_t dtype) {
  if (num_buckets < 0 || heads < 0 || q_len < 0 || k_len < 0) return 0;
  const dim3 g = bias_grid(heads, q_len, k_len, bias_cols(dtype));
  return (size_t)g.x * g.y * g.z * num_buckets * sizeof(float);
}

int mdl_relative_bias_grad(const void* grad, const int32_t* bucket_starts, int32_t num_buckets, int32_t bidirectional,
                           int32_t heads, int64_t q_len, int64_t k_len, int32_t dtype, void* grad_table,
                           void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = bias_check("mdl_relative_bias_grad", heads, q_len, k_len, num_buckets, bidirectional, bucket_starts,
                          dtype))
    return rc;
  if (!grad_table || (q_len > 0 && !grad)) return fail(MDL_ERR_INVALID, "mdl_relative_bias_grad: null pointer");
  const size_t need = mdl_relative_bias_grad_workspace_bytes(num_buckets, heads, q_len, k_len, dtype);
  if (need && (!workspace || workspace_bytes < need))
    return fail(MDL_ERR_WORKSPACE, "mdl_relative_bias_grad: workspace too small");
  const BiasCall a{nullptr, bucket_starts, q_len, k_len, heads, num_buckets,
                   bidirectional ? num_buckets / 2 : num_buckets};
  const dim3 grid = bias_grid(heads, q_len, k_len, bias_cols(dtype));
  const int64_t e = dtype == MDL_BF16 ? 8 : 4;
  const bool vec = reinterpret_cast<uintptr_t>(grad) % 16 == 0 && k_len % e == 0;
  const hipStream_t s = as_stream(stream);
  float* partial = static_cast<float*>(workspace);
  if (q_len > 0) {
    if (dtype == MDL_BF16)
      hipLaunchKernelGGL((vec ? relative_bias_grad_kernel<bf16_t, true> : relative_bias_grad_kernel<bf16_t, false>), grid,
                         dim3(kBiasThreads), 0, s, a, static_cast<const bf16_t*>(grad), partial);
    else
      hipLaunchKernelGGL((vec ? relative_bias_grad_kernel<float, true> : relative_bias_grad_kernel<float, false>), grid,
                         dim3(kBiasThreads), 0, s, a, static_cast<const float*>(grad), partial);
    MDL_CHECK_LAUNCH("relative_bias_grad_kernel");
  }
  return sum_bias_parts(partial, q_len > 0 ? (int64_t)grid.x * grid.y : 0, num_buckets, heads, dtype, grad_table, s);
}

}  // extern "C"
