// The norms around a block, fused with its gate and residual scale:
//
//   r = o / rms(o) * w_post,   y = x + sigmoid(gate) * residual_scale * r,
//   h = y / rms(y) * w_next,   rms(v)^2 = mean(v^2) + eps,
//
// in one pass each way: x, o and gate are read once and y and h written once;
// backward reads x, o, gate, dy and dh once and writes dx, do and dgate once.
// The backward makes y again from x, o and gate (y as it was before rounding)
// instead of reading it: the same bytes, since x would have to be read with it
// for nothing else.  Bytes bound both directions: 262144 rows of 256 in bf16
// take 133 us forward and 210 backward, 5.0 and 5.1 TB/s, the rate of a copy.
//
// A row lies in the registers of a group of lanes (4 to 256, as wide as it
// needs); its two sums are taken across the group.  Sums over rows (the
// gradients of the three weights) stay in each lane's registers for the rows
// it walks, are joined per block in LDS and over blocks by a second launch, in
// a fixed order.
#include "common.cuh"

#include <initializer_list>

namespace mdl {

constexpr int kNormThreads = 256;
constexpr int kNormBlocks = 1024;  // blocks of the backward at most: each leaves three rows of sums

struct NormCall {
  const void *x, *o, *gate, *dy, *dh;
  const void *scale, *w_post, *w_next;
  void *y, *h, *dx, *d_o, *dgate;
  float* rstd;     // [2, rows]: of o, of y
  float* partial;  // [blocks, 3, dim]
  int64_t rows;
  int32_t dim, weight_f32;
  float eps;
};

__device__ __forceinline__ float weight_at(const void* p, int32_t f32, int i) {
  return f32 ? static_cast<const float*>(p)[i] : bf16_to_f32(static_cast<const bf16_t*>(p)[i]);
}

__device__ __forceinline__ float sigmoid(float v) {
  return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * v));
}

// A lane's columns of a row: V pieces of E elements, piece p at column
// (p * L + lane) * E.
template <typename T, int L, int V, bool kVec>
struct NormRow {
  static constexpr int E = 16 / sizeof(T), N = V * E;

  static __device__ __forceinline__ int column(int p) { return (p * L + (int)(threadIdx.x % L)) * E; }

  // A row's pieces as they lie in memory: on their way while the row before is
  // worked on.
  struct Raw {
    u32x4 piece[V];
  };
  static __device__ __forceinline__ void fetch(const void* base, int64_t row, int dim, Raw& r) {
    const T* p = static_cast<const T*>(base) + row * dim;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      r.piece[i] = u32x4{0, 0, 0, 0};
      if (column(i) < dim) r.piece[i] = ld_policy<kStream>(reinterpret_cast<const u32x4*>(p + column(i)));
    }
  }
  static __device__ __forceinline__ void unpack(const Raw& r, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < V; ++i)
#pragma unroll
      for (int k = 0; k < 4; ++k) {
        if constexpr (sizeof(T) == 2) {
          v[i * E + 2 * k] = __uint_as_float(r.piece[i][k] << 16);
          v[i * E + 2 * k + 1] = __uint_as_float(r.piece[i][k] & 0xffff0000u);
        } else {
          v[i * E + k] = __uint_as_float(r.piece[i][k]);
        }
      }
  }

  static __device__ __forceinline__ void load(const void* base, int64_t row, int dim, float (&v)[N]) {
    const T* p = static_cast<const T*>(base) + row * dim;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = column(i);
      if constexpr (kVec) {
        float t[E];
#pragma unroll
        for (int e = 0; e < E; ++e) t[e] = 0.f;
        if (c < dim) RowIO<T, E>::template load<kStream>(p + c, t);
#pragma unroll
        for (int e = 0; e < E; ++e) v[i * E + e] = t[e];
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e) {
          float t = 0.f;
          if (c + e < dim) {
            if constexpr (sizeof(T) == 2) t = bf16_to_f32(*to_global(p + c + e));
            else t = *to_global(p + c + e);
          }
          v[i * E + e] = t;
        }
      }
    }
  }
  static __device__ __forceinline__ void store(void* base, int64_t row, int dim, const float (&v)[N]) {
    T* p = static_cast<T*>(base) + row * dim;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = column(i);
      if constexpr (kVec) {
        if (c < dim) {
          u32x4 w;
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            if constexpr (sizeof(T) == 2) {
              typedef __bf16 pair __attribute__((ext_vector_type(2)));
              const pair b = {(__bf16)v[i * E + 2 * k], (__bf16)v[i * E + 2 * k + 1]};
              w[k] = __builtin_bit_cast(uint32_t, b);
            } else {
              w[k] = __float_as_uint(v[i * E + k]);
            }
          }
          st_policy<kStream>(reinterpret_cast<u32x4*>(p + c), w);
        }
      } else {
#pragma unroll
        for (int e = 0; e < E; ++e)
          if (c + e < dim) {
            if constexpr (sizeof(T) == 2) *to_global(p + c + e) = f32_to_bf16(v[i * E + e]);
            else *to_global(p + c + e) = v[i * E + e];
          }
      }
    }
  }
  // weights of the lane's columns (fill past the row, or without weights)
  static __device__ __forceinline__ void weights(const void* base, int32_t f32, int dim, float fill, float (&v)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int c = column(i / E) + i % E;
      v[i] = base && c < dim ? weight_at(base, f32, c) : fill;
    }
  }
};

// Sum over the row's lanes, in every lane.
template <int L>
struct RowSum {
  float (*smem)[kNormThreads / kWave];  // [2]
  int turn = 0;
  __device__ __forceinline__ float operator()(float v) {
    if constexpr (L <= 32) return group_sum<L>(v);
    v = sum_halves(group_sum<32>(v));
    if constexpr (L == kNormThreads) {
      // two slots in turn: a slot is written again only after the barrier of the sum between
      if (lane_id() == 0) smem[turn][threadIdx.x / kWave] = v;
      __syncthreads();
      v = (smem[turn][0] + smem[turn][1]) + (smem[turn][2] + smem[turn][3]);
      turn ^= 1;
    }
    return v;
  }
};

template <typename T, int L, int V, bool kVec>
__global__ __launch_bounds__(kNormThreads) void norm_forward_kernel(NormCall a) {
  using Row = NormRow<T, L, V, kVec>;
  constexpr int N = Row::N, kGroups = kNormThreads / L;
  __shared__ float smem[2][kNormThreads / kWave];
  RowSum<L> sum{smem};
  float wp[N], wn[N];  // w_post * residual_scale, w_next
  Row::weights(a.w_next, a.weight_f32, a.dim, 1.f, wn);
  if (a.o) {
    Row::weights(a.w_post, a.weight_f32, a.dim, 1.f, wp);
    if (a.scale) {
      float s[N];
      Row::weights(a.scale, a.weight_f32, a.dim, 1.f, s);
#pragma unroll
      for (int i = 0; i < N; ++i) wp[i] *= s[i];
    }
  }
  const float inv_dim = 1.f / (float)a.dim;
  for (int64_t row = (int64_t)blockIdx.x * kGroups + threadIdx.x / L; row < a.rows;
       row += (int64_t)gridDim.x * kGroups) {
    float y[N];
    Row::load(a.x, row, a.dim, y);
    if (a.o) {
      float o[N], g[N];
      Row::load(a.o, row, a.dim, o);
      if (a.gate) Row::load(a.gate, row, a.dim, g);
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) s += o[i] * o[i];
      const float inv = 1.f / sqrtf(sum(s) * inv_dim + a.eps);
#pragma unroll
      for (int i = 0; i < N; ++i) {
        float r = o[i] * inv * wp[i];
        if (a.gate) r *= sigmoid(g[i]);
        y[i] += r;
      }
      if (a.rstd && threadIdx.x % L == 0) a.rstd[row] = inv;
      Row::store(a.y, row, a.dim, y);
    }
    float s = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) s += y[i] * y[i];
    const float inv = 1.f / sqrtf(sum(s) * inv_dim + a.eps);
    if (a.rstd && threadIdx.x % L == 0) a.rstd[a.rows + row] = inv;
#pragma unroll
    for (int i = 0; i < N; ++i) y[i] *= inv * wn[i];
    Row::store(a.h, row, a.dim, y);
  }
}

template <typename T, int L, int V, bool kVec>
__global__ __launch_bounds__(kNormThreads) void norm_backward_kernel(NormCall a) {
  using Row = NormRow<T, L, V, kVec>;
  constexpr int N = Row::N, kGroups = kNormThreads / L;
  __shared__ float smem[2][kNormThreads / kWave];
  __shared__ float joined[kGroups][L * N];
  RowSum<L> sum{smem};
  float wp[N], wn[N], sc[N];
  Row::weights(a.w_next, a.weight_f32, a.dim, 1.f, wn);
  Row::weights(a.o ? a.w_post : nullptr, a.weight_f32, a.dim, 1.f, wp);
  Row::weights(a.o ? a.scale : nullptr, a.weight_f32, a.dim, 1.f, sc);
  float d_scale[N], d_post[N], d_next[N];
#pragma unroll
  for (int i = 0; i < N; ++i) d_scale[i] = d_post[i] = d_next[i] = 0.f;
  const float inv_dim = 1.f / (float)a.dim;
  // the next row is read ahead where registers allow (8 elements a lane: 337 to
  // 212 us for 262144 rows of 256 in bf16)
  constexpr bool kAhead = kVec && N <= 8;
  const int64_t step = (int64_t)gridDim.x * kGroups;
  struct Rows {
    typename Row::Raw x, o, g, dy, dh;
    float inv_o, inv_y;
  } next;
  auto fetch = [&](int64_t row) {
    Row::fetch(a.x, row, a.dim, next.x);
    if (a.o) Row::fetch(a.o, row, a.dim, next.o);
    if (a.gate) Row::fetch(a.gate, row, a.dim, next.g);
    if (a.dh) Row::fetch(a.dh, row, a.dim, next.dh);
    if (a.dy) Row::fetch(a.dy, row, a.dim, next.dy);
    next.inv_o = a.o ? a.rstd[row] : 0.f;
    next.inv_y = a.rstd[a.rows + row];
  };
  const int64_t first = (int64_t)blockIdx.x * kGroups + threadIdx.x / L;
  if constexpr (kAhead)
    if (first < a.rows) fetch(first);
  for (int64_t row = first; row < a.rows; row += step) {
    float y[N], o[N], g[N], dx[N], dh[N], inv_o, inv_y;
    if constexpr (kAhead) {
      Row::unpack(next.x, y);
      if (a.o) Row::unpack(next.o, o);
      if (a.gate) Row::unpack(next.g, g);
      if (a.dh) Row::unpack(next.dh, dh);
      if (a.dy) Row::unpack(next.dy, dx);
      inv_o = next.inv_o;
      inv_y = next.inv_y;
      if (row + step < a.rows) fetch(row + step);
    } else {
      Row::load(a.x, row, a.dim, y);
      if (a.o) Row::load(a.o, row, a.dim, o);
      if (a.gate) Row::load(a.gate, row, a.dim, g);
      if (a.dh) Row::load(a.dh, row, a.dim, dh);
      if (a.dy) Row::load(a.dy, row, a.dim, dx);
      inv_o = a.o ? a.rstd[row] : 0.f;
      inv_y = a.rstd[a.rows + row];
    }
    if (!a.dy) {
#pragma unroll
      for (int i = 0; i < N; ++i) dx[i] = 0.f;
    }
    if (a.o) {
#pragma unroll
      for (int i = 0; i < N; ++i) {
        o[i] *= inv_o;  // the normalised o
        if (a.gate) g[i] = sigmoid(g[i]);
        else g[i] = 1.f;
        y[i] += o[i] * (wp[i] * sc[i]) * g[i];
      }
    }
    if (a.dh) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        y[i] *= inv_y;  // the normalised y
        d_next[i] += dh[i] * y[i];
        dh[i] *= wn[i];
        s += dh[i] * y[i];
      }
      s = sum(s) * inv_dim;
#pragma unroll
      for (int i = 0; i < N; ++i) dx[i] += inv_y * (dh[i] - y[i] * s);
    }
    Row::store(a.dx, row, a.dim, dx);
    if (a.o) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) {
        const float t = dx[i] * g[i] * o[i];
        d_scale[i] += t * wp[i];
        d_post[i] += t * sc[i];
        s += t * (wp[i] * sc[i]);
      }
      s = sum(s) * inv_dim;
      if (a.gate) {
        float dg[N];
#pragma unroll
        for (int i = 0; i < N; ++i) dg[i] = dx[i] * o[i] * (wp[i] * sc[i]) * (g[i] * (1.f - g[i]));
        Row::store(a.dgate, row, a.dim, dg);
      }
#pragma unroll
      for (int i = 0; i < N; ++i) dx[i] = inv_o * (dx[i] * g[i] * (wp[i] * sc[i]) - o[i] * s);
      Row::store(a.d_o, row, a.dim, dx);
    }
  }
  float* part = a.partial + (int64_t)blockIdx.x * 3 * a.dim;
  auto leave = [&](const float (&v)[N], float* to) {
    __syncthreads();
#pragma unroll
    for (int i = 0; i < N; ++i) joined[threadIdx.x / L][Row::column(i / Row::E) + i % Row::E] = v[i];
    __syncthreads();
    for (int c = threadIdx.x; c < a.dim; c += kNormThreads) {
      float s = 0.f;
      for (int k = 0; k < kGroups; ++k) s += joined[k][c];
      to[c] = s;
    }
  };
  if (a.o) {
    leave(d_scale, part);
    leave(d_post, part + a.dim);
  }
  leave(d_next, part + 2 * a.dim);
}

// Weight gradients from the blocks' sums, added in order: 16 columns a block,
// 64 threads each.  which: 0 residual scale, 1 post, 2 next (grid.y).
constexpr int kJoinCols = 16, kJoinParts = 64;
__global__ __launch_bounds__(kJoinCols* kJoinParts) void norm_weight_grads_kernel(const float* partial, int blocks,
                                                                                  int dim, void* d_scale, void* d_post,
                                                                                  void* d_next, int32_t f32) {
  __shared__ float smem[kJoinParts][kJoinCols];
  const int which = blockIdx.y;
  void* to = which == 0 ? d_scale : (which == 1 ? d_post : d_next);
  if (!to) return;
  const int col = threadIdx.x % kJoinCols, part = threadIdx.x / kJoinCols;
  const int c = blockIdx.x * kJoinCols + col;
  float s = 0.f;
  if (c < dim) {
    const float* p = partial + (int64_t)which * dim + c;
#pragma unroll 8
    for (int i = part; i < blocks; i += kJoinParts) s += p[(int64_t)i * 3 * dim];
  }
  smem[part][col] = s;
  __syncthreads();
  if (part == 0 && c < dim) {
    double t = 0.;
    for (int i = 0; i < kJoinParts; ++i) t += (double)smem[i][col];
    if (f32) static_cast<float*>(to)[c] = (float)t;
    else static_cast<bf16_t*>(to)[c] = f32_to_bf16((float)t);
  }
}

// ---------------------------------------------------------------- host side --

struct NormShape {
  int lanes, pieces;
};

// Lanes of a row and pieces per lane: one piece until the row is a wave wide,
// two until it is a block wide, then as many as it needs.
NormShape norm_shape(int dim, int elems) {
  const int n = (dim + elems - 1) / elems;
  if (n <= 4) return {4, 1};
  if (n <= 8) return {8, 1};
  if (n <= 16) return {16, 1};
  if (n <= 32) return {32, 1};
  if (n <= 64) return {64, 1};
  if (n <= 128) return {64, 2};
  if (n <= 256) return {256, 1};
  if (n <= 512) return {256, 2};
  if (n <= 1024) return {256, 4};
  return {0, 0};
}

int norm_blocks(const mdl_block_norm& a) {
  const NormShape n = norm_shape(a.dim, a.dtype == MDL_BF16 ? 8 : 4);
  if (!n.lanes) return 0;
  const int64_t groups = kNormThreads / n.lanes, need = (a.rows + groups - 1) / groups;
  return (int)(need < kNormBlocks ? need : kNormBlocks);
}

template <typename F>
int for_norm(const mdl_block_norm& a, bool vec, F&& f) {
  auto shaped = [&]<typename T, bool kVec>() -> int {
    const NormShape n = norm_shape(a.dim, 16 / sizeof(T));
    switch (n.lanes * 8 + n.pieces) {
      case 4 * 8 + 1: return f.template operator()<T, 4, 1, kVec>();
      case 8 * 8 + 1: return f.template operator()<T, 8, 1, kVec>();
      case 16 * 8 + 1: return f.template operator()<T, 16, 1, kVec>();
      case 32 * 8 + 1: return f.template operator()<T, 32, 1, kVec>();
      case 64 * 8 + 1: return f.template operator()<T, 64, 1, kVec>();
      case 64 * 8 + 2: return f.template operator()<T, 64, 2, kVec>();
      case 256 * 8 + 1: return f.template operator()<T, 256, 1, kVec>();
      case 256 * 8 + 2: return f.template operator()<T, 256, 2, kVec>();
      default: return f.template operator()<T, 256, 4, kVec>();
    }
  };
  if (a.dtype == MDL_BF16)
    return vec ? shaped.template operator()<bf16_t, true>() : shaped.template operator()<bf16_t, false>();
  return vec ? shaped.template operator()<float, true>() : shaped.template operator()<float, false>();
}

int norm_check(const mdl_block_norm* a, const char* what) {
  const std::string w(what);
  if (!a) return fail(MDL_ERR_INVALID, w + ": null descriptor");
  if (a->rows < 0 || a->dim < 1) return fail(MDL_ERR_INVALID, w + ": shape");
  if ((a->dtype != MDL_F32 && a->dtype != MDL_BF16) || (a->weight_dtype != MDL_F32 && a->weight_dtype != MDL_BF16))
    return fail(MDL_ERR_INVALID, w + ": dtype");
  if (!(a->eps >= 0.f)) return fail(MDL_ERR_INVALID, w + ": eps");
  if (!norm_shape(a->dim, a->dtype == MDL_BF16 ? 8 : 4).lanes)
    return fail(MDL_ERR_UNSUPPORTED, w + ": rows of at most 8192 (bf16) or 4096 (fp32) elements");
  if (!a->block_out && (a->gate || a->residual_scale || a->post_weight))
    return fail(MDL_ERR_INVALID, w + ": gate, residual_scale and post_weight belong to a block's output");
  if (a->rows > 0 && (!a->x || !a->rstd)) return fail(MDL_ERR_INVALID, w + ": null pointer");
  return MDL_OK;
}

NormCall norm_call(const mdl_block_norm& a) {
  NormCall c{};
  c.x = a.x; c.o = a.block_out; c.gate = a.gate;
  c.scale = a.residual_scale; c.w_post = a.post_weight; c.w_next = a.next_weight;
  c.rstd = a.rstd;
  c.rows = a.rows;
  c.dim = a.dim;
  c.weight_f32 = a.weight_dtype == MDL_F32;
  c.eps = a.eps;
  return c;
}

bool aligned16(std::initializer_list<const void*> ps) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % 16) return false;
  return true;
}

}  // namespace mdl

using namespace mdl;

extern "C" {

int mdl_block_norm_forward(const mdl_block_norm* a, void* y, void* h, void* stream) {
  if (int rc = norm_check(a, "mdl_block_norm_forward")) return rc;
  if (a->rows == 0) return MDL_OK;
  if (!h || (a->block_out && !y)) return fail(MDL_ERR_INVALID, "mdl_block_norm_forward: null pointer");
  NormCall c = norm_call(*a);
  c.y = y;
  c.h = h;
  const bool vec = a->dim % (a->dtype == MDL_BF16 ? 8 : 4) == 0 && aligned16({c.x, c.o, c.gate, y, h});
  return for_norm(*a, vec, [&]<typename T, int L, int V, bool kVec>() -> int {
    const int64_t groups = kNormThreads / L, need = (c.rows + groups - 1) / groups;
    const unsigned blocks = (unsigned)(need < 4096 ? need : 4096);
    hipLaunchKernelGGL((norm_forward_kernel<T, L, V, kVec>), dim3(blocks), dim3(kNormThreads), 0, as_stream(stream), c);
    MDL_CHECK_LAUNCH("norm_forward_kernel");
    return MDL_OK;
  });
}

size_t mdl_block_norm_backward_workspace_bytes(const mdl_block_norm* a) {
  return a ? (size_t)norm_blocks(*a) * 3 * a->dim * sizeof(float) : 0;
}

int mdl_block_norm_backward(const mdl_block_norm* a, const mdl_block_norm_grads* g, void* workspace,
                            size_t workspace_bytes, void* stream) {
  if (int rc = norm_check(a, "mdl_block_norm_backward")) return rc;
  if (!g) return fail(MDL_ERR_INVALID, "mdl_block_norm_backward: null pointer");
  if (a->rows > 0 && (!g->grad_x || (a->block_out && !g->grad_block_out) || (a->gate && !g->grad_gate)))
    return fail(MDL_ERR_INVALID, "mdl_block_norm_backward: null pointer");
  if (!workspace && a->rows > 0) return fail(MDL_ERR_WORKSPACE, "mdl_block_norm_backward: workspace too small");
  if (workspace_bytes < mdl_block_norm_backward_workspace_bytes(a))
    return fail(MDL_ERR_WORKSPACE, "mdl_block_norm_backward: workspace too small");
  NormCall c = norm_call(*a);
  c.dy = g->grad_y; c.dh = g->grad_h;
  c.dx = g->grad_x; c.d_o = g->grad_block_out; c.dgate = g->grad_gate;
  c.partial = static_cast<float*>(workspace);
  const int blocks = norm_blocks(*a);
  const hipStream_t s = as_stream(stream);
  if (blocks > 0) {
    const bool vec = a->dim % (a->dtype == MDL_BF16 ? 8 : 4) == 0 &&
                     aligned16({c.x, c.o, c.gate, c.dy, c.dh, c.dx, c.d_o, c.dgate});
    if (int rc = for_norm(*a, vec, [&]<typename T, int L, int V, bool kVec>() -> int {
          hipLaunchKernelGGL((norm_backward_kernel<T, L, V, kVec>), dim3((unsigned)blocks), dim3(kNormThreads), 0, s,
                             c);
          MDL_CHECK_LAUNCH("norm_backward_kernel");
          return MDL_OK;
        }))
      return rc;
  }
  if (g->grad_residual_scale || g->grad_post_weight || g->grad_next_weight) {
    const dim3 grid((unsigned)((a->dim + kJoinCols - 1) / kJoinCols), 3);
    hipLaunchKernelGGL(norm_weight_grads_kernel, grid, dim3(kJoinCols * kJoinParts), 0, s, c.partial, blocks, a->dim,
                       g->grad_residual_scale, g->grad_post_weight, g->grad_next_weight, c.weight_f32);
    MDL_CHECK_LAUNCH("norm_weight_grads_kernel");
  }
  return MDL_OK;
}

}  // extern "C"
