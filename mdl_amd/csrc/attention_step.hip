// Attention of one new token a row over a cache of keys and values, and the
// cache's prompt form.
//
// A step reads every visible key and value once and does two multiply-adds
// per element and query head that shares it: bytes bound it (the heads that
// share a key head are answered together, up to 8 of them), so it runs on the
// vector units.  A lane group covers one cached row in 16-byte pieces and
// walks every (groups of the block)-th row with its own running maximum and
// sum; groups, then waves, then blocks are joined at the end.  Few rows with
// long caches are cut into parts over several blocks, joined by a second
// launch.  256 users with up to 1028 rows of 64 (103 MB): 31 us, 3.3 TB/s, the
// longest walks bound it; two users with 62,000 rows of 128 (129 MB): 31 and
// 5 us, 3.6 TB/s together.  (Of caches that other data has driven out of the
// last-level cache, as a model's other layers do.  The figures beside the rules
// below are of loops over two states, of which part stays there: 28, and 26 and 4.)
#include "attention.cuh"

namespace mdl {

constexpr int kJoinThreads = 1024;
// A walk is cut where few of them would leave CUs idle; joining the parts
// costs a launch of 4 to 5 us.  (bf16 caches of 1028 rows of 64, 8 query
// heads on 2 key heads: one user 17 us whole, 16.5 in parts of 512 rows, 13.8
// in four of 257; 100 users, 200 walks: 18.5 whole, 24.6 in two.  Longer caches
// were not measured between kCutUnits walks and one for every CU.)
constexpr int kStepBlocks = 512;   // blocks wanted of walks that are cut
constexpr int kCutUnits = 128;     // walks above which none is cut
constexpr int kStepMinRows = 256;  // cached rows of a part at least

// Rows of a lane group's iteration: twice as many are in flight (the next
// iteration's are read while this one's are worked on).  The more heads share
// a row, the fewer rows fill the registers (4 heads, 2 x 62,000 rows of 128:
// 30.9 us with one, 32.7 with two).
template <int G>
constexpr int step_unroll() { return G == 8 ? 2 : (G == 4 ? 1 : 4); }

struct StepCall {
  const void *q, *k, *v;
  void *cache_k, *cache_v;
  const int64_t* positions;
  const void* table;
  const int32_t* starts;
  float* part;  // [B * Hq, parts, 2 + dim]: maximum, sum, sums of values; NULL with one part
  int64_t q_batch, q_head, k_batch, k_head, v_batch, v_head;
  int64_t ck_batch, ck_head, cv_batch, cv_head, row_k, row_v;  // row_k, row_v: a prompt's row strides
  uint32_t ck_slot, cv_slot;
  int32_t window, sinks, capacity;  // window <= capacity - sinks
  int32_t batch, q_heads, kv_heads, dim, parts, buckets, distances, table_f32;
  float c2;  // scale * log2(e)
};

// The cached rows a token at position n sees, in order: the first tokens,
// then those of the window; the last one is the token itself.
struct StepRows {
  int sinks, count, shift, capacity, ring, first_distance;
  __device__ __forceinline__ StepRows(const StepCall& a, int64_t n) {
    capacity = a.capacity;
    ring = a.capacity - a.sinks;
    sinks = a.sinks < n + 1 ? a.sinks : (int)(n + 1);
    int64_t from = n - a.window + 1;
    if (from < a.sinks) from = a.sinks;
    const int in_window = from <= n ? (int)(n - from + 1) : 0;
    count = sinks + in_window;
    // slot of the window's first row, less its index
    int64_t base = from <= n ? from - a.sinks : 0;
    if (base >= ring) base %= ring;
    shift = (int)base + a.sinks - sinks;
    first_distance = n < INT32_MAX ? (int)n : INT32_MAX;
  }
  __device__ __forceinline__ int slot(int i) const {
    int t = i + (i < sinks ? 0 : shift);
    if (t >= capacity) t -= ring;  // the window is no longer than the ring: one turn at most
    return t;
  }
  __device__ __forceinline__ int distance(int i) const { return (i < sinks ? first_distance : count - 1) - i; }
  // rows of one part, whole parts of at least kStepMinRows
  __device__ __forceinline__ int per_part(int parts) const {
    const int per = (count + parts - 1) / parts;
    return per > kStepMinRows ? per : kStepMinRows;
  }
};

// row + slot * stride (elements); the product has 64 bits, its factors 32.
template <typename T>
__device__ __forceinline__ T* row_at(T* base, int slot, uint32_t stride) {
  return base + (uint64_t)(uint32_t)slot * stride;
}

template <typename T>
__device__ __forceinline__ float element(const typename Frags<T>::Frag& f, int i) {
  return (float)f[i];
}

// Sum over the lane's elements of two rows, in fp32 (bf16 pairs are multiplied
// and added to it by one instruction).
__device__ __forceinline__ float dot(const bf16x8& a, const bf16x8& b) {
  float t = 0.f;
#pragma unroll
  for (int i = 0; i < 4; ++i)
    t = __builtin_amdgcn_fdot2_f32_bf16(bf16x2{a[2 * i], a[2 * i + 1]}, bf16x2{b[2 * i], b[2 * i + 1]}, t, false);
  return t;
}
__device__ __forceinline__ float dot(const f32x4& a, const f32x4& b) {
  float t = a[0] * b[0];
#pragma unroll
  for (int i = 1; i < 4; ++i) t = __builtin_fmaf(a[i], b[i], t);
  return t;
}

// One head group's running softmax over its lanes' values.
template <int G, int E>
struct StepState {
  float m[G], l[G], acc[G][E];
  __device__ __forceinline__ StepState() {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      m[g] = kNoScore;
      l[g] = 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) acc[g][e] = 0.f;
    }
  }
  __device__ __forceinline__ void raise(int g, float top) {
    const float shrink = exp2_fast(m[g] - top);
    m[g] = top;
    l[g] *= shrink;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[g][e] *= shrink;
  }
  __device__ __forceinline__ void join_lanes(int distance) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float m2 = __shfl_xor(m[g], distance);
      raise(g, fmaxf(m[g], m2));
      l[g] += __shfl_xor(l[g], distance);
#pragma unroll
      for (int e = 0; e < E; ++e) acc[g][e] += __shfl_xor(acc[g][e], distance);
    }
  }
};

template <typename T, bool kVec>
__device__ __forceinline__ void store_piece(T* row, int d, int D, const float* v) {
  constexpr int E = Frags<T>::kElems;
#pragma unroll
  for (int i = 0; i < E; ++i)
    if (kVec ? d < D : d + i < D) {
      if constexpr (sizeof(T) == 2) *(gptr<__bf16>)(row + d + i) = (__bf16)v[i];
      else *to_global(row + d + i) = v[i];
    }
}

// Waves of a block: eight for calls of at most two blocks per CU (one with 8
// heads' registers), which end with their longest walk; four where further
// blocks wait for a CU.  (One user's token over 260 rows, 4 heads of 64: 8.7 us
// with four, 7.3 with eight.  512 walks of up to 1028 rows, 4 heads a row: 30.4
// and 27.8; 4096 such walks: 166 and 186.)
template <int G>
constexpr int few_blocks() { return G == 8 ? 256 : 512; }

// What a block's waves leave for its join: (maximum, sum, values) of a lane's
// piece and head.  Beside the bias the largest shape (fp32, 8 heads a row of
// more than 64, 1024 buckets over 2049 distances) takes 84 KB of LDS in all.
template <typename T, int L, int G, int kWaves>
using StepJoin = float[kWaves][L][G][Frags<T>::kElems + 2];

template <typename T, int L, int G, bool kVec, int kWaves>
__global__ __launch_bounds__(kWaves* kWave) void attention_step_kernel(StepCall a, T* out) {
  using F = Frags<T>;
  constexpr int E = F::kElems, kGroups = kWave / L, kStepThreads = kWaves * kWave;
  constexpr int U = step_unroll<G>(), kPass = kGroups * U;  // rows of a wave's iteration
  extern __shared__ __align__(16) char smem[];
  float* lds_table = reinterpret_cast<float*>(smem);           // [buckets][G] bias in powers of two
  uint16_t* lds_bucket = reinterpret_cast<uint16_t*>(lds_table + a.buckets * G);  // [distances]
  __shared__ StepJoin<T, L, G, kWaves> lds_join;

  const int share = a.q_heads / a.kv_heads, groups = (share + G - 1) / G;
  unsigned id = blockIdx.x;
  const int part = (int)(id % a.parts);
  id /= a.parts;
  const int hg = (int)(id % groups);
  id /= groups;
  const int b = (int)(id / a.kv_heads), kv = (int)id - b * a.kv_heads;
  const int head0 = kv * share + hg * G, heads = share - hg * G < G ? share - hg * G : G;
  const int wave = wave_id(), sub = lane_id() % L, group = lane_id() / L;
  const int d = sub * E;
  T* out_row = out + ((int64_t)b * a.q_heads + head0) * a.dim;

  const int64_t n = load_uniform(a.positions + b);
  if (n < 0) {  // no such position: nothing stored, zeros answered
    if (part == 0)
      for (int i = threadIdx.x; i < heads * a.dim; i += kStepThreads) out_row[i] = T(0);
    return;
  }
  const StepRows rows(a, n);
  const int per = rows.per_part(a.parts);
  const int lo = part * per, hi = lo + per < rows.count ? lo + per : rows.count;
  if (lo >= hi) return;

  const T* new_k = static_cast<const T*>(a.k) + b * a.k_batch + kv * a.k_head;
  const T* new_v = static_cast<const T*>(a.v) + b * a.v_batch + kv * a.v_head;
  T* cache_k = static_cast<T*>(a.cache_k) + b * a.ck_batch + kv * a.ck_head;
  T* cache_v = static_cast<T*>(a.cache_v) + b * a.cv_batch + kv * a.cv_head;

  typename F::Frag q[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    q[g] = {};
    if (g < heads)
      q[g] = load_row<T, kVec>(static_cast<const T*>(a.q) + b * a.q_batch + (int64_t)(head0 + g) * a.q_head, d, a.dim);
  }

  const int last = rows.count - 1;
  struct Rows {
    typename F::Frag k[U], v[U];
  };
  auto load = [&](Rows& r, int i0) {
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kGroups + group;
      r.k[u] = {};
      r.v[u] = {};
      if (i < last && i < hi) {
        const int slot = rows.slot(i);
        r.k[u] = load_row<T, kVec>(row_at(cache_k, slot, a.ck_slot), d, a.dim);
        r.v[u] = load_row<T, kVec>(row_at(cache_v, slot, a.cv_slot), d, a.dim);
      }
    }
    if (last < hi && i0 <= last && last < i0 + kPass) {  // the token's own row
#pragma unroll
      for (int u = 0; u < U; ++u)
        if (i0 + u * kGroups + group == last) {
          r.k[u] = load_row<T, kVec>(new_k, d, a.dim);
          r.v[u] = load_row<T, kVec>(new_v, d, a.dim);
        }
    }
  };
  const int first_row = lo + wave * kPass, stride = kWaves * kPass;
  Rows even, odd;
  load(even, first_row);
  // the bias is staged while the first rows are on their way
  if (a.table) {
    for (int i = threadIdx.x; i < a.buckets * G; i += kStepThreads) {
      const int g = i % G;
      float v = 0.f;
      if (g < heads) {
        const int64_t at = (int64_t)(i / G) * a.q_heads + head0 + g;
        v = a.table_f32 ? static_cast<const float*>(a.table)[at]
                        : bf16_to_f32(static_cast<const bf16_t*>(a.table)[at]);
        const bool finite = __builtin_isfinite(v);
        v *= 1.4426950408889634f;
        if (finite) v = fminf(fmaxf(v, kLowScore), -kLowScore);
      }
      lds_table[i] = v;
    }
    // bucket by bucket: every distance from its start to the next one's (of the
    // distances told apart: starts and their number are arguments of their own)
    for (int k = wave; k < a.buckets; k += kWaves) {
      const int from = k == 0 ? 0 : clamp_to(a.starts[k - 1], a.distances);
      const int to = k == a.buckets - 1 ? a.distances : clamp_to(a.starts[k], a.distances);
      for (int x = from + lane_id(); x < to; x += kWave) lds_bucket[x] = (uint16_t)k;
    }
    __syncthreads();
  }


  StepState<G, E> st;
  auto work = [&](const Rows& r, int i0) {
    float s[U][G];
    // distances of the iteration all in the last bucket (the first tokens' are the largest of all)
    const bool far = a.table && rows.distance(i0 + kPass - 1) >= a.distances - 1;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * kGroups + group;
#pragma unroll
      for (int g = 0; g < G; ++g) s[u][g] = group_sum<L>(dot(q[g], r.k[u]));
      if (a.table) {
        const float* bias = lds_table + (a.buckets - 1) * G;
        if (!far) {
          const int x = rows.distance(i < hi ? i : hi - 1);
          if (x < a.distances) bias = lds_table + lds_bucket[x] * G;
        }
#pragma unroll
        for (int g = 0; g < G; ++g) s[u][g] = __builtin_fmaf(s[u][g], a.c2, bias[g]);
      } else {
#pragma unroll
        for (int g = 0; g < G; ++g) s[u][g] *= a.c2;
      }
      if (i0 + kPass > hi) {
#pragma unroll
        for (int g = 0; g < G; ++g) s[u][g] = i < hi ? s[u][g] : -INFINITY;
      }
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float top = s[0][g];
#pragma unroll
      for (int u = 1; u < U; ++u) top = fmaxf(top, s[u][g]);
      if (__any(top > st.m[g] + 8.f)) st.raise(g, fmaxf(st.m[g], top));
#pragma unroll
      for (int u = 0; u < U; ++u) {
        const float p = exp2_fast(s[u][g] - st.m[g]);
        st.l[g] += p;
#pragma unroll
        for (int e = 0; e < E; ++e) st.acc[g][e] = __builtin_fmaf(p, element<T>(r.v[u], e), st.acc[g][e]);
      }
    }
  };
  for (int i0 = first_row; i0 < hi; i0 += 2 * stride) {
    load(odd, i0 + stride);
    work(even, i0);
    if (i0 + stride >= hi) break;
    load(even, i0 + 2 * stride);
    work(odd, i0 + stride);
  }
  // the new token's row takes its slot (this step reads it from the input)
  if (hi == rows.count && hg == 0 && wave == kWaves - 1 && group == 0) {
    const int slot = rows.slot(last);
    const typename F::Frag kf = load_row<T, kVec>(new_k, d, a.dim), vf = load_row<T, kVec>(new_v, d, a.dim);
    float kx[E], vx[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
      kx[e] = element<T>(kf, e);
      vx[e] = element<T>(vf, e);
    }
    store_piece<T, kVec>(row_at(cache_k, slot, a.ck_slot), d, a.dim, kx);
    store_piece<T, kVec>(row_at(cache_v, slot, a.cv_slot), d, a.dim, vx);
  }

#pragma unroll
  for (int x = L; x < kWave; x <<= 1) st.join_lanes(x);
  if (group == 0)
#pragma unroll
    for (int g = 0; g < G; ++g) {
      lds_join[wave][sub][g][0] = st.m[g];
      lds_join[wave][sub][g][1] = st.l[g];
#pragma unroll
      for (int e = 0; e < E; ++e) lds_join[wave][sub][g][2 + e] = st.acc[g][e];
    }
  __syncthreads();
  for (int i = threadIdx.x; i < L * heads; i += kStepThreads) {
    const int g = i / L, at = i % L;
    float m = lds_join[0][at][g][0];
#pragma unroll
    for (int w = 1; w < kWaves; ++w) m = fmaxf(m, lds_join[w][at][g][0]);
    float l = 0.f, v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = 0.f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
      const float f = exp2_fast(lds_join[w][at][g][0] - m);
      l += lds_join[w][at][g][1] * f;
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] += lds_join[w][at][g][2 + e] * f;
    }
    if (a.parts == 1) {
      const float inv = l > 0.f ? 1.f / l : 0.f;
#pragma unroll
      for (int e = 0; e < E; ++e) v[e] *= inv;
      store_piece<T, kVec>(out_row + (int64_t)g * a.dim, at * E, a.dim, v);
    } else {
      float* p = a.part + (((int64_t)b * a.q_heads + head0 + g) * a.parts + part) * (2 + a.dim);
      if (at == 0) {
        p[0] = m;
        p[1] = l;
      }
#pragma unroll
      for (int e = 0; e < E; ++e)
        if (at * E + e < a.dim) p[2 + at * E + e] = v[e];
    }
  }
}

// Joins the parts of a row's walk: one block per row and head.  Waves take every
// kWaves-th part, kAtOnce of them with all loads on their way at once and no
// load waiting for a maximum: the parts come from other XCDs, a trip of about
// a microsecond (128 parts, two users of 8 heads of 128: 4.2 us; 13 with the
// maximum first).
template <typename T>
__global__ __launch_bounds__(kJoinThreads) void attention_step_join_kernel(StepCall a, T* out) {
  constexpr int kWaves = kJoinThreads / kWave, kAtOnce = 8;
  __shared__ float joined[kWaves][2 + 2 * kWave];
  const int64_t at = blockIdx.x;
  const int64_t n = load_uniform(a.positions + blockIdx.x / a.q_heads);
  if (n < 0) return;
  const StepRows rows(a, n);
  const int per = rows.per_part(a.parts);
  const int parts = (rows.count + per - 1) / per, size = 2 + a.dim;
  const float* p = a.part + at * a.parts * size;
  const int wave = wave_id(), lane = lane_id();
  // a lane's two dimensions; those past the last take its value and are not stored
  const int d0 = lane < a.dim ? lane : a.dim - 1, d1 = lane + kWave < a.dim ? lane + kWave : a.dim - 1;
  float m = kNoScore, l = 0.f, v0 = 0.f, v1 = 0.f;
  for (int i0 = wave; i0 < parts; i0 += kWaves * kAtOnce) {
    float pm[kAtOnce], pl[kAtOnce], p0[kAtOnce], p1[kAtOnce];
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const int i = i0 + u * kWaves;
      const float* x = p + (int64_t)(i < parts ? i : i0) * size;
      pm[u] = x[0];
      pl[u] = x[1];
      p0[u] = x[2 + d0];
      p1[u] = x[2 + d1];
    }
    float top = m;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) top = fmaxf(top, pm[u]);
    const float f = exp2_fast(m - top);
    m = top;
    l *= f;
    v0 *= f;
    v1 *= f;
#pragma unroll
    for (int u = 0; u < kAtOnce; ++u) {
      const float w = i0 + u * kWaves < parts ? exp2_fast(pm[u] - m) : 0.f;
      l = __builtin_fmaf(pl[u], w, l);
      v0 = __builtin_fmaf(p0[u], w, v0);
      v1 = __builtin_fmaf(p1[u], w, v1);
    }
  }
  if (lane == 0) {
    joined[wave][0] = m;
    joined[wave][1] = l;
  }
  joined[wave][2 + lane] = v0;
  joined[wave][2 + kWave + lane] = v1;
  __syncthreads();
  const int d = threadIdx.x;
  if (d >= a.dim) return;
  m = joined[0][0];
#pragma unroll
  for (int w = 1; w < kWaves; ++w) m = fmaxf(m, joined[w][0]);
  float o = 0.f;
  l = 0.f;
#pragma unroll
  for (int w = 0; w < kWaves; ++w) {
    const float f = exp2_fast(joined[w][0] - m);
    l = __builtin_fmaf(joined[w][1], f, l);
    o = __builtin_fmaf(joined[w][2 + d], f, o);
  }
  o *= l > 0.f ? 1.f / l : 0.f;
  if constexpr (sizeof(T) == 2) out[at * a.dim + d] = f32_to_bf16(o);
  else out[at * a.dim + d] = o;
}

// The prompt form: rows of k and v at positions 0 .. length - 1 take their
// slots, those that a later one of the same slot replaces left out.  One
// block per (batch row, kWriteRows rows); a thread moves elements of one row.
constexpr int kWriteRows = 64;
template <typename T>
__global__ __launch_bounds__(256) void cache_write_kernel(StepCall a, int64_t len, uint32_t blocks_per_row,
                                                           const int64_t* lengths, int32_t right_aligned) {
  const int b = (int)(blockIdx.x / blocks_per_row);
  int64_t n = lengths[b];
  if (n > len) n = len;
  const int64_t shift = right_aligned ? len - n : 0;
  const int width = a.kv_heads * a.dim;
  const int64_t r0 = (int64_t)(blockIdx.x % blocks_per_row) * kWriteRows;
  for (int64_t i = threadIdx.x; i < kWriteRows * (int64_t)width; i += 256) {
    const int64_t r = r0 + i / width, p = r - shift;
    const int c = (int)(i % width), kv = c / a.dim, d = c % a.dim;
    if (r >= len || p < 0 || p >= n) continue;
    const int ring = a.capacity - a.sinks;
    if (p >= a.sinks && p < n - ring) continue;
    const int64_t slot = p < a.sinks ? p : a.sinks + (p - a.sinks) % ring;
    static_cast<T*>(a.cache_k)[b * a.ck_batch + slot * a.ck_slot + kv * a.ck_head + d] =
        static_cast<const T*>(a.k)[b * a.k_batch + r * a.row_k + kv * a.k_head + d];
    static_cast<T*>(a.cache_v)[b * a.cv_batch + slot * a.cv_slot + kv * a.cv_head + d] =
        static_cast<const T*>(a.v)[b * a.v_batch + r * a.row_v + kv * a.v_head + d];
  }
}

// ---------------------------------------------------------------- host side --

int heads_together(int share) { return share >= 5 ? 8 : (share >= 3 ? 4 : share); }

// Blocks that share a row's walk: one, unless the walks leave half of the CUs
// idle; then as many as give each CU two, of kStepMinRows cached rows or more.
int step_parts(const mdl_attention_step& a) {
  const int share = a.q_heads / a.kv_heads, g = heads_together(share);
  const int64_t units = a.batch * a.kv_heads * ((share + g - 1) / g);
  if (units > kCutUnits) return 1;
  const int64_t most = a.window > 0 && a.window + a.sinks < a.capacity ? a.window + a.sinks : a.capacity;
  int64_t parts = kStepBlocks / (units > 0 ? units : 1);
  const int64_t cap = most / kStepMinRows;
  if (parts > cap) parts = cap;
  return parts < 1 ? 1 : (int)parts;
}

int step_check(const mdl_attention_step* a, const char* what) {
  const std::string w(what);
  if (!a) return fail(MDL_ERR_INVALID, w + ": null descriptor");
  if (a->batch < 0) return fail(MDL_ERR_INVALID, w + ": negative batch");
  if (a->sinks < 0 || a->capacity <= a->sinks)
    return fail(MDL_ERR_INVALID, w + ": the capacity must exceed the first tokens kept");
  if (a->window > 0 && a->window > a->capacity - a->sinks)
    return fail(MDL_ERR_INVALID, w + ": the window must fit the capacity beside the first tokens");
  if (a->q_heads <= 0 || a->kv_heads <= 0 || a->q_heads % a->kv_heads)
    return fail(MDL_ERR_INVALID, w + ": q_heads must be a positive multiple of kv_heads");
  if (a->head_dim <= 0 || a->head_dim > 128) return fail(MDL_ERR_UNSUPPORTED, w + ": head_dim must be 1..128");
  if (a->dtype != MDL_F32 && a->dtype != MDL_BF16) return fail(MDL_ERR_INVALID, w + ": dtype");
  if (a->bias_table) {
    if (a->table_dtype != MDL_F32 && a->table_dtype != MDL_BF16) return fail(MDL_ERR_INVALID, w + ": table_dtype");
    if (a->num_buckets < 1 || (a->num_buckets > 1 && !a->bucket_starts) || a->distances < 1)
      return fail(MDL_ERR_INVALID, w + ": bias buckets");
    if (a->distances > kMaxDistances || a->num_buckets > 1024)
      return fail(MDL_ERR_UNSUPPORTED, w + ": bias buckets must begin at distances up to 2048, at most 1024 of them");
  }
  if (a->capacity > 0x3fffffff || a->ck_slot < 0 || a->cv_slot < 0 || a->ck_slot > 0x7fffffff ||
      a->cv_slot > 0x7fffffff)
    return fail(MDL_ERR_UNSUPPORTED, w + ": at most 2^30 slots, less than 2^31 elements apart");
  if (a->batch > 0 && (!a->k || !a->v || !a->cache_k || !a->cache_v || !a->positions))
    return fail(MDL_ERR_INVALID, w + ": null pointer");
  return MDL_OK;
}

StepCall step_call(const mdl_attention_step& a) {
  StepCall c{};
  c.q = a.q; c.k = a.k; c.v = a.v;
  c.cache_k = a.cache_k; c.cache_v = a.cache_v;
  c.positions = a.positions;
  c.table = a.bias_table;
  c.starts = a.bucket_starts;
  c.q_batch = a.q_batch; c.q_head = a.q_head;
  c.k_batch = a.k_batch; c.k_head = a.k_head;
  c.v_batch = a.v_batch; c.v_head = a.v_head;
  c.ck_batch = a.ck_batch; c.ck_slot = (uint32_t)a.ck_slot; c.ck_head = a.ck_head;
  c.cv_batch = a.cv_batch; c.cv_slot = (uint32_t)a.cv_slot; c.cv_head = a.cv_head;
  c.sinks = (int32_t)a.sinks;
  c.capacity = (int32_t)a.capacity;
  c.window = (int32_t)(a.window > 0 ? a.window : a.capacity - a.sinks);
  c.batch = (int32_t)a.batch; c.q_heads = a.q_heads; c.kv_heads = a.kv_heads; c.dim = a.head_dim;
  c.buckets = a.bias_table ? a.num_buckets : 0;
  c.distances = a.bias_table ? a.distances : 0;
  c.table_f32 = a.table_dtype == MDL_F32;
  c.c2 = (float)((double)a.scale * 1.4426950408889634);
  return c;
}

bool step_vectors(const mdl_attention_step& a) {
  const int64_t e = a.dtype == MDL_BF16 ? 8 : 4;
  auto whole = [&](const void* p, int64_t x, int64_t y, int64_t z) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && x % e == 0 && y % e == 0 && z % e == 0;
  };
  return a.head_dim % e == 0 && whole(a.q, a.q_batch, a.q_head, 0) && whole(a.k, a.k_batch, a.k_head, 0) &&
         whole(a.v, a.v_batch, a.v_head, 0) && whole(a.cache_k, a.ck_batch, a.ck_slot, a.ck_head) &&
         whole(a.cache_v, a.cv_batch, a.cv_slot, a.cv_head);
}

template <typename T, int L, int G, bool kVec, int kWaves>
int launch_step(const StepCall& c, int64_t blocks, void* out, hipStream_t s) {
  const size_t lds = ((size_t)c.buckets * G * 4 + (size_t)c.distances * 2 + 15) & ~size_t(15);
  const auto kernel = attention_step_kernel<T, L, G, kVec, kWaves>;
  if (int rc = allow_lds(reinterpret_cast<const void*>(kernel), lds, sizeof(StepJoin<T, L, G, kWaves>))) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kWaves * kWave), lds, s, c, static_cast<T*>(out));
  MDL_CHECK_LAUNCH("attention_step_kernel");
  return MDL_OK;
}

template <typename T, int L, int G, bool kVec>
int launch_step_blocks(const StepCall& c, void* out, hipStream_t s) {
  const int share = c.q_heads / c.kv_heads;
  const int64_t blocks = (int64_t)c.batch * c.kv_heads * ((share + G - 1) / G) * c.parts;
  if (blocks > 0x7fffffff) return fail(MDL_ERR_UNSUPPORTED, "mdl_attention_step: too many rows");
  if (int rc = blocks <= few_blocks<G>() ? launch_step<T, L, G, kVec, 8>(c, blocks, out, s)
                                    : launch_step<T, L, G, kVec, 4>(c, blocks, out, s))
    return rc;
  if (c.parts > 1) {
    const int64_t joins = (int64_t)c.batch * c.q_heads;
    if (joins > 0x7fffffff) return fail(MDL_ERR_UNSUPPORTED, "mdl_attention_step: too many rows");
    hipLaunchKernelGGL(attention_step_join_kernel<T>, dim3((unsigned)joins), dim3(kJoinThreads), 0, s, c,
                       static_cast<T*>(out));
    MDL_CHECK_LAUNCH("attention_step_join_kernel");
  }
  return MDL_OK;
}

template <typename T, int L, bool kVec>
int launch_step_heads(const StepCall& c, void* out, hipStream_t s) {
  switch (heads_together(c.q_heads / c.kv_heads)) {
    case 1: return launch_step_blocks<T, L, 1, kVec>(c, out, s);
    case 2: return launch_step_blocks<T, L, 2, kVec>(c, out, s);
    case 4: return launch_step_blocks<T, L, 4, kVec>(c, out, s);
    default: return launch_step_blocks<T, L, 8, kVec>(c, out, s);
  }
}

// Lanes per cached row: 16-byte pieces, rounded up to a power of two (4 to 32).
template <typename T, bool kVec>
int launch_step_lanes(const StepCall& c, void* out, hipStream_t s) {
  const int pieces = (c.dim + Frags<T>::kElems - 1) / Frags<T>::kElems;
  if (pieces <= 4) return launch_step_heads<T, 4, kVec>(c, out, s);
  if (pieces <= 8) return launch_step_heads<T, 8, kVec>(c, out, s);
  if (pieces <= 16) return launch_step_heads<T, 16, kVec>(c, out, s);
  if constexpr (sizeof(T) == 4) return launch_step_heads<T, 32, kVec>(c, out, s);
  return MDL_ERR_UNSUPPORTED;
}

}  // namespace mdl

using namespace mdl;

extern "C" {

size_t mdl_attention_step_workspace_bytes(const mdl_attention_step* a) {
  if (!a || step_check(a, "mdl_attention_step")) return 0;
  const int parts = step_parts(*a);
  return parts == 1 ? 0 : (size_t)a->batch * a->q_heads * parts * (2 + a->head_dim) * sizeof(float);
}

int mdl_attention_step_forward(const mdl_attention_step* a, void* out, void* workspace, size_t workspace_bytes,
                               void* stream) {
  if (int rc = step_check(a, "mdl_attention_step_forward")) return rc;
  if (!(a->scale > 0.f) || !(a->scale < INFINITY))
    return fail(MDL_ERR_INVALID, "mdl_attention_step_forward: scale must be positive");
  if (a->batch == 0) return MDL_OK;
  if (a->batch > 0x7fffffff) return fail(MDL_ERR_UNSUPPORTED, "mdl_attention_step_forward: too many rows");
  if (!a->q || !out) return fail(MDL_ERR_INVALID, "mdl_attention_step_forward: null pointer");
  const size_t need = mdl_attention_step_workspace_bytes(a);
  if (need && (!workspace || workspace_bytes < need))
    return fail(MDL_ERR_WORKSPACE, "mdl_attention_step_forward: workspace too small");
  StepCall c = step_call(*a);
  c.parts = step_parts(*a);
  c.part = static_cast<float*>(workspace);
  const hipStream_t s = as_stream(stream);
  if (a->dtype == MDL_BF16)
    return step_vectors(*a) ? launch_step_lanes<bf16_t, true>(c, out, s) : launch_step_lanes<bf16_t, false>(c, out, s);
  return step_vectors(*a) ? launch_step_lanes<float, true>(c, out, s) : launch_step_lanes<float, false>(c, out, s);
}

int mdl_attention_cache_write(const mdl_attention_step* a, int64_t len, int64_t k_row, int64_t v_row,
                              const int64_t* lengths, int32_t right_aligned, void* stream) {
  if (!a || !lengths) return fail(MDL_ERR_INVALID, "mdl_attention_cache_write: null pointer");
  mdl_attention_step with = *a;
  with.positions = lengths;
  with.bias_table = nullptr;
  if (int rc = step_check(&with, "mdl_attention_cache_write")) return rc;
  if (len < 0) return fail(MDL_ERR_INVALID, "mdl_attention_cache_write: negative length");
  if (a->batch == 0 || len == 0) return MDL_OK;
  const int64_t per_row = (len - 1) / kWriteRows + 1;
  if (per_row > 0x7fffffff / a->batch)
    return fail(MDL_ERR_UNSUPPORTED, "mdl_attention_cache_write: too many rows");
  StepCall c = step_call(with);
  c.row_k = k_row;
  c.row_v = v_row;
  const dim3 grid((unsigned)(per_row * a->batch));
  if (a->dtype == MDL_BF16)
    hipLaunchKernelGGL(cache_write_kernel<bf16_t>, grid, dim3(256), 0, as_stream(stream), c, len,
                       (uint32_t)per_row, lengths, right_aligned);
  else
    hipLaunchKernelGGL(cache_write_kernel<float>, grid, dim3(256), 0, as_stream(stream), c, len,
                       (uint32_t)per_row, lengths, right_aligned);
  MDL_CHECK_LAUNCH("cache_write_kernel");
  return MDL_OK;
}

}  // extern "C"
