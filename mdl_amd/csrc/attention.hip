// Attention over histories, forward: a sliding window, first tokens that stay
// visible, and a learned relative position bias.
//
// One pass over the keys with the running maximum m and sum l of the softmax:
// a block owns 128 query rows of one head (32 per wave) and walks key tiles
// that hold a visible column.  Per tile a wave makes x^T = K q^T (its queries
// are the result's columns, so a query's statistics are one value per lane),
// p = exp2(c2 x - c2 m), and out^T += V^T p^T.  Out is divided by l at the
// end; a query without a visible key gets zeros.
//
// The products' operands come from LDS (24 KB a wave and 32 x 64 scores of head
// dimension 128), where rows lie for both readings without bank conflicts, and
// tile t + 1 is on its way while tile t is worked on.  What bounds it: the wave's
// own chain of products, exponentials (a quarter of the vector rate) and
// products; matrix instructions are busy 36 % of the time at dimension 128
// (2 x 8192 rows, window 1024, 16 heads: 178 us, 735 TFLOP/s), 22 % at 64 without
// a window (8 rows of up to 4096, 8 heads: 147 us) and 14 % at 64 with one of 256
// keys, where half of the waves' tiles are partly masked (64 ragged rows of
// 2048, 4 heads: 84 us).
#include "attention.cuh"

namespace mdl {

// ------------------------------------------------------------------- prepare --
//
// What a call's kernels read instead of the mask and the bias table: the
// mask's columns as bits, the first unmasked column of a row, and every
// head's bias by distance, divided by the scale.

template <typename TB>
__device__ __forceinline__ float table_value(const TB* p) {
  if constexpr (sizeof(TB) == 2) return bf16_to_f32(*p);
  else return *p;
}

// Bucket of a distance: the number of starts at or below it.
__device__ __forceinline__ int bucket_of_distance(const int32_t* starts, int buckets, int d) {
  int lo = 0, hi = buckets - 1;  // starts[0 .. hi) of bucket 1 ..
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (starts[mid] <= d) lo = mid + 1;
    else hi = mid;
  }
  return lo;
}

struct PrepareCall {
  const uint8_t* mask;
  int64_t mask_row;
  const void* table;
  const int32_t* starts;
  uint64_t* words;
  int2* bounds;
  float* bias;
  int64_t words_row;
  int32_t batch, k_len, heads, buckets, distances;
  int32_t table_f32, mask_vec;  // mask_vec: mask rows in 16-byte pieces
  float inv_scale;
};

// The four bytes of x that are not 0, as four bits.
__device__ __forceinline__ uint32_t byte_bits(uint32_t x) {
  const uint32_t one = ((((x & 0x7f7f7f7fu) + 0x7f7f7f7fu) | x) >> 7) & 0x01010101u;
  return (one * 0x01020408u) >> 24 & 15u;
}

__global__ __launch_bounds__(256) void attention_prepare_kernel(PrepareCall a) {
  const int wave = threadIdx.x / kWave;
  int64_t block = blockIdx.x;
  if (a.mask) {
    if (block < a.batch) {
      __shared__ int firsts[4], lasts[4];
      const uint8_t* row = a.mask + block * a.mask_row;
      uint64_t* words = a.words + block * a.words_row;
      int first = a.k_len, last = -1;
      auto take = [&](int w, uint64_t word) {
        if (!word) return;
        if (first == a.k_len) first = 64 * w + __builtin_ctzll(word);
        last = 64 * w + 63 - __builtin_clzll(word);
      };
      if (a.mask_vec) {
        // a thread makes a word of its 64 columns' bytes
        for (int w = threadIdx.x; w < a.words_row; w += 256) {
          const int col = 64 * w;
          uint64_t word = 0;
#pragma unroll
          for (int i = 0; i < 4; ++i)
            if (col + 16 * i < a.k_len) {
              const u32x4 x = *(const gptr<u32x4>)(row + col + 16 * i);
#pragma unroll
              for (int k = 0; k < 4; ++k) word |= (uint64_t)byte_bits(x[k]) << (16 * i + 4 * k);
            }
          words[w] = word;
          take(w, word);
        }
      } else {
        // a wave's lanes are the columns of a word
#pragma unroll 4
        for (int w = wave; w < a.words_row; w += 4) {
          const int col = 64 * w + lane_id();
          const uint64_t word = __ballot(col < a.k_len && row[col] != 0);
          if (lane_id() == 0) words[w] = word;
          take(w, word);
        }
      }
      for (int s = 32; s >= 1; s >>= 1) {
        const int f = __shfl_xor(first, s), l = __shfl_xor(last, s);
        first = f < first ? f : first;
        last = l > last ? l : last;
      }
      if (lane_id() == 0) {
        firsts[wave] = first;
        lasts[wave] = last;
      }
      __syncthreads();
      if (threadIdx.x == 0) {
        for (int i = 1; i < 4; ++i) {
          first = firsts[i] < first ? firsts[i] : first;
          last = lasts[i] > last ? lasts[i] : last;
        }
        a.bounds[block] = make_int2(first, last);
      }
      return;
    }
    block -= a.batch;
  }
  const int64_t i = block * 256 + threadIdx.x;
  const int per_head = a.distances + 2 * kBiasEdge;
  if (!a.bias || i >= (int64_t)a.heads * per_head) return;
  const int h = (int)(i / per_head);
  int d = (int)(i % per_head) - kBiasEdge;
  d = d < 0 ? 0 : d;
  const int64_t at = (int64_t)bucket_of_distance(a.starts, a.buckets, d) * a.heads + h;
  const float v = a.table_f32 ? table_value(static_cast<const float*>(a.table) + at)
                              : table_value(static_cast<const bf16_t*>(a.table) + at);
  float x = v * a.inv_scale;
  // an infinite bias hides a key; a finite one never does, however low
  if (__builtin_isfinite(v)) x = fminf(fmaxf(x, kLowScore), -kLowScore);
  a.bias[i] = x;
}

// ------------------------------------------------------------------- forward --

// Raises of a row's maximum below this many powers of two are not applied
// (p stays below 2^8): most tiles then skip the rescaling of out.
constexpr float kLazyRaise = 8.f;

template <typename T, int DP, bool kVec>
__global__ __launch_bounds__(kAttnThreads) void attention_forward_kernel(AttnCall a, T* out, float2* stats) {
  using F = Frags<T>;
  using Stage = TileStage<T, DP, kVec>;
  constexpr int TK = F::kTile, LD = Tile<T, DP>::kLd, kSteps = DP / F::kStep, kSubs = TK / 32;
  constexpr int kStages = tile_stages<T, DP, kVec>();
  extern __shared__ __align__(16) char smem[];
  T* lds = reinterpret_cast<T*>(smem);                                       // [stages][K, V][TK][LD]
  float* lds_bias = reinterpret_cast<float*>(lds + kStages * 2 * TK * LD);  // [stages][kBiasSpan]

  int unit, inner;
  const BlockOrder order = query_blocks(a);
  if (!order.place(blockIdx.x, &unit, &inner)) return;
  const int qb = order.per_unit - 1 - inner;  // last rows first: without a window they walk the most tiles
  const int b = unit / a.q_heads, head = unit - b * a.q_heads;
  const int kv = head / (a.q_heads / a.kv_heads);
  const T* kp = static_cast<const T*>(a.k) + b * a.k_batch + kv * a.k_head;
  const T* vp = static_cast<const T*>(a.v) + b * a.v_batch + kv * a.v_head;
  const float* bias = a.bias ? head_bias(a, head) : nullptr;

  const int off = a.k_len - a.q_len;
  const int wave = wave_id(), l32 = lane_id() & 31, half = lane_id() >> 5;
  const int r0 = qb * kAttnRows;
  const int r_end = r0 + kAttnRows < a.q_len ? r0 + kAttnRows : a.q_len;
  const int row = r0 + 32 * wave + l32, c = row + off;
  const RowMask mask(a, b);
  const KeyWalk walk(a, mask, TK, r0 + off, r_end - 1 + off);
  const int wc_lo = r0 + 32 * wave + off;  // the wave's columns
  const uint32_t q_bits = mask.bits32(wc_lo);
  const bool live = (q_bits >> l32) & 1;

  typename F::Frag q[kSteps];
  load_own_row<T, DP, kVec>(static_cast<const T*>(a.q) + b * a.q_batch + head * a.q_head + (int64_t)row * a.q_row,
                            live, a.dim, q);
  f32x16 acc[DP / 32];
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = (f32x16)(0.f);
  float m = kNoScore, mneg = -(kNoScore * a.c2), l = 0.f;
  const float lazy = kLazyRaise / a.c2;
  const float far_bias = bias ? load_uniform(bias + kBiasEdge + a.distances - 1) : 0.f;

  const Tile<T, DP> read;
  Stage ks, vs;
  ks.open(lds, kp, a.k_row, a.dim);
  vs.open(lds + TK * LD, vp, a.v_row, a.dim);
  const uint32_t bias_to = lds_address(lds_bias + wave * kWave);
  auto fetch = [&](int i, int slot) {
    const int j0 = walk.tile_at(i) * TK;
    const uint64_t bits = mask.bits<TK>(j0);
    const uint32_t past = slot * (2 * TK * LD * (uint32_t)sizeof(T));
    ks.fetch(past, j0 * a.k_row, bits, a.dim);
    vs.fetch(past, j0 * a.v_row, bits, a.dim);
    // lds_bias[i]: distance i + that of the block's first query and the tile's last key
    if (bias)
      copy4_to_lds(bias_to + slot * (kBiasSpan * 4), bias + bias_at(a, r0 + off - j0 - (TK - 1)) + threadIdx.x);
  };
  auto settle = [&](int slot) {
    ks.settle(lds + slot * 2 * TK * LD);
    vs.settle(lds + slot * 2 * TK * LD + TK * LD);
  };
  auto large = [&](float most, float bias_of_all) { return is_large(a, fabsf(most) + fabsf(bias_of_all)); };
  auto work = [&](int i, int slot) {
    const T* lk = lds + slot * 2 * TK * LD;
    const T* lv = lk + TK * LD;
    const int j0 = walk.tile_at(i) * TK, j1 = j0 + TK - 1;
    const bool seen = q_bits && j0 <= wc_lo + 31 && (wc_lo - j1 < a.window || j0 < walk.sink_end);
    if (!seen) return;
    const uint64_t bits = mask.bits<TK>(j0);
    f32x16 x[kSubs];
    // distances of the wave and the tile all in the last bucket, or none told apart
    const bool far = !bias || wc_lo - j1 >= a.distances - 1;
    if (!far) {
#pragma unroll
      for (int s = 0; s < kSubs; ++s) {
        const float* from = lds_bias + slot * kBiasSpan + (32 * wave + l32 + TK - 1 - 32 * s - 4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[s][i] = from[-(8 * (i >> 2) + (i & 3))];
      }
    }
#pragma unroll
    for (int s = 0; s < kSubs; ++s) {
      const NatFrags<T, DP> k(read, lk, s);
      if constexpr (DP > 64) reads_first<T>();
      x[s] = far ? k.times(q, (f32x16)(0.f)) : k.times(q, x[s]);
    }
    const float shift = far ? far_bias : 0.f;  // what x lacks: one bias for the tile is added to the maximum instead
    const TrFrags<T, DP> v0(read, lv, 0);
    const bool whole = q_bits == ~0u && (TK == 64 ? bits == ~0ull : (uint32_t)bits == ~0u) && j1 <= wc_lo &&
                       wc_lo + 31 - j0 < a.window;
    if (!whole) {
#pragma unroll
      for (int s = 0; s < kSubs; ++s) {
        uint32_t vis = live ? visible32(c, j0 + 32 * s, a.window, walk.sink_end, (uint32_t)(bits >> (32 * s))) : 0u;
        vis >>= 4 * half;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[s][i] = keep_bit(vis, 8 * (i >> 2) + (i & 3), x[s][i], -INFINITY);
      }
    }
    float top = x[0][0];
#pragma unroll
    for (int s = 0; s < kSubs; ++s)
#pragma unroll
      for (int i = 0; i < 16; ++i) top = fmaxf(top, x[s][i]);
    top = max_halves(top) + shift;
    if (__any(top > m + lazy)) {
      const float up = fmaxf(m, top);
      const float shrink = exp2_fast((m - up) * a.c2);
      m = up;
      mneg = -(m * a.c2);
      l *= shrink;
#pragma unroll
      for (int i = 0; i < DP / 32; ++i) acc[i] *= shrink;
    }
    float from = __builtin_fmaf(shift, a.c2, mneg);
    if (__any(large(m, shift))) {
      const float add = large(m, shift) ? shift : 0.f, less = large(m, shift) ? m : 0.f;
#pragma unroll
      for (int s = 0; s < kSubs; ++s) x[s] = (x[s] + add) - less;
      from = large(m, shift) ? 0.f : from;
    }
    // the weights take the element type for the second product; their sum does not
    auto weigh = [&](f32x16& w) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        w[i] = exp2_fast(__builtin_fmaf(w[i], a.c2, from));
        l += w[i];
      }
    };
    weigh(x[0]);
    if constexpr (kSubs == 2) {
      const TrFrags<T, DP> v1(read, lv, 1);
      v0.times(x[0], acc);
      weigh(x[1]);
      v1.times(x[1], acc);
    } else {
      v0.times(x[0], acc);
    }
  };
  walk_tiles<kStages, 2 * Stage::kPer, Stage::kDirect>(walk.tiles, bias != nullptr, fetch, settle, work);

  l = sum_halves(l);
  if (row < a.q_len) {
    const int64_t at = (((int64_t)b * a.q_len + row) * a.q_heads + head) * a.dim;
    const float inv = l > 0.f ? 1.f / l : 0.f;
    store_result_row<T, DP>(out + at, acc, inv, a.dim);
    if (stats && half == 0) {
      // -m and -log2 of the sum at the unrounded c2 m; -inf makes every weight of an empty row 0
      const float ll = l > 0.f ? (large(m, 0.f) ? 0.f : __builtin_fmaf(m, a.c2, mneg)) - log2f(l) : -INFINITY;
      stats[((int64_t)b * a.q_heads + head) * a.q_len + row] = make_float2(l > 0.f ? -m : 0.f, ll);
    }
  }
}

template <typename T, int DP, bool kVec>
size_t forward_lds() {
  return tile_stages<T, DP, kVec>() * (2 * Frags<T>::kTile * Tile<T, DP>::kLd * sizeof(T) + kBiasSpan * sizeof(float));
}

template <typename T, int DP, bool kVec>
int launch_forward(const AttnCall& a, void* out, float2* stats, hipStream_t s) {
  const int64_t blocks = query_blocks(a).blocks();
  if (blocks > 0x7fffffff) return fail(MDL_ERR_UNSUPPORTED, "mdl_attention_forward: too many rows");
  const size_t lds = forward_lds<T, DP, kVec>();
  const auto kernel = attention_forward_kernel<T, DP, kVec>;
  if (int rc = allow_lds(reinterpret_cast<const void*>(kernel), lds)) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kAttnThreads), lds, s, a, static_cast<T*>(out), stats);
  MDL_CHECK_LAUNCH("attention_forward_kernel");
  return MDL_OK;
}

// ---------------------------------------------------------------- host side --

size_t align256(size_t n) { return (n + 255) & ~size_t(255); }

int64_t mask_words_row(const mdl_attention& a) { return (a.k_len + 63) / 64 + 1; }

// Where a prepared call's parts lie.
struct PrepareLayout {
  size_t words = 0, bounds = 0, bias = 0, bytes = 0;
  explicit PrepareLayout(const mdl_attention& a) {
    size_t at = 0;
    if (a.mask) {
      words = at;
      at = align256(at + (size_t)a.batch * mask_words_row(a) * 8);
      bounds = at;
      at = align256(at + (size_t)a.batch * 8);
    }
    if (a.bias_table) {
      bias = at;
      at = align256(at + (size_t)a.q_heads * (a.distances + 2 * kBiasEdge) * 4);
    }
    bytes = at;
  }
};

int attention_check(const mdl_attention* a, const char* what) {
  const std::string w(what);
  if (!a) return fail(MDL_ERR_INVALID, w + ": null descriptor");
  if (a->batch < 0 || a->q_len < 0 || a->k_len < a->q_len)
    return fail(MDL_ERR_INVALID, w + ": needs batch >= 0 and 0 <= q_len <= k_len");
  if (a->k_len > 0x3fffffff || (a->batch > 0 && a->q_heads > 0x7fffffff / a->batch)) return fail(MDL_ERR_UNSUPPORTED, w + ": too many rows");
  if (a->q_heads <= 0 || a->kv_heads <= 0 || a->q_heads % a->kv_heads)
    return fail(MDL_ERR_INVALID, w + ": q_heads must be a positive multiple of kv_heads");
  if (a->head_dim <= 0 || a->head_dim > 128) return fail(MDL_ERR_UNSUPPORTED, w + ": head_dim must be 1..128");
  if (a->dtype != MDL_F32 && a->dtype != MDL_BF16) return fail(MDL_ERR_INVALID, w + ": dtype");
  if (!(a->scale > 0.f) || !(a->scale < INFINITY)) return fail(MDL_ERR_INVALID, w + ": scale must be positive");
  if (a->sinks < 0) return fail(MDL_ERR_INVALID, w + ": sinks must not be negative");
  if (a->bias_table) {
    if (a->table_dtype != MDL_F32 && a->table_dtype != MDL_BF16) return fail(MDL_ERR_INVALID, w + ": table_dtype");
    if (a->num_buckets < 1 || (a->num_buckets > 1 && !a->bucket_starts) || a->distances < 1)
      return fail(MDL_ERR_INVALID, w + ": bias buckets");
    if (a->distances > kMaxDistances || a->num_buckets > 1024)
      return fail(MDL_ERR_UNSUPPORTED, w + ": bias buckets must begin at distances up to 2048, at most 1024 of them");
  }
  if (a->batch * a->q_len > 0 && (!a->q || !a->k || !a->v)) return fail(MDL_ERR_INVALID, w + ": null pointer");
  return MDL_OK;
}

AttnCall attention_call(const mdl_attention& a, const void* prepared) {
  const char* p = static_cast<const char*>(prepared);
  const PrepareLayout lay(a);
  AttnCall c{};
  c.q = a.q; c.k = a.k; c.v = a.v;
  c.q_batch = a.q_batch; c.q_row = a.q_row; c.q_head = a.q_head;
  c.k_batch = a.k_batch; c.k_row = a.k_row; c.k_head = a.k_head;
  c.v_batch = a.v_batch; c.v_row = a.v_row; c.v_head = a.v_head;
  if (a.mask) {
    c.words = reinterpret_cast<const uint64_t*>(p + lay.words);
    c.bounds = reinterpret_cast<const int2*>(p + lay.bounds);
    c.words_row = mask_words_row(a);
  }
  if (a.bias_table) c.bias = reinterpret_cast<const float*>(p + lay.bias);
  c.batch = (int32_t)a.batch; c.q_len = (int32_t)a.q_len; c.k_len = (int32_t)a.k_len;
  c.q_heads = a.q_heads; c.kv_heads = a.kv_heads; c.dim = a.head_dim;
  c.distances = a.bias_table ? a.distances : 0;
  c.window = (int32_t)(a.window > 0 && a.window < a.k_len ? a.window : a.k_len);
  // without a window every earlier column is visible as it is
  c.sinks = (int32_t)(c.window >= c.k_len ? 0 : (a.sinks < a.k_len ? a.sinks : a.k_len));
  c.scale = a.scale;
  c.c2 = (float)((double)a.scale * 1.4426950408889634);
  return c;
}

bool attention_vectors(const mdl_attention& a) {
  const int64_t e = a.dtype == MDL_BF16 ? 8 : 4;
  auto whole = [&](const void* p, int64_t b, int64_t r, int64_t h) {
    return reinterpret_cast<uintptr_t>(p) % 16 == 0 && b % e == 0 && r % e == 0 && h % e == 0;
  };
  return a.head_dim % e == 0 && whole(a.q, a.q_batch, a.q_row, a.q_head) && whole(a.k, a.k_batch, a.k_row, a.k_head) &&
         whole(a.v, a.v_batch, a.v_row, a.v_head);
}

int allow_lds(const void* kernel, size_t dynamic, size_t fixed) {
  if (dynamic + fixed <= 64 * 1024) return MDL_OK;
  return check_hip(hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)dynamic),
                   "hipFuncSetAttribute");
}

}  // namespace mdl

using namespace mdl;

extern "C" {

size_t mdl_attention_prepared_bytes(const mdl_attention* a) { return a ? PrepareLayout(*a).bytes : 0; }

int mdl_attention_prepare(const mdl_attention* a, void* prepared, size_t prepared_bytes, void* stream) {
  if (int rc = attention_check(a, "mdl_attention_prepare")) return rc;
  const PrepareLayout lay(*a);
  if (lay.bytes == 0 || a->batch == 0 || a->q_len == 0) return MDL_OK;
  if (!prepared || prepared_bytes < lay.bytes)
    return fail(MDL_ERR_WORKSPACE, "mdl_attention_prepare: prepared buffer too small");
  char* p = static_cast<char*>(prepared);
  PrepareCall c{};
  c.mask = a->mask;
  c.mask_row = a->mask_row;
  c.mask_vec = reinterpret_cast<uintptr_t>(a->mask) % 16 == 0 && a->mask_row % 16 == 0 && a->k_len % 16 == 0;
  c.table = a->bias_table;
  c.starts = a->bucket_starts;
  c.words = reinterpret_cast<uint64_t*>(p + lay.words);
  c.bounds = reinterpret_cast<int2*>(p + lay.bounds);
  c.bias = a->bias_table ? reinterpret_cast<float*>(p + lay.bias) : nullptr;
  c.words_row = mask_words_row(*a);
  c.batch = (int32_t)a->batch;
  c.k_len = (int32_t)a->k_len;
  c.heads = a->q_heads;
  c.buckets = a->num_buckets;
  c.distances = a->bias_table ? a->distances : 0;
  c.table_f32 = a->table_dtype == MDL_F32;
  c.inv_scale = 1.f / a->scale;
  const int64_t blocks = (a->mask ? a->batch : 0) + (c.bias ? ((int64_t)c.heads * (c.distances + 2 * kBiasEdge) + 255) / 256 : 0);
  hipLaunchKernelGGL(attention_prepare_kernel, dim3((unsigned)blocks), dim3(256), 0, as_stream(stream), c);
  MDL_CHECK_LAUNCH("attention_prepare_kernel");
  return MDL_OK;
}

int mdl_attention_forward(const mdl_attention* a, const void* prepared, void* out, float* stats, void* stream) {
  if (int rc = attention_check(a, "mdl_attention_forward")) return rc;
  if (a->batch == 0 || a->q_len == 0) return MDL_OK;
  if (!out || (PrepareLayout(*a).bytes && !prepared))
    return fail(MDL_ERR_INVALID, "mdl_attention_forward: null pointer");
  const AttnCall c = attention_call(*a, prepared);
  return for_attention(*a, attention_vectors(*a), [&]<typename T, int DP, bool kVec>() {
    return launch_forward<T, DP, kVec>(c, out, reinterpret_cast<float2*>(stats), as_stream(stream));
  });
}

}  // extern "C"
