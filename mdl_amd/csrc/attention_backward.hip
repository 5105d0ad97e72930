// Gradients of the history attention.
//
// With p the forward's weights (made again from q, k and the saved row
// statistics), dP = dO . v and delta = sum p dP of a row:
//   dS = p (dP - delta),  dq = scale sum_k dS k,  dk = scale sum_q dS q,
//   dv = sum_q p dO,      dbias[bucket] = sum of dS over the bucket's places.
// Two kernels, so that every sum has one owner and a fixed order: one walks
// the keys of 128 queries (dq and delta), then one the queries of 128 keys (dk
// and dv over all heads that share the keys, and the bias).  Making the
// weights twice costs two products more than making them once; adding dq
// across blocks instead would need atomics, whose order changes results.
//
// delta.  dO . out is delta up to the rounding of out, and of the weights
// that out was made from, to bfloat16: an error of the size of dS's own
// rounding, and larger in rows whose dS cancel.  The first kernel works with it
// all the same, adds the row's dS in fp32 to what it is short of (their sum
// is 0 with the true delta), and takes the share of k that belongs to the
// difference (a fourth product, sum p k) off dq at the end; the second kernel
// reads the corrected delta.  Delta is taken off after the product dP, not put
// in as its start: dP is then the same in every kernel and the difference exact
// where the two are close, so in a row that sees one key dP - delta comes to 0.
// (Unless the terms of that row's dP cancel to a millionth of their size: p, made
// again from the score, need not be 1 exactly, and up to 2^-40 or so of the terms
// can be left.  Its dq is set to 0, since the first kernel's dS still holds the
// first delta.)
// (The residual of out, saved by the forward, would
// spare that product, a tenth of the queries' kernel at dimension 128, for
// another 2 bytes per element of out held until the backward.)
//
// Times: 64 ragged rows of 2048 (4 heads of 64, window 256, bias): 126 us for
// the queries, 158 for the keys, 41 for the first tokens' far pairs; 2 x 8192
// rows (16 heads of 128 on 4, window 1024): 414, 467 and 44.  At dimension 128
// the accumulators leave room for one wave a SIMD, whose chain of LDS reads,
// products and exponentials bounds it (matrix instructions are busy 29 % of the
// time for the queries and 23 % for the keys); at 64 it is the same chain with two
// blocks a CU (17 % and 11 %).  At 128 two waves spill (an eighth longer), and
// the products of one sub-tile under the exponentials of another took longer
// too (466 against 433, without sum p k).
#include "attention.cuh"

namespace mdl {

struct GradCall {
  const void* out;
  const float2* stats;  // -m, -log2 of the sum
  const void* grad_out;
  int64_t g_batch, g_row, g_head;
  void *dq, *dk, *dv;
  float* delta;         // [B, Hq, Lq], negated
  const int32_t* starts;
  int32_t buckets;
  float* bias_partial;  // [Hq, bias_parts, buckets]; NULL: no bias gradient
  int64_t bias_parts, bias_far;  // parts of a head; the first one of the far blocks
  float* far_partial;   // [B, Hkv, far_chunks, sinks, 2, dim]; NULL: no far part
  int32_t far_chunks;
};

constexpr int kSpare = 96;      // distances of one tile and wave past either end of the bias
constexpr int kFarRows = 256;   // query rows of a block of the first tokens' far part
constexpr int kSkew = 64;       // diagonals of a 32x32 product tile, padded
constexpr int kFarFlats = 4;    // sums of the far part's waves in the last bucket

// ------------------------------------------------------ queries: dq, delta --

template <typename T, int DP, bool kVec>
__global__ __launch_bounds__(kAttnThreads) void attention_grad_q_kernel(AttnCall a, GradCall g) {
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
  const int wc_lo = r0 + 32 * wave + off;
  const uint32_t q_bits = mask.bits32(wc_lo);
  const bool live = (q_bits >> l32) & 1;

  typename F::Frag q[kSteps], go[kSteps];
  load_own_row<T, DP, kVec>(static_cast<const T*>(a.q) + b * a.q_batch + head * a.q_head + (int64_t)row * a.q_row,
                            live, a.dim, q);
  load_own_row<T, DP, kVec>(
      static_cast<const T*>(g.grad_out) + b * g.g_batch + head * g.g_head + (int64_t)row * g.g_row, live, a.dim, go);
  float m_neg = 0.f, ll_neg = -INFINITY, delta = 0.f;
  {
    typename F::Frag o[kSteps];
    load_own_row<T, DP, kVec>(static_cast<const T*>(g.out) + (((int64_t)b * a.q_len + row) * a.q_heads + head) * a.dim,
                              live, a.dim, o);
#pragma unroll
    for (int s = 0; s < kSteps; ++s)
#pragma unroll
      for (int i = 0; i < F::kElems; ++i) delta += (float)o[s][i] * (float)go[s][i];
    delta = sum_halves(delta);
    if (row < a.q_len) {
      const float2 st = g.stats[((int64_t)b * a.q_heads + head) * a.q_len + row];
      m_neg = st.x;
      ll_neg = st.y;
    }
  }
  f32x16 acc[DP / 32], pk[DP / 32];  // sums of dS k and of p k
#pragma unroll
  for (int i = 0; i < DP / 32; ++i) acc[i] = pk[i] = (f32x16)(0.f);
  float rest = 0.f;  // sum of dS: delta less dO . out
  uint32_t others = 0;  // not 0: the row sees a key beside its own
  const float far_bias = bias ? load_uniform(bias + kBiasEdge + a.distances - 1) : 0.f;
  // scores start at the bias less the maximum; a large maximum is taken off at the end
  const bool large = bias && is_large(a, m_neg), any_large = __any(large);
  const float far_from = large ? 0.f : far_bias + m_neg, near_from = large ? 0.f : m_neg;

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
    if (bias)
      copy4_to_lds(bias_to + slot * (kBiasSpan * 4), bias + bias_at(a, r0 + off - j0 - (TK - 1)) + threadIdx.x);
  };
  auto settle = [&](int slot) {
    ks.settle(lds + slot * 2 * TK * LD);
    vs.settle(lds + slot * 2 * TK * LD + TK * LD);
  };
  auto work = [&](int i, int slot) {
    const T* lk = lds + slot * 2 * TK * LD;
    const T* lv = lk + TK * LD;
    const int j0 = walk.tile_at(i) * TK, j1 = j0 + TK - 1;
    const bool seen = q_bits && j0 <= wc_lo + 31 && (wc_lo - j1 < a.window || j0 < walk.sink_end);
    if (!seen) return;
    const uint64_t bits = mask.bits<TK>(j0);
    const bool far = !bias || wc_lo - j1 >= a.distances - 1;
    const bool whole = q_bits == ~0u && (TK == 64 ? bits == ~0ull : (uint32_t)bits == ~0u) && j1 <= wc_lo &&
                       wc_lo + 31 - j0 < a.window && !any_large;
    if (whole) others = 1;
#pragma unroll
    for (int s = 0; s < kSubs; ++s) {
      f32x16 x, dp = (f32x16)(0.f);
      if (far) {
        x = (f32x16)(far_from);
      } else {
        const float* from = lds_bias + slot * kBiasSpan + (32 * wave + l32 + TK - 1 - 32 * s - 4 * half);
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = from[-(8 * (i >> 2) + (i & 3))] + near_from;
      }
      {
        const NatFrags<T, DP> kn(read, lk, s), vn(read, lv, s);
        reads_first<T>();
        x = kn.times(q, x);
        dp = vn.times(go, dp);
      }
      const TrFrags<T, DP> kt(read, lk, s);
      reads_first<T>();
      if (!whole) {
        if (any_large) x = (x + (far && large ? far_bias : 0.f)) + (large ? m_neg : 0.f);
        uint32_t vis = live ? visible32(c, j0 + 32 * s, a.window, walk.sink_end, (uint32_t)(bits >> (32 * s))) : 0u;
        const uint32_t own = c - (j0 + 32 * s);
        others |= vis & ~(own < 32 ? 1u << own : 0u);
        vis >>= 4 * half;
#pragma unroll
        for (int i = 0; i < 16; ++i) x[i] = keep_bit(vis, 8 * (i >> 2) + (i & 3), x[i], -INFINITY);
      }
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        x[i] = exp2_fast(__builtin_fmaf(x[i], a.c2, ll_neg));
        dp[i] = (dp[i] - delta) * x[i];
        rest += dp[i];
      }
      // p and dS take the element type for the products with k
      kt.times(dp, acc);
      kt.times(x, pk);
    }
  };
  walk_tiles<kStages, 2 * Stage::kPer, Stage::kDirect>(walk.tiles, bias != nullptr, fetch, settle, work);

  rest = sum_halves(rest);
  if (row >= a.q_len) return;
  if (half == 0) g.delta[((int64_t)b * a.q_heads + head) * a.q_len + row] = -(delta + rest);
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int i = 0; i < 16; ++i) acc[dt][i] = others ? __builtin_fmaf(-rest, pk[dt][i], acc[dt][i]) : 0.f;
  store_result_row<T, DP>(static_cast<T*>(g.dq) + (((int64_t)b * a.q_len + row) * a.q_heads + head) * a.dim, acc,
                          a.scale, a.dim);
}

// ------------------------------------------------------ keys: dk, dv, bias --
//
// The bias gradient sums dS along diagonals (one distance each).  A product
// tile is written to LDS skewed, so that a column holds one distance, and its
// columns are summed by the lanes into four registers each (64 distances of
// which a tile fills 63).  Along the walk the next tile's distances lie 32
// further: half of the sums are complete, cross the lanes and are stored, the
// other half moves down.  (One LDS addition per value instead took 356 us
// where the whole kernel takes 160.)  Tiles wholly in the last bucket
// are summed into one register.

struct DiagonalSums {
  float* skew;   // [32][kSkew] of the wave; places outside the tile's band stay 0
  float* sums;   // of the wave, by distance: sums[distance - shift + kSpare]
  float acc[4];  // distances at - 31 + 4 (lane % 16) + i, rows lane / 16 + 4 k
  float flat;
  int at;        // distance of the tile's corner (row 0, column 0)
  bool open;

  __device__ __forceinline__ void reset() {
    flat = 0.f;
    open = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) acc[i] = 0.f;
  }
  // the 32 distances from `from` on, held by lanes 0 .. 7 of every 16
  __device__ __forceinline__ void leave(int from) {
    f32x4 v;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const auto p = __builtin_amdgcn_permlane16_swap(__float_as_uint(acc[i]), __float_as_uint(acc[i]), false, false);
      v[i] = sum_halves(__uint_as_float(p[0]) + __uint_as_float(p[1]));
    }
    if (lane_id() < 8) *reinterpret_cast<f32x4*>(sums + (from & ~3) + kSpare + 4 * lane_id()) = v;
  }
  __device__ __forceinline__ void move_down() {
#pragma unroll
    for (int i = 0; i < 4; ++i)  // lane i takes lane i + 8 of its 16, zeros above
      acc[i] = __uint_as_float(__builtin_amdgcn_update_dpp(0, __float_as_uint(acc[i]), 0x108, 0xf, 0xf, true));
  }
  // both halves of what is open leave
  __device__ __forceinline__ void close() {
    if (!open) return;
    leave(at - 31);
    move_down();
    leave(at + 1);
    move_down();
    open = false;
  }
  __device__ __forceinline__ void add(const f32x16& ds, int corner) {
    if (open && corner == at + 32) {
      leave(at - 31);
      move_down();
    } else {
      close();
    }
    at = corner;
    open = true;
    // (row q, column n) -> skew[q][q - n + 31]
    float* to = skew + 4 * (lane_id() >> 5) * (kSkew + 1) + 31 - (lane_id() & 31);
#pragma unroll
    for (int i = 0; i < 16; ++i) to[(8 * (i >> 2) + (i & 3)) * (kSkew + 1)] = ds[i];
    wave_sync();
    const float* from = skew + (lane_id() >> 4) * kSkew + 4 * (lane_id() & 15);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const f32x4 v = *reinterpret_cast<const f32x4*>(from + 4 * k * kSkew);
#pragma unroll
      for (int i = 0; i < 4; ++i) acc[i] += v[i];
    }
    wave_sync();
  }
};

// One 32x32 product tile: 32 queries (rows, staged in LDS) and the wave's 32
// keys (columns, one per lane).
template <typename T, int DP>
struct KeyTile {
  using F = Frags<T>;
  static constexpr int kSteps = DP / F::kStep;
  Tile<T, DP> read;
  typename F::Frag k[kSteps], v[kSteps];
  f32x16 dk[DP / 32], dv[DP / 32];

  template <bool kVec>
  __device__ __forceinline__ void open(const AttnCall& a, int b, int kv, int j, bool live) {
    load_own_row<T, DP, kVec>(static_cast<const T*>(a.k) + b * a.k_batch + kv * a.k_head + (int64_t)j * a.k_row, live,
                              a.dim, k);
    load_own_row<T, DP, kVec>(static_cast<const T*>(a.v) + b * a.v_batch + kv * a.v_head + (int64_t)j * a.v_row, live,
                              a.dim, v);
#pragma unroll
    for (int i = 0; i < DP / 32; ++i) dk[i] = dv[i] = (f32x16)(0.f);
  }

  // Adds the tile to dk and dv; returns dS.  q, go: the 32 staged rows; stats,
  // delta: theirs (-m and -log2 sum; -delta); near_bias: the pairs' biases
  // by row (NULL: all far_bias); vis: the visible rows of the lane's key.
  __device__ __forceinline__ f32x16 add(const T* q, const T* go, const float* stats, const float* delta, float far_bias,
                                        const float* near_bias, bool whole, uint32_t vis, const AttnCall& a) {
    const int half = lane_id() >> 5;
    const bool any_large = a.bias && __any(is_large(a, stats[2 * (lane_id() & 31)]));
    stats += 8 * half;
    delta += 4 * half;
    f32x16 x, dp = (f32x16)(0.f);
#pragma unroll
    for (int i = 0; i < 16; ++i) {
      x[i] = stats[2 * (8 * (i >> 2) + (i & 3))];
    }
    if (near_bias) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] += near_bias[8 * (i >> 2) + (i & 3)];
    } else if (far_bias != 0.f) {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] += far_bias;
    }
    if (any_large) {  // rows with a large maximum start without it, and far ones without their bias
#pragma unroll
      for (int i = 0; i < 16; ++i)
        if (is_large(a, stats[2 * (8 * (i >> 2) + (i & 3))])) x[i] = near_bias ? near_bias[8 * (i >> 2) + (i & 3)] : 0.f;
    }
    {
      const NatFrags<T, DP> qn(read, q, 0), gn(read, go, 0);
      reads_first<T>();
      x = qn.times(k, x);
      dp = gn.times(v, dp);
    }
    if (any_large) {
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float m_neg = stats[2 * (8 * (i >> 2) + (i & 3))];
        if (is_large(a, m_neg)) x[i] = (x[i] + (near_bias ? 0.f : far_bias)) + m_neg;
      }
    }
    const TrFrags<T, DP> gt(read, go, 0), qt(read, q, 0);
    reads_first<T>();
    if (!whole) {
      vis >>= 4 * half;
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = keep_bit(vis, 8 * (i >> 2) + (i & 3), x[i], -INFINITY);
    }
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = exp2_fast(__builtin_fmaf(x[i], a.c2, stats[2 * (8 * (i >> 2) + (i & 3)) + 1]));
    gt.times(x, dv);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] *= dp[i] + delta[8 * (i >> 2) + (i & 3)];
    qt.times(x, dk);
    return x;
  }
};

// The bias gradient of a block, one head of its group at a time.
struct BlockBias {
  float *skew, *sums;  // [waves][32][kSkew], [waves][n_pad]
  int n_pad, shift;    // distances of a wave's tiles are alike modulo 32: stored from a multiple of 4
  DiagonalSums diag;

  // any_corner: distance of any tile's corner
  __device__ __forceinline__ void open(const AttnCall& a, float* lds, int any_corner) {
    n_pad = (a.distances + 2 * kSpare + 3) & ~3;
    skew = lds;
    sums = lds + 4 * 32 * kSkew;
    shift = (any_corner + 1) & 3;
    diag.skew = skew + wave_id() * 32 * kSkew;
    diag.sums = sums + wave_id() * n_pad;
    diag.reset();
    for (int i = threadIdx.x; i < 4 * 32 * kSkew; i += kAttnThreads) skew[i] = 0.f;
    for (int i = threadIdx.x; i < 4 * n_pad; i += kAttnThreads) sums[i] = 0.f;
    __syncthreads();
  }
  // Writes the head's sums by bucket and starts anew (every wave calls it).
  __device__ __forceinline__ void leave(const AttnCall& a, const GradCall& g, int head, int64_t part) {
    diag.close();
    float flat = diag.flat;
    for (int s = 32; s >= 1; s >>= 1) flat += __shfl_xor(flat, s);
    __syncthreads();
    if (lane_id() == 0) diag.skew[kSkew - 1] = flat;  // a place no tile fills
    for (int i = threadIdx.x; i < n_pad; i += kAttnThreads)
      sums[i] = (sums[i] + sums[n_pad + i]) + (sums[2 * n_pad + i] + sums[3 * n_pad + i]);
    __syncthreads();
    float* partial = g.bias_partial + ((int64_t)head * g.bias_parts + part) * g.buckets;
    const int sub = threadIdx.x & 7;
    for (int k = threadIdx.x >> 3; k < g.buckets; k += kAttnThreads / 8) {
      const int most = a.distances + kSpare - 4;  // the sums end there, whatever the starts hold
      const int lo = k == 0 ? 0 : clamp_to(g.starts[k - 1], most);
      const int hi = k == g.buckets - 1 ? most : clamp_to(g.starts[k], most);
      float s = 0.f;
      for (int d = lo + sub; d < hi; d += 8) s += sums[d - shift + kSpare];
      for (int x = 4; x >= 1; x >>= 1) s += __shfl_xor(s, x);
      if (k == g.buckets - 1)
        for (int w = 0; w < 4; ++w) s += skew[w * 32 * kSkew + kSkew - 1];
      if (sub == 0) partial[k] = s;
    }
    __syncthreads();
    if (lane_id() == 0) diag.skew[kSkew - 1] = 0.f;
    for (int i = threadIdx.x; i < 4 * n_pad; i += kAttnThreads) sums[i] = 0.f;
    __syncthreads();
    diag.reset();
  }
  __device__ __forceinline__ void add(const f32x16& ds, int corner, bool far) {
    if (far) {
#pragma unroll
      for (int i = 0; i < 16; ++i) diag.flat += ds[i];
    } else {
      diag.add(ds, corner - shift);
    }
  }
};

// A block without a pair: zeros for the heads' parts of the bias gradient.
__device__ __forceinline__ void leave_nothing(const GradCall& g, int head, int heads, int64_t part) {
  for (int i = threadIdx.x; i < heads * g.buckets; i += kAttnThreads)
    g.bias_partial[((int64_t)(head + i / g.buckets) * g.bias_parts + part) * g.buckets + i % g.buckets] = 0.f;
}

// The pairs within a window: 128 keys a block, 32 per wave.
template <typename T, int DP, bool kVec>
__global__ __launch_bounds__(kAttnThreads) void attention_grad_kv_kernel(AttnCall a, GradCall g) {
  using F = Frags<T>;
  using Stage = TileStage<T, DP, kVec>;
  constexpr int TQ = F::kTile, LD = Tile<T, DP>::kLd, kSubs = TQ / 32;
  constexpr int kStages = 2;  // a third would leave LDS for one block beside the bias sums
  extern __shared__ __align__(16) char smem[];
  T* lds = reinterpret_cast<T*>(smem);                                      // [stages][Q, dO][TQ][LD]
  float* lds_row = reinterpret_cast<float*>(lds + kStages * 2 * TQ * LD);  // [stages][(-m, -log2 sum)[TQ], -delta[TQ], ..]
  float* lds_bias = lds_row + kStages * kAttnThreads;                      // [stages][kBiasSpan]

  const int share = a.q_heads / a.kv_heads, off = a.k_len - a.q_len;
  const int key_blocks = (a.k_len + kAttnRows - 1) / kAttnRows;
  int unit, kb;  // first keys first: without a window they walk the most tiles
  if (!key_unit_blocks(a, key_blocks).place(blockIdx.x, &unit, &kb)) return;
  const int b = unit / a.kv_heads, kv = unit - b * a.kv_heads;
  const RowMask mask(a, b);

  const int wave = wave_id(), l32 = lane_id() & 31, half = lane_id() >> 5;
  const int k0 = kb * kAttnRows;
  const int jw = k0 + 32 * wave, j = jw + l32;
  const uint32_t k_bits = mask.bits32(jw);
  const bool live = (k_bits >> l32) & 1;

  // columns of the queries with a pair here, as tiles of query rows
  int c_lo = k0 > mask.first ? k0 : mask.first, c_hi = k0 + kAttnRows - 1 + a.window - 1;
  if (c_hi > mask.last) c_hi = mask.last;
  if (c_lo < off) c_lo = off;
  const int t_first = (c_lo - off) / TQ;
  const bool any = c_lo <= c_hi && k0 <= mask.last && k0 + kAttnRows > mask.first;
  const int per_head = any ? (c_hi - off) / TQ - t_first + 1 : 0;

  KeyTile<T, DP> tile;
  tile.template open<kVec>(a, b, kv, j, live);
  const bool want_bias = g.bias_partial != nullptr;
  const int64_t part = (int64_t)b * key_blocks + kb;
  BlockBias sums;
  if (want_bias) {
    if (any) sums.open(a, lds_bias + kStages * kBiasSpan, off - k0);
    else leave_nothing(g, kv * share, share, part);
  }

  Stage qs, gs;
  qs.open(lds, static_cast<const T*>(a.q) + b * a.q_batch, a.q_row, a.dim);
  gs.open(lds + TQ * LD, static_cast<const T*>(g.grad_out) + b * g.g_batch, g.g_row, a.dim);
  const uint32_t row_to = lds_address(lds_row + wave * kWave), bias_to = lds_address(lds_bias + wave * kWave);
  int fetch_head = 0, fetch_tile = 0;  // the next pair to fetch: head of the group, tile of the walk
  auto fetch = [&](int, int slot) {
    const int head = kv * share + fetch_head, row0 = (t_first + fetch_tile) * TQ;
    if (++fetch_tile == per_head) {
      fetch_tile = 0;
      ++fetch_head;
    }
    const uint64_t bits = mask.bits<TQ>(row0 + off);
    const uint32_t past = slot * (2 * TQ * LD * (uint32_t)sizeof(T));
    qs.fetch(past, head * a.q_head + row0 * a.q_row, bits, a.dim);
    gs.fetch(past, head * g.g_head + row0 * g.g_row, bits, a.dim);
    // one float a thread: the rows' statistics, then their delta (rows past the last one take its)
    {
      const int n = threadIdx.x, most = a.q_len - 1;
      const int r = n < 2 * TQ ? row0 + (n >> 1) : row0 + ((n - 2 * TQ) & (TQ - 1));
      const int64_t at = ((int64_t)b * a.q_heads + head) * a.q_len + (r < most ? r : most);
      const float* from = n < 2 * TQ ? reinterpret_cast<const float*>(g.stats + at) + (n & 1) : g.delta + at;
      copy4_to_lds(row_to + slot * (kAttnThreads * 4), from);
    }
    // lds_bias[i]: distance i + that of the tile's first query and the block's last key
    if (a.bias)
      copy4_to_lds(bias_to + slot * (kBiasSpan * 4),
                   head_bias(a, head) + bias_at(a, row0 + off - k0 - (kAttnRows - 1)) + threadIdx.x);
  };
  auto settle = [&](int slot) {
    qs.settle(lds + slot * 2 * TQ * LD);
    gs.settle(lds + slot * 2 * TQ * LD + TQ * LD);
  };
  int hs = 0, t = 0;
  float far_bias = a.bias ? load_uniform(head_bias(a, kv * share) + kBiasEdge + a.distances - 1) : 0.f;
  auto work = [&](int, int slot) {
    const T* lq = lds + slot * 2 * TQ * LD;
    const T* lg = lq + TQ * LD;
    const float* lr = lds_row + slot * kAttnThreads;
    const float* lb = lds_bias + slot * kBiasSpan;
    const int c0 = (t_first + t) * TQ + off, c1 = c0 + TQ - 1;
    const bool seen = k_bits && c1 >= jw && c0 - (jw + 31) < a.window;
    if (seen) {
      const uint64_t bits = mask.bits<TQ>(c0);
      const bool whole = k_bits == ~0u && (TQ == 64 ? bits == ~0ull : (uint32_t)bits == ~0u) && c0 >= jw + 31 &&
                         c1 - jw < a.window;
#pragma unroll
      for (int s = 0; s < kSubs; ++s) {
        const int col = c0 + 32 * s, corner = col - jw;
        const bool far = !a.bias || corner - 31 >= a.distances - 1;
        uint32_t vis = 0;
        if (!whole)
          vis = live ? ~low_bits(j - col) & low_bits(j + a.window - col) & (uint32_t)(bits >> (32 * s)) : 0u;
        const f32x16 ds =
            tile.add(lq + 32 * s * LD, lg + 32 * s * LD, lr + 64 * s, lr + 2 * TQ + 32 * s, far_bias,
                     far ? nullptr : lb + (kAttnRows - 1 - 32 * wave - l32 + 32 * s + 4 * half), whole, vis, a);
        if (want_bias) sums.add(ds, corner, far);
      }
    }
    if (++t == per_head) {
      if (want_bias) sums.leave(a, g, kv * share + hs, part);
      t = 0;
      ++hs;
      if (a.bias && hs < share)
        far_bias = load_uniform(head_bias(a, kv * share + hs) + kBiasEdge + a.distances - 1);
    }
  };
  walk_tiles<kStages, 2 * Stage::kPer + 1, Stage::kDirect>(per_head * share, a.bias != nullptr, fetch, settle, work);
  // the far parts of the first tokens among the block's keys: summed over their
  // chunks in order by all threads, 32 keys at a time, then taken from LDS
  const int sink_end = mask.first + a.sinks < a.k_len ? mask.first + a.sinks : a.k_len;
  if (g.far_partial && mask.first < k0 + kAttnRows && k0 < sink_end) {
    float* summed = reinterpret_cast<float*>(smem);  // [32][2][dim]: no more than the tiles took
    for (int w = 0; w < kAttnRows / 32; ++w) {
      const int lo = k0 + 32 * w > mask.first ? k0 + 32 * w : mask.first;
      const int hi = k0 + 32 * w + 32 < sink_end ? k0 + 32 * w + 32 : sink_end;
      if (lo >= hi) continue;
      __syncthreads();
      const int n = (hi - lo) * 2 * a.dim;
      const float* far = g.far_partial +
                         (((int64_t)b * a.kv_heads + kv) * g.far_chunks * a.sinks + (lo - mask.first)) * 2 * a.dim;
      const int64_t chunk = (int64_t)a.sinks * 2 * a.dim;
      for (int i = threadIdx.x; i < n; i += kAttnThreads) {
        float s = 0.f;
#pragma unroll 8
        for (int c = 0; c < g.far_chunks; ++c) s += far[c * chunk + i];
        summed[i] = s;
      }
      __syncthreads();
      if (wave == w && j >= lo && j < hi) {
        const float* mine = summed + (j - lo) * 2 * a.dim;
#pragma unroll
        for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
          for (int i = 0; i < 16; ++i) {
            const int d = 32 * dt + result_row(i);
            if (d < a.dim) {
              tile.dk[dt][i] += mine[d];
              tile.dv[dt][i] += mine[a.dim + d];
            }
          }
      }
    }
  }
  if (j >= a.k_len) return;
  const int64_t at = (((int64_t)b * a.k_len + j) * a.kv_heads + kv) * a.dim;
  store_result_row<T, DP>(static_cast<T*>(g.dk) + at, tile.dk, a.scale, a.dim);
  store_result_row<T, DP>(static_cast<T*>(g.dv) + at, tile.dv, 1.f, a.dim);
}

// Whether all pairs a window or more apart lie in the bias's last bucket: their
// gradient is then one sum and needs none of the diagonals' LDS.
__host__ __device__ __forceinline__ bool far_is_flat(const AttnCall& a) { return a.window >= a.distances - 1; }

// Waves of a block that walk: those whose staged rows fit LDS beside the bias.
template <typename T, int DP>
__host__ __device__ constexpr int far_waves() { return sizeof(T) == 4 && DP == 128 ? 2 : 4; }

// The pairs of the first tokens and the queries a window or more past them.
// Every query after a first token sees it, so a block that owned it whole
// would walk the row while the others walk one window: these pairs are cut
// into kFarRows query rows a block, whose parts the block that owns the keys
// adds in order.  A block has 32 first tokens; its waves take 32 query rows
// each in turn, staged in LDS of their own (no barrier in the walk).
template <typename T, int DP, bool kVec>
__global__ __launch_bounds__(kAttnThreads) void attention_grad_far_kernel(AttnCall a, GradCall g) {
  using F = Frags<T>;
  constexpr int LD = Tile<T, DP>::kLd, kPieces = DP / F::kElems, kPer = 32 * kPieces / kWave;
  constexpr int kBias = 64, kWalk = far_waves<T, DP>();
  extern __shared__ __align__(16) char smem[];
  const int wave = wave_id(), l32 = lane_id() & 31, half = lane_id() >> 5;
  T* lq = reinterpret_cast<T*>(smem) + wave * 64 * LD;  // of the wave: [Q, dO][32][LD]
  T* lg = lq + 32 * LD;
  float* lr = reinterpret_cast<float*>(reinterpret_cast<T*>(smem) + kWalk * 64 * LD) + wave * (96 + kBias);
  float* lb = lr + 96;  // lr: (-m, -log2 sum)[32], -delta[32]
  float* joined = reinterpret_cast<float*>(smem);  // [dk, dv][32][dim], after the walk
  __shared__ float flats[kFarFlats];

  const int share = a.q_heads / a.kv_heads, off = a.k_len - a.q_len;
  const int key_blocks = (a.sinks + 31) / 32;
  int unit, inner;
  if (!key_unit_blocks(a, key_blocks * g.far_chunks).place(blockIdx.x, &unit, &inner)) return;
  const int kb = inner % key_blocks, chunk = inner / key_blocks;
  const int b = unit / a.kv_heads, kv = unit - b * a.kv_heads;
  const RowMask mask(a, b);
  const int first = mask.first;
  const int k_end = first + a.sinks < a.k_len ? first + a.sinks : a.k_len;
  const int k0 = first + 32 * kb, j = k0 + l32;
  const uint32_t k_bits = mask.bits32(k0) & low_bits(k_end - k0);
  const bool live = (k_bits >> l32) & 1;

  const int64_t part = g.bias_far + ((int64_t)b * g.far_chunks + chunk) * key_blocks + kb;
  const bool want_bias = g.bias_partial != nullptr;
  float* to = g.far_partial + ((((int64_t)b * a.kv_heads + kv) * g.far_chunks + chunk) * a.sinks + 32 * kb) * 2 * a.dim;
  const int r_first = chunk * kFarRows, r_last = r_first + kFarRows < a.q_len ? r_first + kFarRows : a.q_len;
  if (k0 > mask.last || r_last - 1 + off < k0 + a.window || r_first + off > mask.last) {  // no pair
    for (int i = threadIdx.x; i < 32 * 2 * a.dim; i += kAttnThreads)
      if (32 * kb + i / (2 * a.dim) < a.sinks) to[i] = 0.f;
    if (want_bias) leave_nothing(g, kv * share, share, part);
    return;
  }

  KeyTile<T, DP> tile;
  tile.template open<kVec>(a, b, kv, j, live);
  BlockBias sums;
  const bool all_far = far_is_flat(a);
  if (want_bias && !all_far)
    sums.open(a, reinterpret_cast<float*>(reinterpret_cast<T*>(smem) + kWalk * 64 * LD) + kWalk * (96 + kBias), off - k0);
  if (all_far) sums.diag.flat = 0.f;
  for (int hs = 0; hs < share; ++hs) {
    const int head = kv * share + hs;
    const float far_bias = a.bias ? load_uniform(head_bias(a, head) + kBiasEdge + a.distances - 1) : 0.f;
    const T* qp = static_cast<const T*>(a.q) + b * a.q_batch + head * a.q_head;
    const T* gp = static_cast<const T*>(g.grad_out) + b * g.g_batch + head * g.g_head;
    for (int r0 = r_first + 32 * wave; wave < kWalk && r0 < r_last; r0 += 32 * kWalk) {
      const int col = r0 + off;
      const uint32_t bits = mask.bits32(col);
      if (!k_bits || !bits || col + 31 < k0 + a.window) continue;
      typename F::Frag qr[kPer], gr[kPer];
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int at = i * kWave + lane_id(), row = at / kPieces, d = at % kPieces * F::kElems;
        qr[i] = gr[i] = {};
        if ((bits >> row) & 1) {
          qr[i] = load_row<T, kVec>(qp + (int64_t)(r0 + row) * a.q_row, d, a.dim);
          gr[i] = load_row<T, kVec>(gp + (int64_t)(r0 + row) * g.g_row, d, a.dim);
        }
      }
      float2 st = make_float2(0.f, -INFINITY);
      float delta = 0.f;
      if (r0 + l32 < a.q_len) {
        const int64_t at = ((int64_t)b * a.q_heads + head) * a.q_len + r0 + l32;
        st = g.stats[at];
        delta = g.delta[at];
      }
      const int corner = col - k0;
      const bool far = !a.bias || corner - 31 >= a.distances - 1;
      float near = 0.f;
      if (!far) {
        // lb[i]: distance corner - 31 + i
        near = head_bias(a, head)[bias_at(a, corner - 31) + lane_id()];
      }
      wave_sync();
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int at = i * kWave + lane_id();
        *reinterpret_cast<typename F::Frag*>(lq + Tile<T, DP>::place(at / kPieces, at % kPieces)) = qr[i];
        *reinterpret_cast<typename F::Frag*>(lg + Tile<T, DP>::place(at / kPieces, at % kPieces)) = gr[i];
      }
      if (half == 0) {
        lr[2 * l32] = st.x;
        lr[2 * l32 + 1] = st.y;
        lr[64 + l32] = delta;
      }
      if (!far) lb[lane_id()] = near;
      wave_sync();
      const bool whole = k_bits == ~0u && bits == ~0u && corner - 31 >= a.window;
      const uint32_t vis = live ? ~low_bits(j + a.window - col) & bits : 0u;
      const f32x16 ds =
          tile.add(lq, lg, lr, lr + 64, far_bias, far ? nullptr : lb + 31 - l32 + 4 * half, whole, vis, a);
      if (want_bias) sums.add(ds, corner, far || all_far);
    }
    if (!want_bias) continue;
    if (!all_far) {
      sums.leave(a, g, head, part);
      continue;
    }
    float flat = sums.diag.flat;
    for (int s = 32; s >= 1; s >>= 1) flat += __shfl_xor(flat, s);
    sums.diag.flat = 0.f;
    __syncthreads();
    if (lane_id() == 0) flats[wave] = flat;
    __syncthreads();
    for (int k = threadIdx.x; k < g.buckets; k += kAttnThreads)
      g.bias_partial[((int64_t)head * g.bias_parts + part) * g.buckets + k] =
          k == g.buckets - 1 ? (flats[0] + flats[1]) + (flats[2] + flats[3]) : 0.f;
  }

  // the waves' sums, added in order
  for (int w = 0; w < kWalk; ++w) {
    __syncthreads();
    if (wave == w) {
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
        for (int i = 0; i < 16; ++i) {
          float* at = joined + (32 * dt + result_row(i)) * 32 + l32;
          at[0] = (w ? at[0] : 0.f) + tile.dk[dt][i];
          at[DP * 32] = (w ? at[DP * 32] : 0.f) + tile.dv[dt][i];
        }
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < 32 * 2 * a.dim; i += kAttnThreads) {
    const int key = i / (2 * a.dim), which = i / a.dim & 1, d = i % a.dim;
    if (32 * kb + key < a.sinks) to[(int64_t)key * 2 * a.dim + which * a.dim + d] = joined[which * DP * 32 + d * 32 + key];
  }
}

// ---------------------------------------------------------------- host side --

struct BackwardLayout {
  size_t delta = 0, bias = 0, far = 0, bytes = 0;
  int64_t bias_parts = 0, bias_far = 0;
  int32_t far_chunks = 0;
  explicit BackwardLayout(const mdl_attention& a) {
    auto take = [&](size_t n) {
      const size_t at = bytes;
      bytes = (bytes + n + 255) & ~size_t(255);
      return at;
    };
    delta = take((size_t)a.batch * a.q_heads * a.q_len * 4);
    if (a.window > 0 && a.window < a.k_len && a.sinks > 0) {
      const int64_t sinks = a.sinks < a.k_len ? a.sinks : a.k_len;
      far_chunks = (int32_t)((a.q_len + kFarRows - 1) / kFarRows);
      far = take((size_t)a.batch * a.kv_heads * far_chunks * sinks * 2 * a.head_dim * 4);
      bias_parts = a.batch * far_chunks * ((sinks + 31) / 32);
    }
    if (a.bias_table) {
      bias_far = a.batch * ((a.k_len + kAttnRows - 1) / kAttnRows);
      bias_parts += bias_far;
      bias = take((size_t)bias_parts * a.q_heads * a.num_buckets * 4);
    }
  }
};

template <typename T, int DP, bool kVec>
int launch_backward(const AttnCall& a, const GradCall& g, hipStream_t s) {
  using F = Frags<T>;
  constexpr int kStages = tile_stages<T, DP, kVec>();
  const size_t tiles = kStages * (2 * F::kTile * Tile<T, DP>::kLd * sizeof(T) + kBiasSpan * sizeof(float));
  {
    const int64_t blocks = query_blocks(a).blocks();
    const auto kernel = attention_grad_q_kernel<T, DP, kVec>;
    if (blocks > 0x7fffffff) return fail(MDL_ERR_UNSUPPORTED, "mdl_attention_backward: too many rows");
    if (int rc = allow_lds(reinterpret_cast<const void*>(kernel), tiles)) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kAttnThreads), tiles, s, a, g);
    MDL_CHECK_LAUNCH("attention_grad_q_kernel");
  }
  const size_t bias_lds =
      g.bias_partial ? (size_t)4 * (32 * kSkew + ((a.distances + 2 * kSpare + 3) & ~3)) * sizeof(float) : 0;
  if (g.far_partial) {
    const int64_t blocks = key_unit_blocks(a, (a.sinks + 31) / 32 * g.far_chunks).blocks();
    const size_t walk =
        far_waves<T, DP>() * ((size_t)64 * Tile<T, DP>::kLd * sizeof(T) + (96 + 64) * sizeof(float)) +
        (far_is_flat(a) ? 0 : bias_lds);
    const size_t join = (size_t)2 * DP * 32 * sizeof(float);
    const size_t lds = walk > join ? walk : join;
    const auto kernel = attention_grad_far_kernel<T, DP, kVec>;
    if (blocks > 0x7fffffff) return fail(MDL_ERR_UNSUPPORTED, "mdl_attention_backward: too many rows");
    if (int rc = allow_lds(reinterpret_cast<const void*>(kernel), lds, kFarFlats * sizeof(float))) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kAttnThreads), lds, s, a, g);
    MDL_CHECK_LAUNCH("attention_grad_far_kernel");
  }
  const size_t lds = 2 * (2 * F::kTile * Tile<T, DP>::kLd * sizeof(T) + (kBiasSpan + kAttnThreads) * sizeof(float)) + bias_lds;
  const int64_t blocks = key_unit_blocks(a, (a.k_len + kAttnRows - 1) / kAttnRows).blocks();
  const auto kernel = attention_grad_kv_kernel<T, DP, kVec>;
  if (blocks > 0x7fffffff) return fail(MDL_ERR_UNSUPPORTED, "mdl_attention_backward: too many rows");
  if (int rc = allow_lds(reinterpret_cast<const void*>(kernel), lds)) return rc;
  hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(kAttnThreads), lds, s, a, g);
  MDL_CHECK_LAUNCH("attention_grad_kv_kernel");
  return MDL_OK;
}

}  // namespace mdl

using namespace mdl;

extern "C" {

size_t mdl_attention_backward_workspace_bytes(const mdl_attention* a) { return a ? BackwardLayout(*a).bytes : 0; }

int mdl_attention_backward(const mdl_attention* a, const void* prepared, const mdl_attention_grads* grads,
                           void* workspace, size_t workspace_bytes, void* stream) {
  if (int rc = attention_check(a, "mdl_attention_backward")) return rc;
  if (!grads) return fail(MDL_ERR_INVALID, "mdl_attention_backward: null pointer");
  if (a->batch == 0 || a->q_len == 0) return MDL_OK;
  if (!grads->out || !grads->stats || !grads->grad_out || !grads->grad_q || !grads->grad_k || !grads->grad_v ||
      (mdl_attention_prepared_bytes(a) && !prepared))
    return fail(MDL_ERR_INVALID, "mdl_attention_backward: null pointer");
  if (grads->grad_table && !a->bias_table)
    return fail(MDL_ERR_INVALID, "mdl_attention_backward: grad_table without a bias_table");
  const BackwardLayout lay(*a);
  if (!workspace || workspace_bytes < lay.bytes)
    return fail(MDL_ERR_WORKSPACE, "mdl_attention_backward: workspace too small");
  const AttnCall c = attention_call(*a, prepared);
  char* ws = static_cast<char*>(workspace);
  GradCall g{};
  g.out = grads->out;
  g.stats = reinterpret_cast<const float2*>(grads->stats);
  g.grad_out = grads->grad_out;
  g.g_batch = grads->grad_batch; g.g_row = grads->grad_row; g.g_head = grads->grad_head;
  g.dq = grads->grad_q; g.dk = grads->grad_k; g.dv = grads->grad_v;
  g.delta = reinterpret_cast<float*>(ws + lay.delta);
  g.starts = a->bucket_starts;
  g.buckets = a->num_buckets;
  g.bias_partial = grads->grad_table ? reinterpret_cast<float*>(ws + lay.bias) : nullptr;
  g.bias_parts = lay.bias_parts;
  g.bias_far = lay.bias_far;
  g.far_partial = lay.far_chunks ? reinterpret_cast<float*>(ws + lay.far) : nullptr;
  g.far_chunks = lay.far_chunks;
  const int64_t e = a->dtype == MDL_BF16 ? 8 : 4;
  const bool vec = attention_vectors(*a) && reinterpret_cast<uintptr_t>(g.grad_out) % 16 == 0 &&
                   reinterpret_cast<uintptr_t>(g.out) % 16 == 0 && g.g_batch % e == 0 && g.g_row % e == 0 &&
                   g.g_head % e == 0;
  const hipStream_t s = as_stream(stream);
  if (int rc = for_attention(*a, vec, [&]<typename T, int DP, bool kVec>() {
        return launch_backward<T, DP, kVec>(c, g, s);
      }))
    return rc;
  if (grads->grad_table) {
    return sum_bias_parts(g.bias_partial, lay.bias_parts, a->num_buckets, a->q_heads, a->table_dtype,
                          grads->grad_table, s);
  }
  return MDL_OK;
}

}  // extern "C"
