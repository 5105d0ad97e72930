// What the attention kernels share: the call as the kernels see it, the
// matrix fragments of both element types, tile staging and the visible keys
// of a query.
//
// Shapes.  q [B, Lq, Hq, D], k and v [B, Lk, Hkv, D], any strides over batch,
// row and head.  Query row r stands at column c = r + Lk - Lq.  Column j is
// visible to column c when both are unmasked, j <= c, and c - j < window or
// j < first + sinks (first: the row's first unmasked column).
//
// Units.  Scores are kept divided by the scale: x = q.k + bias / scale, so a
// bias is the matrix product's starting value and costs no instruction; a
// weight is exp2(c2 x - c2 m) with c2 = scale * log2(e).
//
// Fragments.  Every product is a 32x32 tile of the matrix unit whose result
// leaves lane l holding column l % 32 and rows 8 (i / 4) + 4 (l / 32) + i % 4.
// Products are arranged so that this result is, as it stands, the right
// operand of the next product: the order in which the summed index is fed is
// free as long as both operands agree, so the left operand is read from LDS
// in the order the result has.  No value crosses lanes between products.
#pragma once

#include "common.cuh"

namespace mdl {

constexpr int kAttnThreads = 256;
constexpr int kAttnRows = 128;  // rows (queries, or keys in the key gradient) of a block: 32 per wave
constexpr int kMaxDistances = 2049;  // bias distances a call may tell apart

// x of a bias of its type's lowest value: finite, below every real score, and
// a power of two, so that c2 x - round(c2 m) is exact for x = m.
constexpr float kLowScore = -1.2676506002282294e30f;   // -2^100
constexpr float kNoScore = -1.298074214633707e33f;     // -2^110: a row's maximum before its first key

typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x4 __attribute__((ext_vector_type(4)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

struct AttnCall {
  const void *q, *k, *v;
  int64_t q_batch, q_row, q_head, k_batch, k_row, k_head, v_batch, v_row, v_head;  // element strides
  const uint64_t* words;  // unmasked columns, 64 a word, [B, words_row]; NULL: all
  const int32_t* first;   // [B] first unmasked column (Lk: none)
  const float* bias;      // [Hq, distances], divided by the scale; NULL: none
  int64_t words_row;
  int32_t batch, q_len, k_len, q_heads, kv_heads, dim, distances;
  int32_t window;  // >= k_len: none
  int32_t sinks;
  float c2;  // scale * log2(e)
  float scale;
};

// ------------------------------------------------------------- fragments --

template <typename T>
struct Frags;

template <>
struct Frags<bf16_t> {
  static constexpr int kStep = 16;   // summed index per product
  static constexpr int kElems = 8;   // of it per lane
  static constexpr int kTile = 64;   // rows of a staged tile
  // Row padding in LDS, such that eight rows read in 16-byte pieces and four
  // rows of 32 bytes read transposed both fall on different banks.
  static constexpr int pad(int dp) { return dp == 64 ? 8 : 16; }
  typedef bf16x8 Frag;

  static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // result registers 8t .. 8t + 7 as the right operand of product t
  static __device__ __forceinline__ Frag from_result(const f32x16& r, int t) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (__bf16)r[8 * t + i];
    return f;
  }
  static __device__ __forceinline__ int t_offset(int ld) {
    const int l = lane_id();
    return (4 * (l >> 5) + ((l & 15) >> 2)) * ld + ((l >> 4) & 1) * 16 + (l & 3) * 4;
  }
  // rows (in result order) of one column per lane: two transposing reads of
  // four rows each
  static __device__ __forceinline__ Frag load_t(const bf16_t* p, int ld) {
    typedef __attribute__((address_space(3))) bf16x4* lds4;
    const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)p);
    const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(p + 8 * ld));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

template <>
struct Frags<float> {
  static constexpr int kStep = 8;
  static constexpr int kElems = 4;
  static constexpr int kTile = 32;
  static constexpr int pad(int) { return 4; }
  typedef f32x4 Frag;

  static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag from_result(const f32x16& r, int t) {
    return Frag{r[4 * t], r[4 * t + 1], r[4 * t + 2], r[4 * t + 3]};
  }
  static __device__ __forceinline__ int t_offset(int ld) {
    const int l = lane_id();
    return 4 * (l >> 5) * ld + (l & 31);
  }
  static __device__ __forceinline__ Frag load_t(const float* p, int ld) {
    return Frag{p[0], p[ld], p[2 * ld], p[3 * ld]};
  }
};

// A lane's elements of a row, read where they lie (left operand: row of the
// tile; right operand: the lane's own row).
template <typename T>
__device__ __forceinline__ typename Frags<T>::Frag load_frag(const T* p) {
  return *reinterpret_cast<const typename Frags<T>::Frag*>(p);
}

// Rows of a result tile held by a lane: row i of the lane is result_row(i).
__device__ __forceinline__ int result_row(int i) { return 8 * (i >> 2) + 4 * (lane_id() >> 5) + (i & 3); }

// ---------------------------------------------------------------- numerics --

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The maximum of v over this lane and the lane 32 away.
__device__ __forceinline__ float max_halves(float v) {
  const auto p = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
  return fmaxf(__uint_as_float(p[0]), __uint_as_float(p[1]));
}

// Bits [0, n) of a 32-bit word, n any.
__device__ __forceinline__ uint32_t low_bits(int n) {
  return n <= 0 ? 0u : (n >= 32 ? ~0u : (1u << n) - 1u);
}

// v where the bit of mask is set, else fill.
__device__ __forceinline__ float keep_bit(uint32_t mask, int bit, float v, float fill) {
  const uint32_t t = (uint32_t)((int32_t)(mask << (31 - bit)) >> 31);
  return __uint_as_float((t & __float_as_uint(v)) | (~t & __float_as_uint(fill)));
}

// Unmasked columns col .. col + 31 of a row as bits (col >= 0).  A row of
// words has one word of zeros after its last.
__device__ __forceinline__ uint32_t columns32(const AttnCall& a, const uint64_t* words, int col) {
  if (!words) return low_bits(a.k_len - col);
  if (col >= a.k_len) return 0;
  const int w = col >> 6, s = col & 63;
  uint64_t x = words[w] >> s;
  if (s > 32) x |= words[w + 1] << (64 - s);
  return (uint32_t)x;
}

// ----------------------------------------------------------------- staging --

// E elements of a row from column d, zeros from column D on.
template <typename T, bool kVec>
__device__ __forceinline__ typename Frags<T>::Frag load_row(const T* row, int d, int D) {
  constexpr int E = Frags<T>::kElems;
  typename Frags<T>::Frag f = {};
  if constexpr (kVec) {
    if (d < D) f = *(const gptr<typename Frags<T>::Frag>)(row + d);
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i)
      if (d + i < D) {
        if constexpr (sizeof(T) == 2) f[i] = *(const gptr<__bf16>)(row + d + i);
        else f[i] = *to_global(row + d + i);
      }
  }
  return f;
}

// The lane's own row as right operand of the products over the head
// dimension: zeros when absent.
template <typename T, int DP, bool kVec>
__device__ __forceinline__ void load_own_row(const T* row, bool live, int D,
                                             typename Frags<T>::Frag (&f)[DP / Frags<T>::kStep]) {
  using F = Frags<T>;
  const int h = lane_id() >> 5;
#pragma unroll
  for (int s = 0; s < DP / F::kStep; ++s) {
    f[s] = {};
    if (live) f[s] = load_row<T, kVec>(row, s * F::kStep + h * F::kElems, D);
  }
}

// One tile of kTile rows between global memory and LDS: every thread holds
// its 16-byte pieces in registers while the block computes on the tile before.
template <typename T, int DP, bool kVec>
struct TileStage {
  using F = Frags<T>;
  static constexpr int kLd = DP + F::pad(DP);
  static constexpr int kPieces = DP / F::kElems;  // per row
  static constexpr int kPer = F::kTile * kPieces / kAttnThreads;
  static_assert(F::kTile * kPieces % kAttnThreads == 0, "whole pieces per thread");
  typename F::Frag r[kPer];

  // rows row0 .. of base; bits: the live ones (two words of 32)
  __device__ __forceinline__ void load(const T* base, int64_t stride, int row0, uint64_t bits, int D) {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int idx = i * kAttnThreads + threadIdx.x;
      const int row = idx / kPieces, d = idx % kPieces * F::kElems;
      r[i] = {};
      if ((bits >> row) & 1) r[i] = load_row<T, kVec>(base + (int64_t)(row0 + row) * stride, d, D);
    }
  }
  __device__ __forceinline__ void store(T* lds) const {
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const int idx = i * kAttnThreads + threadIdx.x;
      *reinterpret_cast<typename F::Frag*>(lds + idx / kPieces * kLd + idx % kPieces * F::kElems) = r[i];
    }
  }
};

// A result tile's rows are head-dimension elements (transposed outputs): the
// lane's elements 32 dt + result_row(i) of its own row, times scale.
template <typename T, int DP>
__device__ __forceinline__ void store_result_row(T* row, const f32x16 (&acc)[DP / 32], float scale, int D) {
#pragma unroll
  for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int d = 32 * dt + result_row(4 * g);
      float v[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) v[i] = acc[dt][4 * g + i] * scale;
      if ((D & 3) == 0) {
        if (d < D) {
          if constexpr (sizeof(T) == 2) {
            const bf16x4 o = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
            *(gptr<bf16x4>)(row + d) = o;
          } else {
            *(gptr<f32x4>)(row + d) = f32x4{v[0], v[1], v[2], v[3]};
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (d + i < D) {
            if constexpr (sizeof(T) == 2) *(gptr<__bf16>)(row + d + i) = (__bf16)v[i];
            else *to_global(row + d + i) = v[i];
          }
      }
    }
}

// -------------------------------------------------- blocks of query rows --

// What a block of 128 query rows of one head walks: the key tiles with a
// visible column, those of the first tokens and then those of the window.
struct KeyWalk {
  const uint64_t* words;
  int tile, first, sink_end, window_tile, last_tile, last_sink_tile;

  // tile: columns per tile.  c_lo .. c_hi: the block's columns.
  __device__ __forceinline__ KeyWalk(const AttnCall& a, int b, int tile_, int c_lo, int c_hi) : tile(tile_) {
    words = a.words ? a.words + (int64_t)b * a.words_row : nullptr;
    first = a.words ? a.first[b] : 0;
    sink_end = first + a.sinks < a.k_len ? first + a.sinks : a.k_len;
    int lo = c_lo - a.window + 1;
    if (lo < first) lo = first;
    window_tile = lo / tile;
    last_tile = c_hi / tile;
    last_sink_tile = a.sinks > 0 ? (sink_end - 1) / tile : -1;
    if (last_sink_tile >= window_tile) last_sink_tile = window_tile - 1;
    if (last_sink_tile > last_tile) last_sink_tile = last_tile;
  }
  __device__ __forceinline__ uint64_t bits(const AttnCall& a, int t) const {
    const uint32_t lo = columns32(a, words, t * tile);
    if (tile == 32) return lo;
    return lo | (uint64_t)columns32(a, words, t * tile + 32) << 32;
  }
  // the first tile from t on with an unmasked column (last_tile + 1: none)
  __device__ __forceinline__ int seek(const AttnCall& a, int t, uint64_t* b) const {
    for (;; ++t) {
      if (t > last_sink_tile && t < window_tile) t = window_tile;
      if (t > last_tile) return last_tile + 1;
      *b = bits(a, t);
      if (*b) return t;
    }
  }
  __device__ __forceinline__ int begin(const AttnCall& a, uint64_t* b) const {
    return seek(a, last_sink_tile >= 0 ? first / tile : window_tile, b);
  }
};

// Visible columns col .. col + 31 of the query at column c as bits; live: the
// columns' own bits.
__device__ __forceinline__ uint32_t visible32(int c, int col, int window, int sink_end, uint32_t live) {
  const uint32_t past = low_bits(c - col + 1);
  const uint32_t near = ~low_bits(c - window + 1 - col) | low_bits(sink_end - col);
  return past & near & live;
}

// ------------------------------------------------------------- host side --

int attention_check(const mdl_attention* a, const char* what);
AttnCall attention_call(const mdl_attention& a, const void* prepared);
bool attention_vectors(const mdl_attention& a);  // 16-byte rows throughout
int allow_lds(const void* kernel, size_t bytes);

// Calls f.template operator()<T, DP, kVec>() with the element type, the head
// dimension rounded up to 32, 64 or 128 (the columns past it are zeros in LDS
// and registers) and whether rows are read in 16-byte pieces.
template <typename F>
int for_attention(const mdl_attention& a, bool vec, F&& f) {
  auto dims = [&]<typename T, bool kVec>() -> int {
    if (a.head_dim <= 32) return f.template operator()<T, 32, kVec>();
    if (a.head_dim <= 64) return f.template operator()<T, 64, kVec>();
    return f.template operator()<T, 128, kVec>();
  };
  if (a.dtype == MDL_BF16) return vec ? dims.template operator()<bf16_t, true>() : dims.template operator()<bf16_t, false>();
  return vec ? dims.template operator()<float, true>() : dims.template operator()<float, false>();
}

}  // namespace mdl
