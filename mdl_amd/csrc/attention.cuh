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
constexpr int kBiasSpan = 256;   // distances of a tile staged in LDS: one per thread
constexpr int kBiasEdge = kBiasSpan;  // distances of the prepared bias past either end
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
  const int2* bounds;     // [B] first and last unmasked column (Lk, -1: none)
  const float* bias;      // [Hq, distances + 2 kBiasEdge] by distance from -kBiasEdge on, divided by the scale; NULL: none
  int64_t words_row;
  int32_t batch, q_len, k_len, q_heads, kv_heads, dim, distances;
  int32_t window;  // >= k_len: none
  int32_t sinks;
  float c2;  // scale * log2(e)
  float scale;
};

__device__ __forceinline__ int clamp_to(int v, int most) { return v < 0 ? 0 : (v < most ? v : most); }

// ------------------------------------------------------------- fragments --

template <typename T>
struct Frags;

template <>
struct Frags<bf16_t> {
  static constexpr int kStep = 16;   // summed index per product
  static constexpr int kElems = 8;   // of it per lane
  static constexpr int kTile = 64;   // rows of a staged tile
  typedef bf16x8 Frag;

  static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
  }
  // Result registers 8t .. 8t + 7 as the right operand of product t.  Weights
  // and dS are rounded to bf16 here: fp32 products take 16 times as long.  With
  // the rounding of the result itself that leaves 2.2e-3 to 2.4e-3 of the norm
  // against 64 bits, where that last rounding alone makes 1.7e-3.
  static __device__ __forceinline__ Frag from_result(const f32x16& r, int t) {
    Frag f;
#pragma unroll
    for (int i = 0; i < 8; ++i) f[i] = (__bf16)r[8 * t + i];
    return f;
  }
};

template <>
struct Frags<float> {
  static constexpr int kStep = 8;
  static constexpr int kElems = 4;
  static constexpr int kTile = 32;
  typedef f32x4 Frag;

  static __device__ __forceinline__ f32x16 mma(const Frag& a, const Frag& b, f32x16 c) {
#pragma unroll
    for (int i = 0; i < 4; ++i) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[i], b[i], c, 0, 0, 0);
    return c;
  }
  static __device__ __forceinline__ Frag from_result(const f32x16& r, int t) {
    return Frag{r[4 * t], r[4 * t + 1], r[4 * t + 2], r[4 * t + 3]};
  }
};

// ------------------------------------------------------------ tiles in LDS --
//
// How rows of DP elements lie in LDS, and a lane's two ways of reading them:
// nat(tile, sub, d), the elements d * kStep + kElems * (lane / 32) .. of row
// 32 sub + lane % 32 (left operand of a product over the head dimension), and
// tr(tile, row0, dt), column 32 dt + lane % 32 of the rows row0 .. row0 +
// kStep - 1 in result order (left operand of a product over the rows).

template <typename T, int DP>
struct Tile;

// bf16: rows without padding, their 16-byte pieces swapped by the row so that
// both readings use all 64 banks: a row-wise read takes one piece of 16 rows a
// cycle (they must differ modulo the row's banks), a transposing read four
// pieces of four rows (each row another group of four).
template <int DP>
struct Tile<bf16_t, DP> {
  using F = Frags<bf16_t>;
  static constexpr int kLd = DP, kSteps = DP / F::kStep;
  int nat_at[kSteps], tr_at[DP / 32][2];

  static __device__ __forceinline__ int swap(int r) {
    if constexpr (DP == 128) return ((r & 3) << 2) | ((r >> 2) & 3);
    else if constexpr (DP == 64) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    else return (r >> 2) & 3;
  }
  static __device__ __forceinline__ int place(int row, int piece) { return row * DP + 8 * (piece ^ swap(row)); }

  __device__ __forceinline__ Tile() {
    const int l = lane_id(), half = l >> 5;
#pragma unroll
    for (int d = 0; d < kSteps; ++d) nat_at[d] = place(l & 31, 2 * d + half);
    const int row = 4 * half + ((l & 15) >> 2), piece = ((l >> 4) & 1) * 2 + ((l & 3) >> 1);
#pragma unroll
    for (int dt = 0; dt < DP / 32; ++dt)
#pragma unroll
      for (int r = 0; r < 2; ++r) tr_at[dt][r] = place(row + 8 * r, 4 * dt + piece) + 4 * (l & 1);
  }
  __device__ __forceinline__ bf16x8 nat(const bf16_t* tile, int sub, int d) const {
    return *reinterpret_cast<const bf16x8*>(tile + nat_at[d] + 32 * sub * DP);
  }
  __device__ __forceinline__ bf16x8 tr(const bf16_t* tile, int row0, int dt) const {
    typedef __attribute__((address_space(3))) bf16x4* lds4;
    const bf16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(tile + tr_at[dt][0] + row0 * DP));
    const bf16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4bf16((lds4)(tile + tr_at[dt][1] + row0 * DP));
    return __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7);
  }
};

// fp32: rows padded by 16 bytes (16 rows' pieces on different banks).
template <int DP>
struct Tile<float, DP> {
  using F = Frags<float>;
  static constexpr int kLd = DP + 4;
  int nat_at, tr_at;

  static __device__ __forceinline__ int place(int row, int piece) { return row * kLd + 4 * piece; }

  __device__ __forceinline__ Tile() {
    const int l = lane_id(), half = l >> 5;
    nat_at = place(l & 31, half);
    tr_at = 4 * half * kLd + (l & 31);
  }
  __device__ __forceinline__ f32x4 nat(const float* tile, int sub, int d) const {
    return *reinterpret_cast<const f32x4*>(tile + nat_at + 32 * sub * kLd + 8 * d);
  }
  __device__ __forceinline__ f32x4 tr(const float* tile, int row0, int dt) const {
    const float* p = tile + tr_at + row0 * kLd + 32 * dt;
    return f32x4{p[0], p[kLd], p[2 * kLd], p[3 * kLd]};
  }
};

// Nothing moves across: what is read from LDS before it is on its way while
// what follows computes (the compiler would read each operand just before
// its product and wait).  fp32 is bound by its products, which take 16 times
// as long, and has no registers to spare.
template <typename T>
__device__ __forceinline__ void reads_first() {
  if constexpr (sizeof(T) == 2) __builtin_amdgcn_sched_barrier(0);
}

// Every left operand of one 32-row tile over the head dimension, and over the rows.
template <typename T, int DP>
struct NatFrags {
  using F = Frags<T>;
  typename F::Frag f[DP / F::kStep];
  __device__ __forceinline__ NatFrags(const Tile<T, DP>& read, const T* tile, int sub) {
#pragma unroll
    for (int d = 0; d < DP / F::kStep; ++d) f[d] = read.nat(tile, sub, d);
  }
  __device__ __forceinline__ f32x16 times(const typename F::Frag (&right)[DP / F::kStep], f32x16 from) const {
#pragma unroll
    for (int d = 0; d < DP / F::kStep; ++d) from = F::mma(f[d], right[d], from);
    return from;
  }
};
template <typename T, int DP>
struct TrFrags {
  using F = Frags<T>;
  typename F::Frag f[32 / F::kStep][DP / 32];
  __device__ __forceinline__ TrFrags(const Tile<T, DP>& read, const T* tile, int sub) {
#pragma unroll
    for (int p = 0; p < 32 / F::kStep; ++p)
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) f[p][dt] = read.tr(tile, 32 * sub + F::kStep * p, dt);
  }
  // acc += the tile transposed times what a result tile holds
  __device__ __forceinline__ void times(const f32x16& result, f32x16 (&acc)[DP / 32]) const {
#pragma unroll
    for (int p = 0; p < 32 / F::kStep; ++p) {
      const typename F::Frag right = F::from_result(result, p);
#pragma unroll
      for (int dt = 0; dt < DP / 32; ++dt) acc[dt] = F::mma(f[p][dt], right, acc[dt]);
    }
  }
};

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

// v where the bit (a constant) of mask is set, else fill: a bit spread over a
// word and one bitwise selection.  Written out, since the compiler makes it an
// AND, a comparison and a selection that waits for it: four issue slots a score
// instead of two (forward over 64 x 2048 bf16 rows, 4 heads of 64, window 256,
// where half of the waves' tiles are partly masked: 94 us with those, 88 with these).
__device__ __forceinline__ float keep_bit(uint32_t mask, int bit, float v, float fill) {
  uint32_t t;
  asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(t) : "v"(mask), "i"(bit));
  return __uint_as_float((t & __float_as_uint(v)) | (~t & __float_as_uint(fill)));
}

// Weights are 2^(c2 x - c2 m) in one fused multiply-add of the rounded c2 m.
// Where a row's maximum m is past this (biases used as masks, and nothing else
// seen) that rounding would matter, up to overflow: x is then the score and its
// bias added in fp32, whatever that loses, and x - m comes first, in the
// gradients too.
constexpr float kLargeScore = 4096.f;
__device__ __forceinline__ bool is_large(const AttnCall& a, float x) { return fabsf(x) * a.c2 > kLargeScore; }

// Loads of one value per wave, through the scalar cache (read-only data).
template <typename T>
__device__ __forceinline__ T load_uniform(const T* p) {
  return *(const __attribute__((address_space(4))) T*)p;
}

// The unmasked columns of a row.
struct RowMask {
  const uint64_t* words;
  int first, last, k_len;
  __device__ __forceinline__ RowMask(const AttnCall& a, int b) : words(nullptr), first(0), last(a.k_len - 1), k_len(a.k_len) {
    if (!a.words) return;
    words = a.words + (int64_t)b * a.words_row;
    const uint64_t v = load_uniform(reinterpret_cast<const uint64_t*>(a.bounds + b));
    first = (int)(uint32_t)v;
    last = (int)(uint32_t)(v >> 32);
  }
  // columns col .. col + 31 as bits (col >= 0); a row of words has one word of zeros after its last
  __device__ __forceinline__ uint32_t bits32(int col) const {
    if (!words) return low_bits(k_len - col);
    if (col >= k_len) return 0;
    const int w = col >> 6, s = col & 63;
    uint64_t x = load_uniform(words + w) >> s;
    if (s > 32) x |= load_uniform(words + w + 1) << (64 - s);
    return (uint32_t)x;
  }
  // 64 columns (or 32) likewise
  template <int kTile>
  __device__ __forceinline__ uint64_t bits(int col) const {
    if (kTile == 32) return bits32(col);
    if (!words) return low_bits(k_len - col) | (uint64_t)low_bits(k_len - col - 32) << 32;
    if (col >= k_len) return 0;
    const int w = col >> 6, s = col & 63;
    uint64_t x = load_uniform(words + w) >> s;
    if (s) x |= load_uniform(words + w + 1) << (64 - s);
    return x;
  }
};

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

// Starts a copy of 16, or 4, bytes a lane from global memory to LDS, lane l's
// to lds + 16 l or 4 l (lds: one address per wave).  It holds no register;
// wait_fetched ends it.  Written out because the compiler, which knows the
// instruction, would wait for it before any transposing read of LDS,
// whichever buffer that reads; m0, which holds the place, stays the compiler's
// to set (a wait state lies between).
__device__ __forceinline__ uint32_t lds_address(void* lds) {
  typedef __attribute__((address_space(3))) void* lds_void;
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_void)lds);
}
__device__ __forceinline__ void copy16_to_lds(uint32_t lds, const void* from) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"{m0}"(__builtin_amdgcn_readfirstlane(lds)), "v"(from)
               : "memory");
}
__device__ __forceinline__ void copy4_to_lds(uint32_t lds, const void* from) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dword %1, off" ::"{m0}"(__builtin_amdgcn_readfirstlane(lds)), "v"(from)
               : "memory");
}

// All but the wave's last kLeft memory operations have ended: the copies
// before them are in LDS (visible to other waves after a barrier).  Through
// the builtin, so that the compiler counts it as the end of its own loads too
// and adds no wait of its own between a fetch and the products.
template <int kLeft>
__device__ __forceinline__ void wait_fetched() {
  static_assert(kLeft < 64, "six bits");
  asm volatile("" ::: "memory");
  __builtin_amdgcn_s_waitcnt(0x0f70 | (kLeft & 15) | (kLeft >> 4) << 14);
  asm volatile("" ::: "memory");
}

// One tile of kTile rows on its way from global memory to LDS.  bf16 rows in
// whole pieces go there directly (every lane a 16-byte piece, absent ones from
// a row of zeros): the registers they would pass through are free for the
// products, and several tiles can be on their way.  Other rows are held in
// registers from fetch to settle.
template <typename T, int DP, bool kVec>
struct TileStage {
  using F = Frags<T>;
  using Lds = Tile<T, DP>;
  static constexpr bool kDirect = kVec && sizeof(T) == 2;
  static constexpr int kPieces = DP / F::kElems;  // per row
  static constexpr int kPer = F::kTile * kPieces / kAttnThreads;
  static_assert(F::kTile * kPieces % kAttnThreads == 0, "whole pieces per thread");
  static constexpr int kRows = kAttnThreads / kPieces;  // from a piece of a thread to its next
  typename F::Frag r[kDirect ? 1 : kPer];
  const T* mine;    // the thread's first piece (direct) or row, in row 0 of base
  int64_t stride;
  uint32_t to;      // the wave's place in the first buffer
  bool inside, full;

  // lds: the first of the buffers
  __device__ __forceinline__ void open(T* lds, const T* base, int64_t row_stride, int D) {
    stride = row_stride;
    const int row = threadIdx.x / kPieces;
    mine = base + row * stride;
    full = D == DP;
    if constexpr (kDirect) {
      // the lane's place in LDS is given; the piece that belongs there is the same in each of its rows
      static_assert(kRows % 16 == 0, "the swap's period");
      const int d = ((threadIdx.x % kPieces) ^ Lds::swap(row)) * F::kElems;
      mine += d;
      inside = d < D;
      to = lds_address(lds + wave_id() * kWave * F::kElems);
    }
  }
  // A tile to the buffer `past` bytes after the first; first: elements from base
  // to its first row; bits: the live ones.  Scalar offsets from the thread's own
  // place, and no selection where every row is live: with an address made from
  // its row for each piece the walks were a seventh longer (2 x 8192 rows of 16
  // heads of 128: 229, 484 and 545 us, with it 193, 423 and 497).
  __device__ __forceinline__ void fetch(uint32_t past, int64_t first, uint64_t bits, int D) {
    const T* from = mine + first;
    if (kDirect && full && bits == ~0ull) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) copy16_to_lds(to + past + i * kAttnThreads * 16, from + i * kRows * stride);
      return;
    }
#pragma unroll
    for (int i = 0; i < kPer; ++i) {
      const bool live = (bits >> (threadIdx.x / kPieces + i * kRows)) & 1;
      const T* row = from + i * kRows * stride;
      if constexpr (kDirect) {
        copy16_to_lds(to + past + i * kAttnThreads * 16, live && inside ? row : zero_row<T>());
      } else {
        r[i] = {};
        if (live) r[i] = load_row<T, kVec>(row, threadIdx.x % kPieces * F::kElems, D);
      }
    }
  }
  __device__ __forceinline__ void settle(T* lds) const {
    if constexpr (!kDirect) {
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int idx = i * kAttnThreads + threadIdx.x;
        *reinterpret_cast<typename F::Frag*>(lds + Lds::place(idx / kPieces, idx % kPieces)) = r[i];
      }
    }
  }
};

// Tiles of a walk in LDS at once.  A narrow tile is worked off in less time
// than memory takes to answer, so two more are on their way; wide ones would
// not fit LDS a third time beside a second block.
template <typename T, int DP, bool kVec>
__host__ __device__ constexpr int tile_stages() { return kVec && sizeof(T) == 2 && DP <= 64 ? 3 : 2; }

// The walk over n tile pairs that all three kernels make.  fetch(i, slot)
// starts the copies of pair i (kCopies per wave, kSmall more with `small`),
// settle(slot) ends those held in registers, work(i, slot) uses them.
template <int kStages, int kCopies, bool kDirect, typename Fetch, typename Settle, typename Work>
__device__ __forceinline__ void walk_tiles(int n, bool small, Fetch&& fetch, Settle&& settle, Work&& work) {
  constexpr int kAhead = kStages - 1;
#pragma unroll
  for (int i = 0; i < kAhead; ++i)
    if (i < n) fetch(i, i);
  int slot = 0;
  for (int i = 0; i < n; ++i) {
    settle(slot);
    if constexpr (kStages == 3) {
      // pair i + 1 may still be on its way
      if (i + 1 >= n) wait_fetched<0>();
      else if (small) wait_fetched<kCopies + 1>();
      else wait_fetched<kCopies>();
    } else {
      wait_fetched<0>();
    }
    __syncthreads();  // pair i is whole, and the slot of pair i - 1 is no longer read
    int ahead = slot + kAhead;
    if (ahead >= kStages) ahead -= kStages;
    if (i + kAhead < n) fetch(i + kAhead, ahead);
    work(i, slot);
    if (++slot == kStages) slot = 0;
  }
}

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

// ------------------------------------------------------------ block order --

// Blocks are handed to the 8 XCDs in turn.  The blocks of one unit (a row and
// head, whose keys or queries they share) go to one XCD, whose L2 then reads
// them once, and the units to the XCDs in turn: rows of different lengths
// even out (a contiguous range of rows per XCD left all waiting for the XCD of
// the longest row: 255 us for the 170 of the gradients of 64 ragged rows of
// 2048, 4 heads of 64, window 256).  A few units that do not fill
// the XCDs evenly are cut into one contiguous range of blocks per XCD.
constexpr int kXcds = 8, kSpreadUnits = 32;

struct BlockOrder {
  int units, per_unit;  // blocks fit 31 bits (checked by the host)
  __host__ __device__ __forceinline__ bool in_turn() const { return units >= kSpreadUnits || units % kXcds == 0; }
  __host__ __device__ __forceinline__ int64_t blocks() const {
    return (in_turn() ? ((int64_t)units + kXcds - 1) / kXcds * kXcds : (int64_t)units) * per_unit;
  }
  // false: no work for this block
  __device__ __forceinline__ bool place(unsigned block, int* unit, int* inner) const {
    const unsigned per = per_unit;
    if (in_turn()) {
      const unsigned s = block / kXcds, u = s / per;
      *unit = (int)(u * kXcds + block % kXcds);
      *inner = (int)(s - u * per);
    } else {
      const unsigned id = (unsigned)xcd_block(block, (int64_t)units * per), u = id / per;
      *unit = (int)u;
      *inner = (int)(id - u * per);
    }
    return *unit < units;
  }
};

__host__ __device__ __forceinline__ BlockOrder query_blocks(const AttnCall& a) {
  return {a.batch * a.q_heads, (a.q_len + kAttnRows - 1) / kAttnRows};
}
__host__ __device__ __forceinline__ BlockOrder key_unit_blocks(const AttnCall& a, int per_unit) {
  return {a.batch * a.kv_heads, per_unit};
}

// -------------------------------------------------- blocks of query rows --

// What a block of 128 query rows of one head walks: the key tiles with a
// visible column, those of the first tokens and then those of the window.
struct KeyWalk {
  int sink_end, tiles, sink_tiles, sink_tile, window_tile;

  // c_lo .. c_hi: the block's columns
  __device__ __forceinline__ KeyWalk(const AttnCall& a, const RowMask& mask, int tile, int c_lo, int c_hi) {
    sink_end = mask.first + a.sinks < a.k_len ? mask.first + a.sinks : a.k_len;
    tiles = sink_tiles = sink_tile = window_tile = 0;
    if (c_hi < mask.first || c_lo > mask.last) return;
    int lo = c_lo - a.window + 1;
    if (lo < mask.first) lo = mask.first;
    const int hi = c_hi < mask.last ? c_hi : mask.last;
    window_tile = lo / tile;
    if (lo <= hi) tiles = hi / tile - window_tile + 1;
    if (a.sinks > 0) {
      sink_tile = mask.first / tile;
      int last = (sink_end - 1) / tile;
      if (last >= window_tile) last = window_tile - 1;
      if (last > hi / tile) last = hi / tile;
      if (last >= sink_tile) sink_tiles = last - sink_tile + 1;
    }
    tiles += sink_tiles;
  }
  __device__ __forceinline__ int tile_at(int i) const {
    return i < sink_tiles ? sink_tile + i : window_tile + (i - sink_tiles);
  }
};

// Where the bias of a tile of distances from `lowest` on lies in a head's
// prepared row, kBiasSpan of them (tiles wholly in the last bucket read none).
__device__ __forceinline__ int bias_at(const AttnCall& a, int lowest) {
  const int z = lowest + kBiasEdge, most = a.distances + 2 * kBiasEdge - kBiasSpan;
  return z < most ? z : most;
}
__device__ __forceinline__ const float* head_bias(const AttnCall& a, int head) {
  return a.bias + (int64_t)head * (a.distances + 2 * kBiasEdge);
}

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
// Lets a kernel have `dynamic` bytes of LDS beside its own `fixed` ones.
int allow_lds(const void* kernel, size_t dynamic, size_t fixed = 0);

// Calls f.template operator()<T, DP, kVec>() with the element type, the head
// dimension rounded up to 32, 64 or 128 (the columns past it are zeros in LDS
// and registers, and multiplied all the same: 80 pays 1.6 times its products,
// 96 a third more) and whether rows are read in 16-byte pieces.
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
