// A key / value cache in 4 or 8 bits: its rows written (quantised), read back, and attended to by the newest positions.
//
// Format. Along the head dimension a row is cut into blocks of 32 elements. A block keeps a scale byte s and 32 elements of
// 4 bits (E2M1: 0, 0.5, 1, 1.5, 2, 3, 4, 6) or 8 bits (E4M3, up to 448); it stands for element * 2^(s - 127). The scale is
// the smallest power of two under which the block's largest magnitude is at most 7 (464), the upper end of what rounds to
// the largest element: nothing is further from its held value than half a step, and since a division by a power of two is
// exact the codes do not depend on the precision they are computed in. A block that holds an inf or NaN gets scale byte
// 255 and reads back as NaN throughout. Elements round to nearest, ties to even (the conversion instructions' own rule).
//
// Layout. codes [batch, kv_heads, capacity, head_dim * bits / 8], scales [batch, kv_heads, capacity, head_dim / 32]: the rows
// of one head follow each other, so that a tile of 32 positions is one contiguous piece of memory for the kernel that is
// bound by reading it (the decoding step).
#include "gemm_ring.hip.h"
#include <algorithm>

namespace nmtg {
namespace {

constexpr int KV_BLOCK = 32;      // elements per scale
constexpr int KV_TILE = 32;       // positions per step of a wavefront in the attention kernel
constexpr int KV_ROWS = 16;       // query rows per block: the columns of the 16 x 16 x 32 products
constexpr float KV_FLOOR = -5e29f;  // a running maximum before the first visible position: finite, far above the -inf of hidden ones
constexpr float KV_LAZY = 8.f;
constexpr float KV_LOG2E = 1.4426950408889634f;

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef short s16x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x2_t __attribute__((ext_vector_type(2)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

__device__ __forceinline__ int64_t least(int64_t a, int64_t b) { return a < b ? a : b; }
__device__ __forceinline__ int64_t most(int64_t a, int64_t b) { return a > b ? a : b; }

// 2^(byte - 127) as the conversion instructions take it: only the exponent field counts, 0 is 2^-127 and 255 gives NaN
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// Four (4 bits) or two (8 bits) times two elements of a word: pair P as two 16-bit elements of T in one register
template <typename T, int BITS, int P>
__device__ __forceinline__ uint32_t held_pair(uint32_t word, float scale) {
  if constexpr (BITS == 4) {
    if constexpr (elem<T>::dtype == NMTG_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(word, scale, P));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp4(word, scale, P));
  } else {
    if constexpr (elem<T>::dtype == NMTG_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, scale, P != 0));
    else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, scale, P != 0));
  }
}
// all pairs of one word
template <typename T, int BITS>
__device__ __forceinline__ void held_word(uint32_t word, float scale, uint32_t* out) {
  out[0] = held_pair<T, BITS, 0>(word, scale);
  out[1] = held_pair<T, BITS, 1>(word, scale);
  if constexpr (BITS == 4) {
    out[2] = held_pair<T, BITS, 2>(word, scale);
    out[3] = held_pair<T, BITS, 3>(word, scale);
  }
}

// A block whose largest magnitude rounds up can be held as a power of two beyond the type's largest number (fp16: from 57344 on in 4 bits, 63488
// in 8; a cache written in bf16 holds more than fp16 has anyway), which the conversion gives as inf. Scale bytes below the limit cannot.
template <typename T, int BITS> constexpr uint32_t beyond_byte() {
  return 127 + (elem<T>::dtype == NMTG_BF16 ? 128 : 16) - (BITS == 4 ? 2 : 8);      // 4 and 256 are the largest powers of two among the elements
}
// inf in a pair becomes the type's largest number, the nearest to what is held
template <typename T>
__device__ __forceinline__ uint32_t finite_pair(uint32_t w) {
  constexpr uint32_t INF = elem<T>::dtype == NMTG_BF16 ? 0x7f80u : 0x7c00u;
  if ((w & 0x7fffu) == INF) w -= 1;
  if ((w & 0x7fff0000u) == INF << 16) w -= 0x10000u;
  return w;
}

// ------------------------------------------------------------------------------------------------------- write and read
// A block takes a tile of 16-bit rows: 2^tshift neighbouring positions of as many (sequence, head) pairs as 128 (head_dim 64) or
// 64 rows make. In the 16-bit tensors neighbouring pairs lie side by side, in the cache neighbouring positions do: with 8 or 16
// positions a tile is read and written in pieces of at least 256 bytes on both sides. (One row after the other in the order of the
// 16-bit tensors left the cache side with pieces of 32 or 64 bytes, half of a line, and cost 64-bit divisions: 32768 positions of 4 x 8
// heads of 128 in 4 bits read back in 220 us, now 113: 6.0 TB/s.) Rows, codes and results pass by
// the L2, which they would only fill: writing 8192 positions of 8 x 8 heads 86 -> 68 us, 5.0 TB/s.
struct KvRows {
  const void *k, *v;              // write: 16-bit rows [count, batch, kv_heads, head_dim] by three strides
  void *k_out, *v_out;            // read: dense [count, batch, kv_heads, head_dim]
  uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  const int32_t* starts;          // first cache row of every sequence, or null: `start` for all
  int64_t k_st, k_sb, k_sh, v_st, v_sb, v_sh;
  int64_t start, capacity;
  int count, batch, kv_heads, tshift, pair_tiles;
};

template <int D> struct RowTile {
  static constexpr int CH = D / 8, STEP = 256 / CH, PASSES = 4, ROWS = STEP * PASSES;   // rows per pass of the block, rows per tile
};
// Row `row` of the block's tile. held: its cache row, or -1 where `starts` puts it outside.
struct KvRow { int t, b, h; int64_t held; bool live; };
__device__ __forceinline__ KvRow kv_row(const KvRows& a, uint32_t tile, int rows, int row) {
  KvRow r;
  const int t_tile = static_cast<int>(tile / static_cast<uint32_t>(a.pair_tiles)), p_tile = static_cast<int>(tile % static_cast<uint32_t>(a.pair_tiles));
  r.t = (t_tile << a.tshift) + (row & ((1 << a.tshift) - 1));
  const uint32_t pair = static_cast<uint32_t>(p_tile) * static_cast<uint32_t>(rows >> a.tshift) + static_cast<uint32_t>(row >> a.tshift);
  r.live = r.t < a.count && pair < static_cast<uint32_t>(a.batch) * static_cast<uint32_t>(a.kv_heads);
  r.b = static_cast<int>(pair / static_cast<uint32_t>(a.kv_heads));
  r.h = static_cast<int>(pair) - r.b * a.kv_heads;
  const int64_t at = (a.starts != nullptr && r.live ? a.starts[r.b] : a.start) + r.t;
  r.held = at >= 0 && at < a.capacity ? static_cast<int64_t>(pair) * a.capacity + at : -1;
  return r;
}

// One lane per 8 elements, four neighbouring lanes per block of 32; blockIdx.y: keys or values.
template <typename T, int D, int BITS>
__global__ __launch_bounds__(256) void kv_write_kernel(KvRows a) {
  using R = RowTile<D>;
  const bool keys = blockIdx.y == 0;
  const T* src = static_cast<const T*>(keys ? a.k : a.v);
  const int64_t st = keys ? a.k_st : a.v_st, sb = keys ? a.k_sb : a.v_sb, sh = keys ? a.k_sh : a.v_sh;
  const int c = static_cast<int>(threadIdx.x) % R::CH;
  int64_t held[R::PASSES];
  uint32_t w[R::PASSES][4];
#pragma unroll
  for (int i = 0; i < R::PASSES; ++i) {            // all loads on their way before the first is looked at
    const KvRow r = kv_row(a, blockIdx.x, R::ROWS, i * R::STEP + static_cast<int>(threadIdx.x) / R::CH);
    held[i] = r.live ? r.held : -1;
    u32x4_t raw = {0, 0, 0, 0};
    if (held[i] >= 0) raw = __builtin_nontemporal_load(reinterpret_cast<const u32x4_t*>(src + r.t * st + r.b * sb + r.h * sh + 8 * c));
#pragma unroll
    for (int e = 0; e < 4; ++e) w[i][e] = raw[e];
  }
#pragma unroll
  for (int i = 0; i < R::PASSES; ++i) {
    // magnitudes of 16-bit floats compare as integers
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 4; ++e) top = max(top, max(w[i][e] & 0x7fffu, (w[i][e] >> 16) & 0x7fffu));
    top = max(top, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0xB1, 0xf, 0xf, true)));
    top = max(top, static_cast<uint32_t>(__builtin_amdgcn_update_dpp(0, static_cast<int>(top), 0x4E, 0xf, 0xf, true)));
    if (held[i] < 0) continue;                     // the four lanes of a block share a row
    const bool finite = top < (elem<T>::dtype == NMTG_BF16 ? 0x7f80u : 0x7c00u);
    T largest;
    largest.bits = static_cast<uint16_t>(top);
    const uint32_t amax = __float_as_uint(elem<T>::to_float(largest));
    constexpr int EMAX = BITS == 4 ? 2 : 8;
    constexpr uint32_t UP = BITS == 4 ? 0x600000u : 0x680000u;      // fraction of 1.75 (7 / 4) and of 1.8125 (464 / 256)
    const int byte = finite ? max(1, static_cast<int>(amax >> 23) - EMAX + ((amax & 0x7fffffu) > UP ? 1 : 0)) : 255;
    const float scale = scale_of(static_cast<uint32_t>(finite ? byte : 127));
    uint8_t* codes = (keys ? a.k_codes : a.v_codes) + held[i] * (D * BITS / 8) + c * BITS;
    if constexpr (BITS == 4) {
      uint32_t out = 0;
      if constexpr (elem<T>::dtype == NMTG_BF16) {
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(out, __builtin_bit_cast(bf16x2_t, w[i][0]), scale, 0);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(out, __builtin_bit_cast(bf16x2_t, w[i][1]), scale, 1);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(out, __builtin_bit_cast(bf16x2_t, w[i][2]), scale, 2);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_bf16(out, __builtin_bit_cast(bf16x2_t, w[i][3]), scale, 3);
      } else {
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(out, __builtin_bit_cast(f16x2_t, w[i][0]), scale, 0);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(out, __builtin_bit_cast(f16x2_t, w[i][1]), scale, 1);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(out, __builtin_bit_cast(f16x2_t, w[i][2]), scale, 2);
        out = __builtin_amdgcn_cvt_scalef32_pk_fp4_f16(out, __builtin_bit_cast(f16x2_t, w[i][3]), scale, 3);
      }
      __builtin_nontemporal_store(finite ? out : 0u, reinterpret_cast<uint32_t*>(codes));
    } else {
      s16x2_t out[2] = {{0, 0}, {0, 0}};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        if constexpr (elem<T>::dtype == NMTG_BF16) {
          out[e] = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(out[e], __builtin_bit_cast(bf16x2_t, w[i][2 * e]), scale, false);
          out[e] = __builtin_amdgcn_cvt_scalef32_pk_fp8_bf16(out[e], __builtin_bit_cast(bf16x2_t, w[i][2 * e + 1]), scale, true);
        } else {
          out[e] = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(out[e], __builtin_bit_cast(f16x2_t, w[i][2 * e]), scale, false);
          out[e] = __builtin_amdgcn_cvt_scalef32_pk_fp8_f16(out[e], __builtin_bit_cast(f16x2_t, w[i][2 * e + 1]), scale, true);
        }
      }
      const u32x2_t two = {finite ? __builtin_bit_cast(uint32_t, out[0]) : 0u, finite ? __builtin_bit_cast(uint32_t, out[1]) : 0u};
      __builtin_nontemporal_store(two, reinterpret_cast<u32x2_t*>(codes));
    }
    if ((c & 3) == 0) (keys ? a.k_scales : a.v_scales)[held[i] * (D / KV_BLOCK) + c / 4] = static_cast<uint8_t>(byte);
  }
}

template <typename T, int D, int BITS>
__global__ __launch_bounds__(256) void kv_read_kernel(KvRows a) {
  using R = RowTile<D>;
  const bool keys = blockIdx.y == 0;
  const uint8_t *kc = keys ? a.k_codes : a.v_codes, *ksc = keys ? a.k_scales : a.v_scales;
  const int c = static_cast<int>(threadIdx.x) % R::CH;
  int64_t to[R::PASSES];
  uint2 raw[R::PASSES];
  uint32_t byte[R::PASSES];
#pragma unroll
  for (int i = 0; i < R::PASSES; ++i) {
    const KvRow r = kv_row(a, blockIdx.x, R::ROWS, i * R::STEP + static_cast<int>(threadIdx.x) / R::CH);
    to[i] = r.live ? (static_cast<int64_t>(r.t) * a.batch + r.b) * a.kv_heads + r.h : -1;
    raw[i] = make_uint2(0, 0);                     // positions outside the cache: zeros
    byte[i] = 127;
    if (r.live && r.held >= 0) {
      const uint8_t* codes = kc + r.held * (D * BITS / 8) + c * BITS;
      if constexpr (BITS == 4) {
        raw[i].x = __builtin_nontemporal_load(reinterpret_cast<const uint32_t*>(codes));
      } else {
        const u32x2_t two = __builtin_nontemporal_load(reinterpret_cast<const u32x2_t*>(codes));
        raw[i] = make_uint2(two[0], two[1]);
      }
      byte[i] = ksc[r.held * (D / KV_BLOCK) + c / 4];
    }
  }
#pragma unroll
  for (int i = 0; i < R::PASSES; ++i) {
    if (to[i] < 0) continue;
    uint32_t w[4];
    held_word<T, BITS>(raw[i].x, scale_of(byte[i]), w);
    if constexpr (BITS == 8) held_word<T, BITS>(raw[i].y, scale_of(byte[i]), w + 2);
    const u32x4_t row = {w[0], w[1], w[2], w[3]};
    __builtin_nontemporal_store(row, static_cast<u32x4_t*>(keys ? a.k_out : a.v_out) + (to[i] * R::CH + c));
  }
}

// ------------------------------------------------------------------------------------------------------------ attention
// One block per (split, key / value head and group of 16 query rows, sequence). The 16 rows are the newest positions of the
// query heads that share the key / value head: row r is position r / g, head r % g of the group. A wavefront takes tiles of
// 32 positions, each read once from memory into registers one tile ahead:
//   S^T = K Q^T (16 x 16 x 32 products, twice 16 positions): lane (r = lane % 16, g = lane / 16) holds the codes of
//   quarter g of position r, head_dim / 4 consecutive elements as they lie in memory; the products sum over the head
//   dimension in whatever order both operands share, so the queries are read in the same order and no code is moved.
//   The result has one query row per lane column and positions 4 g .. 4 g + 3 (+ 16) in a lane's registers, which is the
//   operand layout of the second product, again with the tile's positions in an order both operands share:
//   O^T = V^T P^T: lane (c, g) holds elements [c D / 16, (c + 1) D / 16) of those eight positions; converted to pairs of
//   neighbouring elements and re-paired by position (one byte permutation per register) they are the operands of D / 16
//   products.
// The running maximum follows lazily (it moves when a score exceeds it by 2^8), the sums stay per lane until the end.
// Memory bounds it, and latency where the cache is short: 856 MB of 32 sequences in 144 us (5.9 TB/s), 5 sequences of 61 positions in 4.4.
struct KvAttn {
  const void* q;
  const uint8_t *k_codes, *k_scales, *v_codes, *v_scales;
  const int32_t* lengths;
  void* out;
  float *part, *part_ml;          // splits > 1: [splits][batch, kv_heads, rows][D] and [..][2] (maximum, sum)
  int64_t q_st, q_sb, q_sh, o_st, o_sb, o_sh;
  int64_t capacity;
  int tq, heads, kv_heads, group, rows, splits;   // group: query heads per key / value head, rows: tq * group
  int window, sinks;              // window beyond every position: none
  float scale_log2;
};

template <typename T> __device__ __forceinline__ f32x4_t mfma_16x16x32(const uint4& a, const uint4& b, f32x4_t c);
template <> __device__ __forceinline__ f32x4_t mfma_16x16x32<bf16_t>(const uint4& a, const uint4& b, f32x4_t c) {
  typedef __bf16 v8 __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}
template <> __device__ __forceinline__ f32x4_t mfma_16x16x32<f16_t>(const uint4& a, const uint4& b, f32x4_t c) {
  typedef _Float16 v8 __attribute__((ext_vector_type(8)));
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(v8, a), __builtin_bit_cast(v8, b), c, 0, 0, 0);
}

template <typename T> struct pair16;
template <> struct pair16<f16_t> { typedef f16x2_t type; };
template <> struct pair16<bf16_t> { typedef bf16x2_t type; };
template <typename T>
__device__ __forceinline__ uint32_t round_pair(float lo, float hi) {
  const f32x2_t v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, typename pair16<T>::type));
}

// The codes and scales of one tile in a lane's registers. STREAM: the codes pass by the L2.
template <int D, int BITS, bool STREAM>
struct KvTile {
  static constexpr int RB = D * BITS / 8, SB = D / KV_BLOCK;        // bytes of a row's codes and scales
  static constexpr int KW = RB / 16;                                // words of a quarter row
  static constexpr int VB = RB / 16, VW = VB >= 4 ? VB / 4 : 1;     // bytes of a sixteenth of a row, words to hold them
  uint32_t k[2][KW], ks[2], v[8][VW], vs[8];
  // the tile's rows start at row `position` of the head's rows; `rows` of its 32 may be read, the others repeat the last of them
  __device__ __forceinline__ void load(const uint8_t* kc, const uint8_t* ksc, const uint8_t* vc, const uint8_t* vsc, int64_t position,
                                       int64_t rows, int lane) {
    const uint8_t *kp = kc + position * RB, *ksp = ksc + position * SB, *vp = vc + position * RB, *vsp = vsc + position * SB;
    const int r = lane & 15, g = lane >> 4;
    if (rows >= KV_TILE) {
#pragma unroll
      for (int m = 0; m < 2; ++m) load_k(m, kp, ksp, static_cast<uint32_t>(16 * m + r), g);
#pragma unroll
      for (int e = 0; e < 8; ++e) load_v(e, vp, static_cast<uint32_t>(16 * (e / 4) + 4 * g + (e & 3)), r);
      // the scales of four neighbouring positions in one load, the lane's block shifted down
#pragma unroll
      for (int m = 0; m < 2; ++m) {
        const uint8_t* p = vsp + static_cast<uint32_t>((16 * m + 4 * g) * SB);
        if constexpr (SB == 4) {
          typedef uint32_t words __attribute__((ext_vector_type(4), aligned(4)));
          const words w = *reinterpret_cast<const words*>(p);
#pragma unroll
          for (int e = 0; e < 4; ++e) vs[4 * m + e] = w[e];
        } else {
          typedef uint32_t words __attribute__((ext_vector_type(2), aligned(2)));
          const words w = *reinterpret_cast<const words*>(p);
#pragma unroll
          for (int e = 0; e < 4; ++e) vs[4 * m + e] = w[e / 2] >> (16 * (e & 1));   // (its lower half counts)
        }
      }
    } else {
      const uint32_t last = static_cast<uint32_t>(rows - 1);
#pragma unroll
      for (int m = 0; m < 2; ++m) load_k(m, kp, ksp, min(static_cast<uint32_t>(16 * m + r), last), g);
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const uint32_t row = min(static_cast<uint32_t>(16 * (e / 4) + 4 * g + (e & 3)), last);
        load_v(e, vp, row, r);
        typedef uint32_t word __attribute__((aligned(1)));
        typedef uint16_t half __attribute__((aligned(1)));
        if constexpr (SB == 4) vs[e] = *reinterpret_cast<const word*>(vsp + row * SB);
        else vs[e] = *reinterpret_cast<const half*>(vsp + row * SB);
      }
    }
  }
  __device__ __forceinline__ void load_k(int m, const uint8_t* kp, const uint8_t* ksp, uint32_t row, int g) {
    constexpr int N = KW >= 4 ? 4 : KW;
#pragma unroll
    for (int i = 0; i < KW; i += N) load_words<N>(k[m] + i, kp + (row * RB + g * (RB / 4)) + 4 * i);
    ks[m] = ksp[row * SB + static_cast<uint32_t>(g) * SB / 4];
  }
  __device__ __forceinline__ void load_v(int e, const uint8_t* vp, uint32_t row, int r) {
    const uint8_t* p = vp + (row * RB + r * VB);
    if constexpr (VB == 2) v[e][0] = *reinterpret_cast<const uint16_t*>(p);
    else load_words<VW>(v[e], p);
  }
  template <int N>
  static __device__ __forceinline__ void load_words(uint32_t* to, const uint8_t* p) {
    typedef uint32_t words __attribute__((ext_vector_type(N)));
    words w;
    if constexpr (STREAM) w = __builtin_nontemporal_load(reinterpret_cast<const words*>(p));
    else w = *reinterpret_cast<const words*>(p);
    __builtin_memcpy(to, &w, 4 * N);
  }
  // scale of the lane's elements of position e, byte r SB / 16 of its scales, rotated into the exponent's place. What else
  // the word holds lands in sign and fraction, which the conversion instructions do not look at.
  __device__ __forceinline__ float v_scale(int e, int r) const {
    return __uint_as_float(__builtin_amdgcn_alignbit(vs[e], vs[e], static_cast<uint32_t>(8 * (r * SB / 16) + 9) & 31u));
  }
};

// Wavefronts per block: 4 or 8, see attn_plan(). Head dimension 64 in 4 bits keeps to the 128 registers of four wavefronts on a SIMD (32
// sequences of 16384 to 32768 positions, 8 heads: 103 us, 136 with 129 registers and three).
template <typename T, int D, int BITS, bool STREAM>
__global__ __launch_bounds__(512, D == 64 && BITS == 4 ? 4 : 2) void kv_attn_kernel(KvAttn a) {
  constexpr int NK = D / 32, NV = D / 16;
  using Tile = KvTile<D, BITS, STREAM>;
  extern __shared__ __align__(16) float lds_attn[];                 // [waves][KV_ROWS][2] maximum and sum, [waves][rows][D + 4]
  const int waves = static_cast<int>(blockDim.x) >> 6;
  const int lane = static_cast<int>(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int b = static_cast<int>(blockIdx.z), kvh = static_cast<int>(blockIdx.y) % a.kv_heads;
  const int row0 = static_cast<int>(blockIdx.y) / a.kv_heads * KV_ROWS, split = static_cast<int>(blockIdx.x);
  const int nrows = min(KV_ROWS, a.rows - row0);
  const int len = static_cast<int>(least(most(a.lengths[b], 0), a.capacity));
  // this lane's query row, its position, and the positions of the block's first and last row
  const int row = row0 + min(r, nrows - 1);
  const int qpos = len - a.tq + row / a.group;
  const int qfirst = len - a.tq + row0 / a.group, qlast = len - a.tq + (row0 + nrows - 1) / a.group;

  // tiles of the sinks, then tiles from the first row's window on
  const int end = max(qlast + 1, 0), tiles_end = (end + KV_TILE - 1) / KV_TILE;
  const int lo = min(max(qfirst - a.window + 1, 0) / KV_TILE, tiles_end);
  const int ns = min((min(a.sinks, end) + KV_TILE - 1) / KV_TILE, lo);
  const int tiles = ns + tiles_end - lo;
  const int per = (tiles + a.splits - 1) / a.splits, t0 = min(split * per, tiles), t1 = min(t0 + per, tiles);

  const int64_t bh = static_cast<int64_t>(b) * a.kv_heads + kvh;
  const uint8_t *kc = a.k_codes + bh * a.capacity * Tile::RB, *ksc = a.k_scales + bh * a.capacity * Tile::SB;
  const uint8_t *vc = a.v_codes + bh * a.capacity * Tile::RB, *vsc = a.v_scales + bh * a.capacity * Tile::SB;
  uint4 qf[NK];
  {
    const T* qp = static_cast<const T*>(a.q) + static_cast<int64_t>(row / a.group) * a.q_st + static_cast<int64_t>(b) * a.q_sb +
                  static_cast<int64_t>(kvh * a.group + row % a.group) * a.q_sh + g * (D / 4);
#pragma unroll
    for (int s = 0; s < NK; ++s) qf[s] = *reinterpret_cast<const uint4*>(qp + 8 * s);
  }
  f32x4_t o[NV];
#pragma unroll
  for (int j = 0; j < NV; ++j) o[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  float m = KV_FLOOR, l = 0.f;
  const float hidden = a.scale_log2 >= 0.f ? -INFINITY : INFINITY;

  auto position_of = [&](int i) { return (i < ns ? i : i - ns + lo) * KV_TILE; };
  auto fetch = [&](Tile& to, int i) {
    const int64_t position = position_of(i);
    to.load(kc, ksc, vc, vsc, position, a.capacity - position, lane);
  };
  uint64_t far_keys = 0;                                           // lanes that met a key that may be beyond the type's largest number
  // exact: held values beyond the type's largest number become that number
  const auto visit = [&](int t, Tile& tile, Tile& next, auto exact) __attribute__((always_inline)) {
    const int position = position_of(t);
    if (t + waves < t1) fetch(next, t + waves);
    if constexpr (!exact) far_keys |= __builtin_amdgcn_ballot_w64(max(tile.ks[0], tile.ks[1]) >= beyond_byte<T, BITS>());
    float sc[8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      f32x4_t s = {0.f, 0.f, 0.f, 0.f};
      const float scale = scale_of(tile.ks[h]);
      uint32_t kw[4 * NK];
#pragma unroll
      for (int w = 0; w < Tile::KW; ++w) held_word<T, BITS>(tile.k[h][w], scale, kw + w * (BITS == 4 ? 4 : 2));
      if constexpr (exact) {
#pragma unroll
        for (int w = 0; w < 4 * NK; ++w) kw[w] = finite_pair<T>(kw[w]);
      }
#pragma unroll
      for (int x = 0; x < NK; ++x) s = mfma_16x16x32<T>(make_uint4(kw[4 * x], kw[4 * x + 1], kw[4 * x + 2], kw[4 * x + 3]), qf[x], s);
#pragma unroll
      for (int e = 0; e < 4; ++e) sc[4 * h + e] = s[e];
    }
    // positions that some row does not see: only where the tile crosses the newest positions or an edge of a window
    if (position + KV_TILE - 1 > qfirst || (position <= qlast - a.window && position + KV_TILE > a.sinks)) {
      const int first = position + 4 * g;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int at = first + 16 * (e / 4) + (e & 3);
        sc[e] = (at > qpos) | ((at <= qpos - a.window) & (at >= a.sinks)) ? hidden : sc[e];
        // What no row of the block sees (rows behind the newest, not written yet, among it) must not meet its probability of
        // zero: an inf or NaN there would come through the product.
        const bool unseen = (at > qlast) | ((at <= qfirst - a.window) & (at >= a.sinks));
#pragma unroll
        for (int w = 0; w < Tile::VW; ++w) tile.v[e][w] = unseen ? 0u : tile.v[e][w];
        tile.vs[e] = unseen ? 0x7f7f7f7fu : tile.vs[e];
      }
    }
    float top = sc[0];
    if (a.scale_log2 >= 0.f) {
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fmaxf(top, sc[e]);
    } else {
#pragma unroll
      for (int e = 1; e < 8; ++e) top = fminf(top, sc[e]);
    }
    top *= a.scale_log2;
    if (__builtin_amdgcn_ballot_w64(top > m + KV_LAZY) != 0) {
      top = fmaxf(top, __shfl_xor(top, 16));
      top = fmaxf(top, __shfl_xor(top, 32));
      const float m_new = top > m + KV_LAZY ? top : m;      // the same in the four lanes of a query row
      const float alpha = fast_exp2(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int j = 0; j < NV; ++j) o[j] *= alpha;
    }
    float p[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) p[e] = fast_exp2(__builtin_fmaf(sc[e], a.scale_log2, -m));
    // Probabilities rounded to the 16-bit type of the product (relative to a maximum at most 2^8 below the true one); their sum is
    // that of the rounded ones, so that the weights the values get add up to one.
    const uint4 pf = make_uint4(round_pair<T>(p[0], p[1]), round_pair<T>(p[2], p[3]), round_pair<T>(p[4], p[5]), round_pair<T>(p[6], p[7]));
    constexpr uint32_t ONES = elem<T>::dtype == NMTG_BF16 ? 0x3f803f80u : 0x3c003c00u;
    l = dot2<T>(pf.x, ONES, dot2<T>(pf.y, ONES, dot2<T>(pf.z, ONES, dot2<T>(pf.w, ONES, l))));
    // two positions at a time: pairs of neighbouring elements become pairs of neighbouring positions
    uint32_t vw[NV][4];
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
      uint32_t x[NV / 2], y[NV / 2];
      const float sx = tile.v_scale(e, r), sy = tile.v_scale(e + 1, r);
      if constexpr (Tile::VB == 2) {
        x[0] = held_pair<T, BITS, 0>(tile.v[e][0], sx);
        x[1] = held_pair<T, BITS, 1>(tile.v[e][0], sx);
        y[0] = held_pair<T, BITS, 0>(tile.v[e + 1][0], sy);
        y[1] = held_pair<T, BITS, 1>(tile.v[e + 1][0], sy);
      } else {
#pragma unroll
        for (int w = 0; w < Tile::VW; ++w) {
          held_word<T, BITS>(tile.v[e][w], sx, x + w * (BITS == 4 ? 4 : 2));
          held_word<T, BITS>(tile.v[e + 1][w], sy, y + w * (BITS == 4 ? 4 : 2));
        }
      }
#pragma unroll
      for (int j = 0; j < NV / 2; ++j) {
        vw[2 * j][e / 2] = __builtin_amdgcn_perm(y[j], x[j], 0x05040100u);
        vw[2 * j + 1][e / 2] = __builtin_amdgcn_perm(y[j], x[j], 0x07060302u);
      }
    }
    if constexpr (exact) {
#pragma unroll
      for (int j = 0; j < NV; ++j)
#pragma unroll
        for (int w = 0; w < 4; ++w) vw[j][w] = finite_pair<T>(vw[j][w]);
    }
#pragma unroll
    for (int j = 0; j < NV; ++j) o[j] = mfma_16x16x32<T>(make_uint4(vw[j][0], vw[j][1], vw[j][2], vw[j][3]), pf, o[j]);
  };
  // two sets of registers in turn, so that nothing is moved from one to the other
  const auto pass = [&](auto exact) __attribute__((always_inline)) {
    Tile even, odd;
    if (t0 + wave < t1) fetch(even, t0 + wave);
    for (int t = t0 + wave; t < t1; t += 2 * waves) {
      visit(t, even, odd, exact);
      if (t + waves < t1) visit(t + waves, odd, even, exact);
    }
  };
  pass(std::false_type{});
  // Where a key may have been inf, or a value was (whatever its probability, its product is inf or NaN and stays in the sums), this wavefront's
  // tiles once more, exactly. (As a branch in every tile the question cost 2 to 7%.)
  float spoilt = 0.f;
#pragma unroll
  for (int j = 0; j < NV; ++j)
#pragma unroll
    for (int i = 0; i < 4; ++i) spoilt = __builtin_fmaf(o[j][i], 0.f, spoilt);
  if ((far_keys | __builtin_amdgcn_ballot_w64(spoilt != spoilt)) != 0) {
#pragma unroll
    for (int j = 0; j < NV; ++j) o[j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
    m = KV_FLOOR;
    l = 0.f;
    pass(std::true_type{});
  }

  // the wavefronts' results: lane (r, g) holds elements (4 g + i) D / 16 + j of query row r in o[j][i]
  l += __shfl_xor(l, 16);
  l += __shfl_xor(l, 32);
  float* lds_o = lds_attn + waves * KV_ROWS * 2;
  if (g == 0) { lds_attn[(wave * KV_ROWS + r) * 2] = m; lds_attn[(wave * KV_ROWS + r) * 2 + 1] = l; }
  if (r < nrows) {
    float* to = lds_o + (wave * nrows + r) * (D + 4);
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < NV; ++j) to[(4 * g + i) * NV + j] = o[j][i];
  }
  __syncthreads();
  for (int i = static_cast<int>(threadIdx.x); i < nrows * D; i += static_cast<int>(blockDim.x)) {
    const int rr = i / D, d = i % D;
    float top = KV_FLOOR;
    for (int w = 0; w < waves; ++w) top = fmaxf(top, lds_attn[(w * KV_ROWS + rr) * 2]);
    float sum = 0.f, val = 0.f;
    for (int w = 0; w < waves; ++w) {
      const float f = fast_exp2(lds_attn[(w * KV_ROWS + rr) * 2] - top);
      sum += f * lds_attn[(w * KV_ROWS + rr) * 2 + 1];
      val += f * lds_o[(w * nrows + rr) * (D + 4) + d];
    }
    const int qrow = row0 + rr;
    if (a.splits == 1) {
      T* op = static_cast<T*>(a.out) + static_cast<int64_t>(qrow / a.group) * a.o_st + static_cast<int64_t>(b) * a.o_sb +
              static_cast<int64_t>(kvh * a.group + qrow % a.group) * a.o_sh;
      op[d] = elem<T>::from_float(sum == 0.f ? 0.f : val / sum);      // (a NaN stays one)
    } else {
      const int64_t at = (split * (static_cast<int64_t>(gridDim.z) * a.kv_heads) + bh) * a.rows + qrow;
      a.part[at * D + d] = val;
      if (d == 0) { a.part_ml[2 * at] = top; a.part_ml[2 * at + 1] = sum; }
    }
  }
}

// The splits of every query row added up, one block per row: a thread per split for its weight, then every split's row by D / 4 threads,
// 256 / (D / 4) splits at a time, added up in that order. Latency bounds it, so that nothing waits on a chain over the splits: 2 sequences
// of 26506 positions, 103 splits each: 6.9 us with its events, 48.7 as a loop over them per element.
constexpr int KV_SPLITS = 256;
template <typename T, int D>
__global__ __launch_bounds__(256) void kv_attn_join_kernel(KvAttn a, int64_t rows_all) {
  constexpr int LANES = D / 4, GROUPS = 256 / LANES;
  __shared__ float weight[KV_SPLITS], wave_top[4], wave_sum[4];
  __shared__ float4 rows[256];
  const int64_t at = blockIdx.x;
  const int t = static_cast<int>(threadIdx.x), wave = t >> 6;
  float m = KV_FLOOR, l = 0.f;
  if (t < a.splits) {
    const float2 ml = *reinterpret_cast<const float2*>(a.part_ml + 2 * (t * rows_all + at));
    m = ml.x; l = ml.y;
  }
  float top = m;
  for (int x = 32; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor(top, x, 64));
  if ((t & 63) == 0) wave_top[wave] = top;
  __syncthreads();
  top = fmaxf(fmaxf(wave_top[0], wave_top[1]), fmaxf(wave_top[2], wave_top[3]));
  const float f = fast_exp2(m - top);
  weight[t] = f;
  float sum = f * l;
  for (int x = 32; x > 0; x >>= 1) sum += __shfl_xor(sum, x, 64);
  if ((t & 63) == 0) wave_sum[wave] = sum;
  __syncthreads();
  const int c = t % LANES, g = t / LANES;
  float4 val = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int s = g; s < a.splits; s += GROUPS) {
    const float4 v = *reinterpret_cast<const float4*>(a.part + (s * rows_all + at) * D + 4 * c);
    const float w = weight[s];
    val.x += w * v.x; val.y += w * v.y; val.z += w * v.z; val.w += w * v.w;
  }
  rows[t] = val;
  __syncthreads();
  if (t >= LANES) return;
  sum = wave_sum[0] + wave_sum[1] + wave_sum[2] + wave_sum[3];
  for (int i = 1; i < min(GROUPS, a.splits); ++i) {
    const float4 v = rows[i * LANES + c];
    val.x += v.x; val.y += v.y; val.z += v.z; val.w += v.w;
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  const int qrow = static_cast<int>(at % a.rows);
  const int64_t bh = at / a.rows, b = bh / a.kv_heads, kvh = bh % a.kv_heads;
  T* op = static_cast<T*>(a.out) + static_cast<int64_t>(qrow / a.group) * a.o_st + b * a.o_sb + (kvh * a.group + qrow % a.group) * a.o_sh;
  const float out[4] = {val.x * inv, val.y * inv, val.z * inv, val.w * inv};
#pragma unroll
  for (int i = 0; i < 4; ++i) op[4 * c + i] = elem<T>::from_float(out[i]);
}

constexpr int64_t KV_MOST_BLOCKS = 0xffffffffll / 256;                 // a launch holds less than 2^32 threads

int check_format(const char* what, int64_t batch, int64_t kv_heads, int64_t head_dim, int64_t capacity, int bits, int dtype) {
  NMTG_REQUIRE(batch >= 0 && kv_heads >= 1 && capacity >= 0, "%s: bad shape batch=%lld kv_heads=%lld capacity=%lld", what, (long long)batch,
               (long long)kv_heads, (long long)capacity);
  NMTG_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head dimension %lld (64 and 128 are built)", what, (long long)head_dim);
  NMTG_REQUIRE(bits == 4 || bits == 8, "%s: %d bits per element (4 and 8 are built)", what, bits);
  NMTG_REQUIRE(dtype == NMTG_F16 || dtype == NMTG_BF16, "%s: fp16 or bf16 tensors required", what);
  NMTG_REQUIRE(batch <= 65535 && kv_heads <= 65535 && capacity < (1ll << 30), "%s: more than 65535 sequences or heads, or 2^30 positions", what);
  return 0;
}
bool rows_view_ok(const void* p, int64_t st, int64_t sb, int64_t sh) {
  return aligned16(p) && st % 8 == 0 && sb % 8 == 0 && sh % 8 == 0 && st >= 0 && sb >= 0 && sh >= 0;
}

// the tiles of a write or read: as many positions as there are, up to 8 (head_dim 128) or 16
int row_tiles(const char* what, KvRows& a, const int32_t* starts, int64_t start, int64_t count, int64_t batch, int64_t kv_heads, int64_t capacity,
              int64_t head_dim, dim3& grid) {
  const int64_t rows = head_dim == 64 ? RowTile<64>::ROWS : RowTile<128>::ROWS;
  a.starts = starts; a.start = start; a.capacity = capacity;
  a.count = static_cast<int>(count); a.batch = static_cast<int>(batch); a.kv_heads = static_cast<int>(kv_heads);
  a.tshift = 0;
  while ((2 << a.tshift) <= (head_dim == 64 ? 16 : 8) && (1 << a.tshift) < count) ++a.tshift;
  const int64_t pairs = batch * kv_heads, pairs_per = rows >> a.tshift, pair_tiles = (pairs + pairs_per - 1) / pairs_per;
  const int64_t tiles = ((count + (1 << a.tshift) - 1) >> a.tshift) * pair_tiles;
  NMTG_REQUIRE(pairs < (1ll << 31) && tiles <= KV_MOST_BLOCKS, "%s: too many rows in one call", what);
  a.pair_tiles = static_cast<int>(pair_tiles);
  grid = dim3(static_cast<unsigned>(tiles), 2);
  return 0;
}

#define KV_DISPATCH(head_dim, bits, dtype, GO)                                                        \
  if (dtype == NMTG_F16) {                                                                            \
    if (head_dim == 64) { if (bits == 4) GO(f16_t, 64, 4); else GO(f16_t, 64, 8); }                   \
    else { if (bits == 4) GO(f16_t, 128, 4); else GO(f16_t, 128, 8); }                                \
  } else {                                                                                            \
    if (head_dim == 64) { if (bits == 4) GO(bf16_t, 64, 4); else GO(bf16_t, 64, 8); }                 \
    else { if (bits == 4) GO(bf16_t, 128, 4); else GO(bf16_t, 128, 8); }                              \
  }

template <typename K>
int attn_launch(K kern, dim3 grid, int waves, int lds, const KvAttn& a, hipStream_t st) {
  if (lds > 64 * 1024) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return fail(NMTG_ERR_LAUNCH, "kv_cache_attn: cannot reserve %d bytes of LDS: %s", lds, hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kern, grid, dim3(64 * waves), lds, st, a);
  return 0;
}

// How the positions of a sequence are shared out. Up to 2048 positions in reach one block of eight wavefronts takes them all: a second
// launch to join parts costs what more blocks would save (64 sequences of 1024 positions in reach, 4 heads of 64 in 8 bits: 17.1 us
// with four blocks each, 9.7 with one). Beyond, blocks of four wavefronts share them, as many as give every compute unit
// four, each wavefront two tiles or more; fewer leave ragged lengths unbalanced (32 sequences of 16384 to 32768 positions, 8 heads of
// 128 in 4 bits: 154 us with four, 162 with two), more cost in the join. Such a reach does not stay in the caches from one step to the
// next, and its codes pass by the L2 (144 us, 5.9 TB/s); a short one mostly does (9.7 us, 10.0 past the L2).
struct AttnPlan { int waves, splits; bool stream; };
AttnPlan attn_plan(int64_t tq, int64_t batch, int64_t heads, int64_t kv_heads, int64_t longest, int64_t window, int64_t sinks) {
  const int64_t rows = tq * (heads / kv_heads), blocks = batch * kv_heads * ((rows + KV_ROWS - 1) / KV_ROWS);
  const int64_t reach = window > 0 ? std::min(longest, window + tq + sinks) : longest;
  const int64_t tiles = (reach + KV_TILE - 1) / KV_TILE;
  if (tiles <= 64) return {8, 1, false};
  const int64_t splits = std::min((4 * num_cus() + blocks - 1) / std::max<int64_t>(blocks, 1), tiles / 8);
  return {4, static_cast<int>(std::max<int64_t>(1, std::min<int64_t>(splits, KV_SPLITS))), true};
}

}  // namespace
}  // namespace nmtg

using namespace nmtg;

extern "C" int nmtg_kv_cache_write(const void* k, int64_t k_stride_t, int64_t k_stride_b, int64_t k_stride_h, const void* v, int64_t v_stride_t,
                                   int64_t v_stride_b, int64_t v_stride_h, uint8_t* k_codes, uint8_t* k_scales, uint8_t* v_codes,
                                   uint8_t* v_scales, const int32_t* starts, int64_t start, int64_t count, int64_t batch, int64_t kv_heads,
                                   int64_t head_dim, int64_t capacity, int bits, int dtype, void* stream) {
  if (int rc = check_format("kv_cache_write", batch, kv_heads, head_dim, capacity, bits, dtype)) return rc;
  NMTG_REQUIRE(count >= 0 && count < (1ll << 31), "kv_cache_write: %lld rows", (long long)count);
  NMTG_REQUIRE(starts != nullptr || (start >= 0 && start + count <= capacity), "kv_cache_write: rows %lld .. %lld of a cache of %lld positions",
               (long long)start, (long long)(start + count), (long long)capacity);
  if (batch == 0 || count == 0 || capacity == 0) return 0;
  NMTG_REQUIRE(k && v && k_codes && k_scales && v_codes && v_scales, "kv_cache_write: null pointer argument");
  NMTG_REQUIRE(rows_view_ok(k, k_stride_t, k_stride_b, k_stride_h) && rows_view_ok(v, v_stride_t, v_stride_b, v_stride_h),
               "kv_cache_write: k and v must be 16-byte aligned [count, batch, kv_heads, head_dim] views with a contiguous head_dim and "
               "strides that are multiples of 8 elements");
  NMTG_REQUIRE(aligned16(k_codes) && aligned16(v_codes), "kv_cache_write: 16-byte aligned codes required");
  KvRows a = {};
  a.k = k; a.v = v; a.k_codes = k_codes; a.k_scales = k_scales; a.v_codes = v_codes; a.v_scales = v_scales;
  a.k_st = k_stride_t; a.k_sb = k_stride_b; a.k_sh = k_stride_h; a.v_st = v_stride_t; a.v_sb = v_stride_b; a.v_sh = v_stride_h;
  dim3 grid;
  if (int rc = row_tiles("kv_cache_write", a, starts, start, count, batch, kv_heads, capacity, head_dim, grid)) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  TraceScope trace("kv_cache_write", st);
#define GO(T, D, B) hipLaunchKernelGGL((kv_write_kernel<T, D, B>), grid, dim3(256), 0, st, a)
  KV_DISPATCH(head_dim, bits, dtype, GO)
#undef GO
  NMTG_CHECK_LAUNCH("kv_cache_write");
  return 0;
}

extern "C" int nmtg_kv_cache_read(const uint8_t* k_codes, const uint8_t* k_scales, const uint8_t* v_codes, const uint8_t* v_scales, void* k,
                                  void* v, const int32_t* starts, int64_t start, int64_t count, int64_t batch, int64_t kv_heads,
                                  int64_t head_dim, int64_t capacity, int bits, int dtype, void* stream) {
  if (int rc = check_format("kv_cache_read", batch, kv_heads, head_dim, capacity, bits, dtype)) return rc;
  NMTG_REQUIRE(count >= 0 && count < (1ll << 31), "kv_cache_read: %lld rows", (long long)count);
  NMTG_REQUIRE(starts != nullptr || (start >= 0 && start + count <= capacity), "kv_cache_read: rows %lld .. %lld of a cache of %lld positions",
               (long long)start, (long long)(start + count), (long long)capacity);
  if (batch == 0 || count == 0) return 0;
  NMTG_REQUIRE(k && v && (capacity == 0 || (k_codes && k_scales && v_codes && v_scales)), "kv_cache_read: null pointer argument");
  NMTG_REQUIRE(aligned16(k) && aligned16(v) && aligned16(k_codes) && aligned16(v_codes), "kv_cache_read: 16-byte aligned codes and results required");
  KvRows a = {};
  a.k_out = k; a.v_out = v;
  a.k_codes = const_cast<uint8_t*>(k_codes); a.k_scales = const_cast<uint8_t*>(k_scales);
  a.v_codes = const_cast<uint8_t*>(v_codes); a.v_scales = const_cast<uint8_t*>(v_scales);
  dim3 grid;
  if (int rc = row_tiles("kv_cache_read", a, starts, start, count, batch, kv_heads, capacity, head_dim, grid)) return rc;
  hipStream_t st = static_cast<hipStream_t>(stream);
  TraceScope trace("kv_cache_read", st);
#define GO(T, D, B) hipLaunchKernelGGL((kv_read_kernel<T, D, B>), grid, dim3(256), 0, st, a)
  KV_DISPATCH(head_dim, bits, dtype, GO)
#undef GO
  NMTG_CHECK_LAUNCH("kv_cache_read");
  return 0;
}

extern "C" int64_t nmtg_kv_cache_attn_workspace_bytes(int64_t tq, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t longest,
                                                      int64_t window, int64_t sinks) {
  if (tq <= 0 || batch <= 0 || heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || head_dim <= 0) return 0;
  const int64_t splits = attn_plan(tq, batch, heads, kv_heads, longest, window, sinks).splits;
  return splits == 1 ? 0 : splits * tq * batch * heads * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
}

extern "C" int nmtg_kv_cache_attn(const void* q, int64_t q_stride_t, int64_t q_stride_b, int64_t q_stride_h, const uint8_t* k_codes,
                                  const uint8_t* k_scales, const uint8_t* v_codes, const uint8_t* v_scales, const int32_t* lengths, void* out,
                                  int64_t out_stride_t, int64_t out_stride_b, int64_t out_stride_h, int64_t tq, int64_t batch, int64_t heads,
                                  int64_t kv_heads, int64_t head_dim, int64_t capacity, int64_t longest, int64_t window, int64_t sinks,
                                  float scale, int bits, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "kv_cache_attn";
  if (int rc = check_format(what, batch, kv_heads, head_dim, capacity, bits, dtype)) return rc;
  NMTG_REQUIRE(tq >= 0 && heads >= kv_heads && heads % kv_heads == 0, "%s: %lld query heads do not share %lld key / value heads evenly", what,
               (long long)heads, (long long)kv_heads);
  NMTG_REQUIRE(longest >= 0 && longest <= capacity, "%s: longest sequence %lld in a cache of %lld positions", what, (long long)longest, (long long)capacity);
  NMTG_REQUIRE(window >= 0 && sinks >= 0 && window < (1ll << 40) && sinks < (1ll << 40), "%s: window %lld, sinks %lld", what, (long long)window, (long long)sinks);
  NMTG_REQUIRE(scale >= -1e6f && scale <= 1e6f, "%s: scale %g", what, (double)scale);
  if (batch == 0 || tq == 0) return 0;
  NMTG_REQUIRE(q && lengths && out && (capacity == 0 || (k_codes && k_scales && v_codes && v_scales)), "%s: null pointer argument", what);
  NMTG_REQUIRE(rows_view_ok(q, q_stride_t, q_stride_b, q_stride_h), "%s: q must be a 16-byte aligned [tq, batch, heads, head_dim] view with a contiguous "
               "head_dim and strides that are multiples of 8 elements", what);
  NMTG_REQUIRE(aligned16(k_codes) && aligned16(v_codes), "%s: 16-byte aligned codes required", what);
  const int64_t group = heads / kv_heads, rows = tq * group, row_blocks = (rows + KV_ROWS - 1) / KV_ROWS;
  NMTG_REQUIRE(rows < (1 << 24) && row_blocks * kv_heads <= 65535, "%s: too many query rows in one call", what);
  KvAttn a = {};
  a.q = q; a.k_codes = k_codes; a.k_scales = k_scales; a.v_codes = v_codes; a.v_scales = v_scales; a.lengths = lengths; a.out = out;
  a.q_st = q_stride_t; a.q_sb = q_stride_b; a.q_sh = q_stride_h; a.o_st = out_stride_t; a.o_sb = out_stride_b; a.o_sh = out_stride_h;
  a.capacity = capacity;
  a.tq = static_cast<int>(tq); a.heads = static_cast<int>(heads); a.kv_heads = static_cast<int>(kv_heads); a.group = static_cast<int>(group);
  a.rows = static_cast<int>(rows); a.scale_log2 = scale == 0.f ? 1e-30f : scale * KV_LOG2E;   // (hidden scores are infinite, and stay so under a scale this small)
  // both fit 31 bits: nothing lies behind the capacity
  a.window = static_cast<int>(window > 0 ? std::min(window, capacity + tq) : capacity + tq);
  a.sinks = static_cast<int>(window > 0 ? std::min(sinks, capacity) : 0);
  const AttnPlan plan = attn_plan(tq, batch, heads, kv_heads, longest, window, sinks);
  a.splits = plan.splits;
  const int64_t rows_all = batch * kv_heads * rows;
  if (a.splits > 1) {
    const int64_t need = a.splits * rows_all * (head_dim + 2) * static_cast<int64_t>(sizeof(float));
    NMTG_REQUIRE(workspace != nullptr && aligned16(workspace) && workspace_bytes >= need,
                 "%s: a 16-byte aligned workspace of %lld bytes required (nmtg_kv_cache_attn_workspace_bytes)", what, (long long)need);
    NMTG_REQUIRE(rows_all <= KV_MOST_BLOCKS, "%s: too many query rows in one call", what);
    a.part = static_cast<float*>(workspace);
    a.part_ml = a.part + a.splits * rows_all * head_dim;
  }
  hipStream_t st = static_cast<hipStream_t>(stream);
  const dim3 grid(static_cast<unsigned>(a.splits), static_cast<unsigned>(kv_heads * row_blocks), static_cast<unsigned>(batch));
  {
    TraceScope trace("kv_cache_attn", st);
    const int lds = plan.waves * (KV_ROWS * 2 + static_cast<int>(std::min<int64_t>(rows, KV_ROWS) * (head_dim + 4))) * static_cast<int>(sizeof(float));
    int launched = 0;
#define GO(T, D, B) launched = plan.stream ? attn_launch(kv_attn_kernel<T, D, B, true>, grid, plan.waves, lds, a, st) : attn_launch(kv_attn_kernel<T, D, B, false>, grid, plan.waves, lds, a, st)
    KV_DISPATCH(head_dim, bits, dtype, GO)
#undef GO
    if (launched) return launched;
  }
  if (a.splits > 1) {
    TraceScope trace("kv_cache_attn_join", st);
    const dim3 rows_grid(static_cast<unsigned>(rows_all));
    if (dtype == NMTG_F16) {
      if (head_dim == 64) hipLaunchKernelGGL((kv_attn_join_kernel<f16_t, 64>), rows_grid, dim3(256), 0, st, a, rows_all);
      else hipLaunchKernelGGL((kv_attn_join_kernel<f16_t, 128>), rows_grid, dim3(256), 0, st, a, rows_all);
    } else {
      if (head_dim == 64) hipLaunchKernelGGL((kv_attn_join_kernel<bf16_t, 64>), rows_grid, dim3(256), 0, st, a, rows_all);
      else hipLaunchKernelGGL((kv_attn_join_kernel<bf16_t, 128>), rows_grid, dim3(256), 0, st, a, rows_all);
    }
  }
  NMTG_CHECK_LAUNCH(what);
  return 0;
}
