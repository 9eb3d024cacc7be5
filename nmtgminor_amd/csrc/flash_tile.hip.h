// What the tiled attention kernels share: the two LDS images of a tile of 64 rows, their reads as matrix-core operands, the way of
// an accumulator tile into the operand of the next product, and the way of a result out of the registers.
#pragma once
#include "gemm_ring.hip.h"

namespace nmtg {
namespace {

constexpr int FA_ROWS = 128;   // queries (forward, dQ) or keys (dK/dV) per block: 32 per wavefront
constexpr int FA_TILE = 64;    // rows of the streamed operand per LDS tile
constexpr int FA_THREADS = 256;
constexpr float FA_NEG = -1e30f;
constexpr float FA_LAZY = 8.f;   // log2 of the growth of a row maximum that moves the softmax's reference point
constexpr float FA_LOG2E = 1.4426950408889634f;

typedef unsigned int u32x2_t __attribute__((ext_vector_type(2)));
typedef short s16x4_t __attribute__((ext_vector_type(4)));

// lanes 32..63 of `a` change places with lanes 0..31 of `b`
__device__ __forceinline__ void swap_halves(uint32_t& a, uint32_t& b) {
  const u32x2_t r = __builtin_amdgcn_permlane32_swap(a, b, false, false);
  a = r[0];
  b = r[1];
}
// f(own value, value of lane ^ 32)
__device__ __forceinline__ float pair_max(float v) {
  uint32_t a = __float_as_uint(v), b = a;
  swap_halves(a, b);
  return fmaxf(__uint_as_float(a), __uint_as_float(b));
}
__device__ __forceinline__ float pair_sum(float v) {
  uint32_t a = __float_as_uint(v), b = a;
  swap_halves(a, b);
  return __uint_as_float(a) + __uint_as_float(b);
}

// two floats rounded (to nearest even) into one register of two 16-bit elements, one conversion instruction
typedef float f32x2_t __attribute__((ext_vector_type(2)));
template <typename T> struct pair_of;
template <> struct pair_of<f16_t> { typedef _Float16 type __attribute__((ext_vector_type(2))); };
template <> struct pair_of<bf16_t> { typedef __bf16 type __attribute__((ext_vector_type(2))); };
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  const f32x2_t v = {lo, hi};
  return __builtin_bit_cast(uint32_t, __builtin_convertvector(v, typename pair_of<T>::type));
}

// Accumulator registers r0 .. r0+7 of a 32 x 32 tile (lane (col, half) holds rows 8 (r / 4) + 4 half + r % 4) as the
// B operand of the next product: lane (col, half) holds rows 16 (r0 / 8) + 8 half .. + 7.
template <typename T>
__device__ __forceinline__ uint4 acc_to_operand(const float* p) {
  uint32_t g0a = pack2<T>(p[0], p[1]), g0b = pack2<T>(p[2], p[3]), g1a = pack2<T>(p[4], p[5]), g1b = pack2<T>(p[6], p[7]);
  swap_halves(g0a, g1a);
  swap_halves(g0b, g1b);
  return make_uint4(g0a, g0b, g1a, g1b);
}

// ---- LDS images of a [64 rows][D] tile, rows of D 16-bit elements = D / 8 chunks of 16 bytes ----
// "row image": chunk c of row r at position c ^ (r & 7); read as the A operand (lane = row, 8 consecutive columns).
// "transposed image": chunk c of row r at position c ^ 2 (r & 3); read with ds_read_b64_tr_b16 as the A operand of the
// transposed tile (lane = column, 8 consecutive rows).
template <int D>
__device__ __forceinline__ uint32_t row_image_at(int r, int c) { return static_cast<uint32_t>(r * (2 * D) + ((c ^ (r & 7)) * 16)); }
template <int D>
__device__ __forceinline__ uint32_t tr_image_at(int r, int c) { return static_cast<uint32_t>(r * (2 * D) + ((c ^ (2 * (r & 3))) * 16)); }

template <int D>
struct Staged {
  static constexpr int CH = D / 8;
  static constexpr int N = FA_TILE * CH / FA_THREADS;
  uint4 v[N];
  // rows row0 .. row0+63 of a sequence of `len` rows that starts at `base` (head offset applied); rows past the end are zeros
  template <typename T>
  __device__ __forceinline__ void load(const T* base, int64_t stride, int row0, int len) {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = (static_cast<int>(threadIdx.x) & (FA_THREADS - 1)) + FA_THREADS * i;   // a block may hold several groups of FA_THREADS
      const int r = id / CH, c = id % CH;
      v[i] = make_uint4(0, 0, 0, 0);
      if (row0 + r < len) v[i] = *reinterpret_cast<const uint4*>(base + static_cast<int64_t>(row0 + r) * stride + 8 * c);
    }
  }
  __device__ __forceinline__ void store_rows(uint8_t* img) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = (static_cast<int>(threadIdx.x) & (FA_THREADS - 1)) + FA_THREADS * i;   // a block may hold several groups of FA_THREADS
      *reinterpret_cast<uint4*>(img + row_image_at<D>(id / CH, id % CH)) = v[i];
    }
  }
  __device__ __forceinline__ void store_transposed(uint8_t* img) const {
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int id = (static_cast<int>(threadIdx.x) & (FA_THREADS - 1)) + FA_THREADS * i;   // a block may hold several groups of FA_THREADS
      *reinterpret_cast<uint4*>(img + tr_image_at<D>(id / CH, id % CH)) = v[i];
    }
  }
};

// A operand from the row image: rows 32 i + (lane & 31), columns 16 s + 8 (lane >> 5) .. + 7
template <int D>
__device__ __forceinline__ uint4 read_rows(const uint8_t* img, int i, int s, int lane) {
  return *reinterpret_cast<const uint4*>(img + row_image_at<D>(32 * i + (lane & 31), 2 * s + (lane >> 5)));
}
// A operand of the transposed tile: columns 32 i + (lane & 31), rows 16 kk + 8 (lane >> 5) .. + 7. Within 16 lanes the
// transposing read takes 4 rows x 16 columns and hands each lane the 4 rows of its own column.
template <int D>
__device__ __forceinline__ uint4 read_transposed(const uint8_t* img, int i, int kk, int lane) {
  const int r = 16 * kk + 8 * (lane >> 5) + ((lane >> 2) & 3);
  const int c = 4 * i + 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
  const uint8_t* p = img + tr_image_at<D>(r, c) + (lane & 1) * 8;      // r + 4 has the same r & 3: same swizzle
  const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(p));
  const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4_t*)(p + 4 * 2 * D));
  union { s16x4_t s[2]; uint4 u; } cv;
  cv.s[0] = lo;
  cv.s[1] = hi;
  return cv.u;
}

// The wavefront's 32 resident rows as the B operand: lane (row, half) holds columns 16 s + 8 half .. + 7
template <typename T, int D>
__device__ __forceinline__ void load_resident(uint4 (&f)[D / 16], const T* base, int64_t stride, int row, int len, int lane) {
  const T* p = base + static_cast<int64_t>(row) * stride + 8 * (lane >> 5);
#pragma unroll
  for (int s = 0; s < D / 16; ++s) f[s] = row < len ? *reinterpret_cast<const uint4*>(p + 16 * s) : make_uint4(0, 0, 0, 0);
}

// Touches the rows that stay in registers for a whole tile loop (the queries of the inference kernel), in front of the
// loop and outside any branch. They are loaded under conditions, and without a use that the compiler sees on every path
// it repeats the wait for them inside the loop, behind the loads of the next tile: every tile then waits for its own
// prefetch. Not for the training kernels: behind a statement like this one (or a wait instruction of our own) the
// compiler no longer reads wave-uniform values (tile classes, dropout bits) through the scalar cache but with vector
// loads, each waited for on the spot.
template <int N>
__device__ __forceinline__ void registers_landed(const uint4 (&f)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) asm volatile("" ::"v"(f[i].x), "v"(f[i].y), "v"(f[i].z), "v"(f[i].w));
}

// Writes the wavefront's 32 rows x D accumulators (acc[i][r]: column 32 i + 8 (r / 4) + 4 half + r % 4 of row lane & 31)
// through its own LDS patch as whole 16-byte chunks, rows past `len` skipped.
template <typename T, int D>
__device__ __forceinline__ void store_rows_out(const acc16_t (&acc)[D / 32], float mul, uint8_t* patch, T* base, int64_t stride,
                                               int row0, int len, int lane) {
  const int half = lane >> 5, row = lane & 31;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g) {
      const int col = 32 * i + 8 * g + 4 * half;
      uint2 w;
      w.x = pack2<T>(acc[i][4 * g + 0] * mul, acc[i][4 * g + 1] * mul);
      w.y = pack2<T>(acc[i][4 * g + 2] * mul, acc[i][4 * g + 3] * mul);
      *reinterpret_cast<uint2*>(patch + row_image_at<D>(row, col / 8) + (col % 8) * 2) = w;
    }
  __syncthreads();
  constexpr int CH = D / 8;
#pragma unroll
  for (int i = 0; i < 32 * CH / 64; ++i) {
    const int id = lane + 64 * i;
    const int r = id / CH, c = id % CH;
    if (row0 + r < len)
      *reinterpret_cast<uint4*>(base + static_cast<int64_t>(row0 + r) * stride + 8 * c) =
          *reinterpret_cast<const uint4*>(patch + row_image_at<D>(r, c));
  }
}

}  // namespace
}  // namespace nmtg
