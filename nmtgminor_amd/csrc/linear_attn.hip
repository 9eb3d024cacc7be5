// Linear attention with a decay for each head, forward and backward in chunks on the matrix cores, and the recurrence itself for the newest
// positions of a decoder (gfx950).
//
//   S_t = lambda S_(t-1) + k_t v_t^T,   o_t = scale S_t^T q_t,   lambda = exp(log_decay)
//
// A walk takes rows x, y, z in chunks of 32 and computes, with X the state in front of the chunk,
//   out_i = scale (lambda^(i+e) X^T x_i + sum_(j<=i) lambda^(i-j) (x_i . y_j) z_j),    X <- lambda^m X + sum_j lambda^(m-j-e) y_j z_j^T
// for the m rows i, j of a chunk. Four walks are the whole operator:
//   out   x, y, z = q, k, v,    forwards, e = 1, X = S
//   dq              dout, v, k, forwards, e = 1, X = S^T
//   dv              k, q, dout, backwards, e = 0, X = R = sum_(t>=j) lambda^(t-j) q_t dout_t^T + lambda^.. dS / scale, decayed once more
//   dk              v, dout, q, backwards, e = 0, X = R^T
// and what R is in front of the first position is the gradient of the state that was given.
//
// A block has a head's state X in its accumulators, 32 columns a wavefront, and goes through its rows chunk by chunk: rows straight into LDS a
// chunk ahead, X rounded to 16 bits from the accumulators into the operands of its product with the rows, the scores of a chunk from
// accumulators into operands (S^T = Y X^T, so that a lane has one row's), X updated in 32 bits. Chunks of 32 rows: one tile of scores.
// Where heads are too few to fill the GPU, sequences are split into segments (LaPlan): a first launch finds what each segment adds to the
// state, a scan, or the blocks of heads of 64 themselves, put the states together. The forward keeps its states for the backward (64 KB per
// segment and head of 128), whose first launch then reads queries and output gradients alone.
//
// Rounding. The state, sums and powers are in 32 bits; a power of lambda is one exponential, a state's decay over many chunks the product of
// few (LA_OWED). Scores and the state are rounded to 16 bits where the products take them: about as much error as rounding the result
// adds (bf16: 0.0023 of the norm instead of 0.0017). What is added to the state is carried to 22 bits (fp16) or 24 (bf16, where the state is a
// result; 16 otherwise): states and their gradients are off by 4e-7. fp16 takes scores relative to a row's largest, the state to a slice's
// and lambda^.. z to a chunk's largest, by powers of two, so that scores and states far beyond its range give the outputs that are in it.
//
// What bounds it (MI355X; a large copy: 5.2 to 5.4 TB/s). Memory, where the GPU is full: 16384 positions, 32 heads of 128: outputs 115 us, 575 MB past the
// L2, 5.0 TB/s; the segments' states 68 us, 283 MB, 4.2 TB/s, with the matrix cores and the vector units at 43% each. 2 x 8192 positions, 32
// heads of 128, three walks: 293 us, 1.46 GB past the L2 (dK's and dV's blocks share rows there), 5.0 TB/s. Without the products that update the state the
// same three kernels would take 111, 65 and 261 us. 8 x 2048, 16 heads of 64: 28 us (145 MB, 5.2 TB/s) and 63 (328 MB, 5.2 TB/s). A block alone on a
// compute unit takes 1.5 us a chunk (head dimension 64: 1.1), which bounds few heads. What did not help: rows two chunks ahead (201 -> 204 us for a
// prompt, 117 -> 118 for 8 x 2048), operands of the next chunk read into registers before the barrier (201 -> 202; alone 1.5 -> 2.2 us a chunk), z's parts between
// the products by hand, wave priorities. No atomics, and sums in a fixed order: results do not depend on scheduling.
#include "flash_tile.hip.h"
#include <algorithm>
#include <type_traits>

namespace nmtg {
namespace {

constexpr int LA_CHUNK = 32;
constexpr float LA_OWED = 8.f;      // bits: a state in the registers is at most 2^16 times its value

struct LaView { const void* p; int64_t st, sb, sh; };   // [len, batch, heads, head_dim], head_dim contiguous

struct LaWalk {
  LaView x, y, z, o;
  const float* state_in;       // of a walk that is not split: the state in front, or null
  float* state_out;            // the state behind the last position, or null
  float* parts;                // [batch * heads][segments][head_dim][head_dim]: the state given, then what segments 0 .. add; behind a scan
                               // the state in front of every segment
  float mul_in, mul_out;       // of state_in and state_out
  bool backwards, transposed;  // transposed: state_in and parts hold X^T
  bool exact;                  // the state is a result
};
struct LaArgs {
  LaWalk walk[3];
  const float* log_decay;
  const int32_t* lengths;
  int walks, len, batch, heads, segments, segment;   // segment: positions of one, a multiple of LA_CHUNK
  bool folded;                                       // see LaPlan
  float scale;
};

// Consecutive blocks of a launch go round the eight XCDs, each with an L2 of its own: item i of `total` in launch order, re-counted so
// that every XCD gets a contiguous piece.
__device__ __forceinline__ uint32_t xcd_piece(uint32_t i, uint32_t total) {
  const uint32_t xcd = i & 7, share = total >> 3, more = total & 7;
  return xcd * share + min(xcd, more) + (i >> 3);
}

template <typename T>
__device__ __forceinline__ const T* la_head(const LaView& v, int b, int h) {
  return static_cast<const T*>(v.p) + static_cast<int64_t>(b) * v.sb + static_cast<int64_t>(h) * v.sh;
}
__device__ __forceinline__ int la_length(const LaArgs& a, int b) { return a.lengths != nullptr ? min(max(a.lengths[b], 0), a.len) : a.len; }
// log(lambda), at most 0; the lower bound keeps -inf times 0 from being NaN
__device__ __forceinline__ float la_decay(const float* log_decay, int h) {
  const float d = log_decay[h];
  return d > 0.f ? 0.f : d < -1e30f ? -1e30f : d;
}

// ---- the LDS image of 32 rows: the 16-byte chunks of row r change places by an exclusive-or with la_swizzle(r) ----
template <int D>
__device__ __forceinline__ int la_swizzle(int r) { return D == 64 ? (4 * ((r >> 1) & 1) | ((r >> 2) & 3)) : (4 * (r & 3) | ((r >> 2) & 3)); }
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
template <typename V>
__device__ __forceinline__ const __attribute__((address_space(3))) V* lds_ptr(uint32_t at) {
  return reinterpret_cast<const __attribute__((address_space(3))) V*>(at);
}
template <int D>
struct LaReader {
  uint32_t rows, columns;
  __device__ __forceinline__ LaReader(uint32_t base, int lane) {
    const int r = lane & 31, rt = 4 * (lane >> 5) + ((lane >> 2) & 3), ct = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
    rows = base + static_cast<uint32_t>(r * (2 * D) + ((lane >> 5) ^ la_swizzle<D>(r)) * 16);
    columns = base + static_cast<uint32_t>(rt * (2 * D) + (ct ^ la_swizzle<D>(rt)) * 16 + (lane & 1) * 8);
  }
  // hides that the addresses do not change, or the compiler would keep one register per piece of an operand through the loop
  __device__ __forceinline__ void per_chunk() { asm volatile("" : "+v"(rows), "+v"(columns)); }
  // row lane & 31, columns 16 s + 8 (lane >> 5) .. + 7
  __device__ __forceinline__ uint4 row_operand(int img, int s) const {
    const u32x4_t v = *lds_ptr<u32x4_t>((rows ^ static_cast<uint32_t>(32 * s)) + static_cast<uint32_t>(img));
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
  // Column 32 i + (lane & 31), of every 16 rows those that a lane has of an accumulator tile, 4 (lane >> 5) .. + 3 and 8 + 4 (lane >> 5) .. + 3:
  // the scores go from accumulators into operands in the lanes that hold them.
  __device__ __forceinline__ uint4 column_operand(int img, int i, int kk) const {
    const uint32_t at = columns ^ static_cast<uint32_t>(64 * i), off = static_cast<uint32_t>(img + 16 * kk * 2 * D);
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(const_cast<__attribute__((address_space(3))) s16x4_t*>(lds_ptr<s16x4_t>(at + off)));
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(const_cast<__attribute__((address_space(3))) s16x4_t*>(lds_ptr<s16x4_t>((at ^ 32u) + (off + 8 * 2 * D))));
    union { s16x4_t s[2]; uint4 u; } cv;
    cv.s[0] = lo;
    cv.s[1] = hi;
    return cv.u;
  }
};

// Transfers of the m rows of a chunk into an image, shared out over the block's wavefronts: lane l of transfer n fills chunk 64 n + l.
// Rows behind the last are read as the last (in bounds; their weights are zero and their results are not kept).
template <typename T, int D>
struct LaLoader {
  static constexpr int CH = D / 8, N = 2;     // D / 32 wavefronts
  int row[N];
  uint32_t col[N];
  uint32_t to;
  __device__ __forceinline__ LaLoader(int wave, int lane) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int id = 64 * (wave * N + n) + lane;
      row[n] = id / CH;
      col[n] = static_cast<uint32_t>(((id % CH) ^ la_swizzle<D>(row[n])) * 16);
    }
    to = static_cast<uint32_t>(wave * N * 1024);
  }
  // rows at walked positions u .. u + m - 1 of a sequence of n
  __device__ __forceinline__ void start(const T* head, int64_t stride, int u, int m, int n, bool backwards, uint32_t img) const {
    const T* base = head + static_cast<int64_t>(backwards ? n - u - m : u) * stride;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      const int r = min(row[i], m - 1);
      dma16(static_cast<uint32_t>((backwards ? m - 1 - r : r) * static_cast<int>(stride)) * 2 + col[i], base, img + to + 1024 * i);
    }
  }
};

// 2^k with k so that `largest`, if it is at least 2^LOWEST, times it is at least 2^14 and below 2^15, and its inverse: where fp16 holds
// all its bits, and two of its numbers 22. room: as many powers of two less; up is 2^(14 - least) at most
struct Pow2 { float up, down; };
__device__ __forceinline__ int exponent_of(float x) { return static_cast<int>(__float_as_uint(x) >> 23) - 127; }      // x >= 0
template <int LOWEST>
__device__ __forceinline__ Pow2 to_half_range(float largest, int room = 0, int least = LOWEST) {
  const int e = max(max(exponent_of(largest), LOWEST) + room, least);
  return {__uint_as_float(static_cast<uint32_t>(141 - e) << 23), __uint_as_float(static_cast<uint32_t>(113 + e) << 23)};
}

// x rounded to 16 bits, and what that took from it
template <typename T>
__device__ __forceinline__ uint4 round_to(const float (&x)[8]) {
  return make_uint4(pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7]));
}
template <typename T>
__device__ __forceinline__ void subtract(float (&x)[8], const uint4& rounded) {
  const uint32_t words[4] = {rounded.x, rounded.y, rounded.z, rounded.w};
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    T t;
    t.bits = static_cast<uint16_t>(words[j / 2] >> (16 * (j & 1)));
    x[j] -= elem<T>::to_float(t);
  }
}

// OUT: the walk of a segment, its outputs written. Otherwise what a segment adds to the state, from zero.
template <typename T, int D, bool OUT>
__global__ __launch_bounds__(2 * D, 2) void linear_walk_kernel(LaArgs a) {
  extern __shared__ __align__(256) uint8_t lds_raw[];
  constexpr bool HALF = elem<T>::dtype == NMTG_F16;
  constexpr int IMG = LA_CHUNK * D * 2, YIMG = 0, ZIMG = IMG, XIMG = 2 * IMG, BUF = (OUT ? 3 : 2) * IMG;
  const int lane = static_cast<int>(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6);
  const int half = lane >> 5, li = lane & 31;
  const uint32_t id = xcd_piece(blockIdx.x, gridDim.x);
  const int segments = OUT ? a.segments : a.segments - 1;
  const LaWalk& w = a.walk[id % a.walks];
  const uint32_t rest = id / a.walks;
  const int seg = static_cast<int>(rest % segments), bh = static_cast<int>(rest / segments), b = bh / a.heads, h = bh % a.heads;
  const int n = la_length(a, b), u0 = seg * a.segment, u1 = min(u0 + a.segment, n);
  const T *x = OUT ? la_head<T>(w.x, b, h) : nullptr, *y = la_head<T>(w.y, b, h), *z = la_head<T>(w.z, b, h);
  const bool backwards = w.backwards, exact = w.exact;
  const int64_t x_stride = w.x.st, y_stride = w.y.st, z_stride = w.z.st, o_stride = w.o.st;
  const LaLoader<T, D> loader(wave, lane);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds_raw)));
  const LaReader<D> lane_reader(lds0, lane);
  auto start = [&](int u, int buffer) __attribute__((always_inline)) {
    const int m = min(LA_CHUNK, u1 - u);
    const uint32_t to = lds0 + static_cast<uint32_t>(buffer) * BUF;
    loader.start(y, y_stride, u, m, n, backwards, to + YIMG);
    loader.start(z, z_stride, u, m, n, backwards, to + ZIMG);
    if constexpr (OUT) loader.start(x, x_stride, u, m, n, backwards, to + XIMG);
  };
  if (u0 < u1) start(u0, 0);

  // the state: rows 32 i + 8 (r / 4) + 4 half + r % 4 of column `col` in register r of tile i
  const int col = 32 * wave + li;
  const float l2 = la_decay(a.log_decay, h) * FA_LOG2E;
  acc16_t s[D / 32];
  // s <- from mul for the first, s <- keep s + from for those behind
  const auto add_state = [&](const float* from, float keep, float mul, auto first) __attribute__((always_inline)) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int row = 32 * i + 8 * g + 4 * half;
        float v[4] = {0.f, 0.f, 0.f, 0.f};
        if (from != nullptr) {
          if (w.transposed) load_pack<float, 4>(from + col * D + row, v);
          else {
#pragma unroll
            for (int j = 0; j < 4; ++j) v[j] = from[(row + j) * D + col];
          }
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) s[i][4 * g + j] = decltype(first)::value ? v[j] * mul : s[i][4 * g + j] * keep + v[j];
      }
  };
  float* const parts = w.parts + static_cast<int64_t>(bh) * a.segments * (D * D);
  const float* given = w.state_in != nullptr ? w.state_in + static_cast<int64_t>(bh) * (D * D) : nullptr;
  if constexpr (OUT) {
    const bool whole = a.segments == 1, later = !a.folded && seg > 0;
    add_state(whole ? given : later ? parts + seg * (D * D) : given != nullptr ? parts : nullptr, 0.f, whole ? w.mul_in : 1.f, std::true_type{});
    if (D == 64 && a.folded) {
      for (int i = 1; i <= seg; ++i)
        add_state(parts + i * (D * D), __builtin_amdgcn_exp2f(static_cast<float>(min(max(n - (i - 1) * a.segment, 0), a.segment)) * l2), 1.f,
                  std::false_type{});
    }
  } else {
    add_state(nullptr, 0.f, 1.f, std::true_type{});
    const int copied = a.folded && seg == 0 && given != nullptr ? D * D : 0;      // (the walk may write its last state over the one given)
    for (int i = static_cast<int>(threadIdx.x) * 4; i < copied; i += 8 * D) {
      float v[4];
      load_pack<float, 4>(given + i, v);
#pragma unroll
      for (int j = 0; j < 4; ++j) v[j] *= w.mul_in;
      store_pack<float, 4>(parts + i, v);
    }
  }

  const int e = backwards ? 0 : 1;
  float apart[16], left[16];                                    // of a whole chunk: scale lambda^(i - j) of row i = li, lambda^(32 - j - e)
#pragma unroll
  for (int r = 0; r < 16; ++r) {
    const int j = 8 * (r / 4) + 4 * half + r % 4;
    if constexpr (OUT) apart[r] = j <= li ? __builtin_amdgcn_exp2f(static_cast<float>(li - j) * l2) * a.scale : 0.f;
    left[r] = __builtin_amdgcn_exp2f(static_cast<float>(LA_CHUNK - j - e) * l2);
  }
  const float front = __builtin_amdgcn_exp2f(static_cast<float>(li + e) * l2) * a.scale;
  // The registers hold the state times 2^owed unit.up: decays are owed to it until they come to 2^-LA_OWED (the weights of what is added
  // grow instead), which is less work, and no factor of a chunk multiplies its own rounding over the chunks. unit: fp16's
  // numbers, which lambda^.. z is split into, have their bits where the chunk's largest z is, and the state in the registers, whatever it was given
  // as, stays below 2^126 (where segments begin with zero, 2^24 positions of fp16's values make 2^94 at most).
  float owed = 0.f;
  Pow2 unit = {1.f, 1.f};
  const bool lean = !HALF && LA_CHUNK * -l2 <= LA_OWED;
  T* const out_rows = OUT ? const_cast<T*>(la_head<T>(w.o, b, h)) + 32 * wave + 8 * half : nullptr;

  // LEAN: a whole chunk of a head whose decay within it may be owed: one block of code, in which the products of one part run under the
  // arithmetic of another. Otherwise any chunk.
  const auto visit = [&](int u, auto buffer, auto lean_tag) __attribute__((always_inline)) {
    constexpr bool LEAN = decltype(lean_tag)::value;
    constexpr int img = decltype(buffer)::value * BUF;
    const int m = LEAN ? LA_CHUNK : min(LA_CHUNK, u1 - u);
    if (OUT && u > u0) wait_vmcnt<counted_stores(2)>();         // the chunk is there (the outputs of the one before left after it)
    else wait_vmcnt<0>();
    ring_barrier();                                             // for every wavefront, and the one before has been read
    if (u + LA_CHUNK < u1) start(u + LA_CHUNK, 1 - buffer);
    LaReader<D> reader = lane_reader;
    reader.per_chunk();
    const auto scale_state = [&](float f) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
#pragma unroll
        for (int r = 0; r < 16; ++r) s[i][r] *= f;
    };
    if (LEAN && owed > LA_OWED) {
      scale_state(__builtin_amdgcn_exp2f(-owed));
      owed = 0.f;
    }

    uint4 zf[2];                                                // z: column `col`, 16 rows each
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) zf[kk] = reader.column_operand(img + ZIMG, wave, kk);
    float out[16], highest = 0.f;                               // highest: of the state in the registers (fp16)
    if constexpr (OUT) {
      uint4 xf[D / 16], yf[D / 16];
#pragma unroll
      for (int ss = 0; ss < D / 16; ++ss) {
        xf[ss] = reader.row_operand(img + XIMG, ss);
        yf[ss] = reader.row_operand(img + YIMG, ss);
      }
      acc16_t p, o;
#pragma unroll
      for (int r = 0; r < 16; ++r) { p[r] = 0.f; o[r] = 0.f; }
      Pow2 range = {1.f, 1.f};
      if constexpr (HALF) {
        float top = 0.f;
#pragma unroll
        for (int i = 0; i < D / 32; ++i)
#pragma unroll
          for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(s[i][r]));
        top = wave_max(top);
        if (top == INFINITY) {                                  // the columns without an inf go on
          top = 0.f;
#pragma unroll
          for (int i = 0; i < D / 32; ++i)
#pragma unroll
            for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(s[i][r]) == INFINITY ? 0.f : fabsf(s[i][r]));
          top = wave_max(top);
        }
        range = to_half_range<-112>(top);
        highest = top;
      }
#pragma unroll
      for (int ss = 0; ss < D / 16; ++ss) {
        float v[8];
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = HALF ? s[ss / 2][8 * (ss % 2) + j] * range.up : s[ss / 2][8 * (ss % 2) + j];
        mfma<T>::run(acc_to_operand<T>(v), xf[ss], o);
        mfma<T>::run(yf[ss], xf[ss], p);
      }
#pragma unroll
      for (int r = 0; r < 16; ++r) p[r] *= apart[r];
      const float f1 = front * __builtin_amdgcn_exp2f(-owed) * (HALF ? range.down * unit.down : 1.f);
      if constexpr (HALF) {
        float top = 0.f;
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(p[r]));
        const Pow2 row = to_half_range<-112>(pair_max(top));
        acc16_t within;
#pragma unroll
        for (int r = 0; r < 16; ++r) within[r] = 0.f;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = p[8 * kk + j] * row.up;
          mfma<T>::run(zf[kk], round_to<T>(v), within);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) out[r] = o[r] * f1 + within[r] * row.down;
      } else {
#pragma unroll
        for (int r = 0; r < 16; ++r) o[r] *= f1;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
          float v[8];
#pragma unroll
          for (int j = 0; j < 8; ++j) v[j] = p[8 * kk + j];
          mfma<T>::run(zf[kk], round_to<T>(v), o);
        }
#pragma unroll
        for (int r = 0; r < 16; ++r) out[r] = o[r];
      }
    }

    float zv[2][8];
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      const uint32_t words[4] = {zf[kk].x, zf[kk].y, zf[kk].z, zf[kk].w};
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        T t;
        t.bits = static_cast<uint16_t>(words[j / 2] >> (16 * (j & 1)));
        zv[kk][j] = elem<T>::to_float(t);
      }
    }
    owed -= static_cast<float>(m) * l2;
    if constexpr (!LEAN) {
      if (m < LA_CHUNK) {
#pragma unroll
        for (int r = 0; r < 16; ++r) {
          const int j = 8 * (r / 4) + 4 * half + r % 4;
          left[r] = j < m ? __builtin_amdgcn_exp2f(static_cast<float>(m - j - e) * l2) : 0.f;
        }
      }
      float pay = 1.f;
      if (owed > LA_OWED) {
        pay = __builtin_amdgcn_exp2f(-owed);
        owed = 0.f;
      }
      if constexpr (HALF) {
        float top = 0.f;
#pragma unroll
        for (int kk = 0; kk < 2; ++kk)
#pragma unroll
          for (int j = 0; j < 8; ++j) top = fmaxf(top, fabsf(zv[kk][j]));
        const int least = OUT ? exponent_of(highest * pay) - exponent_of(unit.up) - 111 : -24;
        const Pow2 next = to_half_range<-24>(fminf(wave_max(top), 65504.f), static_cast<int>(ceilf(owed)), least);
        pay *= unit.down * next.up;
        unit = next;
      }
      if (pay != 1.f) scale_state(pay);
    }
    const float grown = __builtin_amdgcn_exp2f(owed) * unit.up;
    // lambda^.. z as the sum of two numbers of 16 bits (fp16: 22 bits), of three for bf16 where the state is a result in 32 bits (24 bits);
    // one that only goes into products, which take it in 8 bits, has 16
#pragma unroll
    for (int kk = 0; kk < 2; ++kk) {
      uint4 yt[D / 32];
#pragma unroll
      for (int i = 0; i < D / 32; ++i) yt[i] = reader.column_operand(img + YIMG, i, kk);
      float v[8];
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = zv[kk][j] * (left[8 * kk + j] * grown);
      const uint4 first = round_to<T>(v);
      subtract<T>(v, first);
      const uint4 second = round_to<T>(v);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) mfma<T>::run(yt[i], second, s[i]);
#pragma unroll
      for (int i = 0; i < D / 32; ++i) mfma<T>::run(yt[i], first, s[i]);
      if (!HALF && exact) {
        subtract<T>(v, second);
        const uint4 third = round_to<T>(v);
#pragma unroll
        for (int i = 0; i < D / 32; ++i) mfma<T>::run(yt[i], third, s[i]);
      }
    }
    if constexpr (OUT) {
      // row li: columns 32 wave + 16 kk + 8 half .. + 7
      T* to = out_rows + static_cast<int64_t>(backwards ? n - 1 - u - li : u + li) * o_stride;
      const uint4 lo = acc_to_operand<T>(out), hi = acc_to_operand<T>(out + 8);
      if (LEAN || li < m) {
        *reinterpret_cast<uint4*>(to) = lo;
        *reinterpret_cast<uint4*>(to + 16) = hi;
      }
    }
  };
  const auto walk = [&](int u, int end, auto lean_tag) __attribute__((always_inline)) {
    for (; u < end; u += 2 * LA_CHUNK) {
      visit(u, std::integral_constant<int, 0>{}, lean_tag);
      if (u + LA_CHUNK < end) visit(u + LA_CHUNK, std::integral_constant<int, 1>{}, lean_tag);
    }
  };
  // whole pairs of chunks, so that the rest begins with the first buffer
  const int split_at = lean ? u0 + max(u1 - u0, 0) / (2 * LA_CHUNK) * (2 * LA_CHUNK) : u0;
  if constexpr (!HALF) walk(u0, split_at, std::true_type{});
  walk(split_at, u1, std::false_type{});

  if constexpr (OUT) {
    // positions behind the sequence's end
    constexpr int CH = D / 8;
    T* to = const_cast<T*>(la_head<T>(w.o, b, h));
    const int first = max(n, u0), count = (min(u0 + a.segment, a.len) - first) * CH;
    for (int i = static_cast<int>(threadIdx.x); i < count; i += 2 * D)
      *reinterpret_cast<uint4*>(to + static_cast<int64_t>(first + i / CH) * w.o.st + i % CH * 8) = make_uint4(0, 0, 0, 0);
  }
  float* end = nullptr;
  float mul = 1.f;
  if constexpr (!OUT) end = parts + (seg + 1) * (D * D);
  else if (w.state_out != nullptr && seg == segments - 1) { end = w.state_out + static_cast<int64_t>(bh) * (D * D); mul = w.mul_out; }
  mul *= unit.down * __builtin_amdgcn_exp2f(-owed);
  if (end != nullptr) {
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) end[(32 * i + 8 * (r / 4) + 4 * half + r % 4) * D + col] = s[i][r] * mul;
  }
}

// parts: what the segments in front of segments 1 .. add -> the states in front of segments 0 .., in place
__global__ __launch_bounds__(256) void linear_scan_kernel(LaArgs a, int elements) {
  const int walk = static_cast<int>(blockIdx.z), bh = static_cast<int>(blockIdx.x), b = bh / a.heads;
  const LaWalk& w = a.walk[walk];
  const int at = (static_cast<int>(blockIdx.y) * 256 + static_cast<int>(threadIdx.x)) * 4, n = la_length(a, b);
  const float l2 = la_decay(a.log_decay, bh % a.heads) * FA_LOG2E;
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  if (w.state_in != nullptr) {
    load_pack<float, 4>(w.state_in + static_cast<int64_t>(bh) * elements + at, s);
#pragma unroll
    for (int j = 0; j < 4; ++j) s[j] *= w.mul_in;
  }
  float* p = w.parts + static_cast<int64_t>(bh) * a.segments * elements + at;
  if (w.state_in != nullptr) store_pack<float, 4>(p, s);        // (the walk may write its last state over the one given)
  // eight segments at a time: their loads do not wait for the stores between them (64 segments of one head: with the events around them 20.5 -> 10.7 us)
  constexpr int AHEAD = 8;
  for (int i0 = 0; i0 < a.segments - 1; i0 += AHEAD) {
    float v[AHEAD][4];
#pragma unroll
    for (int i = 0; i < AHEAD; ++i)
      load_pack<float, 4>(p + static_cast<int64_t>(min(i0 + i, a.segments - 2) + 1) * elements, v[i]);
#pragma unroll
    for (int i = 0; i < AHEAD; ++i) {
      if (i0 + i >= a.segments - 1) break;
      const float keep = __builtin_amdgcn_exp2f(static_cast<float>(min(max(n - (i0 + i) * a.segment, 0), a.segment)) * l2);
#pragma unroll
      for (int j = 0; j < 4; ++j) s[j] = s[j] * keep + v[i][j];
      store_pack<float, 4>(p + static_cast<int64_t>(i0 + i + 1) * elements, s);
    }
  }
}

// ------------------------------------------------------------------------------------------------------------ recurrence
struct LaStep {
  LaView q, k, v, o;
  const float *log_decay, *in;
  float* out;
  const int32_t* counts;
  int len, heads;
  float scale;
};

// COLS columns of the state of one head, 4 columns and D COLS / 1024 rows a thread: every byte of the state once in and once out, in
// 32 bits throughout, whatever the number of positions. Bound by memory: 128 x 32 heads of 128, 104 us for 537 MB, 5.2 TB/s; half a
// head a block, so that a beam's few heads have twice the blocks (5 x 8 heads of 64: 3.7 us).
template <typename T, int D, int COLS>
__global__ __launch_bounds__(256) void linear_step_kernel(LaStep a) {
  constexpr int LANES = COLS / 4, GROUPS = 256 / LANES, ROWS = D / GROUPS;
  __shared__ float sums[2][4][COLS];
  const int bh = static_cast<int>(blockIdx.x), b = bh / a.heads, h = bh % a.heads;
  const int lane = static_cast<int>(threadIdx.x) & 63, wave = static_cast<int>(threadIdx.x) >> 6;
  const int group = static_cast<int>(threadIdx.x) / LANES, c = static_cast<int>(threadIdx.x) % LANES * 4, col = static_cast<int>(blockIdx.y) * COLS + c;
  const int n = a.counts != nullptr ? min(max(a.counts[b], 0), a.len) : a.len;
  const int64_t at = static_cast<int64_t>(bh) * (D * D) + static_cast<int64_t>(group) * ROWS * D + col;
  float s[ROWS][4];
#pragma unroll
  for (int i = 0; i < ROWS; ++i) {
    s[i][0] = s[i][1] = s[i][2] = s[i][3] = 0.f;
    if (a.in != nullptr) load_pack<float, 4>(a.in + at + i * D, s[i]);
  }
  const float keep = expf(la_decay(a.log_decay, h));
  const T *q = la_head<T>(a.q, b, h) + group * ROWS, *k = la_head<T>(a.k, b, h) + group * ROWS, *v = la_head<T>(a.v, b, h) + col;
  T* out = const_cast<T*>(la_head<T>(a.o, b, h)) + col;
  for (int t = 0; t < n; ++t) {
    float qf[ROWS], kf[ROWS], vf[4], o[4] = {0.f, 0.f, 0.f, 0.f};
    load_pack<T, ROWS>(q + static_cast<int64_t>(t) * a.q.st, qf);
    load_pack<T, ROWS>(k + static_cast<int64_t>(t) * a.k.st, kf);
    load_pack<T, 4>(v + static_cast<int64_t>(t) * a.v.st, vf);
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        s[i][j] = s[i][j] * keep + kf[i] * vf[j];
        o[j] += qf[i] * s[i][j];
      }
#pragma unroll
    for (int m = LANES; m < 64; m *= 2)
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] += __shfl_xor(o[j], m);
    if (lane < LANES) {
#pragma unroll
      for (int j = 0; j < 4; ++j) sums[t & 1][wave][c + j] = o[j];
    }
    __syncthreads();                                            // (two buffers: the next position's sums do not wait for this one's readers)
    if (threadIdx.x < LANES) {
#pragma unroll
      for (int j = 0; j < 4; ++j) o[j] = a.scale * ((sums[t & 1][0][c + j] + sums[t & 1][1][c + j]) + (sums[t & 1][2][c + j] + sums[t & 1][3][c + j]));
      store_pack<T, 4>(out + static_cast<int64_t>(t) * a.o.st, o);
    }
  }
  if (threadIdx.x < LANES) {
    const float none[4] = {0.f, 0.f, 0.f, 0.f};
    for (int t = n; t < a.len; ++t) store_pack<T, 4>(out + static_cast<int64_t>(t) * a.o.st, none);
  }
#pragma unroll
  for (int i = 0; i < ROWS; ++i) store_pack<float, 4>(a.out + at + i * D, s[i]);
}

// ---------------------------------------------------------------------------------------------------------------- host
// How sequences are split. Segments of a sequence run side by side, at the price of a pass that finds what each adds to the state and of
// states in memory: as many as give two blocks of 256 threads to a compute unit, or three of 128, and at least eight chunks each. us, forward
// and backward, head dimension 128: 16384 positions of 32 heads (forward) 302 in 4 segments, 186 in 8, 187 in 16, 221 in 32; 2 x 8192 of 32
// heads 772 whole, 595 in 4, 634 in 8, 718 in 16 (before the forward's states were kept; 625, 611 and 676 with them); head dimension 64:
// 8 x 2048 of 16 heads 166 whole, 127 in 4, 127 in 6, 137 in 8; one head of 16384 92 in 32, 85 in 64. Short sequences stay whole: 13 x 509
// of 8 heads of 64 take 64 us whole and 71 in 3, 4 x 900 of 8 heads of 128 90 whole and 79 in 3.
// folded: heads of 64 add up to seven states in front of their segment themselves (122 -> 117 us for 8 x 2048), which costs those of 128,
// with states four times as large, more than the scan (603 -> 636).
struct LaPlan {
  int segments, segment;
  bool folded;
  LaPlan(int64_t len, int64_t heads, int64_t head_dim) {
    const int64_t chunks = (len + LA_CHUNK - 1) / LA_CHUNK, fill = head_dim == 128 ? 512 : 768;
    int64_t want = chunks < 24 ? 1 : std::max<int64_t>(1, std::min(fill / std::max<int64_t>(1, heads), chunks / 8));
    const int64_t each = std::max<int64_t>(1, (chunks + want - 1) / want);
    segment = static_cast<int>(each * LA_CHUNK);
    segments = static_cast<int>(std::max<int64_t>(1, (chunks + each - 1) / each));
    folded = head_dim == 64 && segments <= 8;
  }
  int64_t floats(int64_t heads, int64_t head_dim) const { return segments > 1 ? segments * heads * head_dim * head_dim : 0; }
};

int la_check(const char* what, int64_t len, int64_t batch, int64_t heads, int64_t head_dim, float scale, int dtype) {
  NMTG_REQUIRE(len >= 0 && batch >= 0 && heads >= 1, "%s: bad shape len=%lld batch=%lld heads=%lld", what, (long long)len, (long long)batch, (long long)heads);
  NMTG_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head dimension %lld (64 and 128 are built)", what, (long long)head_dim);
  NMTG_REQUIRE(dtype == NMTG_F16 || dtype == NMTG_BF16, "%s: fp16 or bf16 tensors required (matrix-core kernel)", what);
  const float size = scale < 0.f ? -scale : scale;
  NMTG_REQUIRE(size >= 1e-6f && size <= 1e6f, "%s: scale %g (1e-6 to 1e6 in magnitude)", what, (double)scale);
  NMTG_REQUIRE(len <= (1 << 24) && heads <= (1 << 22) && batch <= (1 << 22) && batch * heads <= (1 << 22), "%s: more than 2^24 positions, or 2^22 heads of sequences",
               what);
  return 0;
}
int la_views(const char* what, LaView* views, const void* const* pointers, const int64_t* strides, int count, int64_t len) {
  for (int i = 0; i < count; ++i) {
    const int64_t s[3] = {len == 1 ? 0 : strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]};
    NMTG_REQUIRE(pointers[i] != nullptr, "%s: null pointer argument", what);
    NMTG_REQUIRE(aligned16(pointers[i]) && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0 && s[0] >= 0 && s[1] >= 0 && s[2] >= 0 && s[0] < (1 << 24),
                 "%s: every tensor must be a 16-byte aligned [len, batch, heads, head_dim] view with a contiguous head_dim and strides that are "
                 "multiples of 8 elements (position stride below 2^24)", what);
    views[i] = {pointers[i], s[0], s[1], s[2]};
  }
  return 0;
}
int la_states(const char* what, const float* in, const float* out, bool may_be_one, int64_t floats) {
  NMTG_REQUIRE(aligned16(in) && aligned16(out), "%s: states must be 16-byte aligned", what);
  const bool apart = in == nullptr || out == nullptr || in + floats <= out || out + floats <= in;
  NMTG_REQUIRE(apart || (may_be_one && in == out), "%s: the states overlap", what);
  return 0;
}

template <typename T, int D, bool OUT>
int la_walk(const LaArgs& a, hipStream_t st, const char* what) {
  constexpr int lds = 2 * (OUT ? 3 : 2) * LA_CHUNK * D * 2;
  const int64_t blocks = static_cast<int64_t>(a.batch) * a.heads * (OUT ? a.segments : a.segments - 1) * a.walks;
  if (blocks > (1 << 24) - 1) return fail(NMTG_ERR_UNSUPPORTED, "%s: too many blocks in one launch", what);
  TraceScope trace(what, st);
  hipLaunchKernelGGL((linear_walk_kernel<T, D, OUT>), dim3(static_cast<unsigned>(blocks)), dim3(2 * D), lds, st, a);
  return 0;
}
int la_scan(const LaArgs& a, int d, hipStream_t st, const char* what) {
  TraceScope trace(what, st);
  hipLaunchKernelGGL(linear_scan_kernel, dim3(static_cast<unsigned>(a.batch * a.heads), static_cast<unsigned>(d * d / 1024), static_cast<unsigned>(a.walks)), dim3(256), 0,
                     st, a, d * d);
  return 0;
}
template <typename T, int D>
int la_forward(const LaArgs& a, hipStream_t st) {
  if (a.segments > 1) {
    if (int rc = la_walk<T, D, false>(a, st, "linear_attn_fwd_states")) return rc;
    if (!a.folded) {
      if (int rc = la_scan(a, D, st, "linear_attn_fwd_scan")) return rc;
    }
  }
  return la_walk<T, D, true>(a, st, "linear_attn_fwd");
}
template <typename T, int D>
int la_backward(const LaArgs& a, const LaArgs& states, hipStream_t st) {
  if (a.segments > 1) {
    if (int rc = la_walk<T, D, false>(states, st, "linear_attn_bwd_states")) return rc;
    if (!a.folded) {
      if (int rc = la_scan(states, D, st, "linear_attn_bwd_scan")) return rc;
    }
  }
  return la_walk<T, D, true>(a, st, "linear_attn_bwd");
}
template <typename T>
int la_step(const LaStep& a, int64_t heads, int64_t head_dim, hipStream_t st) {
  TraceScope trace("linear_attn_step", st);
  const unsigned blocks = static_cast<unsigned>(heads);
  if (head_dim == 64) hipLaunchKernelGGL((linear_step_kernel<T, 64, 32>), dim3(blocks, 2), dim3(256), 0, st, a);
  else hipLaunchKernelGGL((linear_step_kernel<T, 128, 64>), dim3(blocks, 2), dim3(256), 0, st, a);
  return 0;
}
#define LA_DISPATCH(call) (dtype == NMTG_F16 ? (head_dim == 64 ? call<f16_t, 64> : call<f16_t, 128>) : (head_dim == 64 ? call<bf16_t, 64> : call<bf16_t, 128>))

}  // namespace
}  // namespace nmtg

using namespace nmtg;

extern "C" int64_t nmtg_linear_attn_fwd_workspace_bytes(int64_t len, int64_t batch, int64_t heads, int64_t head_dim) {
  if (len <= 0 || batch <= 0 || heads <= 0 || head_dim <= 0) return 0;
  return LaPlan(len, batch * heads, head_dim).floats(batch * heads, head_dim) * static_cast<int64_t>(sizeof(float));
}

extern "C" int nmtg_linear_attn_fwd(const void* q, const void* k, const void* v, void* out, const float* log_decay, const int32_t* lengths,
                                    const float* state_in, float* state_out, const int64_t* strides, int64_t len, int64_t batch, int64_t heads,
                                    int64_t head_dim, float scale, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "linear_attn_fwd";
  if (int rc = la_check(what, len, batch, heads, head_dim, scale, dtype)) return rc;
  if (batch == 0 || (len == 0 && state_out == nullptr)) return 0;
  NMTG_REQUIRE(log_decay && strides, "%s: null pointer argument", what);
  if (int rc = la_states(what, state_in, state_out, true, batch * heads * head_dim * head_dim)) return rc;
  const LaPlan plan(len, batch * heads, head_dim);
  NMTG_REQUIRE(plan.segments == 1 || (workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 256 == 0 &&
                                      workspace_bytes >= nmtg_linear_attn_fwd_workspace_bytes(len, batch, heads, head_dim)),
               "%s: a 256-byte aligned workspace of nmtg_linear_attn_fwd_workspace_bytes bytes required", what);
  LaView views[4] = {};
  const void* pointers[4] = {q, k, v, out};
  if (len > 0) {
    if (int rc = la_views(what, views, pointers, strides, 4, len)) return rc;
  }
  LaArgs a = {};
  a.walk[0] = {views[0], views[1], views[2], views[3], state_in, state_out, static_cast<float*>(workspace), 1.f, 1.f, false, false, state_out != nullptr};
  a.walks = 1; a.log_decay = log_decay; a.lengths = lengths; a.len = static_cast<int>(len); a.batch = static_cast<int>(batch); a.heads = static_cast<int>(heads);
  a.segments = plan.segments; a.segment = plan.segment; a.folded = plan.folded; a.scale = scale;
  if (int rc = LA_DISPATCH(la_forward)(a, static_cast<hipStream_t>(stream))) return rc;
  NMTG_CHECK_LAUNCH(what);
  return 0;
}

extern "C" int64_t nmtg_linear_attn_bwd_workspace_bytes(int64_t len, int64_t batch, int64_t heads, int64_t head_dim) {
  if (len <= 0 || batch <= 0 || heads <= 0 || head_dim <= 0) return 0;
  return nmtg_linear_attn_fwd_workspace_bytes(len, batch, heads, head_dim);
}

extern "C" int nmtg_linear_attn_bwd(const void* dout, const void* q, const void* k, const void* v, void* dq, void* dk, void* dv, const float* log_decay,
                                    const int32_t* lengths, const float* state_in, const float* states, const float* dstate_out, float* dstate_in, const int64_t* strides,
                                    int64_t len, int64_t batch, int64_t heads, int64_t head_dim, float scale, int dtype, void* workspace,
                                    int64_t workspace_bytes, void* stream) {
  const char* what = "linear_attn_bwd";
  if (int rc = la_check(what, len, batch, heads, head_dim, scale, dtype)) return rc;
  if (batch == 0 || (len == 0 && dstate_in == nullptr)) return 0;
  NMTG_REQUIRE(log_decay && strides, "%s: null pointer argument", what);
  const int64_t all = batch * heads;
  if (int rc = la_states(what, dstate_out, dstate_in, false, all * head_dim * head_dim)) return rc;
  if (int rc = la_states(what, state_in, dstate_in, false, all * head_dim * head_dim)) return rc;
  const LaPlan plan(len, all, head_dim);
  NMTG_REQUIRE(plan.segments == 1 || (workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 256 == 0 &&
                                      workspace_bytes >= nmtg_linear_attn_bwd_workspace_bytes(len, batch, heads, head_dim)),
               "%s: a 256-byte aligned workspace of nmtg_linear_attn_bwd_workspace_bytes bytes required", what);
  NMTG_REQUIRE(plan.segments == 1 || (states != nullptr && aligned16(states)), "%s: the states that the forward left in its workspace required", what);
  LaView views[7] = {};
  const void* pointers[7] = {dout, q, k, v, dq, dk, dv};
  if (len > 0) {
    if (int rc = la_views(what, views, pointers, strides, 7, len)) return rc;
  }
  const LaView &vg = views[0], &vq = views[1], &vk = views[2], &vv = views[3];
  float *s_parts = const_cast<float*>(states), *r_parts = static_cast<float*>(workspace);
  LaArgs a = {};
  a.log_decay = log_decay; a.lengths = lengths; a.len = static_cast<int>(len); a.batch = static_cast<int>(batch); a.heads = static_cast<int>(heads);
  a.segments = plan.segments; a.segment = plan.segment; a.folded = plan.folded; a.scale = scale;
  LaArgs r = a;
  r.walks = 1;
  r.walk[0] = {vk, vq, vg, vv, dstate_out, nullptr, r_parts, 1.f / scale, scale, true, false, dstate_in != nullptr};
  a.walks = 3;
  a.walk[0] = {vg, vv, vk, views[4], state_in, nullptr, s_parts, 1.f, 1.f, false, true, false};
  a.walk[1] = {vv, vg, vq, views[5], dstate_out, nullptr, r_parts, 1.f / scale, 1.f, true, true, false};
  a.walk[2] = {vk, vq, vg, views[6], dstate_out, dstate_in, r_parts, 1.f / scale, scale, true, false, dstate_in != nullptr};
  if (int rc = LA_DISPATCH(la_backward)(a, r, static_cast<hipStream_t>(stream))) return rc;
  NMTG_CHECK_LAUNCH(what);
  return 0;
}

extern "C" int nmtg_linear_attn_step(const void* q, const void* k, const void* v, void* out, const float* log_decay, const int32_t* counts,
                                     const float* state_in, float* state_out, const int64_t* strides, int64_t len, int64_t batch, int64_t heads,
                                     int64_t head_dim, float scale, int dtype, void* stream) {
  const char* what = "linear_attn_step";
  if (int rc = la_check(what, len, batch, heads, head_dim, scale, dtype)) return rc;
  if (batch == 0) return 0;
  NMTG_REQUIRE(log_decay && strides && state_out, "%s: null pointer argument", what);
  if (int rc = la_states(what, state_in, state_out, true, batch * heads * head_dim * head_dim)) return rc;
  LaView views[4] = {};
  const void* pointers[4] = {q, k, v, out};
  if (len > 0) {
    if (int rc = la_views(what, views, pointers, strides, 4, len)) return rc;
  }
  const LaStep a = {views[0], views[1], views[2], views[3], log_decay, state_in, state_out, counts, static_cast<int>(len), static_cast<int>(heads), scale};
  hipStream_t st = static_cast<hipStream_t>(stream);
  if (int rc = dtype == NMTG_F16 ? la_step<f16_t>(a, batch * heads, head_dim, st) : la_step<bf16_t>(a, batch * heads, head_dim, st)) return rc;
  NMTG_CHECK_LAUNCH(what);
  return 0;
}
