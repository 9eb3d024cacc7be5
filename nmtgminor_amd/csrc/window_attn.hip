// Attention with a sliding window and a few first tokens that stay visible (sinks), forward and backward: query i of a
// sequence sees key j where j <= i and (j > i - window or j < sinks). Work and memory grow with len * (window + sinks); there
// is no mask tensor. Query heads may share a key / value head (heads = group * kv_heads), sequences may end early (lengths):
// positions behind the end see nothing and are seen by nobody, their outputs and gradients are zeros.
//
//   forward     O_i = sum_j P_ij V_j,  P_ij = exp(s_ij - lse_i),  s_ij = scale Q_i . K_j
//   backward    D_i = dO_i . O_i,  dS = P (dP - D),  dP_ij = dO_i . V_j
//               dQ = scale dS K,  dK = scale dS^T Q,  dV = P^T dO   (dK, dV summed over the heads of a group)
//
// The tiling is that of the other tiled attention kernels (flash_tile.hip.h): scores as S^T = K Q^T on 32 x 32 x 16 products,
// one query per lane pair and 32 keys in a lane's registers, so that the softmax's maximum and sum are scalars of a lane;
// probabilities go from accumulators into operands with two lane exchanges per 16 keys. A block visits the tiles that hold
// sinks, then the tiles from its first query's window to its last query. What is different here:
//   - Tiles go from memory straight into LDS (no registers in between), one tile ahead.
//   - A tile lies in LDS once and is read both by rows and transposed: the 16-byte chunks of row r change places by an
//     exclusive-or with img_swizzle(r), under which both kinds of reads spread over all 64 banks (without conflicts; those
//     counted, 1 to 5% of the LDS cycles, are the output patches').
//   - A wavefront that sees nothing of a tile skips it; masks are computed only where a tile crosses an edge.
// Backward in two kernels of three and four products, seven where one kernel would do five: summing dQ over the blocks of keys, or dK
// and dV over those of queries, takes atomics, whose order changes results, or a [blocks, len, head_dim] tensor in 32 bits.
//
// Rounding. Scores, the softmax's statistics, D and all sums are in 32 bits. P and dS are rounded to the tensors' type, which the
// products take: about as much error as rounding the result adds, so that gradients are off by 1.4 times what sums in 32 bits
// rounded once are. D is that of O before its rounding: the forward of a training step leaves what the rounding took in 8 bits
// per element, a byte each that is kept until then. That takes 2.0 to 2.2% of the time of forward and backward; without it gradients of values
// of unit variance are off by 1.5 times instead of 1.45, and those of values with a large common part by up to thirty times as much.
// Exponents are differences of products in 32 bits, the backward's also of the kept logarithm: off by 2^-23 of a score, so that scores beyond
// 10^4 or so in magnitude cost more than the roundings above.
//
// What bounds them (MI355X; shares of the cycles in which a compute unit is busy). Head dimension 128: the matrix cores, busy 46 to 57%, at the
// 1.9 to 2.1 GHz that the power limit leaves: one kernel's time shrinks when another of the step waits more. Forward over 16384 positions,
// window 4096, 32 heads: 925 us, 1.04 PFLOP/s (a large library product: 1.43). Head dimension 64, 8 x 2048 positions, window 512, 16
// heads, a pass of 228 us: forward and dQ the vector instructions, 70 and 61% beside 32 and 37% of products (6.7 and 7.9 per score
// that is computed, masks and the blocks' beginnings and ends among them; a score is half the products of head dimension 128). dK and dV
// wait: 46% of the wavefronts' cycles, with the vector units at 42%, the matrix cores at 35 and the LDS at 29. Operands are read in front of
// their products: four reads ahead take 16 registers, of which three wavefronts on a SIMD leave 6. 61, 73 and 99 us where counters ran.
// No atomics, and what blocks leave to be added up is added in a fixed order: results do not depend on scheduling.
#include "flash_tile.hip.h"
#include <algorithm>

namespace nmtg {
namespace {

constexpr int WA_WAVES = 4, WA_ROWS = 32 * WA_WAVES;   // of a block: 128 queries (forward, dQ) or keys (dK, dV), 32 per wavefront

// Consecutive blocks of a launch go round the eight XCDs, each with an L2 of its own: item i of `total` in launch order, re-counted so
// that every XCD gets a contiguous piece, in which blocks that read the same keys and values are neighbours.
__device__ __forceinline__ uint32_t xcd_item(uint32_t i, uint32_t total) {
  const uint32_t xcd = i & 7, share = total >> 3, more = total & 7;
  return xcd * share + min(xcd, more) + (i >> 3);
}
// Query block x of head h, sequence b. First those with a whole window in front of them, the heads of a group together, then the blocks
// of a sequence; at last the shorter ones, longest first, so that the launch ends evenly (forward, us, before and after: 16384 positions in
// one window 1259 and 1053, 8 x 2048 positions with a window of 512 80 and 71).
struct WaBlock { int x, h, b; };
__device__ __forceinline__ WaBlock query_block(int blocks, int group, int kv_heads, int window) {
  const uint32_t all = gridDim.x / blocks, part = min(blocks, (window + WA_ROWS - 1) / WA_ROWS), whole = all * (blocks - part);
  if (blockIdx.x < whole) {
    const uint32_t id = xcd_item(blockIdx.x, whole), rest = id / group, kv = rest / (blocks - part);
    return {static_cast<int>(part + rest % (blocks - part)), static_cast<int>(kv % kv_heads * group + id % group), static_cast<int>(kv / kv_heads)};
  }
  const uint32_t id = blockIdx.x - whole, head = id % all, kv = head / group;
  return {static_cast<int>(part - 1 - id / all), static_cast<int>(kv % kv_heads * group + head % group), static_cast<int>(kv / kv_heads)};
}

typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
typedef _Float16 f16x2_t __attribute__((ext_vector_type(2)));
typedef short s16x2_t __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4_t __attribute__((ext_vector_type(4)));
typedef float f32x4_t __attribute__((ext_vector_type(4)));

struct WaView { const void* p; int64_t st, sb, sh; };   // [len, batch, heads, head_dim], head_dim contiguous

struct WaArgs {
  WaView q, k, v, o, d_o, dq, dk, dv;
  uint8_t* rest;             // what rounding took from o, or null: see rest_at()
  float* lse;                // [batch, heads, len]
  float* stats;              // backward: [batch, heads][2][stat_rows], log-sum-exp in units of log2 and -D, rows up to a whole block
  int stat_rows;
  const int32_t* lengths;    // [batch] or null: every sequence fills `len`
  int len, batch, heads, kv_heads, group;
  int window, sinks;         // at most len + 1 and len: beyond, nothing changes
  float scale, scale_log2;
  // backward, dK and dV in parts (see DkvPlan): fp32 [parts][batch, kv_heads, part_rows][2][head_dim] of the key blocks, then
  // [chunks][batch, kv_heads, sink_rows][2][head_dim] of the blocks that hold sinks
  float *part, *sink_part;
  int key_blocks, sink_blocks, parts, chunks, part_rows, sink_rows;
};

template <typename T>
__device__ __forceinline__ const T* at_head(const WaView& x, int b, int h) {
  return static_cast<const T*>(x.p) + static_cast<int64_t>(b) * x.sb + static_cast<int64_t>(h) * x.sh;
}
template <typename T>
__device__ __forceinline__ T* out_head(const WaView& x, int b, int h) { return const_cast<T*>(at_head<T>(x, b, h)); }

__device__ __forceinline__ int seq_len(const WaArgs& a, int b) {
  return a.lengths != nullptr ? min(max(a.lengths[b], 0), a.len) : a.len;
}

// ---- what rounding took from O ----
// In 8 bits (E4M3, a sixteenth of it at most is lost again) and units of a power of two per row: 2^-8 (bf16, 2^-11 fp16: half a unit in
// the last place) of the power of two in the row's largest |O| is 256 units, the most that any of its elements lost, so that the conversion,
// which overflows to NaN above 464, cannot. The unit is taken from the rounded O, which the backward reads anyway. Elements below 2^-15 of the
// row's largest lose their rest, of which D would not see anything. A row that is not finite has a D that is not, with a rest or without.
// 32 rows of a head by column chunks of 8, [batch, heads, ceil(len / 32)][head_dim / 8][32][8] bytes, which the accumulators' lanes write
// and the queries' lanes read in whole lines without going through LDS.
template <int D>
__device__ __forceinline__ uint8_t* rest_at(const WaArgs& a, int bh, int row0, int row) {
  return a.rest + ((static_cast<int64_t>(bh) * ((a.len + 31) / 32) + row0 / 32) * (D / 8) * 32 + row) * 8;
}
// the unit of a row whose largest magnitude, rounded, is `largest`. Below fp16's normal range the last place stays where it is, and below
// 2^-110 the unit of bf16 would leave that of 32 bits: the exponents stop there.
template <typename T>
__device__ __forceinline__ float rest_unit(uint32_t largest) {
  constexpr uint32_t UNITS = elem<T>::dtype == NMTG_BF16 ? 16 : 19, LOWEST = elem<T>::dtype == NMTG_BF16 ? 17 : 127 - 14;
  T x;
  x.bits = static_cast<uint16_t>(largest);
  return __uint_as_float((max(__float_as_uint(elem<T>::to_float(x)) >> 23, LOWEST) - UNITS) << 23);
}
__device__ __forceinline__ uint32_t rest_word(const float (&x)[4], float unit) {
  s16x2_t w = {0, 0};
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[0], x[1], unit, false);
  w = __builtin_amdgcn_cvt_scalef32_pk_fp8_f32(w, x[2], x[3], unit, true);
  return __builtin_bit_cast(uint32_t, w);
}
template <typename T, bool HIGH>
__device__ __forceinline__ uint32_t rest_pair(uint32_t word, float unit) {
  if constexpr (elem<T>::dtype == NMTG_BF16) return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(word, unit, HIGH));
  else return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(word, unit, HIGH));
}
// rest . dO of a lane's half row, o the rounded O. fp16 holds the units' numbers, not the units: they come in at the end.
template <typename T, int N>
__device__ __forceinline__ float rest_dot(const uint4 (&o)[N], const uint2 (&rest)[N], const uint4 (&g)[N]) {
  typedef uint16_t u16x2_t __attribute__((ext_vector_type(2)));
  u16x2_t most = {0, 0};                                        // magnitudes of 16-bit floats compare as integers
  const auto look = [&](uint32_t w) __attribute__((always_inline)) { most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2_t, w & 0x7fff7fffu)); };
#pragma unroll
  for (int s = 0; s < N; ++s) { look(o[s].x); look(o[s].y); look(o[s].z); look(o[s].w); }
  uint32_t mine = max(most[0], most[1]), other = mine;
  swap_halves(mine, other);
  const float unit = rest_unit<T>(max(mine, other)), held = elem<T>::dtype == NMTG_BF16 ? unit : 1.f;
  float sum = 0.f;
#pragma unroll
  for (int s = 0; s < N; ++s) {
    sum = dot2<T>(rest_pair<T, false>(rest[s].x, held), g[s].x, dot2<T>(rest_pair<T, true>(rest[s].x, held), g[s].y, sum));
    sum = dot2<T>(rest_pair<T, false>(rest[s].y, held), g[s].z, dot2<T>(rest_pair<T, true>(rest[s].y, held), g[s].w, sum));
  }
  return elem<T>::dtype == NMTG_BF16 ? sum : sum * unit;
}

// ---- the LDS image ----
template <int D>
__device__ __forceinline__ int img_swizzle(int r) { return D == 64 ? (4 * ((r >> 1) & 1) | ((r >> 2) & 3)) : (4 * (r & 3) | ((r >> 2) & 3)); }

// The lane's LDS addresses, which differ between the pieces of an operand by an exclusive-or and a constant: two registers
// instead of one per piece, which the compiler would keep through the loop (per_tile() hides from it that they do not change).
template <typename V>
__device__ __forceinline__ const __attribute__((address_space(3))) V* lds_ptr(uint32_t at) {
  return reinterpret_cast<const __attribute__((address_space(3))) V*>(at);
}
template <int D>
struct ImgReader {
  uint32_t rows, columns;
  // base: LDS address of the images, a multiple of 256
  __device__ __forceinline__ ImgReader(uint32_t base, int lane) {
    const int r = lane & 31, rt = 8 * (lane >> 5) + ((lane >> 2) & 3), ct = 2 * ((lane >> 4) & 1) + ((lane >> 1) & 1);
    rows = base + static_cast<uint32_t>(r * (2 * D) + ((lane >> 5) ^ img_swizzle<D>(r)) * 16);
    columns = base + static_cast<uint32_t>(rt * (2 * D) + (ct ^ img_swizzle<D>(rt)) * 16 + (lane & 1) * 8);
  }
  // the same `offset` bytes on (a multiple of 256)
  __device__ __forceinline__ ImgReader at(int offset) const {
    ImgReader r = *this;
    r.rows += static_cast<uint32_t>(offset);
    r.columns += static_cast<uint32_t>(offset);
    return r;
  }
  __device__ __forceinline__ void per_tile() { asm volatile("" : "+v"(rows), "+v"(columns)); }
  // A operand: rows 32 i + (lane & 31), columns 16 s + 8 (lane >> 5) .. + 7 of the image at `img`
  __device__ __forceinline__ uint4 row_operand(int img, int i, int s) const {
    const u32x4_t v = *lds_ptr<u32x4_t>((rows ^ static_cast<uint32_t>(32 * s)) + static_cast<uint32_t>(img + 32 * i * 2 * D));
    return make_uint4(v[0], v[1], v[2], v[3]);
  }
  // A operand of the transposed image: columns 32 i + (lane & 31), rows 16 kk + 8 (lane >> 5) .. + 7
  __device__ __forceinline__ uint4 column_operand(int img, int i, int kk) const {
    const uint32_t at = columns ^ static_cast<uint32_t>(64 * i), off = static_cast<uint32_t>(img + 16 * kk * 2 * D);
    const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16(const_cast<__attribute__((address_space(3))) s16x4_t*>(lds_ptr<s16x4_t>(at + off)));
    const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16(const_cast<__attribute__((address_space(3))) s16x4_t*>(lds_ptr<s16x4_t>((at ^ 16u) + (off + 4 * 2 * D))));
    union { s16x4_t s[2]; uint4 u; } cv;
    cv.s[0] = lo;
    cv.s[1] = hi;
    return cv.u;
  }
};

// Lane l copies the 4 bytes at sbase + voff(l) to LDS address lds_addr + 4 l (dma16's sibling).
__device__ __forceinline__ void dma4(uint32_t voff, const void* sbase, uint32_t lds_addr) {
  asm volatile("s_mov_b32 m0, %2\n\ts_nop 0\n\tglobal_load_lds_dword %0, %1"
               :
               : "v"(voff), "s"(sbase), "s"(lds_addr)
               : "memory", "m0");
}

// Transfers of one tile of ROWS rows into an image, shared out over the block's wavefronts: lane l of transfer n fills chunk
// 64 n + l. Rows behind `last` are read as row `last` (in bounds, finite where the sequence is; they are masked by the caller).
template <typename T, int D, int ROWS = FA_TILE>
struct TileLoader {
  static constexpr int CH = D / 8, N = ROWS * CH / 64 / WA_WAVES;
  uint32_t voff[N];
  int wave, lane;
  __device__ __forceinline__ TileLoader(int64_t stride_t, int wave_, int lane_) : wave(wave_), lane(lane_) {
#pragma unroll
    for (int n = 0; n < N; ++n) {
      const int id = 64 * (wave * N + n) + lane, r = id / CH, c = (id % CH) ^ img_swizzle<D>(r);
      voff[n] = static_cast<uint32_t>(r * stride_t * 2 + c * 16);
    }
  }
  __device__ __forceinline__ void start(const T* head, int64_t stride_t, int first, int last, uint32_t img) const {
    const T* base = head + static_cast<int64_t>(first) * stride_t;
    const uint32_t to = img + static_cast<uint32_t>(wave * N * 1024);
    if (first + ROWS - 1 <= last) {
#pragma unroll
      for (int n = 0; n < N; ++n) dma16(voff[n], base, to + 1024 * n);
    } else {
#pragma unroll
      for (int n = 0; n < N; ++n) {
        const int id = 64 * (wave * N + n) + lane, behind = first + id / CH - last;
        dma16(voff[n] - static_cast<uint32_t>(max(behind, 0) * stride_t * 2), base, to + 1024 * n);
      }
    }
  }
};

// visit(i, buffer) for i from i0 to i1, the two buffers in turn: constants, so that LDS addresses need no arithmetic per tile.
template <typename F>
__device__ __forceinline__ void in_turn(int i0, int i1, const F& visit) {
  for (int i = i0; i < i1; i += 2) {
    visit(i, std::integral_constant<int, 0>{});
    if (i + 1 < i1) visit(i + 1, std::integral_constant<int, 1>{});
  }
}

// The next tile's transfers have landed for the whole block, and the block's reads of the tile before are done. (Transfers two
// tiles ahead, into three buffers, gained nothing: LDS for fewer blocks on a compute unit cost as much as the longer lead gave.)
__device__ __forceinline__ void next_tile() {
  wait_vmcnt<0>();
  ring_barrier();
}

// the tiles of a block whose queries are first .. last: those of the sinks, then those from the first query's window on
template <int TILE = FA_TILE>
struct TileList {
  int sinks, lo, count;
  __device__ __forceinline__ TileList(const WaArgs& a, int first, int end) {
    const int tiles = (end + TILE - 1) / TILE;
    lo = min(max(first - a.window + 1, 0) / TILE, tiles);
    sinks = min((min(a.sinks, end) + TILE - 1) / TILE, lo);
    count = sinks + tiles - lo;
  }
  __device__ __forceinline__ int operator[](int i) const { return i < sinks ? i : i - sinks + lo; }
};

// Whether queries first .. last of a sequence of n see nothing, or do not see everything, of the tile of keys from k0 on.
template <int TILE = FA_TILE>
__device__ __forceinline__ bool nothing_seen(const WaArgs& a, int n, int first, int last, int k0) {
  return k0 > last || first >= n || (k0 + TILE - 1 <= first - a.window && k0 >= a.sinks);
}
template <int TILE = FA_TILE>
__device__ __forceinline__ bool some_hidden(const WaArgs& a, int n, int first, int last, int k0) {
  return k0 + TILE - 1 > first || last >= n || (k0 <= last - a.window && k0 + TILE > a.sinks);
}

// Scores of the queries first .. first + 31 (one a lane pair, qrow) against the 32 keys from k0 on, 8 (r / 4) + r % 4 + 4 half in
// register r: those that a query does not see become `hidden`, the infinity that the scale turns negative, whose probability is zero.
// Most tiles at an edge are at one of them, so that each edge is a pass of its own: a comparison and a select per score.
__device__ __forceinline__ void hide_keys(acc16_t& s, const WaArgs& a, int n, int first, int qrow, int half, int k0, float hidden) {
  asm volatile("" : "+v"(qrow), "+v"(half));                   // so that no bounds are kept in registers through the loops
  const int key0 = k0 + 4 * half;
  if (k0 + 31 > first || first + 31 >= n) {                    // the diagonal, or the end of the sequence
    const int to = (qrow < n ? qrow : -1) - key0;
#pragma unroll
    for (int r = 0; r < 16; ++r) s[r] = 8 * (r / 4) + r % 4 > to ? hidden : s[r];
  }
  if (k0 <= first + 31 - a.window && k0 + 31 >= a.sinks) {     // keys up to `from` are in front of the window
    const int from = qrow - a.window - key0, sinks = a.sinks - key0;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      const int key = 8 * (r / 4) + r % 4;
      s[r] = (key <= from) & (key >= sinks) ? hidden : s[r];    // (a short-circuit test became a branch per element)
    }
  }
}

// ------------------------------------------------------------------------------------------------------------- forward
constexpr float WA_FLOOR = -5e29f;   // a running maximum before the first visible key: finite, and far above the -inf of hidden ones

// Key tiles of 64, or of 32 for head_dim 128: with the scores of 32 keys a wavefront needs at most 168 registers there, and three of them
// share a SIMD (32 KB of LDS a block). What bounds the kernel is how much of the softmax runs under other wavefronts' products:
// prompt of 16384 positions, window 4096, 32 heads of 128: 1088 us with two wavefronts and tiles of 64, 1023 with three, 925 as it is. (For
// head_dim 64 tiles of 32 keys take as long as tiles of 64.)
template <int D> constexpr int fwd_tile() { return D == 64 ? 64 : 32; }

template <typename T, int D>
__global__ __launch_bounds__(64 * WA_WAVES, 3) void window_fwd_kernel(WaArgs a) {
  extern __shared__ __align__(256) uint8_t lds_raw[];
  constexpr int TILE = fwd_tile<D>(), IMG = TILE * D * 2;
  const WaBlock block = query_block((a.len + WA_ROWS - 1) / WA_ROWS, a.group, a.kv_heads, a.window);
  const int b = block.b, h = block.h, q0 = block.x * WA_ROWS;
  const int lane = static_cast<int>(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6), half = lane >> 5;
  const int n = seq_len(a, b), bh = b * a.heads + h;
  const int end = min(q0 + WA_ROWS, n), qw = q0 + 32 * wave, qrow = qw + (lane & 31);
  const T *kb = at_head<T>(a.k, b, h / a.group), *vb = at_head<T>(a.v, b, h / a.group);

  const TileList<TILE> tiles(a, q0, end > q0 ? end : 0);
  const int count = end > q0 ? tiles.count : 0;
  const TileLoader<T, D, TILE> ldk(a.k.st, wave, lane), ldv(a.v.st, wave, lane);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds_raw)));
  const ImgReader<D> reader(lds0, lane);
  auto start = [&](int i, int buffer) {
    const int row = tiles[i] * TILE;
    const uint32_t to = lds0 + static_cast<uint32_t>(buffer) * 2 * IMG;
    ldk.start(kb, a.k.st, row, n - 1, to);
    ldv.start(vb, a.v.st, row, n - 1, to + IMG);
  };
  if (count > 0) start(0, 0);                                    // before the queries: the two latencies are one
  uint4 qf[D / 16];
  load_resident<T, D>(qf, at_head<T>(a.q, b, h), a.q.st, qrow, n, lane);
  acc16_t o[D / 32];
  float m = WA_FLOOR, l = 0.f;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) o[i][r] = 0.f;
  registers_landed(qf);
  const int first = qw, last = qw + 31;                         // the wavefront's queries
  const float hidden = a.scale_log2 >= 0.f ? -INFINITY : INFINITY;
  constexpr uint32_t ONES = elem<T>::dtype == NMTG_BF16 ? 0x3f803f80u : 0x3c003c00u;
  const auto visit = [&](int i, auto buffer) __attribute__((always_inline)) {
    const int k0 = tiles[i] * TILE;
    next_tile();
    if (i + 1 < count) start(i + 1, 1 - buffer);
    constexpr int kimg = decltype(buffer)::value * 2 * IMG, vimg = kimg + IMG;
    ImgReader<D> img = reader;
    img.per_tile();
    if (nothing_seen<TILE>(a, n, first, last, k0)) return;
    acc16_t s[TILE / 32];
#pragma unroll
    for (int nn = 0; nn < TILE / 32; ++nn)
#pragma unroll
      for (int r = 0; r < 16; ++r) s[nn][r] = 0.f;
    uint4 kf[TILE / 32][D / 16];                                // all read before the first product, which otherwise waits for each in turn
#pragma unroll
    for (int ss = 0; ss < D / 16; ++ss)
#pragma unroll
      for (int nn = 0; nn < TILE / 32; ++nn) kf[nn][ss] = img.row_operand(kimg, nn, ss);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int ss = 0; ss < D / 16; ++ss)
#pragma unroll
      for (int nn = 0; nn < TILE / 32; ++nn) mfma<T>::run(kf[nn][ss], qf[ss], s[nn]);
    if (some_hidden<TILE>(a, n, first, last, k0)) {
#pragma unroll
      for (int nn = 0; nn < TILE / 32; ++nn) hide_keys(s[nn], a, n, first, qrow, half, k0 + 32 * nn, hidden);
    }
    // the tile's maximum from the extreme raw score
    float top = s[0][0];
    if (a.scale_log2 >= 0.f) {
#pragma unroll
      for (int nn = 0; nn < TILE / 32; ++nn)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fmaxf(top, s[nn][r]);
    } else {
#pragma unroll
      for (int nn = 0; nn < TILE / 32; ++nn)
#pragma unroll
        for (int r = 0; r < 16; ++r) top = fminf(top, s[nn][r]);
    }
    const float mx = pair_max(top * a.scale_log2);
    // The reference point follows the maximum lazily: it moves when a row's maximum has grown by more than 2^8, so that
    // probabilities relative to it stay below 256 and most tiles rescale nothing.
    const bool grow = mx > m + FA_LAZY;
    if (__builtin_amdgcn_ballot_w64(grow) != 0) {
      const float m_new = grow ? mx : m;
      const float alpha = fast_exp2(m - m_new);
      m = m_new;
      l *= alpha;
#pragma unroll
      for (int j = 0; j < D / 32; ++j)
#pragma unroll
        for (int r = 0; r < 16; ++r) o[j][r] *= alpha;
    }
#pragma unroll
    for (int kk = 0; kk < TILE / 16; ++kk) {
      float pv[8];
#pragma unroll
      for (int e = 0; e < 8; ++e) pv[e] = fast_exp2(__builtin_fmaf(s[kk / 2][8 * (kk % 2) + e], a.scale_log2, -m));
      const uint4 pf = acc_to_operand<T>(pv);
      // The sum is that of the rounded probabilities: the weights that the values get add up to one, and two of them cost
      // one instruction.
      l = dot2<T>(pf.x, ONES, dot2<T>(pf.y, ONES, dot2<T>(pf.z, ONES, dot2<T>(pf.w, ONES, l))));
#pragma unroll
      for (int j = 0; j < D / 32; ++j) mfma<T>::run(img.column_operand(vimg, j, kk), pf, o[j]);
    }
  };
  in_turn(0, count, visit);
  __syncthreads();                                              // every wavefront is done with the images
  const float sum = pair_sum(l);
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  if (half == 0 && qrow < a.len)
    a.lse[static_cast<int64_t>(bh) * a.len + qrow] = sum > 0.f ? (m + log2f(sum)) * (1.0f / FA_LOG2E) : sum == 0.f ? -INFINITY : sum;
  // O is rounded twice, for the result and for what that takes: both from one product in 32 bits. (Left to itself the compiler rounds the
  // second from the unrounded product, and the rest of a mean that lies between two numbers is then that of the wrong one.)
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) {
      float whole = o[i][r] * inv;
      asm volatile("" : "+v"(whole));
      o[i][r] = whole;
    }
  if (a.rest != nullptr && qw < a.len) {
    uint8_t* to = rest_at<D>(a, bh, qw, lane & 31) + 4 * half;
    float top = 0.f;
#pragma unroll
    for (int i = 0; i < D / 32; ++i)
#pragma unroll
      for (int r = 0; r < 16; ++r) top = fmaxf(top, fabsf(o[i][r]));
    const float unit = rest_unit<T>(elem<T>::from_float(pair_max(top)).bits);
#pragma unroll
    for (int m = 0; m < D / 8; ++m) {
      float x[4];
#pragma unroll
      for (int e = 0; e < 4; ++e) {
        const float whole = o[m / 4][4 * (m % 4) + e];
        x[e] = whole - elem<T>::to_float(elem<T>::from_float(whole));
      }
      *reinterpret_cast<uint32_t*>(to + 256 * m) = rest_word(x, unit);
    }
  }
  store_rows_out<T, D>(o, 1.f, lds_raw + wave * (32 * D * 2), out_head<T>(a.o, b, h), a.o.st, qw, a.len, lane);
}

// ------------------------------------------------------------------------------------ backward: dQ, and D = rowsum(dO O)
// Queries in registers, tiles of 64 keys and values as in the forward. Head dimension 64: four wavefronts on a SIMD (128 registers, none
// spilt), 128: two. 2 x 8192 positions, window 1024, 32 heads of 128: 440 us, 0.9 PFLOP/s of its three products.
template <typename T, int D>
__global__ __launch_bounds__(64 * WA_WAVES, D == 64 ? 4 : 2) void window_bwd_dq_kernel(WaArgs a) {
  extern __shared__ __align__(256) uint8_t lds_raw[];
  constexpr int IMG = FA_TILE * D * 2;
  const WaBlock block = query_block((a.len + WA_ROWS - 1) / WA_ROWS, a.group, a.kv_heads, a.window);
  const int b = block.b, h = block.h, q0 = block.x * WA_ROWS;
  const int lane = static_cast<int>(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6), half = lane >> 5;
  const int n = seq_len(a, b), bh = b * a.heads + h;
  const int end = min(q0 + WA_ROWS, n), qw = q0 + 32 * wave, qrow = qw + (lane & 31);
  const T *kb = at_head<T>(a.k, b, h / a.group), *vb = at_head<T>(a.v, b, h / a.group);

  const TileList<> tiles(a, q0, end > q0 ? end : 0);
  const int count = end > q0 ? tiles.count : 0;
  const TileLoader<T, D> ldk(a.k.st, wave, lane), ldv(a.v.st, wave, lane);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds_raw)));
  const ImgReader<D> reader(lds0, lane);
  auto start = [&](int i) {
    const int row = tiles[i] * FA_TILE;
    const uint32_t to = lds0 + static_cast<uint32_t>(i & 1) * 2 * IMG;
    ldk.start(kb, a.k.st, row, n - 1, to);
    ldv.start(vb, a.v.st, row, n - 1, to + IMG);
  };
  if (count > 0) start(0);
  uint4 qf[D / 16], gf[D / 16];
  load_resident<T, D>(qf, at_head<T>(a.q, b, h), a.q.st, qrow, n, lane);
  load_resident<T, D>(gf, at_head<T>(a.d_o, b, h), a.d_o.st, qrow, n, lane);
  float delta = 0.f, lse2 = -FA_NEG;                            // rows behind the end: probability 0
  {
    uint4 of[D / 16];
    uint2 rf[D / 16];
    load_resident<T, D>(of, at_head<T>(a.o, b, h), a.o.st, qrow, n, lane);
    if (a.rest != nullptr) {
#pragma unroll
      for (int s = 0; s < D / 16; ++s) rf[s] = qrow < n ? *reinterpret_cast<const uint2*>(rest_at<D>(a, bh, qw, lane & 31) + 256 * (2 * s + half)) : make_uint2(0, 0);
    }
    if (qrow < n) {
      const float v = a.lse[static_cast<int64_t>(bh) * a.len + qrow];
      lse2 = v == -INFINITY ? -FA_NEG : v * FA_LOG2E;
    }
#pragma unroll
    for (int s = 0; s < D / 16; ++s) {
      delta = dot2<T>(of[s].x, gf[s].x, dot2<T>(of[s].y, gf[s].y, delta));
      delta = dot2<T>(of[s].z, gf[s].z, dot2<T>(of[s].w, gf[s].w, delta));
    }
    if (a.rest != nullptr) delta += rest_dot<T>(of, rf, gf);
    delta = pair_sum(delta);
    // for the kernel of dK and dV: whole blocks of rows, so that it reads tiles without looking at lengths
    float* to = a.stats + static_cast<int64_t>(bh) * 2 * a.stat_rows + qrow;
    if (half == 0) to[0] = lse2;
    else to[a.stat_rows] = -delta;
  }
  acc16_t dq[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) dq[i][r] = 0.f;
  registers_landed(qf);
  const int first = qw, last = qw + 31;
  const float hidden = a.scale_log2 >= 0.f ? -INFINITY : INFINITY;
  for (int i = 0; i < count; ++i) {
    const int k0 = tiles[i] * FA_TILE;
    next_tile();
    if (i + 1 < count) start(i + 1);
    // 32 keys at a time, so that scores, score gradients and their operands need half the registers; what is not seen is left out.
    // At head dimension 128 the products of dP start from -D, which takes the subtraction out (2%); at 64 there are no registers for
    // that (25 spilt, half as fast again).
#pragma unroll 1
    for (int kn = k0; kn < k0 + FA_TILE; kn += 32) {
      if (nothing_seen<32>(a, n, first, last, kn)) continue;
      const ImgReader<D> img = reader.at((i & 1) * (2 * IMG) + (kn - k0) * (2 * D));
      acc16_t s, dp;
#pragma unroll
      for (int r = 0; r < 16; ++r) { s[r] = 0.f; dp[r] = D == 128 ? -delta : 0.f; }
#pragma unroll
      for (int ss = 0; ss < D / 16; ss += 2) {
        uint4 kf[2], vf[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) { kf[x] = img.row_operand(0, 0, ss + x); vf[x] = img.row_operand(IMG, 0, ss + x); }
        if constexpr (D == 128) __builtin_amdgcn_sched_barrier(0);   // four reads ahead: 4%; at head dimension 64 there are no registers for them
#pragma unroll
        for (int x = 0; x < 2; ++x) {
          mfma<T>::run(kf[x], qf[ss + x], s);
          mfma<T>::run(vf[x], gf[ss + x], dp);
        }
      }
      hide_keys(s, a, n, first, qrow, half, kn, hidden);
#pragma unroll
      for (int r = 0; r < 16; ++r) s[r] = fast_exp2(__builtin_fmaf(s[r], a.scale_log2, -lse2)) * (D == 128 ? dp[r] : dp[r] - delta);
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        float dsv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) dsv[e] = s[8 * kk + e];
        const uint4 df = acc_to_operand<T>(dsv);
#pragma unroll
        for (int j = 0; j < D / 32; ++j) mfma<T>::run(img.column_operand(0, j, kk), df, dq[j]);
      }
    }
  }
  __syncthreads();
  store_rows_out<T, D>(dq, a.scale, lds_raw + wave * (32 * D * 2), out_head<T>(a.dq, b, h), a.dq.st, qw, a.len, lane);
}

// ------------------------------------------------------------------------------------------------- backward: dK and dV
// One key per lane pair: a block holds 128 keys of a key / value head, the queries of every head of its group come in tiles.
// The work is laid out so that blocks are alike (DkvPlan): the queries behind the windows of a block that holds sinks, up to
// the sequence's end, are shared out over `chunks` more blocks, and where the key blocks would not fill the chip each is
// shared out over `parts`. Such blocks leave fp32 sums that a last kernel adds in a fixed order.

// accumulators of the wavefront's 32 rows as fp32 rows of D elements, `pitch` floats apart
template <int D>
__device__ __forceinline__ void store_part(const acc16_t (&acc)[D / 32], float mul, float* base, int64_t pitch, int row0, int rows, int lane) {
  const int half = lane >> 5, row = row0 + (lane & 31);
  if (row >= rows) return;
  float* p = base + static_cast<int64_t>(row) * pitch + 4 * half;
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int g = 0; g < 4; ++g)
      *reinterpret_cast<float4*>(p + 32 * i + 8 * g) = make_float4(acc[i][4 * g] * mul, acc[i][4 * g + 1] * mul, acc[i][4 * g + 2] * mul, acc[i][4 * g + 3] * mul);
}

// Query tiles of 64, or of 32 for head_dim 128: two wavefronts of that size on a SIMD leave 256 registers each, which the
// accumulators of 32 keys half fill, so the keys of a block are read from LDS (32 KB, which the smaller tiles make room for)
// and only the values stay in registers. With both in registers there was one wavefront on a SIMD, and nothing ran
// under the waits of the other: 1.5 times the time. 2 x 8192 positions, window 1024, 32 heads of 128: 565 us, 1.0 PFLOP/s of its products.
template <int D> constexpr int dkv_tile() { return D == 64 ? 64 : 32; }
template <int D> constexpr int dkv_buf() { return 2 * dkv_tile<D>() * D * 2 + 2 * dkv_tile<D>() * 4; }   // Q, dO, lse2, -D
template <int D> constexpr int dkv_keys() { return D == 64 ? 0 : WA_ROWS * D * 2; }

template <typename T, int D>
__global__ __launch_bounds__(64 * WA_WAVES, D == 64 ? 3 : 2) void window_bwd_dkv_kernel(WaArgs a) {
  extern __shared__ __align__(256) uint8_t lds_raw[];
  constexpr int TILE = dkv_tile<D>(), IMG = TILE * D * 2, BUF = dkv_buf<D>();
  constexpr bool KEYS_IN_LDS = dkv_keys<D>() > 0;
  // First the parts of key blocks with a whole window of queries behind them, then those of the shorter blocks, longest first, at last
  // the chunks of queries that see a block's keys as sinks only.
  const uint32_t heads = static_cast<uint32_t>(a.kv_heads) * a.batch, shorter = min(a.key_blocks, (a.window + WA_ROWS - 1) / WA_ROWS);
  const uint32_t whole = (a.key_blocks - shorter) * a.parts, own = a.key_blocks * a.parts;
  const bool sink_chunk = blockIdx.x >= own * heads;
  uint32_t head, block, share, shares = a.parts;
  if (sink_chunk) {
    const uint32_t id = xcd_item(blockIdx.x - own * heads, gridDim.x - own * heads), per_head = a.sink_blocks * a.chunks;
    shares = a.chunks;
    head = id / per_head; block = id % per_head / shares; share = id % per_head % shares;
  } else if (blockIdx.x < whole * heads) {
    const uint32_t id = xcd_item(blockIdx.x, whole * heads);
    head = id / whole; block = id % whole / shares; share = id % whole % shares;
  } else {
    const uint32_t id = blockIdx.x - whole * heads;
    share = id % shares; head = id / shares % heads; block = a.key_blocks - shorter + id / shares / heads;
  }
  const int h = static_cast<int>(head % a.kv_heads), b = static_cast<int>(head / a.kv_heads), k0 = static_cast<int>(block) * WA_ROWS;
  const int lane = static_cast<int>(threadIdx.x) & 63, wave = __builtin_amdgcn_readfirstlane(static_cast<int>(threadIdx.x) >> 6), half = lane >> 5;
  const int n = seq_len(a, b), kw = k0 + 32 * wave, krow = kw + (lane & 31);
  const uint32_t lds0 = __builtin_amdgcn_readfirstlane(static_cast<uint32_t>(reinterpret_cast<uintptr_t>(lds_raw)));
  const ImgReader<D> reader(lds0, lane);
  acc16_t dk[D / 32], dv[D / 32];
#pragma unroll
  for (int i = 0; i < D / 32; ++i)
#pragma unroll
    for (int r = 0; r < 16; ++r) { dk[i][r] = 0.f; dv[i][r] = 0.f; }

  // the query tiles up to the end of the last key's window, and those behind it
  const int tw = (min(k0 + WA_ROWS - 1 + a.window, n) + TILE - 1) / TILE, tn = (n + TILE - 1) / TILE;
  const int t0 = sink_chunk ? tw : k0 / TILE, t1 = sink_chunk ? tn : tw;
  const int per = k0 < n ? t1 - t0 : 0, all = per * a.group;
  // this block's share of the (head, tile) pairs
  const int i0 = static_cast<int>(static_cast<int64_t>(all) * share / static_cast<int>(shares)), i1 = static_cast<int>(static_cast<int64_t>(all) * (share + 1) / static_cast<int>(shares));
  const TileLoader<T, D, TILE> ldq(a.q.st, wave, lane), ldg(a.d_o.st, wave, lane);
  const float hidden = a.scale_log2 >= 0.f ? -INFINITY : INFINITY;
  // Beside a tile's rows, what the backward keeps of its queries: log-sum-exp, -D. Tiles of 64: 64 floats a transfer, by two
  // wavefronts each (the same values); of 32: both in one, by all four.
  const uint32_t stat_off = TILE == 64 ? static_cast<uint32_t>((wave & 1) * a.stat_rows + lane) * 4 : static_cast<uint32_t>((lane >> 5) * a.stat_rows + (lane & 31)) * 4;
  // (head, tile) of the next transfers and of the next products
  struct Cursor { int head, tile; };
  auto advance = [&](Cursor& c) {
    if (++c.tile == t1) { c.tile = t0; ++c.head; }
  };
  Cursor ahead = {h * a.group + (per > 0 ? i0 / per : 0), t0 + (per > 0 ? i0 % per : 0)}, here = ahead;
  auto start = [&](int buffer) {
    const int hq = ahead.head, q0 = ahead.tile * TILE;
    advance(ahead);
    const uint32_t to = lds0 + static_cast<uint32_t>(buffer) * BUF;
    ldq.start(at_head<T>(a.q, b, hq), a.q.st, q0, n - 1, to);
    ldg.start(at_head<T>(a.d_o, b, hq), a.d_o.st, q0, n - 1, to + IMG);
    dma4(stat_off, a.stats + (static_cast<int64_t>(b) * a.heads + hq) * 2 * a.stat_rows + q0, to + 2 * IMG + (TILE == 64 ? (wave & 1) * 256 : 0));
  };
  if (i0 < i1) start(0);
  uint4 kf[KEYS_IN_LDS ? 1 : D / 16], vf[D / 16];
  if constexpr (KEYS_IN_LDS) {
    if (k0 < n) TileLoader<T, D, WA_ROWS>(a.k.st, wave, lane).start(at_head<T>(a.k, b, h), a.k.st, k0, n - 1, lds0 + 2 * BUF);
  } else {
    load_resident<T, D>(kf, at_head<T>(a.k, b, h), a.k.st, krow, n, lane);
  }
  load_resident<T, D>(vf, at_head<T>(a.v, b, h), a.v.st, krow, n, lane);
  wait_vmcnt<0>();      // the resident rows: waited for at their first use, they would be in every tile, behind its transfers
  const auto visit = [&](int i, auto buffer) __attribute__((always_inline)) {
    const int q0 = here.tile * TILE;
    advance(here);
    next_tile();
    if (i + 1 < i1) start(1 - buffer);
    constexpr int qimg = decltype(buffer)::value * BUF, gimg = qimg + IMG, stats = gimg + IMG;
    ImgReader<D> img = reader;
    img.per_tile();
    const int klast = kw + 31;
    // 32 queries at a time, so that scores, their gradients and their operands need half the registers
#pragma unroll
    for (int nn = 0; nn < TILE / 32; ++nn) {
      const int qn = q0 + 32 * nn;
      if (qn + 31 < kw || kw >= n || (qn - a.window >= klast && kw >= a.sinks)) continue;
      acc16_t s, dp;
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int ql = 32 * nn + 8 * g;
        const f32x4_t dl = *lds_ptr<f32x4_t>(lds0 + 16 * half + static_cast<uint32_t>(stats + 4 * (TILE + ql)));
#pragma unroll
        for (int e = 0; e < 4; ++e) { s[4 * g + e] = 0.f; dp[4 * g + e] = dl[e]; }
      }
#pragma unroll
      for (int ss = 0; ss < D / 16; ++ss) {
        uint4 key;
        if constexpr (KEYS_IN_LDS) key = img.row_operand(2 * BUF, wave, ss);
        else key = kf[ss];
        mfma<T>::run(img.row_operand(qimg, nn, ss), key, s);
        mfma<T>::run(img.row_operand(gimg, nn, ss), vf[ss], dp);
      }
      if constexpr (D == 64) __builtin_amdgcn_sched_barrier(0);   // exponentials among the products would need more registers than there are
      // queries that do not see this lane's key: in front of it, or behind its window (a sink has none)
      const int at = qn + 4 * half;
      if (qn < klast || klast >= n) {
        const int from = krow < n ? krow - at : n;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 8 * (r / 4) + r % 4 < from ? hidden : s[r];
      }
      if (qn + 31 - a.window >= kw && klast >= a.sinks) {
        const int to = (krow < a.sinks ? n : min(krow + a.window, n)) - at;
#pragma unroll
        for (int r = 0; r < 16; ++r) s[r] = 8 * (r / 4) + r % 4 >= to ? hidden : s[r];
      }
#pragma unroll
      for (int g = 0; g < 4; ++g) {
        const int ql = 32 * nn + 8 * g + 4 * half;            // first of four consecutive queries, within the tile
        const f32x4_t lse2 = *lds_ptr<f32x4_t>(lds0 + 16 * half + static_cast<uint32_t>(stats + 4 * (ql - 4 * half)));
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const int r = 4 * g + e;
          const float p = fast_exp2(__builtin_fmaf(s[r], a.scale_log2, -lse2[e]));
          s[r] = p * dp[r];
          dp[r] = p;
        }
      }
#pragma unroll
      for (int kk = 0; kk < 2; ++kk) {
        float pv[8], dsv[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) { pv[e] = dp[8 * kk + e]; dsv[e] = s[8 * kk + e]; }
        const uint4 pf = acc_to_operand<T>(pv), df = acc_to_operand<T>(dsv);
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          mfma<T>::run(img.column_operand(gimg, j, 2 * nn + kk), pf, dv[j]);
          mfma<T>::run(img.column_operand(qimg, j, 2 * nn + kk), df, dk[j]);
        }
      }
    }
  };
  in_turn(i0, i1, visit);
  wait_vmcnt<0>();                                              // of a share without a tile: the keys' transfers
  // What is still to be joined: all rows in parts, or those of the sinks, which the join then writes over.
  if (sink_chunk || a.parts > 1 || k0 < a.sink_rows) {
    const int rows = sink_chunk ? a.sink_rows : a.part_rows;
    float* base = (sink_chunk ? a.sink_part : a.part) +
                  ((static_cast<int64_t>(share) * a.batch + b) * a.kv_heads + h) * rows * (2 * D);
    store_part<D>(dk, a.scale, base, 2 * D, kw, rows, lane);
    store_part<D>(dv, 1.f, base + D, 2 * D, kw, rows, lane);
    if (sink_chunk || a.parts > 1) return;
  }
  __syncthreads();
  uint8_t* patch = lds_raw + wave * (32 * D * 2);
  store_rows_out<T, D>(dk, a.scale, patch, out_head<T>(a.dk, b, h), a.dk.st, kw, a.len, lane);
  __syncthreads();
  store_rows_out<T, D>(dv, 1.f, patch, out_head<T>(a.dv, b, h), a.dv.st, kw, a.len, lane);
}

// The sums of the parts, rounded: D / 4 threads per row of keys and as many for its row of values.
template <typename T, int D>
__global__ __launch_bounds__(256) void window_dkv_join_kernel(WaArgs a, int64_t total) {
  const int64_t id = static_cast<int64_t>(blockIdx.x) * 256 + threadIdx.x;
  if (id >= total) return;
  constexpr int CH = 2 * D / 4;
  const int c = static_cast<int>(id % CH), h = static_cast<int>(blockIdx.y), b = static_cast<int>(blockIdx.z);
  const int row = static_cast<int>(id / CH);
  const int64_t bh = static_cast<int64_t>(b) * a.kv_heads + h, bhs = static_cast<int64_t>(gridDim.z) * a.kv_heads;
  float4 sum = make_float4(0.f, 0.f, 0.f, 0.f);
  const auto add = [&](const float* base, int i, int pitch) __attribute__((always_inline)) {
    const float4 v = *reinterpret_cast<const float4*>(base + ((i * bhs + bh) * pitch + row) * (2 * D) + 4 * c);
    sum.x += v.x; sum.y += v.y; sum.z += v.z; sum.w += v.w;
  };
  for (int i = 0; i < a.parts; ++i) add(a.part, i, a.part_rows);
  if (row < a.sink_rows) {
#pragma unroll 8
    for (int i = 0; i < a.chunks; ++i) add(a.sink_part, i, a.sink_rows);   // few threads and many chunks: loads ahead of their sums
  }
  T* out = c < CH / 2 ? out_head<T>(a.dk, b, h) + static_cast<int64_t>(row) * a.dk.st + 4 * c
                      : out_head<T>(a.dv, b, h) + static_cast<int64_t>(row) * a.dv.st + 4 * (c - CH / 2);
  *reinterpret_cast<uint2*>(out) = make_uint2(pack2<T>(sum.x, sum.y), pack2<T>(sum.z, sum.w));
}

// ---------------------------------------------------------------------------------------------------------------- host
constexpr int64_t WA_MOST_BLOCKS = 0xffffffffll / (64 * WA_WAVES);     // a launch holds less than 2^32 threads

int check_call(const char* what, int64_t len, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t window, int64_t sinks,
               float scale, int dtype) {
  NMTG_REQUIRE(len >= 0 && batch >= 0 && heads >= 1 && kv_heads >= 1, "%s: bad shape len=%lld batch=%lld heads=%lld kv_heads=%lld", what,
               (long long)len, (long long)batch, (long long)heads, (long long)kv_heads);
  NMTG_REQUIRE(heads % kv_heads == 0, "%s: %lld query heads do not share %lld key / value heads evenly", what, (long long)heads, (long long)kv_heads);
  NMTG_REQUIRE(head_dim == 64 || head_dim == 128, "%s: head dimension %lld (64 and 128 are built)", what, (long long)head_dim);
  NMTG_REQUIRE(dtype == NMTG_F16 || dtype == NMTG_BF16, "%s: fp16 or bf16 tensors required (matrix-core kernel)", what);
  NMTG_REQUIRE(window >= 1 && sinks >= 0 && window < (1ll << 40) && sinks < (1ll << 40), "%s: window %lld (at least 1), sinks %lld (at least 0)", what,
               (long long)window, (long long)sinks);
  NMTG_REQUIRE(scale >= -1e6f && scale <= 1e6f, "%s: scale %g", what, (double)scale);
  NMTG_REQUIRE(heads <= 65535 && batch <= 65535 && len <= (1 << 24), "%s: more than 65535 heads or sequences, or 2^24 positions", what);
  NMTG_REQUIRE((len + WA_ROWS - 1) / WA_ROWS * heads * batch <= WA_MOST_BLOCKS, "%s: too many blocks in one launch", what);
  return 0;
}
// Views whose tile of up to 128 rows lies within 32-bit offsets of its first row. A single position has no stride.
int check_views(const char* what, WaView* views, const void* const* pointers, const int64_t* strides, int count, int64_t len) {
  for (int i = 0; i < count; ++i) {
    const int64_t s[3] = {len == 1 ? 0 : strides[3 * i], strides[3 * i + 1], strides[3 * i + 2]};
    NMTG_REQUIRE(aligned16(pointers[i]) && s[0] % 8 == 0 && s[1] % 8 == 0 && s[2] % 8 == 0 && s[0] >= 0 && s[1] >= 0 && s[2] >= 0 && s[0] < (1 << 24),
                 "%s: every tensor must be a 16-byte aligned [len, batch, heads, head_dim] view with a contiguous head_dim and strides that are "
                 "multiples of 8 elements (position stride below 2^24)", what);
    views[i] = {pointers[i], s[0], s[1], s[2]};
  }
  return 0;
}

// a scale of zero as one so small that every score is: hidden scores are infinite, and infinity times it stays so
float log2_scale(float scale) { return scale == 0.f ? 1e-30f : scale * FA_LOG2E; }

template <typename K>
int launch_tiled(K kern, int lds, dim3 grid, const WaArgs& a, hipStream_t st, const char* what) {
  if (lds > 64 * 1024) {
    hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(kern), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return fail(NMTG_ERR_LAUNCH, "%s: cannot reserve %d bytes of LDS: %s", what, lds, hipGetErrorString(e));
  }
  hipLaunchKernelGGL(kern, grid, dim3(64 * WA_WAVES), lds, st, a);
  return 0;
}
template <int D, int TILE> constexpr int tiles_lds() { return std::max(4 * TILE * D * 2, WA_WAVES * 32 * D * 2); }
template <int D> constexpr int dkv_lds() { return std::max(2 * dkv_buf<D>() + dkv_keys<D>(), WA_WAVES * 32 * D * 2); }
dim3 linear_grid(const WaArgs& a, int64_t blocks, int64_t heads) { return dim3(static_cast<unsigned>(blocks * heads * a.batch)); }
int64_t row_blocks(const WaArgs& a) { return (a.len + WA_ROWS - 1) / WA_ROWS; }

template <typename T, int D>
int fwd_launch(const WaArgs& a, hipStream_t st) {
  TraceScope trace("window_attn_fwd", st);
  return launch_tiled(window_fwd_kernel<T, D>, tiles_lds<D, fwd_tile<D>()>(), linear_grid(a, row_blocks(a), a.heads), a, st, "window_attn_fwd");
}
// How the blocks of dK and dV are laid out, and the floats they leave behind.
struct DkvPlan {
  int key_blocks, sink_blocks, parts, chunks, part_rows, sink_rows;
  int64_t part_floats, sink_floats;
  DkvPlan(int64_t len, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t window, int64_t sinks) {
    const int64_t blocks = (len + WA_ROWS - 1) / WA_ROWS, group = heads / kv_heads;
    const int64_t tiles = (std::min(len, window + WA_ROWS) + FA_TILE - 1) / FA_TILE;      // query tiles of a key block, per head
    key_blocks = static_cast<int>(blocks);
    // some query stands behind the window of a block's first sinks
    sink_blocks = len > WA_ROWS - 1 + window ? static_cast<int>(std::min(blocks, (std::min(sinks, len) + WA_ROWS - 1) / WA_ROWS)) : 0;
    // The queries behind, in chunks of eight tiles: shorter than a block of its own, so that the last ones of a launch end it soon, and where
    // the sinks are one wavefront's keys the other three only wait (2 x 8192 positions, window 1024, 4 sinks: 570 us, 580 with 16
    // tiles, 650 with 72; 4096 positions of one key head, 33 sinks: 42, 53, 133). Every chunk leaves the sums of all sinks in 32 bits:
    // with more than 256 of them twice as long (2048 sinks, 2 x 8192 positions: 210 us, 236 with eight), and no more than 64 chunks or
    // 32768 rows, but 16 in any case (2048 sinks, 16384 positions: 710 us, 884 with four).
    const int64_t behind = (len - std::min(len, window) + FA_TILE - 1) / FA_TILE * group, chunk = sinks <= 256 ? 8 : 16;
    const int64_t most = std::min<int64_t>(64, std::max<int64_t>(16, 32768 / std::max<int64_t>(sinks, 1)));
    chunks = sink_blocks > 0 ? static_cast<int>(std::max<int64_t>(1, std::min((behind + chunk - 1) / chunk, most))) : 0;
    // About two blocks for every compute unit, each with at least four tiles; four where most blocks are shorter than a whole window's,
    // so that the short ones even out the long (8192 positions in one window, 512 blocks of up to 516 tiles: 1480 us in one part, 1100
    // in two), if they are long enough (128 blocks of up to 48 tiles: 61 us in four parts, 84 in seven). But the sums of every part of
    // every block pass through memory in 32 bits, while what a split saves is a block's own tiles: no more parts than 18 tiles per block
    // / blocks (us of dK, dV and join, head dimension 128: 208 blocks of 12 tiles: 46 in one part, 64 in two; 104 of 24: 52 in three,
    // 47 in four, 53 in five).
    const int64_t all = std::max<int64_t>(blocks * batch * kv_heads, 1), pairs = tiles * group;
    const int64_t fill = (2 * std::min(blocks, (window + WA_ROWS - 1) / WA_ROWS) > blocks && pairs >= 96 ? 4 : 2) * num_cus();
    parts = static_cast<int>(std::max<int64_t>(1, std::min({(fill + all / 2) / all, pairs / 4, (18 * pairs + all / 2) / all, int64_t(16)})));
    sink_rows = sink_blocks > 0 ? static_cast<int>(std::min(sinks, len)) : 0;
    part_rows = parts > 1 ? static_cast<int>(len) : sink_rows;
    part_floats = batch * kv_heads * parts * part_rows * 2 * head_dim;
    sink_floats = batch * kv_heads * chunks * sink_rows * 2 * head_dim;
  }
};
int stat_rows(int64_t len) { return static_cast<int>((len + WA_ROWS - 1) / WA_ROWS * WA_ROWS); }
int64_t stat_floats(int64_t len, int64_t batch, int64_t heads) { return batch * heads * 2 * stat_rows(len); }

template <typename T, int D>
int bwd_launch(const WaArgs& a, hipStream_t st) {
  {
    TraceScope trace("window_attn_bwd_dq", st);
    if (int rc = launch_tiled(window_bwd_dq_kernel<T, D>, tiles_lds<D, FA_TILE>(), linear_grid(a, row_blocks(a), a.heads), a, st, "window_attn_bwd")) return rc;
  }
  {
    TraceScope trace("window_attn_bwd_dkv", st);
    const dim3 grid = linear_grid(a, a.key_blocks * a.parts + a.sink_blocks * a.chunks, a.kv_heads);
    if (int rc = launch_tiled(window_bwd_dkv_kernel<T, D>, dkv_lds<D>(), grid, a, st, "window_attn_bwd")) return rc;
  }
  if (a.part_rows > 0) {
    TraceScope trace("window_attn_bwd_join", st);
    const int64_t total = static_cast<int64_t>(a.part_rows) * (2 * D / 4);
    hipLaunchKernelGGL((window_dkv_join_kernel<T, D>), dim3(static_cast<unsigned>((total + 255) / 256), static_cast<unsigned>(a.kv_heads), static_cast<unsigned>(a.batch)),
                       dim3(256), 0, st, a, total);
  }
  return 0;
}

}  // namespace
}  // namespace nmtg

using namespace nmtg;

extern "C" int nmtg_window_attn_fwd(const void* q, const void* k, const void* v, void* out, uint8_t* out_rest, float* softmax_lse,
                                    const int32_t* lengths, const int64_t* strides, int64_t len, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                    int64_t window, int64_t sinks, float softmax_scale, int dtype, void* stream) {
  const char* what = "window_attn_fwd";
  if (int rc = check_call(what, len, batch, heads, kv_heads, head_dim, window, sinks, softmax_scale, dtype)) return rc;
  if (len == 0 || batch == 0) return 0;
  NMTG_REQUIRE(q && k && v && out && softmax_lse && strides, "%s: null pointer argument", what);
  NMTG_REQUIRE(aligned16(out_rest), "%s: out_rest must be 16-byte aligned", what);
  WaView views[4];
  const void* pointers[4] = {q, k, v, out};
  if (int rc = check_views(what, views, pointers, strides, 4, len)) return rc;
  WaArgs a = {};
  a.q = views[0]; a.k = views[1]; a.v = views[2]; a.o = views[3];
  a.rest = out_rest;
  a.lse = softmax_lse; a.lengths = lengths; a.len = static_cast<int>(len); a.batch = static_cast<int>(batch); a.heads = static_cast<int>(heads); a.kv_heads = static_cast<int>(kv_heads);
  a.group = static_cast<int>(heads / kv_heads); a.window = static_cast<int>(std::min(window, len + 1)); a.sinks = static_cast<int>(std::min(sinks, len)); a.scale = softmax_scale; a.scale_log2 = log2_scale(softmax_scale);
  hipStream_t st = static_cast<hipStream_t>(stream);
  int rc;
  if (dtype == NMTG_F16) rc = head_dim == 64 ? fwd_launch<f16_t, 64>(a, st) : fwd_launch<f16_t, 128>(a, st);
  else rc = head_dim == 64 ? fwd_launch<bf16_t, 64>(a, st) : fwd_launch<bf16_t, 128>(a, st);
  if (rc) return rc;
  NMTG_CHECK_LAUNCH(what);
  return 0;
}

extern "C" int64_t nmtg_window_attn_bwd_workspace_bytes(int64_t len, int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim,
                                                        int64_t window, int64_t sinks) {
  if (len <= 0 || batch <= 0 || heads <= 0 || kv_heads <= 0 || head_dim <= 0 || window <= 0 || sinks < 0) return 0;
  if (heads % kv_heads != 0) return 0;
  const DkvPlan plan(len, batch, heads, kv_heads, head_dim, window, sinks);
  return (stat_floats(len, batch, heads) + plan.part_floats + plan.sink_floats) * static_cast<int64_t>(sizeof(float));
}

extern "C" int nmtg_window_attn_bwd(const void* dout, const void* q, const void* k, const void* v, const void* out, const uint8_t* out_rest,
                                    const float* softmax_lse, void* dq, void* dk, void* dv, const int32_t* lengths, const int64_t* strides, int64_t len,
                                    int64_t batch, int64_t heads, int64_t kv_heads, int64_t head_dim, int64_t window, int64_t sinks,
                                    float softmax_scale, int dtype, void* workspace, int64_t workspace_bytes, void* stream) {
  const char* what = "window_attn_bwd";
  if (int rc = check_call(what, len, batch, heads, kv_heads, head_dim, window, sinks, softmax_scale, dtype)) return rc;
  if (len == 0 || batch == 0) return 0;
  NMTG_REQUIRE(dout && q && k && v && out && softmax_lse && dq && dk && dv && strides, "%s: null pointer argument", what);
  NMTG_REQUIRE(aligned16(out_rest), "%s: out_rest must be 16-byte aligned", what);
  NMTG_REQUIRE(workspace != nullptr && reinterpret_cast<uintptr_t>(workspace) % 256 == 0 &&
                   workspace_bytes >= nmtg_window_attn_bwd_workspace_bytes(len, batch, heads, kv_heads, head_dim, window, sinks),
               "%s: a 256-byte aligned workspace of nmtg_window_attn_bwd_workspace_bytes bytes required", what);
  WaView views[8];
  const void* pointers[8] = {dout, q, k, v, out, dq, dk, dv};
  if (int rc = check_views(what, views, pointers, strides, 8, len)) return rc;
  WaArgs a = {};
  a.d_o = views[0]; a.q = views[1]; a.k = views[2]; a.v = views[3]; a.o = views[4]; a.dq = views[5]; a.dk = views[6]; a.dv = views[7];
  a.rest = const_cast<uint8_t*>(out_rest);
  a.lse = const_cast<float*>(softmax_lse); a.stats = static_cast<float*>(workspace);
  a.stat_rows = stat_rows(len);
  const DkvPlan plan(len, batch, heads, kv_heads, head_dim, window, sinks);
  NMTG_REQUIRE((static_cast<int64_t>(plan.key_blocks) * plan.parts + static_cast<int64_t>(plan.sink_blocks) * plan.chunks) * kv_heads * batch <= WA_MOST_BLOCKS,
               "%s: too many blocks in one launch", what);
  a.part = a.stats + stat_floats(len, batch, heads);
  a.sink_part = a.part + plan.part_floats;
  a.key_blocks = plan.key_blocks; a.sink_blocks = plan.sink_blocks; a.parts = plan.parts; a.chunks = plan.chunks;
  a.part_rows = plan.part_rows; a.sink_rows = plan.sink_rows;
  a.lengths = lengths; a.len = static_cast<int>(len);
  a.batch = static_cast<int>(batch); a.heads = static_cast<int>(heads); a.kv_heads = static_cast<int>(kv_heads); a.group = static_cast<int>(heads / kv_heads);
  a.window = static_cast<int>(std::min(window, len + 1)); a.sinks = static_cast<int>(std::min(sinks, len)); a.scale = softmax_scale; a.scale_log2 = log2_scale(softmax_scale);
  hipStream_t st = static_cast<hipStream_t>(stream);
  int rc;
  if (dtype == NMTG_F16) rc = head_dim == 64 ? bwd_launch<f16_t, 64>(a, st) : bwd_launch<f16_t, 128>(a, st);
  else rc = head_dim == 64 ? bwd_launch<bf16_t, 64>(a, st) : bwd_launch<bf16_t, 128>(a, st);
  if (rc) return rc;
  NMTG_CHECK_LAUNCH(what);
  return 0;
}
