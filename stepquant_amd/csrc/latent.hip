// MI355X (gfx950) kernels of latent attention: one shared vector a token (the
// latent, `W` dims, and a rope key of 64) in 16 bits in pages; the write that
// turns the rope key on the way, the dense rows of requests, attention over the
// pages with the heads' projections absorbed into queries and outputs, and
// attention over keys and values that were expanded from the latents.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>

#include "internal.h"
#include "rotary.h"
#include "stepquant_hip.h"

// every fused multiply-add is written out
#pragma clang fp contract(off)

namespace {

typedef __bf16 bf16x2_v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_v __attribute__((ext_vector_type(8)));
typedef _Float16 half2_v __attribute__((ext_vector_type(2)));
typedef _Float16 half8_v __attribute__((ext_vector_type(8)));
typedef short short4_v __attribute__((ext_vector_type(4)));
typedef float f32x2_v __attribute__((ext_vector_type(2)));
typedef float f32x4_v __attribute__((ext_vector_type(4)));
typedef float f32x16_v __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void *lds_t;

constexpr int kRope = 64;
constexpr int kTile = 64;        // keys of a plan's tile, and of the expanded form's
constexpr float kNone = -3e38f;    // a row's unit before it has seen a finite score
constexpr float kUnseen = -3.2e38f;  // before it has seen a key
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLarge = 0x1p19f;  // scores from here on (in log2) hold few fractions

// Weights are in units of 2^m, m at most `top` and, once it is set, `bias` below the
// largest score that the row has seen: it is raised only where a score passes
// `top`, so that outputs are seldom rescaled.  A half then holds all bits of a
// weight down to 2^-21 of the row's largest.  Weights in bfloat16, whose range is that
// of 32 bits, are 2^-36 of those: sums over a million of the largest values stay within
// 32 bits, and products with values down to 2^-97 normal numbers.

__device__ __forceinline__ int64_t load_index(const void *p, int dtype, int64_t i) {
  return dtype == SQ_I64 ? ((const int64_t *)p)[i] : (int64_t)((const int32_t *)p)[i];
}

// the two 16-bit types
template <bool BF16>
struct Half;

template <>
struct Half<true> {
  static constexpr uint32_t exponent = 0x7f80u;
  static constexpr float bias = -29.f, top = -21.f;
  static __device__ __forceinline__ f32x4_v mul32(u32x4_v a, u32x4_v b, f32x4_v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16_v mul(u32x4_v a, u32x4_v b, f32x16_v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_v){x, y}, bf16x2_v));
  }
  // a pair's sum, as rounded, and l
  static __device__ __forceinline__ float add(uint32_t w, float l) {
    return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2_v, w), (bf16x2_v){(__bf16)1.f, (__bf16)1.f}, l, false);
  }
};

template <>
struct Half<false> {
  static constexpr uint32_t exponent = 0x7c00u;
  static constexpr float bias = 7.f, top = 15.f;
  static __device__ __forceinline__ f32x4_v mul32(u32x4_v a, u32x4_v b, f32x4_v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_v, a), __builtin_bit_cast(half8_v, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16_v mul(u32x4_v a, u32x4_v b, f32x16_v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_v, a), __builtin_bit_cast(half8_v, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_v){x, y}, half2_v));
  }
  static __device__ __forceinline__ float add(uint32_t w, float l) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_v, w), (half2_v){(_Float16)1.f, (_Float16)1.f}, l, false);
  }
};

// What a row's outputs are multiplied by.  A row that sees nothing is zero; where it sees
// keys and every weight is 0, all scores are -infinity and it is no number.
__device__ __forceinline__ float inverse_sum(float sum, float m) { return sum != 0.f ? 1.f / sum : m < kNone ? 0.f : NAN; }

__device__ __forceinline__ float max2(float x) {  // over the lanes l and l ^ 32
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum2(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
template <int CTRL>
__device__ __forceinline__ float dpp(float x) {
  return __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(x), CTRL, 0xf, 0xf, true));
}
// over the 8 or 16 lanes of a row: the lane 1, 2, 7 - l and 15 - l away
template <int LANES>
__device__ __forceinline__ float row_max(float x) {
  x = fmaxf(x, dpp<0xb1>(x));
  x = fmaxf(x, dpp<0x4e>(x));
  x = fmaxf(x, dpp<0x141>(x));
  return LANES == 8 ? x : fmaxf(x, dpp<0x140>(x));
}
template <int LANES>
__device__ __forceinline__ float row_sum(float x) {
  x += dpp<0xb1>(x);
  x += dpp<0x4e>(x);
  x += dpp<0x141>(x);
  return LANES == 8 ? x : x + dpp<0x140>(x);
}

// ------------------------------------------------------------ pages

struct LatentAppend {
  sq_latent_cache c;
  sq_latent_append_args a;
  sq_rotary r;  // dim 0: rope keys go in as they are
  sq_rotary_rows q;
  int rows_blocks, q_lanes;
};

// A thread moves 16 bytes of a token's latent, or turns 16 dims of its rope
// key; the workgroups behind turn the queries.  It moves memory and nothing else bounds
// it; a decode step's is smaller than a launch (256 requests, 32 heads: 10 us with the
// host's share, 300 as five calls of the library with the rotation written out).
template <int T>
__global__ __launch_bounds__(256) void latent_append_kernel(LatentAppend d) {
  const uint32_t block = blockIdx.x;
  if (block >= (uint32_t)d.rows_blocks) {
    rotary::rotate_rows_typed<T, 1>(d.r, d.q, d.q_lanes, (block - d.rows_blocks) * 256 + threadIdx.x);
    return;
  }
  const uint32_t groups = d.c.latent / 8, threads = groups + kRope / 16, id = block * 256 + threadIdx.x;
  const uint32_t token = id / threads, g = id - token * threads;
  if (token >= d.a.tokens) return;
  const int64_t slot = d.a.slots[token];
  if (slot < d.c.page_tokens || slot >= d.c.num_pages * d.c.page_tokens) return;  // (none, or the padding page)
  uint16_t *dst = (uint16_t *)d.c.data + slot * (d.c.latent + kRope);
  if (g < groups) {
    *(u32x4_v *)(dst + 8 * g) = *(const u32x4_v *)((const uint16_t *)d.a.latent + token * d.a.latent_stride + 8 * g);
    return;
  }
  const int item = g - groups;
  const uint16_t *src = (const uint16_t *)d.a.rope + token * d.a.rope_stride;
  dst += d.c.latent;
  int ga = 2 * item, gb = 2 * item + 1;
  if (d.r.dim) rotary::groups(d.r, item, ga, gb);
  rotary::Eight<T> xa, xb;
  xa.load(src, 8 * ga), xb.load(src, 8 * gb);
  if (item < d.r.dim / 16) {
    const int position = d.a.positions[token];
    rotary::Angles t;
    t.at(d.r, item, (uint64_t)(int64_t)position);
    float x[16];
    xa.widen(x), xb.widen(x + 8);
    rotary::rotate(d.r.interleaved, t, x);
    xa.narrow(x), xb.narrow(x + 8);
  }
  xa.store(dst, 8 * ga), xb.store(dst, 8 * gb);
}

// Rows of all requests, request after request, 32 of them a workgroup, which
// sums the requests' lengths for itself, so that nothing is read back and one launch does:
// a workgroup reads up to 16 KB of lengths from its L2 beside 36 KB of rows.  Each row
// is read and written once, all of a thread's loads before its stores (6 requests of up to 9100, 32,000 rows
// in all: 20 us, 3.7 TB/s with pages in any order; 25 with 64 rows a workgroup and four loads at a time).
constexpr int kGatherRows = 32;

template <int W>
__global__ __launch_bounds__(256) void latent_gather_kernel(sq_latent_cache c, sq_latent_gather_args a) {
  extern __shared__ int64_t ends[];  // of the requests' rows, [batch]
  __shared__ int64_t waves[4];
  __shared__ int64_t source[kGatherRows];
  const int tid = threadIdx.x, B = a.batch, items = (B + 255) / 256, b0 = min(B, tid * items), b1 = min(B, b0 + items);
  int64_t sum = 0;
  for (int b = b0; b < b1; b++) sum += max(a.lens[b], 0);
  int64_t upto = sum;
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) {
    const int64_t x = __shfl_up(upto, k, 64);
    if ((tid & 63) >= k) upto += x;
  }
  if ((tid & 63) == 63) waves[tid >> 6] = upto;
  __syncthreads();
  int64_t at = upto - sum;
  for (int w = 0; w < tid >> 6; w++) at += waves[w];
  for (int b = b0; b < b1; b++) ends[b] = at += max(a.lens[b], 0);
  __syncthreads();
  if (blockIdx.x == 0) {
    // (starts stop at the rows that there are)
    if (tid == 0) a.starts[0] = 0;
    for (int b = tid; b < B; b += 256) a.starts[b + 1] = (int32_t)min(ends[b], a.rows_out);
  }
  const int64_t first = (int64_t)blockIdx.x * kGatherRows;
  if (tid < kGatherRows) {
    const int64_t r = first + tid;
    int lo = 0, hi = B;
    while (lo < hi) {
      const int mid = (lo + hi) >> 1;
      if (ends[mid] > r) hi = mid;
      else lo = mid + 1;
    }
    int64_t from = -1;
    if (lo < B) {
      const int64_t row = load_index(a.rows, a.rows_dtype, lo), pos = r - (lo ? ends[lo - 1] : 0);
      const int64_t block = pos / c.page_tokens;
      if (row >= 0 && row < a.requests && block < a.width) {
        const int64_t page = a.table[row * a.width + block];
        if (page > 0 && page < c.num_pages) from = page * c.page_tokens + (pos - block * c.page_tokens);
      }
    }
    source[tid] = from;
  }
  __syncthreads();
  constexpr int groups = (W + kRope) / 8, N = (kGatherRows * groups + 255) / 256;
  const int rows = (int)min((int64_t)kGatherRows, a.rows_out - first);
  u32x4_v x[N];
#pragma unroll
  for (int k = 0; k < N; k++) {
    const int i = 256 * k + tid, r = i / groups, g = i - r * groups;
    const int64_t from = r < rows ? source[r] : -1;
    x[k] = from < 0 ? (u32x4_v){0, 0, 0, 0} : *(const u32x4_v *)((const uint16_t *)c.data + from * (W + kRope) + 8 * g);
  }
#pragma unroll
  for (int k = 0; k < N; k++) {
    const int i = 256 * k + tid, r = i / groups, g = i - r * groups;
    if (r >= rows) break;
    if (8 * g < W) *(u32x4_v *)((uint16_t *)a.latent + (first + r) * W + 8 * g) = x[k];
    else *(u32x4_v *)((uint16_t *)a.rope + (first + r) * kRope + 8 * g - W) = x[k];
  }
}

// ------------------------------------------------------------ tiles in LDS
//
// LDS has 64 banks, 256 bytes.  A wave reads 16 bytes a lane in four cycles, of the
// lanes 0-3, 12-15, 20-23 and 24-27, of 4-11, 16-19 and 28-31, and of the same 32 on;
// the transposing load of 8 bytes a lane takes lanes 0-31 and 32-63.  (Taken from the
// counters of conflicts of single reads.)  Rows of 16-byte groups lie one after
// the other, and a row's groups are exchanged by an exclusive or, so that neither kind of
// read meets a bank twice: 16 rows at four adjacent groups as lanes 16 g + row,
// and 32 bytes of the rows 0-3 and 8-11, or 4-7 and 12-15.  The load from memory
// to LDS puts 64 lanes' groups side by side, so a lane asks for the group whose place it has.

// Cached tiles: rows are an odd number of 128 bytes long, the last 128 of them the rope key.
template <int W>
__device__ __forceinline__ int place_of(int row, int at) {
  return at ^ (row & 3) << 1 ^ (at < W / 8 ? ((row >> 3 ^ row) & 1) << 3 : 0);
}

// rows of 32 scores (128 bytes) and of 32 weights (64)
__device__ __forceinline__ int score_place(int row, int at) { return at ^ (row & 2) ^ (row >> 1 & 4); }
__device__ __forceinline__ int weight_place(int row, int at) { return at ^ (row >> 2 & 2); }

// 16 bytes a lane from memory to LDS at `lds` + 16 lane.  The compiler does not
// count these loads: it would wait for all of them before any write to LDS; the
// waits are written out.  M0 holds the place in LDS, and is to be there an instruction before.
__device__ __forceinline__ void to_lds(uint32_t lds, const uint8_t *base, uint32_t offset) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"{m0}"(lds), "v"(offset), "s"(base) : "memory");
}

// the same, of what nothing else will read (64 requests of up to 8192: 8% faster)
__device__ __forceinline__ void to_lds_once(uint32_t lds, const uint8_t *base, uint32_t offset) {
  asm volatile("s_nop 0\n\tglobal_load_lds_dwordx4 %1, %2 nt" ::"{m0}"(lds), "v"(offset), "s"(base) : "memory");
}

// a word that the whole wave reads and no kernel running beside writes, by the scalar cache
__device__ __forceinline__ int uniform_word(const int32_t *p) {
  return *(const __attribute__((address_space(4))) int32_t *)(uintptr_t)p;
}

template <int N>
__device__ __forceinline__ void wait_loads() {  // until at most N are under way
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}

__device__ __forceinline__ uint32_t lds_address(const void *p) {
  return __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)(lds_t)p);
}

// Four consecutive rows' elements of one column, transposed: of 16 lanes, lane i
// addresses row i / 4, columns 4 (i % 4) to 4 (i % 4) + 3, and lane j gets column j
// of the four rows.
__device__ __forceinline__ short4_v read_column(uint32_t lds) {
  return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) short4_v *)lds);
}

template <typename T>
__device__ __forceinline__ const __attribute__((address_space(3))) T *from_lds(uint32_t lds) {
  return (const __attribute__((address_space(3))) T *)lds;
}

// A value that the compiler takes for a new one: what is made from it is made where
// it is used, and keeps no registers in loops around.
template <typename T>
__device__ __forceinline__ T anew(T x) {
  asm volatile("" : "+v"(x));
  return x;
}

template <typename T>
__device__ __forceinline__ __attribute__((address_space(3))) T *to_lds_at(uint32_t lds) {
  return (__attribute__((address_space(3))) T *)lds;
}

// infinities and NaN of two halves as zero
template <bool BF16>
__device__ __forceinline__ uint32_t only_finite(uint32_t w) {
  constexpr uint32_t e = Half<BF16>::exponent;
  const uint32_t lo = (w & e) == e ? 0u : 0xffffu, hi = (w & e << 16) == e << 16 ? 0u : 0xffff0000u;
  return w & (lo | hi);
}

template <bool BF16>
__device__ __forceinline__ void store4(uint16_t *dst, f32x4_v x) {
  *(uint2 *)dst = make_uint2(Half<BF16>::pack(x[0], x[1]), Half<BF16>::pack(x[2], x[3]));
}

// ------------------------------------------------------------ absorbed
//
// out[t, h] = sum_j softmax_j(scale (q[t, h] . c_j + q_rope[t, h] . r_j)) c_j: one
// key and value for all heads, so a row is a token's head and the rows of a
// token share every key that is read.  S^T = K Q^T and O^T = C^T P^T run as matrix
// products whose columns are rows of queries, and the softmax by rows between them.
//
// Weights are rounded to the cache's type for the second product, by 2^-8 (bf16) or
// 2^-11 of each at most, and their sum is that of the rounded ones, so that the error is
// of the spread of the values alone; scores, sums and outputs are held in 32 bits.
//
// What bounds it: with up to 32 rows (a decode step of 32 heads) the pages, 1152 bytes a token
// that are read once.  64 requests of up to 8191 take 69 us, 4.9 TB/s; of equal lengths
// it is 5.9 (16 heads 6.5; a large copy reaches 5, reading alone 6.5).  What is missing are
// units' starts, which wait for queries and all tiles under way, and the parts of cut keys, 20 MB
// written and read again (311 of 314 units).  With 128 rows (32 requests of up to
// 16,383: 144 us) it is the two steps below, 0.7 us each of a tile of 32 keys, in
// which the matrix cores are busy for a quarter of the time: each waits for the barrier,
// for its weights and first operands from LDS, and for its last scores.

struct AbsorbedDev {
  sq_latent_cache c;
  const uint16_t *q, *rope;
  uint16_t *out;
  float *ws;
  const int32_t *table, *units, *merges, *starts;
  int64_t requests, tokens, q_stride, q_head_stride, rope_stride, rope_head_stride;
  int32_t width, heads, causal, max_partials, max_units, max_workers, unit_rows;
  float scale;
};

struct Unit {
  int row, q0, f0, rows, pos0, kv0, kv1, part;
};

// rows at_row to at_row + most - 1 of a unit
__device__ __forceinline__ Unit read_unit(const AbsorbedDev &a, int i, int at_row, int most) {
  const int32_t *u = a.units + 8 * (int64_t)i;
  const auto word = [&](int k) { return uniform_word(u + k); };
  Unit x = {word(0), word(1), word(2), word(3), word(4), word(5), word(6), word(7)};
  if (x.rows <= 0 || x.rows > a.unit_rows || x.q0 < 0 || x.f0 < 0 || x.kv0 < 0 ||
      x.q0 + (int64_t)(x.f0 + x.rows - 1) / a.heads >= a.tokens)
    x.rows = 0;
  x.f0 += at_row, x.rows = max(0, min(x.rows - at_row, most));
  x.kv0 &= ~(kTile - 1);  // (a tile lies within a page)
  // a row of the table that does not exist holds no keys
  const bool held = x.rows > 0 && x.row >= 0 && x.row < a.requests;
  x.kv1 = held ? (int)min((int64_t)x.kv1, (int64_t)a.width * a.c.page_tokens) : 0;
  return x;
}

// Tiles of 32 keys pass through a ring in LDS, for one or two groups of four waves
// with up to 16 NR rows each.  A group takes a tile through two steps:
//
//   products  outputs with the tile before, every wave for a quarter of the dims
//             (so outputs need no joining); then scores with this tile, every
//             wave for 16 keys and half of the dims, as sums in 32 bits;
//   softmax   by rows: 8 or 16 lanes have a row's 32 scores, and alone know its
//             unit and its sum; rounded weights and what the row's outputs are
//             to be multiplied by go to LDS.
//
// Two groups run a step apart, so that one's products have the matrix cores while
// the other waits for scores and exponentials; a barrier ends each step.  The
// late group loads.  PAIR: units of 128 rows have two workgroups, which run
// side by side on one XCD (8 apart, blocks go to the 8 in turn) so that its L2 gives one
// of them the keys (349 MB of pages: half of the reads hit, 364 MB come from memory); others
// are read past the caches' later use.
template <int W_, int RG_, int NR_, bool PAIR_ = false>
struct Absorbed {
  static constexpr int W = W_, TK = 32, RG = RG_, NR = NR_, NW = 4 * RG, threads = 64 * NW, RING = W == 512 ? 4 : 6;
  static constexpr bool PAIR = PAIR_, HALVES = NR == 1;  // two waves share 16 rows' scores: half of the dims each
  static constexpr int R = 16 * RG * NR, TILE = TK * 2 * (W + kRope), SROW = 4 * TK, PROW = 2 * TK;
  static constexpr size_t lds = RING * TILE + R * ((HALVES ? 2 : 1) * SROW + PROW + 4) + 16;
  static_assert(lds <= 163840, "LDS of a CU");
};

template <typename S, bool BF16>
__device__ __forceinline__ void absorbed_attend(const AbsorbedDev &a) {
  typedef Half<BF16> H;
  constexpr int W = S::W, TK = S::TK, RG = S::RG, NR = S::NR, NW = S::NW, RING = S::RING, TILE = S::TILE, R = S::R;
  constexpr int KD = W + kRope, ROW = 2 * KD, KS = KD / (S::HALVES ? 64 : 32), DB = W / 64;
  constexpr int SROW = S::SROW, PROW = S::PROW;
  constexpr int LOADS = TILE / 4096;                           // of a tile, of a wave of the group that loads
  constexpr int LANES = 256 / (16 * NR), KEYS = TK / LANES;    // of a row's softmax, and of a lane
  extern __shared__ __attribute__((aligned(128))) uint8_t smem[];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), lane = tid & 63;
  const int rg = wave >> 2, share = wave & 3, kg = wave & 1, half = wave >> 1 & 1;
  const bool late = RG == 2 && rg == 1, loads = rg == RG - 1;
  const int worker = S::PAIR ? (blockIdx.x >> 4) * 8 + (blockIdx.x & 7) : (int)blockIdx.x;
  const int at_row = S::PAIR ? R * (blockIdx.x >> 3 & 1) : 0;
  if (worker >= a.max_workers) return;
  const int unit0 = max(0, uniform_word(a.starts + worker)), unit1 = min(uniform_word(a.starts + worker + 1), a.max_units);
  if (unit0 >= unit1) return;
  const int G = a.heads, P = a.c.page_tokens;
  const uint32_t tiles_at = lds_address(smem);
  const uint32_t scores = tiles_at + RING * TILE;  // [HALVES ? 2 : 1][R] rows of TK
  const uint32_t weights = scores + (S::HALVES ? 2 : 1) * R * SROW;  // [R] rows of TK
  const uint32_t factors = weights + R * PROW;     // [R]
  const uint32_t bad_at = factors + 4 * R;         // [4] keys of a tile that the waves cleaned
  // Where a lane's operands lie: its key's steps of 32 dims (four of them 256 bytes;
  // the last two may be the rope key's), and its four keys of the wave's 16 dims of
  // every 64 (two of them 256 bytes, and four keys on a constant way).
  const int c = lane & 15, g = lane >> 4, token = 8 * g + (c >> 2);
  const int step0 = S::HALVES ? KS * half : 0;
  auto key_step = [&](int k) {
    const int row = 16 * kg + c;
    return tiles_at + row * ROW + 16 * place_of<W>(row, 4 * (step0 + k) + g);
  };
  const uint32_t key_at[4] = {key_step(0), key_step(1), key_step(2), key_step(3)};
  const uint32_t last_at[2] = {key_step(KS - 2), key_step(KS - 1)};
  auto four_keys = [&](int e) { return tiles_at + token * ROW + 16 * place_of<W>(token, 8 * e + 2 * share + (c >> 1 & 1)) + 8 * (c & 1); };
  const uint32_t value_at[2] = {four_keys(0), four_keys(1)};
  uint32_t from[LOADS];  // the groups of a tile's eight rows that a lane loads
#pragma unroll
  for (int k = 0; k < LOADS; k++) {
    const int n = 64 * k + lane, row = n / (KD / 8), at = n - row * (KD / 8);
    from[k] = (row + 8 * share) * ROW + 16 * place_of<W>(row + 8 * share, at);
  }
  const int row0 = 16 * NR * rg, q_row = row0 + (S::HALVES ? 0 : 16 * half) + c;  // of the group; of the lane's scores
  const uint32_t score_to = scores + ((S::HALVES ? R * half : 0) + q_row) * SROW + 16 * score_place(c, 4 * kg + g);
  const uint32_t weight_at = weights + (row0 + c) * PROW + 16 * weight_place(c, g), factor_at = factors + 4 * (row0 + c);
  // the lane's row of the softmax, and its keys there
  const int mine = row0 + (tid & 255) / LANES, part = tid % LANES;
  const uint32_t score_at = scores + mine * SROW + 16 * score_place(mine, KEYS * part / 4) + 4 * (KEYS * part % 4);
  const uint32_t weight_to = weights + mine * PROW + 16 * weight_place(mine, KEYS * part / 8) + 2 * (KEYS * part % 8);

  // the tile that is loaded next: its page, the tokens before it there
  struct Place {
    const int32_t *entry;
    int page, in_page, n;
  };
  auto place = [&](const Unit &u) {
    Place x = {a.table, 0, 0, max(0, (u.kv1 - u.kv0 + TK - 1) / TK)};
    if (x.n) {
      const int block = u.kv0 / P;
      x.entry += (int64_t)u.row * a.width + block;
      x.in_page = u.kv0 - block * P;
      x.page = uniform_word(x.entry);
    }
    return x;
  };
  Unit u = read_unit(a, unit0, at_row, R);
  Place next = place(u);
  int n = 0, loaded = 0;  // tiles of the unit, and how many of them are on their way
  uint32_t known = 0;     // bit i % 32: tile i has a page
  uint32_t load_slot = 0; // where the next tile goes
  auto after_slot = [&](uint32_t slot) { return slot + TILE == RING * TILE ? 0u : slot + TILE; };
  auto load = [&]() {
    const int i = loaded++;
    const bool there = next.page > 0 && next.page < a.c.num_pages;
    known = known & ~(1u << (i & 31)) | (uint32_t)there << (i & 31);
    if (loads) {
      const uint8_t *base = (const uint8_t *)a.c.data + ((there ? (int64_t)next.page * P : 0) + next.in_page) * ROW;
      const uint32_t to = tiles_at + load_slot + TILE / 4 * share;
#pragma unroll
      for (int k = 0; k < LOADS; k++) {
        if constexpr (S::PAIR) to_lds(to + 1024 * k, base, from[k]);
        else to_lds_once(to + 1024 * k, base, from[k]);
      }
    }
    load_slot = after_slot(load_slot);
    next.in_page += TK;
    if (next.in_page == P && i + 1 < n) next.in_page = 0, next.page = uniform_word(++next.entry);
  };
  // until tile i is there, with MOST tiles behind it on their way as a rule
  auto wait_tile = [&](auto MOST, int i) {
    constexpr int most = decltype(MOST)::value;
    if (!loads) return;
    if (loaded - 1 - i >= most) wait_loads<most * LOADS>();
    else wait_loads<0>();
  };
  auto begin = [&]() {
    n = next.n, loaded = 0, load_slot = 0;
#pragma unroll
    for (int i = 0; i < RING - 1; i++)
      if (i < n) load();
  };
  begin();
  for (int unit_at = unit0; unit_at < unit1; unit_at++) {
    u32x4_v q[KS];
    f32x4_v o[NR][DB];
    {
      const int fresh = anew(lane), row = q_row - c + (fresh & 15), f = u.f0 + row;
      const bool live = row < u.rows;
      const int t = live ? f / G : 0, head = live ? f - t * G : 0, d0 = 32 * step0 + 8 * (fresh >> 4);
      const uint16_t *src = a.q + (u.q0 + t) * a.q_stride + head * a.q_head_stride;
      const uint16_t *rope = a.rope + (u.q0 + t) * a.rope_stride + head * a.rope_head_stride;
#pragma unroll
      for (int s = 0; s < KS; s++) {
        const int d = d0 + 32 * s;
        q[s] = live ? *(const u32x4_v *)(32 * (step0 + s) < W ? src + d : rope + d - W) : (u32x4_v){0, 0, 0, 0};
      }
    }
    const Unit following = read_unit(a, min(unit_at + 1, unit1 - 1), at_row, R);
    const Place after = place(following);
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
      for (int e = 0; e < DB; e++) o[r][e] = (f32x4_v){0, 0, 0, 0};
    // (the queries' loads are waited for here, and the tiles' that were issued before them, as loads
    // return in order, but not those of later tiles by a wait in the loop)
#pragma unroll
    for (int s = 0; s < KS; s++) asm volatile("" : "+v"(q[s]));
    const float mult = a.scale * kLog2e;
    // the keys that the lane's row sees, and those that every row of the unit sees
    const int hi = mine >= u.rows ? 0 : a.causal ? min(u.kv1, u.pos0 + (u.f0 + mine) / G + 1) : u.kv1;
    const int all_hi = u.rows <= 0 ? 0 : a.causal ? min(u.kv1, u.pos0 + u.f0 / G + 1) : u.kv1;
    auto whole = [&](int i) { return (known >> (i & 31) & 1) && u.kv0 + TK * (i + 1) <= all_hi; };
    float m = whole(0) ? kNone : kUnseen, l = 0.f;

    // Outputs with the tile at `values` (OUT) and scores with the one at `keys` (IN), their products in turn;
    // operands are read some products ahead.
    auto products = [&](auto OUT, auto IN, uint32_t values, uint32_t keys) {
      constexpr int NO = decltype(OUT)::value ? DB : 0, NI = decltype(IN)::value ? KS : 0, N = NO + NI;
      constexpr int AHEAD_K = NI < 4 ? NI : 4, AHEAD_V = NO < 2 ? NO : 2;
      u32x4_v p[NR], kw[AHEAD_K + 1], vw[AHEAD_V + 1];
      f32x4_v s[2] = {{0, 0, 0, 0}, {0, 0, 0, 0}};
      auto read_key = [&](int k) { return *from_lds<u32x4_v>(k < KS - 2 ? key_at[k & 3] + keys + 256 * (k >> 2) : last_at[k - KS + 2] + keys); };
      auto read_value = [&](int e) {
        uint2 w[2];
#pragma unroll
        for (int z = 0; z < 2; z++)
          w[z] = __builtin_bit_cast(uint2, read_column(value_at[e & 1] + values + 256 * (e >> 1) + 4 * z * ROW));
        return (u32x4_v){w[0].x, w[0].y, w[1].x, w[1].y};
      };
      if constexpr (NO > 0) {
        float f[NR];
        bool raised = false;
#pragma unroll
        for (int r = 0; r < NR; r++) {
          f[r] = *from_lds<float>(factor_at + 64 * r);
          p[r] = *from_lds<u32x4_v>(weight_at + 16 * r * PROW);
          raised |= f[r] != 1.f;
        }
        if (__any(raised)) {
#pragma unroll
          for (int r = 0; r < NR; r++)
#pragma unroll
            for (int e = 0; e < DB; e++) o[r][e] *= f[r];
        }
      }
#pragma unroll
      for (int k = 0; k < AHEAD_K; k++) kw[k] = read_key(k);
#pragma unroll
      for (int e = 0; e < AHEAD_V; e++) vw[e] = read_value(e);
#pragma unroll
      for (int j = 0; j < N; j++) {
        const int e = NO ? j * NO / N : 0;  // products of outputs before this one
        if (NO && (j + 1) * NO / N > e) {
          if (e + AHEAD_V < NO) vw[(e + AHEAD_V) % (AHEAD_V + 1)] = read_value(e + AHEAD_V);
#pragma unroll
          for (int r = 0; r < NR; r++) o[r][e] = H::mul32(vw[e % (AHEAD_V + 1)], p[r], o[r][e]);
        } else {
          const int k = j - e;
          if (k + AHEAD_K < NI) kw[(k + AHEAD_K) % (AHEAD_K + 1)] = read_key(k + AHEAD_K);
          s[k & 1] = H::mul32(kw[k % (AHEAD_K + 1)], q[k], s[k & 1]);
        }
      }
      __builtin_amdgcn_sched_group_barrier(0x100, AHEAD_K + 2 * AHEAD_V, 0);  // LDS reads
#pragma unroll
      for (int j = 0; j < N; j++) {
        const int e = NO ? j * NO / N : 0;
        if (NO && (j + 1) * NO / N > e) {
          if (e + AHEAD_V < NO) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
          __builtin_amdgcn_sched_group_barrier(0x8, NR, 0);  // products
        } else {
          if (j - e + AHEAD_K < NI) __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);
        }
      }
      if constexpr (NI > 0) *to_lds_at<f32x4_v>(score_to) = s[0] + s[1];
    };
    // What some row does not see has a weight of 0 there; infinities and NaN would
    // still reach its outputs.  They are taken out, and rows that do see such a latent are
    // NaN (its score may be -infinity, of which neither sum nor outputs would tell).
    auto clean = [&](int i, uint32_t slot) {
      const int first = u.kv0 + TK * i, r0 = known >> (i & 31) & 1 ? max(0, min(TK, all_hi - first)) : 0;
      uint32_t bad = 0;
      for (int j = r0 * (W / 8) + (tid & 255); j < TK * (W / 8); j += 256) {
        const int row = j / (W / 8);
        const uint32_t at = tiles_at + slot + row * ROW + 16 * (j % (W / 8));
        u32x4_v w = *from_lds<u32x4_v>(at);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const uint32_t x = only_finite<BF16>(w[k]);
          bad |= x != w[k] ? 1u << row : 0u;
          w[k] = x;
        }
        *to_lds_at<u32x4_v>(at) = w;
      }
      if (__any(bad != 0))
#pragma unroll
        for (int k = 1; k < 64; k <<= 1) bad |= (uint32_t)__shfl_xor((int)bad, k, 64);
      *to_lds_at<uint32_t>(bad_at + 4 * share) = bad;
    };
    auto poison = [&](int i) {
      const int seen = known >> (i & 31) & 1 ? hi - (u.kv0 + TK * i) : 0;
      const u32x4_v w = *from_lds<u32x4_v>(bad_at);
      const uint32_t bad = w[0] | w[1] | w[2] | w[3];
      if (seen > 0 && (bad & (seen >= TK ? ~0u : (1u << seen) - 1))) l = NAN;
    };
    auto softmax = [&](int i, bool all) {
      const int first = u.kv0 + TK * i;
      typedef float vec __attribute__((ext_vector_type(KEYS)));
      vec x = *from_lds<vec>(score_at);
      if constexpr (S::HALVES) x += *from_lds<vec>(score_at + R * SROW);
      x *= mult;
      if (!all) {
        const int held = known >> (i & 31) & 1 ? hi - first : 0, seen = held - KEYS * part;
#pragma unroll
        for (int k = 0; k < KEYS; k++) x[k] = k < seen ? x[k] : -INFINITY;
        m = fmaxf(m, held > 0 ? kNone : kUnseen);
      }
      float best = x[0];
#pragma unroll
      for (int k = 1; k < KEYS; k++) best = fmaxf(best, x[k]);
      best = row_max<LANES>(best);
      float factor = 1.f;
      if (best - m > H::top) {
        const float raised = best - H::bias;
        factor = __builtin_amdgcn_exp2f(m - raised);
        m = raised;
        l *= factor;
      }
      uint32_t w[KEYS / 2];
#pragma unroll
      for (int k = 0; k < KEYS / 2; k++) {
        w[k] = H::pack(__builtin_amdgcn_exp2f(x[2 * k] - m), __builtin_amdgcn_exp2f(x[2 * k + 1] - m));
        l = H::add(w[k], l);
      }
      typedef uint32_t words __attribute__((ext_vector_type(2)));
      if constexpr (KEYS == 4) *to_lds_at<words>(weight_to) = (words){w[0], w[1]};
      else *to_lds_at<uint32_t>(weight_to) = w[0];
      if (part == 0) *to_lds_at<float>(factors + 4 * mine) = factor;
    };

    uint32_t slot = 0;  // of tile i
    if (n > 0) {
      typedef std::integral_constant<int, RING - 2> Issued;          // tiles behind the one that is waited for
      typedef std::integral_constant<int, RING - 1 - RG> Issued_late;  // (the late group has not loaded in this step)
      wait_tile(Issued{}, 0);
      __syncthreads();
      // a step apart
      if (late) {
        wait_tile(Issued{}, 0);
        __syncthreads();
      }
      products(std::false_type{}, std::true_type{}, 0, 0);
      for (int i = 0;; i++) {
        if (late && i + 1 < n) wait_tile(Issued_late{}, i + 1);
        __syncthreads();
        const bool all = whole(i);
        if (late && !all) {
          clean(i, slot);
          __syncthreads();
        }
        if (loaded < n) load();  // where the tile before this one was
        softmax(i, all);
        if (RG == 1) {
          if (!all) clean(i, slot);
          if (i + 1 < n) wait_tile(Issued{}, i + 1);
        }
        __syncthreads();
        if (RG == 2 && !late && !all) __syncthreads();  // the other group cleans the tile
        if (!all) poison(i);
        if (i + 1 == n) break;
        const uint32_t following_slot = after_slot(slot);
        products(std::true_type{}, std::true_type{}, slot, following_slot);
        slot = following_slot;
      }
    }
    // the next unit's first tiles load while this one's outputs leave
    const Unit done = u;
    const int last = n;
    if (last > 0) products(std::true_type{}, std::false_type{}, slot, 0);
    if (RG == 2 && !late && last > 0) __syncthreads();
    __syncthreads();
    u = following, next = after;
    if (unit_at + 1 < unit1) begin();
    // rows' units and sums, by way of LDS
    l = row_sum<LANES>(l);
    if (part == 0) {
      *to_lds_at<float>(weights + 4 * mine) = m;
      *to_lds_at<float>(weights + 4 * (R + mine)) = l;
    }
    __syncthreads();
    const int fresh_o = anew(lane), go = fresh_o >> 4;
#pragma unroll
    for (int r = 0; r < NR; r++) {
      const int row = row0 + 16 * r + (fresh_o & 15), d = 16 * share + 4 * go;
      const float unit = *from_lds<float>(weights + 4 * row), all = *from_lds<float>(weights + 4 * (R + row));
      if (row >= done.rows) continue;
      if (done.part < 0) {
        const float f = inverse_sum(all, unit);
        uint16_t *dst = a.out + (done.q0 * (int64_t)G + done.f0 + row) * W + d;
#pragma unroll
        for (int e = 0; e < DB; e++) store4<BF16>(dst + 64 * e, o[r][e] * f);
      } else {
        const int64_t slot = (int64_t)done.part * a.unit_rows + at_row + row;
#pragma unroll
        for (int e = 0; e < DB; e++) *(f32x4_v *)(a.ws + slot * W + d + 64 * e) = o[r][e];
        if (share == 0 && go == 0)
          *(float2 *)(a.ws + (int64_t)a.max_partials * a.unit_rows * W + 2 * slot) = make_float2(unit, all);
      }
    }
    __syncthreads();  // before the next unit's weights
  }
}

// Plans of sets of 64 and 128 may hold sets of 32 instead, where there is little work.
template <typename S, bool BF16>
__global__ __launch_bounds__(S::threads, S::RG) void latent_attend_kernel(AbsorbedDev a) {
  if constexpr (S::NR > 1) {
    typedef Absorbed<S::W, 2, 1> Few;
    static_assert(Few::threads == S::threads && Few::lds <= S::lds, "one launch for both");
    if (uniform_word(a.starts + a.max_workers + 1) == Few::R) return absorbed_attend<Few, BF16>(a);
  }
  absorbed_attend<S, BF16>(a);
}

// Joins the parts of query rows whose keys were cut.  Few rows (a long sequence by itself,
// hundreds of parts): one workgroup per merge, row and 128 dims; 32 lanes read a part,
// 16 parts at a time.
template <int W, bool BF16>
__global__ __launch_bounds__(512) void latent_merge_kernel(AbsorbedDev a) {
  constexpr int L = 32, GR = 512 / L;
  __shared__ f32x4_v part_o[GR][L];
  __shared__ float2 part_s[GR];
  const int tid = threadIdx.x, j = blockIdx.y, lane = tid % L, grp = tid / L, d = 4 * (L * (int)blockIdx.z + lane);
  const int32_t *u = a.merges + 8 * (int64_t)blockIdx.x;
  const int q0 = u[0], f0 = u[1], rows = u[2], p0 = u[3], n = u[4];
  if (j >= rows) return;
  const float *ml = a.ws + (int64_t)a.max_partials * a.unit_rows * W;
  f32x4_v x = {0, 0, 0, 0};
  float sum = 0, mm = kUnseen;
#pragma unroll 4
  for (int i = grp; i < n; i += GR) {
    const int64_t slot = (int64_t)(p0 + i) * a.unit_rows + j;
    const float2 stat = *(const float2 *)(ml + 2 * slot);
    const f32x4_v y = *(const f32x4_v *)(a.ws + slot * W + d);
    const float high = fmaxf(mm, stat.x), was = __builtin_amdgcn_exp2f(mm - high), w = __builtin_amdgcn_exp2f(stat.x - high);
    mm = high;
    sum = fmaf(sum, was, stat.y * w);
    x = x * was + y * w;
  }
  part_o[grp][lane] = x;
  if (lane == 0) part_s[grp] = make_float2(mm, sum);
  __syncthreads();
  if (grp) return;
#pragma unroll
  for (int i = 1; i < GR; i++) mm = fmaxf(mm, part_s[i].x);
  sum = 0;
  x = (f32x4_v){0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < GR; i++) {
    const float w = __builtin_amdgcn_exp2f(part_s[i].x - mm);
    x += part_o[i][lane] * w;
    sum = fmaf(part_s[i].y, w, sum);
  }
  store4<BF16>(a.out + (q0 * (int64_t)a.heads + f0 + j) * W + d, x * inverse_sum(sum, mm));
}

// The same of many rows, with a few parts each: a wave a row, so that a plan's merges that there
// are none of cost little (181 of 128 rows: 10.6 us with a workgroup a row, 3.1 so).
template <int W, bool BF16>
__global__ __launch_bounds__(512) void latent_merge_rows_kernel(AbsorbedDev a) {
  constexpr int N = W / 256;
  const int j = 8 * blockIdx.y + (threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int32_t *u = a.merges + 8 * (int64_t)blockIdx.x;
  const int q0 = u[0], f0 = u[1], rows = u[2], p0 = u[3], n = u[4];
  if (j >= rows) return;
  const float *ml = a.ws + (int64_t)a.max_partials * a.unit_rows * W;
  f32x4_v x[N];
#pragma unroll
  for (int k = 0; k < N; k++) x[k] = (f32x4_v){0, 0, 0, 0};
  float sum = 0, mm = kUnseen;
#pragma unroll 4
  for (int i = 0; i < n; i++) {
    const int64_t slot = (int64_t)(p0 + i) * a.unit_rows + j;
    const float2 stat = *(const float2 *)(ml + 2 * slot);
    f32x4_v y[N];
#pragma unroll
    for (int k = 0; k < N; k++) y[k] = *(const f32x4_v *)(a.ws + slot * W + 4 * lane + 256 * k);
    const float high = fmaxf(mm, stat.x), was = __builtin_amdgcn_exp2f(mm - high), w = __builtin_amdgcn_exp2f(stat.x - high);
    mm = high;
    sum = fmaf(sum, was, stat.y * w);
#pragma unroll
    for (int k = 0; k < N; k++) x[k] = x[k] * was + y[k] * w;
  }
  uint16_t *dst = a.out + (q0 * (int64_t)a.heads + f0 + j) * W + 4 * lane;
#pragma unroll
  for (int k = 0; k < N; k++) store4<BF16>(dst + 256 * k, x[k] * inverse_sum(sum, mm));
}

// ------------------------------------------------------------ expanded
//
// Every head has keys of its own, D dims beside the shared rope key, and values
// of D dims, packed request after request.  A unit is up to 256 rows (tokens) of
// one head, 32 for each of eight waves, against a range of keys; tiles of 64 keys pass through LDS.
//
// Two waves share a SIMD, one of each half of the workgroup, and the halves run a
// step apart: while one issues its products (the tile before's values, this tile's
// keys), the other one's vector instructions (the softmax) have the SIMD.  A barrier ends
// each step.  The late half loads.
//
// It is bound by the products: a prompt of 8192 tokens and 16 heads of 128 + 64 dims takes
// 347 us, 990 TFLOP/s (16,384 tokens of 8 heads 645 to 663 us, 1036 to 1066; a large matrix product of the
// library reaches 1364); less is reached where rows do not fill sets of 256 or
// see few tiles, whose starts and partial results nothing covers (2048 tokens 54 us, 394
// TFLOP/s; 4 chunks of up to 701 tokens over 12,000 171 us, 614).  Heads of 64 dims are
// bound by the softmax, which is as long for them (8192 tokens 241 us, 857 TFLOP/s; vector
// instructions 47% of the cycles, products 37%).

struct ExpandedDev {
  const uint16_t *q, *k, *v, *rope;
  uint16_t *out;
  float *ws;
  const int32_t *cu, *starts, *units, *merges, *unit_starts;
  int64_t tokens, rows, q_stride, q_head_stride, k_stride, k_head_stride, v_stride, v_head_stride, rope_stride;
  int32_t batch, heads, causal, max_partials, max_units, max_workers, unit_rows;
  float scale;
};

// Where 16-byte groups lie in LDS: rows of 128 dims of a key (256 bytes) and of 64 (128 bytes)
// are read as 32 rows at one group, values as 64 bytes of four rows.
template <int DIMS>
__device__ __forceinline__ int key_place(int row, int at) { return at ^ (DIMS == 128 ? row & 15 : row >> 1 & 7); }
template <int DIMS>
__device__ __forceinline__ int value_place(int row, int at) { return at ^ (DIMS == 128 ? (row & 3) << 2 : (row >> 1 & 1) << 2); }

template <int D>
struct Expanded {
  static constexpr int KTILE = 64 * 2 * D, RTILE = 64 * 2 * kRope, VTILE = 64 * 2 * D, RING = 3;
  static constexpr int KEYS = KTILE + RTILE;
  static constexpr int OUT = 2 * D + 16;  // bytes from row to row of the outputs' way out
  static constexpr size_t tiles = RING * (KEYS + VTILE), lds = tiles + 16;
  static_assert(256 * OUT <= tiles, "outputs leave by way of the tiles' place");
};

template <int D, bool BF16>
__global__ __launch_bounds__(512, 2) void expanded_attend_kernel(ExpandedDev a) {
  typedef Half<BF16> H;
  typedef Expanded<D> S;
  constexpr int KS = (D + kRope) / 16, KK = D / 16, DT = D / 32, RING = S::RING;
  constexpr int KL = S::KTILE / 4096, RL = S::RTILE / 4096, VL = S::VTILE / 4096, BATCH = KL + RL + VL;  // loads of a wave
  constexpr int ROWS = 1024 / (2 * D);  // of keys or values that a load takes
  extern __shared__ __attribute__((aligned(256))) uint8_t smem[];
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), share = wave & 3;
  const int lane = tid & 63, c = lane & 31, hl = lane >> 5;
  const bool late = wave >= 4;
  const int h = blockIdx.x % a.heads, worker = blockIdx.x / a.heads;
  const int unit0 = max(0, uniform_word(a.unit_starts + worker)), unit1 = min(uniform_word(a.unit_starts + worker + 1), a.max_units);
  const uint32_t at = lds_address(smem), keys_at = at, values_at = at + RING * S::KEYS;
  const uint32_t bad_at = at + S::tiles;  // two masks of keys whose values are not numbers
  // a lane's first operands: its key's groups (those of other steps flip bits 5 and on, or 4 and
  // on of 64 dims), the rope key's, its four keys' values (other blocks of 32 dims flip bits 6 and on)
  const uint32_t key_lane = c * (2 * D) + 16 * key_place<D>(c, hl), rope_lane = S::KTILE + c * 128 + 16 * key_place<64>(c, hl);
  const int token = 4 * hl + (lane >> 2 & 3);
  const uint32_t value_lane = token * (2 * D) + 16 * value_place<D>(token, 2 * (lane >> 4 & 1) + (lane >> 1 & 1)) + 8 * (lane & 1);

  // the lanes hold where the first 64 requests' queries end and their keys begin
  const int ends = a.cu[min(lane, a.batch - 1) + 1];
  const int2 keys_of = make_int2(a.starts[min(lane, a.batch - 1)], a.starts[min(lane, a.batch - 1) + 1]);

  for (int unit_at = unit0; unit_at < unit1; unit_at++) {
    const int32_t *u = a.units + 8 * (int64_t)unit_at;
    const int q0 = uniform_word(u + 1), f0 = uniform_word(u + 2), rows = uniform_word(u + 3), pos0 = uniform_word(u + 4);
    const int kv0 = uniform_word(u + 5), unit_end = uniform_word(u + 6), part = uniform_word(u + 7);
    if (rows <= 0 || rows > a.unit_rows || q0 < 0 || f0 < 0 || kv0 < 0 || (int64_t)q0 + f0 + rows > a.tokens) continue;
    // the request: the last one that starts at q0 or before
    int64_t start = 0, end = 0;
    const unsigned long long past = __ballot(lane < a.batch && ends > q0);
    if (past) {
      const int b = __builtin_ctzll(past);
      start = __builtin_amdgcn_readlane(keys_of.x, b), end = __builtin_amdgcn_readlane(keys_of.y, b);
    } else {
      for (int i = 64; i < a.batch; i += 64) {
        const unsigned long long there = __ballot(i + lane < a.batch && a.cu[min(i + lane, a.batch - 1) + 1] > q0);
        if (!there) continue;
        const int b = i + __builtin_ctzll(there);
        start = uniform_word(a.starts + b), end = uniform_word(a.starts + b + 1);
        break;
      }
    }
    start = max(start, (int64_t)0);
    const int held = (int)max((int64_t)0, min(end, a.rows) - start);
    const int kv1 = min(unit_end, held), n = max(0, (kv1 - kv0 + kTile - 1) / kTile);

    // Loads of tile i's keys, or values; past the last key the last again, whose scores are masked.
    // Offsets from a tile's first row fit 32 bits (the host checks the strides).
    auto load_rows = [&](auto COUNT, auto PLACE, const uint16_t *base, int64_t stride, int per, uint32_t to, int i) {
      constexpr int count = decltype(COUNT)::value;
      const int first = kv0 + kTile * i, last = kv1 - 1 - first, from = anew(lane);
      const uint8_t *src = (const uint8_t *)(base + (start + first) * stride);
      const int lanes = 64 / per, row_in = from / lanes, group = from % lanes;
#pragma unroll
      for (int k = 0; k < count; k++) {
        const int row = per * (count * share + k) + row_in;
        const uint32_t offset = (uint32_t)min(row, last) * (uint32_t)(2 * stride) + 16 * PLACE(row, group);
        to_lds(to + 1024 * (count * share + k), src, offset);
      }
    };
    auto load_keys = [&](int i, uint32_t slot) {
      if (i >= n) return;
      load_rows(std::integral_constant<int, KL>{}, key_place<D>, a.k + h * a.k_head_stride, a.k_stride, ROWS, keys_at + slot, i);
      load_rows(std::integral_constant<int, RL>{}, key_place<64>, a.rope, a.rope_stride, 8, keys_at + slot + S::KTILE, i);
    };
    auto load_values = [&](int i, uint32_t slot) {
      if (i >= n) return;
      load_rows(std::integral_constant<int, VL>{}, value_place<D>, a.v + h * a.v_head_stride, a.v_stride, ROWS, values_at + slot, i);
    };
    if (late) {
      load_keys(0, 0);
      load_keys(1, S::KEYS);
      load_values(0, 0);
      load_keys(2, 2 * S::KEYS);
      load_values(1, S::VTILE);
    }
    if (tid < 2) *to_lds_at<uint32_t>(bad_at + 4 * tid) = 0;
    const int mine = 32 * wave + c;
    const bool live = mine < rows;
    u32x4_v q[KS];
    {
      const uint16_t *src = a.q + (int64_t)(q0 + f0 + (live ? mine : 0)) * a.q_stride + h * a.q_head_stride + 8 * hl;
      // scores keep their order when they are scaled: the sign goes to the query
      const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
      for (int s = 0; s < KS; s++) q[s] = (live ? *(const u32x4_v *)(src + 16 * s) : (u32x4_v){0, 0, 0, 0}) ^ flip;
    }
#pragma unroll
    for (int s = 0; s < KS; s++) asm volatile("" : "+v"(q[s]));
    const int hi = live ? a.causal ? min(kv1, pos0 + f0 + mine + 1) : kv1 : 0;
    const int all_hi = a.causal ? min(kv1, pos0 + f0 + 1) : kv1;  // keys that every row of the unit sees
    // (a factor of 0 would make NaN of masked scores; the least number leaves no score past 2^-21)
    const float mult = a.scale == 0.f ? 0x1p-149f : fabsf(a.scale) * kLog2e;
    // (rows that see none of the unit's keys keep a unit that no branch below is taken for)
    float m = hi > kv0 ? kNone : -H::bias, l = 0.f;
    // (keys that are the plan's own new rows are not all that a request sees that held others before)
    bool poisoned = a.starts == a.cu && pos0 > 0;
    f32x16_v o[DT], s[2];
    u32x4_v p[4];
#pragma unroll
    for (int e = 0; e < DT; e++)
#pragma unroll
      for (int k = 0; k < 16; k++) o[e][k] = 0.f;
    auto whole = [&](int i) { return kv0 + kTile * (i + 1) <= all_hi; };

    // Outputs with the values at `values` (OUT), then scores with the keys at `keys` (IN);
    // operands are read DEEP products ahead.
    auto products = [&](auto OUT, auto IN, uint32_t values, uint32_t keys) {
      constexpr int NO = decltype(OUT)::value ? 4 * DT : 0, N = NO + (decltype(IN)::value ? 2 * KS : 0), DEEP = 4;
      const uint32_t vat = values_at + values + value_lane, kat = keys_at + keys + key_lane, rat = keys_at + keys + rope_lane;
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int k = 0; k < 16; k++) s[t][k] = 0.f;
      u32x4_v w[DEEP];
      auto read = [&](int i) {
        if (i < NO) {
          const int e = i % DT, j = i / DT;
          const uint2 x = __builtin_bit_cast(uint2, read_column((vat ^ 64 * e) + 16 * j * (2 * D)));
          const uint2 y = __builtin_bit_cast(uint2, read_column((vat ^ 64 * e) + (16 * j + 8) * (2 * D)));
          return (u32x4_v){x.x, x.y, y.x, y.y};
        }
        const int t = (i - NO) % 2, k = (i - NO) / 2;
        return *from_lds<u32x4_v>(k < KK ? (kat ^ 32 * k) + 32 * t * (2 * D) : (rat ^ 32 * (k - KK)) + 32 * t * 128);
      };
#pragma unroll
      for (int i = 0; i < DEEP; i++) w[i] = read(i);
#pragma unroll
      for (int i = 0; i < N; i++) {
        if (i < NO) o[i % DT] = H::mul(w[i % DEEP], p[i / DT], o[i % DT]);
        else s[(i - NO) % 2] = H::mul(w[i % DEEP], q[(i - NO) / 2], s[(i - NO) % 2]);
        if (i + DEEP < N) w[i % DEEP] = read(i + DEEP);
      }
      __builtin_amdgcn_sched_group_barrier(0x100, NO ? 2 * DEEP : DEEP, 0);  // LDS reads
#pragma unroll
      for (int i = 0; i < N - DEEP; i++) {
        __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);  // a product
        if (i + DEEP < NO) __builtin_amdgcn_sched_group_barrier(0x100, 2, 0);
        else __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
      }
      __builtin_amdgcn_sched_group_barrier(0x8, DEEP, 0);
    };
    // Values that are not numbers would reach rows that do not see their key (0 times
    // infinity); they are taken out, and rows that do see the key are NaN.
    auto clean = [&](int i, uint32_t slot) {
      for (int j = tid & 255; j < S::VTILE / 16; j += 256) {
        const uint32_t place = values_at + slot + 16 * j;
        const u32x4_v w = *from_lds<u32x4_v>(place);
        u32x4_v x;
        uint32_t off = 0;
#pragma unroll
        for (int k = 0; k < 4; k++) x[k] = only_finite<BF16>(w[k]), off |= x[k] ^ w[k];
        if (off) {
          const int row = j / (D / 8);
          *to_lds_at<u32x4_v>(place) = x;
          __hip_atomic_fetch_or(to_lds_at<uint32_t>(bad_at + 8 * (i & 1) + 4 * (row >> 5)), 1u << (row & 31), __ATOMIC_RELAXED,
                                __HIP_MEMORY_SCOPE_WORKGROUP);
        }
      }
    };
    auto poison = [&](int i) {
      const int seen = hi - (kv0 + kTile * i);
#pragma unroll
      for (int k = 0; k < 2; k++) {
        const uint32_t bad = *from_lds<uint32_t>(bad_at + 8 * (i & 1) + 4 * k);
        const int some = seen - 32 * k;
        poisoned |= some > 0 && (bad & (some >= 32 ? ~0u : (1u << some) - 1)) != 0;
      }
    };
    auto softmax = [&](int i, bool all) {
      if (!all) {
        const int above = hi - (kv0 + kTile * i) - 4 * hl;
#pragma unroll
        for (int k = 0; k < 32; k++) {
          // all ones where the key is seen; as conditions, 32 of them would spill scalar registers
          int seen = (32 * (k >> 4) + 8 * (k >> 2 & 3) + (k & 3) - above) >> 31;
          asm("" : "+v"(seen));
          const uint32_t x = __float_as_uint(s[k >> 4][k & 15]);
          s[k >> 4][k & 15] = __uint_as_float((x & seen) | (0xff800000u & ~seen));
        }
      }
      float best = s[0][0];
#pragma unroll
      for (int k = 1; k < 32; k++) best = fmaxf(best, s[k >> 4][k & 15]);
      best = max2(best) * mult;
      float f = mult, less = m;
      // (or scores past 2^19, m of which hold no fine fractions)
      if (__any(fmaxf(best - m, fmaf(fabsf(m), 15.f / kLarge, H::top - 15.f)) > H::top)) {
        const float raised = best - m > H::top ? best - H::bias : m, shrink = __builtin_amdgcn_exp2f(m - raised);
        m = less = raised;
        l *= shrink;
#pragma unroll
        for (int e = 0; e < DT; e++) o[e] *= shrink;
        if (__any(fabsf(m) > kLarge && m > kNone)) {
          // rounded before the difference, as the maximum is, so that no weight passes what a half holds
          // (rows without a finite score need no such care, and leave the others' rounding as it is)
#pragma unroll
          for (int k = 0; k < 32; k++) s[k >> 4][k & 15] = s[k >> 4][k & 15] * mult - m;
          f = 1.f, less = 0.f;
        }
      }
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int x = 8 * j + 2 * k;
          p[j][k] = H::pack(__builtin_amdgcn_exp2f(fmaf(s[x >> 4][x & 15], f, -less)), __builtin_amdgcn_exp2f(fmaf(s[x >> 4][(x & 15) + 1], f, -less)));
          l = H::add(p[j][k], l);
        }
    };

    if (n > 0) {
      auto next_keys = [](uint32_t x) { return x + S::KEYS == RING * S::KEYS ? 0u : x + S::KEYS; };
      auto next_values = [](uint32_t x) { return x + S::VTILE == RING * S::VTILE ? 0u : x + S::VTILE; };
      uint32_t keys = 0, values = 0;  // tile i's places
      // Loads go in batches, a tile's keys and the values of the one before; the first keys by themselves.
      // The early half cleans a tile's values beside its softmax, so they are waited for a step
      // before their products (prompts of 2048 and 4096 tokens 54 and 134 us; with a step of its own 59 and 144).
      if (late) {
        if (n > 2) wait_loads<2 * BATCH>();
        else wait_loads<0>();
      }
      __syncthreads();
      if (late) {
        if (n > 2) wait_loads<BATCH>();
        else wait_loads<0>();
        __syncthreads();
      }
      products(std::false_type{}, std::true_type{}, 0, 0);
      for (int i = 0;; i++) {
        const bool all = whole(i);
        __syncthreads();
        if (late) {
          const uint32_t k3 = keys, v2 = values >= S::VTILE ? values - S::VTILE : values + (RING - 1) * S::VTILE;
          load_keys(i + 3, k3);
          load_values(i + 2, v2);
        }
        softmax(i, all);
        if (late) {
          if (i + 3 < n) wait_loads<BATCH>();
          else wait_loads<0>();
        } else if (!all) {
          clean(i, values);
        }
        __syncthreads();
        if (!all) poison(i);
        if (tid < 2) *to_lds_at<uint32_t>(bad_at + 8 * (~i & 1) + 4 * tid) = 0;  // of the next tile
        if (i + 1 == n) break;
        const uint32_t k1 = next_keys(keys);
        products(std::true_type{}, std::true_type{}, values, k1);
        keys = k1, values = next_values(values);
      }
      products(std::true_type{}, std::false_type{}, values, 0);
      if (!late) __syncthreads();
      __syncthreads();  // the outputs go where the tiles were
    }
    l = sum2(l);
    if (part < 0) {
      // through LDS, by the wave alone, so that whole rows go out 16 bytes a lane
      const float f = poisoned ? NAN : inverse_sum(l, hi > kv0 ? m : kUnseen);
      const uint32_t mine_at = at + wave * (32 * S::OUT);
#pragma unroll
      for (int e = 0; e < DT; e++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          typedef uint32_t words __attribute__((ext_vector_type(2)));
          *to_lds_at<words>(mine_at + c * S::OUT + 64 * e + 16 * k + 8 * hl) =
              (words){H::pack(o[e][4 * k] * f, o[e][4 * k + 1] * f), H::pack(o[e][4 * k + 2] * f, o[e][4 * k + 3] * f)};
        }
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      __builtin_amdgcn_wave_barrier();
      constexpr int LANES = D / 8;
#pragma unroll
      for (int i = 0; i < 32 * LANES / 64; i++) {
        const int r = (64 * i + lane) / LANES, g = (64 * i + lane) % LANES;
        const u32x4_v x = *from_lds<u32x4_v>(mine_at + r * S::OUT + 16 * g);
        if (32 * wave + r < rows) *(u32x4_v *)(a.out + ((int64_t)(q0 + f0 + 32 * wave + r) * a.heads + h) * D + 8 * g) = x;
      }
    } else {
      // as the registers hold them
      typedef float vec __attribute__((ext_vector_type(DT)));
      const int64_t slot = (int64_t)part * a.heads + h;
      float *dst = a.ws + ((slot * 8 + wave) * (16 * 64) + lane) * DT;
#pragma unroll
      for (int k = 0; k < 16; k++) {
        vec x;
#pragma unroll
        for (int e = 0; e < DT; e++) x[e] = o[e][k];
        *(vec *)(dst + k * 64 * DT) = x;
      }
      if (live && hl == 0)
        *(float2 *)(a.ws + (int64_t)a.max_partials * a.heads * a.unit_rows * D + 2 * (slot * a.unit_rows + mine)) =
            make_float2(hi > kv0 ? m : kUnseen, poisoned ? NAN : l);
    }
    __syncthreads();  // before the next unit's tiles
  }
}

// Joins the parts of units whose keys were cut: one workgroup per (merge, head) and wave of 32 rows.
template <int D, bool BF16>
__global__ __launch_bounds__(256) void expanded_merge_kernel(ExpandedDev a) {
  constexpr int DT = D / 32;
  typedef float vec __attribute__((ext_vector_type(DT)));
  const int h = blockIdx.x % a.heads, wave = blockIdx.y;
  const int32_t *u = a.merges + 8 * (int64_t)(blockIdx.x / a.heads);
  const int q0 = u[0], f0 = u[1], rows = u[2], p0 = u[3], n = u[4];
  const int lane = threadIdx.x & 63, c = lane & 31, hl = lane >> 5, four = threadIdx.x >> 6, mine = 32 * wave + c;
  if (32 * wave >= rows) return;
  const float *ml = a.ws + (int64_t)a.max_partials * a.heads * a.unit_rows * D + 2 * (int64_t)min(mine, rows - 1);
  vec x[4];
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = (vec)(0.f);
  float sum = 0, mm = kUnseen;
#pragma unroll 2
  for (int i = 0; i < n; i++) {
    const int64_t slot = (int64_t)(p0 + i) * a.heads + h;
    const float2 stat = *(const float2 *)(ml + 2 * slot * a.unit_rows);
    vec y[4];
#pragma unroll
    for (int k = 0; k < 4; k++) y[k] = *(const vec *)(a.ws + (((slot * 8 + wave) * 16 + 4 * four + k) * 64 + lane) * DT);
    const float high = fmaxf(mm, stat.x), was = __builtin_amdgcn_exp2f(mm - high), w = __builtin_amdgcn_exp2f(stat.x - high);
    mm = high;
    sum = fmaf(sum, was, stat.y * w);
#pragma unroll
    for (int k = 0; k < 4; k++) x[k] = x[k] * was + y[k] * w;
  }
  if (mine >= rows) return;
  const float f = inverse_sum(sum, mm);
  uint16_t *dst = a.out + ((int64_t)(q0 + f0 + mine) * a.heads + h) * D;
#pragma unroll
  for (int e = 0; e < DT; e++)
    store4<BF16>(dst + 32 * e + 8 * four + 4 * hl, (f32x4_v){x[0][e], x[1][e], x[2][e], x[3][e]} * f);
}

// ------------------------------------------------------------ host side

int fail(int code, const char *msg) { return sq_internal_fail(code, msg); }

int check_cache(const sq_latent_cache *c) {
  if (!c || !c->data || ((uintptr_t)c->data & 15)) return fail(SQ_EINVAL, "latent cache: null or misaligned pages");
  if ((c->latent != 256 && c->latent != 512) || c->rope != kRope)
    return fail(SQ_ESHAPE, "latent cache: a latent has 256 or 512 dims, a rope key 64");
  if (c->page_tokens <= 0 || c->page_tokens % kTile || c->page_tokens > 4096)
    return fail(SQ_ESHAPE, "latent cache: page_tokens must be a multiple of 64, at most 4096");
  if (c->dtype != SQ_BF16 && c->dtype != SQ_F16) return fail(SQ_ESTORAGE, "latent cache: pages are bf16 or fp16");
  if (c->num_pages <= 0 || c->num_pages > 0x7fffffff) return fail(SQ_EINVAL, "latent cache: page count");
  return 0;
}

std::atomic<uint64_t> g_raised[20];

// Raises a kernel's limit of dynamic LDS, once per kernel (each with an id of its own) and device.
int dynamic_lds(const void *kernel, int id, size_t most, const char *what) {
  if (most <= 65536) return 0;
  int dev = -1;
  hipError_t e = hipGetDevice(&dev);
  if (e != hipSuccess) return fail((int)e, what);
  const uint64_t bit = dev >= 0 && dev < 64 ? (uint64_t)1 << dev : 0;
  if (g_raised[id].load(std::memory_order_relaxed) & bit) return 0;
  e = hipFuncSetAttribute(kernel, hipFuncAttributeMaxDynamicSharedMemorySize, (int)most);
  if (e != hipSuccess) return fail((int)e, what);
  g_raised[id].fetch_or(bit, std::memory_order_relaxed);
  return 0;
}

template <int W, bool BF16>
int launch_absorbed(const AbsorbedDev &d, const sq_kv_schedule &s, hipStream_t st) {
  constexpr int id = 8 * (W == 512) + 4 * BF16;
  auto go = [&](auto kernel, int which, auto shape) {
    typedef decltype(shape) S;
    const int rc = dynamic_lds((const void *)kernel, id + which, S::lds, "latent attend: LDS attribute");
    if (rc) return rc;
    const unsigned grid = S::PAIR ? ((unsigned)s.max_workers + 7) / 8 * 16 : (unsigned)s.max_workers;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(S::threads), S::lds, st, d);
    return sq_internal_launched("latent_attend_kernel");
  };
  typedef Absorbed<W, 1, 1> S16;
  typedef Absorbed<W, 2, 1> S32;
  typedef Absorbed<W, 2, 2> S64;
  typedef Absorbed<W, 2, 2, true> S128;
  const int rc = s.rows == 16   ? go(latent_attend_kernel<S16, BF16>, 0, S16{})
                 : s.rows == 32 ? go(latent_attend_kernel<S32, BF16>, 1, S32{})
                 : s.rows == 64 ? go(latent_attend_kernel<S64, BF16>, 2, S64{})
                                : go(latent_attend_kernel<S128, BF16>, 3, S128{});
  if (rc) return rc;
  // Up to here empty workgroups cost less than parts in a row: two requests of 8000 tokens and 128 heads
  // (1408) 35.6 us, 38.8 by rows; one of 65,536 and 32 heads 32, 41; 32 drafts (7680) 30.8, 27.3 by rows.
  if ((int64_t)s.max_merges * s.merge_rows <= 1536)
    hipLaunchKernelGGL((latent_merge_kernel<W, BF16>), dim3((unsigned)s.max_merges, (unsigned)s.merge_rows, W / 128), dim3(512), 0, st, d);
  else
    hipLaunchKernelGGL((latent_merge_rows_kernel<W, BF16>), dim3((unsigned)s.max_merges, (unsigned)(s.merge_rows + 7) / 8), dim3(512), 0, st, d);
  return sq_internal_launched("latent_merge_kernel");
}

template <int D, bool BF16>
int launch_expanded(const ExpandedDev &d, const sq_kv_schedule &s, hipStream_t st) {
  constexpr size_t lds = Expanded<D>::lds;
  const int rc = dynamic_lds((const void *)expanded_attend_kernel<D, BF16>, 16 + 2 * (D == 128) + BF16, lds, "expanded attention: LDS attribute");
  if (rc) return rc;
  hipLaunchKernelGGL((expanded_attend_kernel<D, BF16>), dim3((unsigned)d.max_workers * d.heads), dim3(512), lds, st, d);
  const int e = sq_internal_launched("expanded_attend_kernel");
  if (e) return e;
  hipLaunchKernelGGL((expanded_merge_kernel<D, BF16>), dim3((unsigned)s.max_merges * d.heads, (unsigned)(s.merge_rows + 31) / 32), dim3(256), 0, st, d);
  return sq_internal_launched("expanded_merge_kernel");
}

}  // namespace

extern "C" {

int sq_latent_append(const sq_latent_cache *c, const sq_latent_append_args *a, const sq_rotary *r, const sq_rotary_rows *rows,
                     void *stream) {
  int rc = check_cache(c);
  if (rc) return rc;
  if (!a) return fail(SQ_EINVAL, "latent append: null arguments");
  const bool turned = rows && rows->tokens;
  if (turned && !r) return fail(SQ_EINVAL, "latent append: queries are turned by a rotary");
  if (turned && rows->dtype != c->dtype) return fail(SQ_EINVAL, "latent append: queries have the cache's type");
  if (r && r->dim > kRope) return fail(SQ_ESHAPE, "latent append: the rotation turns more dims than a rope key has");
  if (a->tokens == 0) return turned ? sq_rotary_apply(r, rows, stream) : 0;
  if (!a->latent || !a->rope || !a->slots || a->tokens < 0) return fail(SQ_EINVAL, "latent append: null pointer or size");
  if ((a->latent_stride | a->rope_stride) & 7 || (((uintptr_t)a->latent | (uintptr_t)a->rope) & 15))
    return fail(SQ_EINVAL, "latent append: strides must be multiples of 8 and starts 16-byte aligned");
  if (a->latent_stride < 0 || a->rope_stride < 0) return fail(SQ_EINVAL, "latent append: negative stride");
  LatentAppend d = {*c, *a, {}, {}, 0, 0};
  const int64_t threads = a->tokens * (c->latent / 8 + kRope / 16);
  int64_t blocks = (threads + 255) / 256;
  d.rows_blocks = (int)blocks;
  if (r) {
    rc = rotary::check(r);
    if (rc) return rc;
    if (!a->positions) return fail(SQ_EINVAL, "latent append: null positions");
    d.r = *r;
  }
  if (turned) {
    rc = rotary::check_rows(r, rows);
    if (rc) return rc;
    d.q = *rows;
    d.q_lanes = rows->heads;
    const int64_t more = rows->tokens * rows->heads * rotary::row_items(*r, *rows, false);
    if (more >= (int64_t)1 << 31) return fail(SQ_EINVAL, "latent append: too many queries for one call");
    blocks += (more + 255) / 256;
  }
  if (threads >= (int64_t)1 << 31 || blocks >= 1 << 24) return fail(SQ_EINVAL, "latent append: too many tokens for one call");
  if (c->dtype == SQ_BF16) hipLaunchKernelGGL(latent_append_kernel<SQ_BF16>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, d);
  else hipLaunchKernelGGL(latent_append_kernel<SQ_F16>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, d);
  return sq_internal_launched("latent_append_kernel");
}

int sq_latent_gather(const sq_latent_cache *c, const sq_latent_gather_args *a, void *stream) {
  const int rc = check_cache(c);
  if (rc) return rc;
  if (!a || !a->rows || !a->lens || !a->table || !a->starts || a->batch <= 0 || a->batch > SQ_KV_MAX_REQUESTS || a->requests <= 0 ||
      a->width <= 0 || a->rows_out < 0 || a->rows_out > 0x7fffffff)
    return fail(SQ_EINVAL, "latent gather: null pointer or size");
  if (a->rows_dtype != SQ_I32 && a->rows_dtype != SQ_I64) return fail(SQ_EINVAL, "latent gather: rows are int32 or int64");
  if (a->rows_out && (!a->latent || !a->rope || (((uintptr_t)a->latent | (uintptr_t)a->rope) & 15)))
    return fail(SQ_EINVAL, "latent gather: null or misaligned outputs");
  int64_t blocks = (a->rows_out + kGatherRows - 1) / kGatherRows;
  if (blocks < 1) blocks = 1;  // (starts)
  if (blocks >= 1 << 24) return fail(SQ_EINVAL, "latent gather: too many rows for one call");
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, dim3((unsigned)blocks), dim3(256), sizeof(int64_t) * (size_t)a->batch, (hipStream_t)stream, *c, *a);
  };
  c->latent == 512 ? go(latent_gather_kernel<512>) : go(latent_gather_kernel<256>);
  return sq_internal_launched("latent_gather_kernel");
}

int sq_latent_attend(const sq_latent_cache *c, const sq_latent_attend_args *a, void *stream) {
  int rc = check_cache(c);
  if (rc) return rc;
  if (!a) return fail(SQ_EINVAL, "latent attend: null arguments");
  if (a->tokens == 0) return 0;
  if (!a->q || !a->q_rope || !a->out || !a->table || a->tokens < 0 || a->requests <= 0 || a->width <= 0)
    return fail(SQ_EINVAL, "latent attend: null pointer or size");
  if ((a->q_stride | a->q_head_stride | a->rope_stride | a->rope_head_stride) & 7 ||
      (((uintptr_t)a->q | (uintptr_t)a->q_rope | (uintptr_t)a->out) & 15))
    return fail(SQ_EINVAL, "latent attend: strides must be multiples of 8 and starts 16-byte aligned");
  if (a->q_stride < 0 || a->q_head_stride < 0 || a->rope_stride < 0 || a->rope_head_stride < 0)
    return fail(SQ_EINVAL, "latent attend: negative stride");
  if (!(a->scale > -2e38f && a->scale < 2e38f)) return fail(SQ_EINVAL, "latent attend: scale must be finite, below 2e38");
  const sq_kv_schedule &s = a->schedule;
  rc = sq_internal_check_schedule(&s, a->tokens, 1);
  if (rc) return rc;
  if (s.kv_heads != 1 || s.window || (s.rows != 16 && s.rows != 32 && s.rows != 64 && s.rows != 128))
    return fail(SQ_ESHAPE, "latent attend: the schedule is for another kind of attention");
  if (!a->workspace || ((uintptr_t)a->workspace & 15)) return fail(SQ_EINVAL, "latent attend: null or misaligned workspace");
  const AbsorbedDev d = {*c, (const uint16_t *)a->q, (const uint16_t *)a->q_rope, (uint16_t *)a->out, a->workspace, a->table,
                         s.units, s.merges, s.starts, a->requests, a->tokens, a->q_stride, a->q_head_stride, a->rope_stride,
                         a->rope_head_stride, a->width, s.q_heads, s.causal, s.max_partials, s.max_units, s.max_workers, s.rows, a->scale};
  hipStream_t st = (hipStream_t)stream;
  const bool bf16 = c->dtype == SQ_BF16;
  if (c->latent == 256) return bf16 ? launch_absorbed<256, true>(d, s, st) : launch_absorbed<256, false>(d, s, st);
  return bf16 ? launch_absorbed<512, true>(d, s, st) : launch_absorbed<512, false>(d, s, st);
}

int sq_expanded_attend(const sq_expanded_attend_args *a, void *stream) {
  if (!a) return fail(SQ_EINVAL, "expanded attention: null arguments");
  if (a->tokens == 0) return 0;
  if (!a->q || !a->k || !a->v || !a->rope || !a->out || !a->cu || !a->starts || a->tokens < 0 || a->rows < 0)
    return fail(SQ_EINVAL, "expanded attention: null pointer or size");
  if (!a->workspace || ((uintptr_t)a->workspace & 15)) return fail(SQ_EINVAL, "expanded attention: null or misaligned workspace");
  if (a->dim != 64 && a->dim != 128) return fail(SQ_ESHAPE, "expanded attention: heads have 64 or 128 dims");
  if (a->dtype != SQ_BF16 && a->dtype != SQ_F16) return fail(SQ_EINVAL, "expanded attention: operands are bf16 or fp16");
  if (a->batch <= 0 || a->batch > SQ_KV_MAX_REQUESTS) return fail(SQ_EINVAL, "expanded attention: batch must be in [1, 4096]");
  if ((a->q_stride | a->q_head_stride | a->k_stride | a->k_head_stride | a->v_stride | a->v_head_stride | a->rope_stride) & 7 ||
      (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->rope | (uintptr_t)a->out) & 15))
    return fail(SQ_EINVAL, "expanded attention: strides must be multiples of 8 and starts 16-byte aligned");
  if (a->q_stride < 0 || a->q_head_stride < 0 || a->k_stride < 0 || a->k_head_stride < 0 || a->v_stride < 0 ||
      a->v_head_stride < 0 || a->rope_stride < 0)
    return fail(SQ_EINVAL, "expanded attention: negative stride");
  if (a->k_stride >= 1 << 24 || a->v_stride >= 1 << 24 || a->rope_stride >= 1 << 24)
    return fail(SQ_EINVAL, "expanded attention: rows of keys and values must be fewer than 2^24 elements apart");
  if (!(a->scale > -2e38f && a->scale < 2e38f)) return fail(SQ_EINVAL, "expanded attention: scale must be finite, below 2e38");
  const sq_kv_schedule &s = a->schedule;
  const int rc = sq_internal_check_schedule(&s, a->tokens, a->batch);
  if (rc) return rc;
  if (s.kv_heads != s.q_heads || s.window || s.few_work || s.rows != 256)
    return fail(SQ_ESHAPE, "expanded attention: the schedule is for another kind of attention");
  const ExpandedDev d = {(const uint16_t *)a->q, (const uint16_t *)a->k, (const uint16_t *)a->v, (const uint16_t *)a->rope,
                         (uint16_t *)a->out, a->workspace, a->cu, a->starts, s.units, s.merges, s.starts, a->tokens, a->rows,
                         a->q_stride, a->q_head_stride, a->k_stride, a->k_head_stride, a->v_stride, a->v_head_stride,
                         a->rope_stride, a->batch, s.q_heads, s.causal, s.max_partials, s.max_units, s.max_workers, s.rows, a->scale};
  hipStream_t st = (hipStream_t)stream;
  const bool bf16 = a->dtype == SQ_BF16;
  if (a->dim == 64) return bf16 ? launch_expanded<64, true>(d, s, st) : launch_expanded<64, false>(d, s, st);
  return bf16 ? launch_expanded<128, true>(d, s, st) : launch_expanded<128, false>(d, s, st);
}

}  // extern "C"
