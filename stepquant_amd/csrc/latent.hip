// MI355X (gfx950) kernels of latent attention: one shared vector a token (the
// latent, `W` dims, and a rope key of 64) in 16 bits in pages; the write that
// turns the rope key on the way, the dense rows of requests, attention over the
// pages with the heads' projections absorbed into queries and outputs, and
// attention over keys and values that were expanded from the latents.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>

#include "internal.h"
#include "rotary.h"
#include "stepquant_hip.h"

namespace {

typedef __bf16 bf16x2_v __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x8_v __attribute__((ext_vector_type(8)));
typedef _Float16 half2_v __attribute__((ext_vector_type(2)));
typedef _Float16 half4_v __attribute__((ext_vector_type(4)));
typedef _Float16 half8_v __attribute__((ext_vector_type(8)));
typedef short short4_v __attribute__((ext_vector_type(4)));
typedef float f32x2_v __attribute__((ext_vector_type(2)));
typedef float f32x4_v __attribute__((ext_vector_type(4)));
typedef float f32x16_v __attribute__((ext_vector_type(16)));
typedef uint32_t u32x4_v __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) void *lds_t;

constexpr int kRope = 64;
constexpr int kTile = 64;        // keys of a plan's tile
constexpr float kNone = -3e38f;  // below every score
constexpr float kLog2e = 1.4426950408889634f;

// Weights are in units of 2^m, m at most kTop and, once it is set, kBias below the
// largest score that the row has seen: it is raised only where a score passes
// kTop, so that outputs are seldom rescaled.  A half then holds all bits of a
// weight down to 2^-21 of the row's largest.
constexpr float kBias = 7.f, kTop = 15.f;

__device__ __forceinline__ int64_t load_index(const void *p, int dtype, int64_t i) {
  return dtype == SQ_I64 ? ((const int64_t *)p)[i] : (int64_t)((const int32_t *)p)[i];
}

// the two 16-bit types
template <bool BF16>
struct Half;

template <>
struct Half<true> {
  static constexpr uint32_t exponent = 0x7f80u;
  static __device__ __forceinline__ f32x4_v mul32(u32x4_v a, u32x4_v b, f32x4_v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4_v mul16(short4_v a, uint2 b, f32x4_v c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(a, __builtin_bit_cast(short4_v, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16_v mul(u32x4_v a, u32x4_v b, f32x16_v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8_v, a), __builtin_bit_cast(bf16x8_v, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_v){x, y}, bf16x2_v));
  }
  // a pair's sum, as rounded
  static __device__ __forceinline__ float sum(uint32_t w) { return __uint_as_float(w << 16) + __uint_as_float(w & 0xffff0000u); }
};

template <>
struct Half<false> {
  static constexpr uint32_t exponent = 0x7c00u;
  static __device__ __forceinline__ f32x4_v mul32(u32x4_v a, u32x4_v b, f32x4_v c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(half8_v, a), __builtin_bit_cast(half8_v, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x4_v mul16(short4_v a, uint2 b, f32x4_v c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(half4_v, a), __builtin_bit_cast(half4_v, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ f32x16_v mul(u32x4_v a, u32x4_v b, f32x16_v c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(half8_v, a), __builtin_bit_cast(half8_v, b), c, 0, 0, 0);
  }
  static __device__ __forceinline__ uint32_t pack(float x, float y) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector((f32x2_v){x, y}, half2_v));
  }
  static __device__ __forceinline__ float sum(uint32_t w) {
    return __builtin_amdgcn_fdot2(__builtin_bit_cast(half2_v, w), (half2_v){(_Float16)1.f, (_Float16)1.f}, 0.f, false);
  }
};

__device__ __forceinline__ float max2(float x) {  // over the lanes l and l ^ 32
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum2(float x) {
  const auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}
__device__ __forceinline__ float max4(float x) {  // over the lanes l, l ^ 16, l ^ 32, l ^ 48
  x = max2(x);
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}
__device__ __forceinline__ float sum4(float x) {
  x = sum2(x);
  const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
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
// key; the workgroups behind turn the queries.
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

// Rows of all requests, request after request, 64 of them a workgroup, which
// sums the requests' lengths for itself.
constexpr int kGatherRows = 64;

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
  const int W = c.latent, groups = (W + kRope) / 8;
  const int rows = (int)min((int64_t)kGatherRows, a.rows_out - first);
#pragma unroll 4
  for (int i = tid; i < rows * groups; i += 256) {
    const int r = i / groups, g = i - r * groups;
    const int64_t from = source[r];
    const u32x4_v x = from < 0 ? (u32x4_v){0, 0, 0, 0} : *(const u32x4_v *)((const uint16_t *)c.data + from * (W + kRope) + 8 * g);
    if (8 * g < W) *(u32x4_v *)((uint16_t *)a.latent + (first + r) * W + 8 * g) = x;
    else *(u32x4_v *)((uint16_t *)a.rope + (first + r) * kRope + 8 * g - W) = x;
  }
}

// ------------------------------------------------------------ tiles in LDS
//
// Rows of 16-byte groups lie one after the other, each row's groups of eight
// exchanged by an exclusive or with `mix` of the row: 16 bytes of one group of 8
// consecutive rows, and 32 of 4 consecutive rows (the transposing load of the
// values), then fall on all banks.  The load that goes from memory to LDS puts
// 64 lanes' groups side by side, so a lane asks for the group whose place it has.
__device__ __forceinline__ int mix(int row) { return (row & 3) << 1 | (row >> 2 & 1); }

// 16 bytes a lane from memory to LDS at `lds` + 16 lane.  The compiler does not
// count these loads: it would wait for all of them before any write to LDS; the
// waits are written out.  M0, which holds the place in LDS, has no other use in these kernels.
__device__ __forceinline__ void to_lds(uint32_t lds, const uint8_t *base, uint32_t offset) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" ::"s"(lds), "v"(offset), "s"(base) : "memory");
}

__device__ __forceinline__ void to_lds(uint32_t lds, const void *lane_at) {
  asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, off" ::"s"(lds), "v"(lane_at) : "memory");
}

// a word that the whole wave reads and no kernel running beside writes, by the scalar cache
__device__ __forceinline__ int uniform_word(const int32_t *p) {
  return *(const __attribute__((address_space(4))) int32_t *)(uintptr_t)p;
}

template <int N>
__device__ __forceinline__ void wait_loads() {  // until at most N are under way
  asm volatile("s_waitcnt vmcnt(%0)" ::"i"(N) : "memory");
}

// until at most N are under way, or none where fewer may be
template <int N>
__device__ __forceinline__ void wait_ring(bool some) {
  if (N && some) wait_loads<N>();
  else wait_loads<0>();
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
// products whose columns are rows of queries: a lane keeps scores, statistics
// and outputs of one row, and the rounded weights of the first product are the
// operand of the second without leaving their registers.

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

__device__ __forceinline__ Unit read_unit(const AbsorbedDev &a, int i) {
  const int32_t *u = a.units + 8 * (int64_t)i;
  const auto word = [&](int k) { return __builtin_amdgcn_readfirstlane(u[k]); };
  Unit x = {word(0), word(1), word(2), word(3), word(4), word(5), word(6), word(7)};
  if (x.rows <= 0 || x.rows > a.unit_rows || x.q0 < 0 || x.f0 < 0 || x.kv0 < 0 ||
      x.q0 + (int64_t)(x.f0 + x.rows - 1) / a.heads >= a.tokens)
    x.rows = 0;
  x.kv0 &= ~(kTile - 1);  // (a tile lies within a page)
  // a row of the table that does not exist holds no keys
  const bool held = x.rows > 0 && x.row >= 0 && x.row < a.requests;
  x.kv1 = held ? (int)min((int64_t)x.kv1, (int64_t)a.width * a.c.page_tokens) : 0;
  return x;
}

// A workgroup has RG groups of four waves and units of up to 16 RG NR rows.  Of a
// tile of 64 keys, in a ring of tiles in LDS, each wave of a group takes the
// scores of 16 keys and of the group's NR times 16 rows; the weights pass through
// LDS, and each wave of the workgroup takes the outputs of its own share of the
// dims, for all rows.  So keys are read from LDS once for each group, values once, and
// outputs need no joining.
template <int W, int RG, int NR, bool BF16>
__global__ __launch_bounds__(256 * RG, RG) void latent_attend_kernel(AbsorbedDev a) {
  typedef Half<BF16> H;
  constexpr int KD = W + kRope, ROW = 2 * KD, TILE = kTile * ROW, RING = W == 512 ? 2 : 3;
  constexpr int NW = 4 * RG, LOADS = TILE / 1024 / NW, EIGHT = KD / 64;  // loads of a wave's tile, of 8 rows
  constexpr int KS = KD / 32, DB = W / NW / 16, RT = RG * NR, R = 16 * RT, PROW = 2 * kTile + 16;
  extern __shared__ uint8_t smem[];
  uint8_t *const weights = smem + RING * TILE;           // [R] rows of 64 weights
  float *const peaks = (float *)(weights + R * PROW);    // [4][R] largest scores of 16 keys
  float *const sums = peaks + 4 * R;                     // [4][R]
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6), kg = wave & 3, rg = wave >> 2;
  const int lane = tid & 63;
  const int unit0 = max(0, __builtin_amdgcn_readfirstlane(a.starts[blockIdx.x]));
  const int unit1 = min(__builtin_amdgcn_readfirstlane(a.starts[blockIdx.x + 1]), a.max_units);
  if (unit0 >= unit1) return;
  const int G = a.heads, P = a.c.page_tokens;
  const uint32_t ring_at = lds_address(smem) + wave * (LOADS * 1024);

  const uint32_t tiles_at = lds_address(smem);
  Unit u = read_unit(a, unit0);
  int n = 0, page = 0, in_page = 0;  // of the tile that is loaded next
  const int32_t *entry = a.table;
  auto load = [&](int i) {  // tile i, into its place of the ring
    const bool known = page > 0 && page < a.c.num_pages;
    const uint8_t *base = (const uint8_t *)a.c.data + ((known ? (int64_t)page * P : 0) + in_page + wave * (kTile / NW)) * ROW;
    const uint32_t to = ring_at + i % RING * TILE;
    // a wave has 8 or 16 rows of the tile; the offsets of 8 rows' groups are made anew, too
    const int from = anew(lane);
#pragma unroll
    for (int k = 0; k < EIGHT; k++) {
      const int n = 64 * k + from, row = n / (KD / 8), at = n - row * (KD / 8);
      const uint32_t offset = row * ROW + 16 * ((at & ~7) | ((at & 7) ^ mix(row)));
#pragma unroll
      for (int j = 0; j < LOADS / EIGHT; j++) to_lds(to + 1024 * (j * EIGHT + k), base + j * (8 * ROW), offset);
    }
    in_page += kTile;
    if (in_page == P && i + 1 < n) in_page = 0, page = uniform_word(++entry);
    return known;
  };
  uint32_t known = 0;  // bit i % RING: tile i has a page
  auto begin = [&]() {
    n = max(0, (u.kv1 - u.kv0 + kTile - 1) / kTile);
    known = 0;
    if (n) {
      const int block = u.kv0 / P;
      entry = a.table + (int64_t)u.row * a.width + block;
      in_page = u.kv0 - block * P;
      page = uniform_word(entry);
    }
#pragma unroll
    for (int i = 0; i < RING; i++)
      if (i < n && load(i)) known |= 1u << i;
  };
  begin();
  for (int unit_at = unit0; unit_at < unit1; unit_at++) {
    u32x4_v q[NR][KS];
    int hi[NR];
    float l[NR], m[RT];
    f32x4_v o[RT][DB];
    const int lane_q = anew(lane), cq = lane_q & 15, gq = lane_q >> 4;
#pragma unroll
    for (int r = 0; r < NR; r++) {
      const int row = 16 * (rg * NR + r) + cq, f = u.f0 + row;
      const bool live = row < u.rows;
      const int t = live ? f / G : 0, head = live ? f - t * G : 0;
      const uint16_t *src = a.q + (u.q0 + t) * a.q_stride + head * a.q_head_stride + 8 * gq;
      const uint16_t *rope = a.rope + (u.q0 + t) * a.rope_stride + head * a.rope_head_stride + 8 * gq;
#pragma unroll
      for (int s = 0; s < KS; s++)
        q[r][s] = live ? *(const u32x4_v *)(s < W / 32 ? src + 32 * s : rope + 32 * s - W) : (u32x4_v){0, 0, 0, 0};
      hi[r] = live ? a.causal ? min(u.kv1, u.pos0 + t + 1) : u.kv1 : 0;
      l[r] = 0.f;
    }
#pragma unroll
    for (int r = 0; r < RT; r++) {
      m[r] = kNone;
#pragma unroll
      for (int e = 0; e < DB; e++) o[r][e] = (f32x4_v){0, 0, 0, 0};
    }
    // (their loads are waited for here, not by a wait for all loads in the loop)
#pragma unroll
    for (int r = 0; r < NR; r++)
#pragma unroll
      for (int s = 0; s < KS; s++) asm volatile("" : "+v"(q[r][s]));
    const float mult = a.scale * kLog2e;
    // keys that every row of the unit sees
    const int all_hi = u.rows <= 0 ? 0 : a.causal ? min(u.kv1, u.pos0 + u.f0 / G + 1) : u.kv1;
    wait_ring<LOADS * (RING - 1)>(n >= RING);
    __syncthreads();

    for (int i = 0; i < n; i++) {
      const int first = u.kv0 + kTile * i, at = i % RING * TILE;
      constexpr int CHAINS = NR == 1 ? 2 : 1;
      f32x4_v s[NR][2];
#pragma unroll
      for (int r = 0; r < NR; r++) s[r][0] = s[r][1] = (f32x4_v){0, 0, 0, 0};
      // (a lane's offsets are made anew in each part of a tile: two waves on a SIMD
      // leave no registers for them)
      const int lane_k = anew(lane), c = lane_k & 15, g = lane_k >> 4;
      // a lane's key: other steps of 32 dims flip bit 6, or lie 128 bytes on
      const uint32_t keys = tiles_at + at + (16 * kg + c) * ROW + 16 * (g ^ mix(c & 7));
#pragma unroll
      for (int k = 0; k < KS; k++) {
        const u32x4_v w = *from_lds<u32x4_v>((keys ^ 64 * (k & 1)) + 128 * (k >> 1));
#pragma unroll
        for (int r = 0; r < NR; r++) s[r][k % CHAINS] = H::mul32(w, q[r][k], s[r][k % CHAINS]);
      }
      const bool there = known >> (i % RING) & 1, whole = there && first + kTile <= all_hi;
      float x[NR][4];
#pragma unroll
      for (int r = 0; r < NR; r++) {
        float best = -INFINITY;
#pragma unroll
        for (int k = 0; k < 4; k++) {
          x[r][k] = (s[r][0][k] + s[r][1][k]) * mult;
          if (!whole) x[r][k] = there && first + 16 * kg + 4 * g + k < hi[r] ? x[r][k] : -INFINITY;
          best = fmaxf(best, x[r][k]);
        }
        best = max4(best);
        if (g == 0) peaks[kg * R + 16 * (rg * NR + r) + c] = best;
      }
      __syncthreads();
      if (!whole) {
        // What some row does not see has a weight of 0 there; infinities and NaN
        // would still reach its outputs.  (Rows that see them have them in their scores.)
        const int r0 = there ? max(0, min(kTile, all_hi - first)) : 0;
        for (int j = r0 * (KD / 8) + tid; j < kTile * (KD / 8); j += 256 * RG) {
          u32x4_v *p = (u32x4_v *)(smem + at + 16 * j);
          u32x4_v w = *p;
#pragma unroll
          for (int k = 0; k < 4; k++) w[k] = only_finite<BF16>(w[k]);
          *p = w;
        }
      }
      const int lane_p = anew(lane), cp = lane_p & 15, gp = lane_p >> 4;
#pragma unroll
      for (int r = 0; r < RT; r++) {
        const float *peak = peaks + 16 * r + cp;
        const float best = fmaxf(fmaxf(peak[0], peak[R]), fmaxf(peak[2 * R], peak[3 * R]));
        if (__any(best - m[r] > kTop)) {
          const float raised = best - m[r] > kTop ? best - kBias : m[r], shrink = __builtin_amdgcn_exp2f(m[r] - raised);
          m[r] = raised;
          if (r / NR == rg) l[r % NR] *= shrink;
#pragma unroll
          for (int e = 0; e < DB; e++) o[r][e] *= shrink;
        }
      }
#pragma unroll
      for (int r = 0; r < NR; r++) {
        float unit = m[r];
#pragma unroll
        for (int k = 1; k < RG; k++) unit = rg == k ? m[k * NR + r] : unit;
        float p[4];
#pragma unroll
        for (int k = 0; k < 4; k++) p[k] = __builtin_amdgcn_exp2f(x[r][k] - unit);
        const uint2 w = make_uint2(H::pack(p[0], p[1]), H::pack(p[2], p[3]));
        l[r] += H::sum(w.x) + H::sum(w.y);
        *(uint2 *)(weights + (16 * (rg * NR + r) + cp) * PROW + 2 * (16 * kg + 4 * gp)) = w;
      }
      __syncthreads();
      // a lane's four keys of the wave's first 16 dims: four blocks of 16 flip bits 5
      // and 6, four keys on flip bit 4
      const int lane_v = anew(lane), cv = lane_v & 15, gv = lane_v >> 4, row_v = 8 * gv + (cv >> 2);
      const uint32_t values = tiles_at + at + row_v * ROW + 128 * (wave * DB >> 2) +
                              16 * ((2 * (wave * DB & 3) + (cv >> 1 & 1)) ^ mix(row_v & 7)) + 8 * (cv & 1);
#pragma unroll
      for (int j = 0; j < 2; j++) {
        u32x4_v p[RT];
#pragma unroll
        for (int r = 0; r < RT; r++) p[r] = *(const u32x4_v *)(weights + (16 * r + cv) * PROW + 64 * j + 16 * gv);
#pragma unroll
        for (int e = 0; e < DB; e++) {
          uint2 w[2];
#pragma unroll
          for (int z = 0; z < 2; z++)
            w[z] = __builtin_bit_cast(uint2, read_column((values ^ (32 * (e & 3) + 16 * z)) + 128 * (e >> 2) + (32 * j + 4 * z) * ROW));
          const u32x4_v v = {w[0].x, w[0].y, w[1].x, w[1].y};
#pragma unroll
          for (int r = 0; r < RT; r++) o[r][e] = H::mul32(v, p[r], o[r][e]);
        }
      }
      if (i + 1 < n) wait_ring<LOADS * (RING - 2)>(i + RING <= n);
      __syncthreads();
      if (i + RING < n) {
        const uint32_t bit = 1u << (i % RING);
        known = load(i + RING) ? known | bit : known & ~bit;
      }
    }
    // the next unit's first tiles load while this one's outputs leave
    const Unit done = u;
    const int lane_o = anew(lane), co = lane_o & 15, go = lane_o >> 4;
    if (unit_at + 1 < unit1) {
      u = read_unit(a, unit_at + 1);
      begin();
    }
#pragma unroll
    for (int r = 0; r < NR; r++) {
      const float sum = sum4(l[r]);
      if (go == 0) sums[kg * R + 16 * (rg * NR + r) + co] = sum;
    }
    __syncthreads();
#pragma unroll
    for (int r = 0; r < RT; r++) {
      const int row = 16 * r + co, d = wave * (W / NW) + 4 * go;
      const float *part = sums + row;
      const float all = (part[0] + part[R]) + (part[2 * R] + part[3 * R]);
      if (row >= done.rows) continue;
      if (done.part < 0) {
        const float f = all == 0.f ? 0.f : 1.f / all;
        uint16_t *dst = a.out + (done.q0 * (int64_t)G + done.f0 + row) * W + d;
#pragma unroll
        for (int e = 0; e < DB; e++) store4<BF16>(dst + 16 * e, o[r][e] * f);
      } else {
        const int64_t slot = (int64_t)done.part * a.unit_rows + row;
#pragma unroll
        for (int e = 0; e < DB; e++) *(f32x4_v *)(a.ws + slot * W + d + 16 * e) = o[r][e];
        if (wave == 0 && go == 0)
          *(float2 *)(a.ws + (int64_t)a.max_partials * a.unit_rows * W + 2 * slot) = make_float2(m[r], all);
      }
    }
  }
}

// Joins the parts of query rows whose keys were cut: one workgroup per merge and row.
template <int W, bool BF16>
__global__ __launch_bounds__(512) void latent_merge_kernel(AbsorbedDev a) {
  constexpr int LANES = W / 4, GROUPS = 512 / LANES;
  __shared__ f32x4_v part_o[GROUPS][LANES];
  __shared__ float part_l[GROUPS], part_m[GROUPS];
  const int tid = threadIdx.x, j = blockIdx.y;
  const int32_t *u = a.merges + 8 * (int64_t)blockIdx.x;
  const int q0 = u[0], f0 = u[1], rows = u[2], p0 = u[3], n = u[4];
  if (j >= rows) return;
  const int lane = tid % LANES, grp = tid / LANES;
  const float *ml = a.ws + (int64_t)a.max_partials * a.unit_rows * W;
  f32x4_v x = {0, 0, 0, 0};
  float sum = 0, mm = kNone;
#pragma unroll 2
  for (int i = grp; i < n; i += GROUPS) {
    const int64_t slot = (int64_t)(p0 + i) * a.unit_rows + j;
    const float2 stat = *(const float2 *)(ml + 2 * slot);
    const f32x4_v y = *(const f32x4_v *)(a.ws + slot * W + 4 * lane);
    const float high = fmaxf(mm, stat.x), was = __builtin_amdgcn_exp2f(mm - high), w = __builtin_amdgcn_exp2f(stat.x - high);
    mm = high;
    sum = fmaf(sum, was, stat.y * w);
    x = x * was + y * w;
  }
  part_o[grp][lane] = x;
  if (lane == 0) part_l[grp] = sum, part_m[grp] = mm;
  __syncthreads();
  if (grp) return;
#pragma unroll
  for (int i = 1; i < GROUPS; i++) mm = fmaxf(mm, part_m[i]);
  sum = 0;
  x = (f32x4_v){0, 0, 0, 0};
#pragma unroll
  for (int i = 0; i < GROUPS; i++) {
    const float w = __builtin_amdgcn_exp2f(part_m[i] - mm);
    x += part_o[i][lane] * w;
    sum = fmaf(part_l[i], w, sum);
  }
  store4<BF16>(a.out + (q0 * (int64_t)a.heads + f0 + j) * W + 4 * lane, x * (sum == 0.f ? 0.f : 1.f / sum));
}

// ------------------------------------------------------------ expanded
//
// Every head has keys of its own, D dims beside the shared rope key, and values
// of D dims, packed request after request.  A unit is up to 256 rows (tokens) of
// one head, 32 a wave; the tiles of 64 keys pass through LDS.

struct ExpandedDev {
  const uint16_t *q, *k, *v, *rope;
  uint16_t *out;
  const int32_t *cu, *starts, *units, *unit_starts;
  int64_t tokens, rows, q_stride, q_head_stride, k_stride, k_head_stride, v_stride, v_head_stride, rope_stride;
  int32_t batch, heads, causal, max_units, max_workers, unit_rows;
  float scale;
};

template <int D, bool BF16>
__global__ __launch_bounds__(512, 2) void expanded_attend_kernel(ExpandedDev a) {
  typedef Half<BF16> H;
  constexpr int KD = D + kRope, KROW = 2 * KD, VROW = 2 * D, KTILE = 64 * KROW, VTILE = 64 * VROW;
  constexpr int KLOADS = KTILE / 8192, VLOADS = VTILE / 8192, KS = KD / 16, DT = D / 32;
  extern __shared__ uint8_t smem[];
  __shared__ unsigned long long bad_keys[2];
  uint8_t *const kt = smem, *const vt = smem + 2 * KTILE;
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, c = lane & 31, hl = lane >> 5;
  const int h = blockIdx.x % a.heads, worker = blockIdx.x / a.heads;
  const int unit0 = max(0, a.unit_starts[worker]), unit1 = min(a.unit_starts[worker + 1], a.max_units);
  const uint32_t kt_at = lds_address(kt), vt_at = lds_address(vt);

  for (int unit_at = unit0; unit_at < unit1; unit_at++) {
    const int32_t *u = a.units + 8 * (int64_t)unit_at;
    const int q0 = u[1], f0 = u[2], rows = u[3], pos0 = u[4];
    if (rows <= 0 || rows > a.unit_rows || q0 < 0 || f0 < 0 || u[5] < 0 || (int64_t)q0 + f0 + rows > a.tokens) continue;
    // the request: the last one that starts at q0 or before
    int b = -1;
    for (int i = 0; i < a.batch && b < 0; i += 64) {
      const unsigned long long past = __ballot(i + lane < a.batch && a.cu[i + lane + 1] > q0);
      if (past) b = i + __builtin_ctzll(past);
    }
    const int64_t start = b >= 0 ? max(a.starts[b], 0) : 0;
    const int held = b >= 0 ? (int)max((int64_t)0, min((int64_t)a.starts[b + 1], a.rows) - start) : 0;
    const int kv0 = u[5], kv1 = min(u[6], held), n = max(0, (kv1 - kv0 + kTile - 1) / kTile);

    // (past the last key the last again; its scores are masked)
    auto load = [&](int i) {
      const int first = kv0 + kTile * i;
#pragma unroll
      for (int k = 0; k < KLOADS; k++) {
        const int j = 512 * k + tid, row = j / (KD / 8), at = j - row * (KD / 8);
        const int g = (at & ~7) | ((at & 7) ^ mix(row & 7));
        const int64_t key = start + min(first + row, kv1 - 1);
        const uint16_t *src = g < D / 8 ? a.k + key * a.k_stride + h * a.k_head_stride + 8 * g : a.rope + key * a.rope_stride + 8 * g - D;
        to_lds(kt_at + (i & 1) * KTILE + 8192 * k + 1024 * wave, src);
      }
#pragma unroll
      for (int k = 0; k < VLOADS; k++) {
        const int j = 512 * k + tid, row = j / (D / 8), at = j - row * (D / 8);
        const int g = (at & ~7) | ((at & 7) ^ mix(row & 7));
        const int64_t key = start + min(first + row, kv1 - 1);
        to_lds(vt_at + (i & 1) * VTILE + 8192 * k + 1024 * wave, a.v + key * a.v_stride + h * a.v_head_stride + 8 * g);
      }
    };
    if (n > 0) load(0);
    const int mine = 32 * wave + c;
    const bool live = mine < rows;
    u32x4_v q[KS];
    {
      const uint16_t *src = a.q + (int64_t)(q0 + f0 + (live ? mine : 0)) * a.q_stride + h * a.q_head_stride + 8 * hl;
#pragma unroll
      for (int s = 0; s < KS; s++) q[s] = live ? *(const u32x4_v *)(src + 16 * s) : (u32x4_v){0, 0, 0, 0};
    }
    const int hi = live ? a.causal ? min(kv1, pos0 + f0 + mine + 1) : kv1 : 0;
    const int all_hi = a.causal ? min(kv1, pos0 + f0 + 1) : kv1;  // keys that every row of the unit sees
    const float mult = a.scale * kLog2e;
    float m = kNone, l = 0.f;
    bool poisoned = false;
    f32x16_v o[DT];
#pragma unroll
    for (int e = 0; e < DT; e++)
#pragma unroll
      for (int k = 0; k < 16; k++) o[e][k] = 0.f;

    for (int i = 0; i < n; i++) {
      const int first = kv0 + kTile * i;
      const bool whole = first + kTile <= all_hi;
      wait_loads<0>();
      if (tid == 0) bad_keys[i & 1] = 0;
      __syncthreads();
      if (i + 1 < n) load(i + 1);
      const uint8_t *keys = kt + (i & 1) * KTILE, *values = vt + (i & 1) * VTILE;
      const uint32_t values_at = vt_at + (i & 1) * VTILE;
      if (!whole) {
        // Values that are not numbers would reach rows that do not see their key
        // (0 times infinity); they are taken out, and rows that do see the key are NaN.
#pragma unroll
        for (int k = 0; k < VLOADS; k++) {
          const int j = 512 * k + tid, row = j / (D / 8);
          u32x4_v *p = (u32x4_v *)(values + 16 * j);
          const u32x4_v w = *p;
          u32x4_v x;
          uint32_t off = 0;
#pragma unroll
          for (int e = 0; e < 4; e++) x[e] = only_finite<BF16>(w[e]), off |= x[e] ^ w[e];
          if (off) {
            *p = x;
            atomicOr(&bad_keys[i & 1], 1ull << row);
          }
        }
        __syncthreads();
        const int seen = hi - first;
        const unsigned long long bad = bad_keys[i & 1];
        poisoned |= seen > 0 && (bad & (seen >= 64 ? ~0ull : (1ull << seen) - 1));
      }
      f32x16_v s[2];
#pragma unroll
      for (int t = 0; t < 2; t++)
#pragma unroll
        for (int k = 0; k < 16; k++) s[t][k] = 0.f;
#pragma unroll
      for (int k = 0; k < KS; k++)
#pragma unroll
        for (int t = 0; t < 2; t++) {
          const int row = 32 * t + c, g = 2 * k + hl;
          const u32x4_v w = *(const u32x4_v *)(keys + row * KROW + 16 * ((g & ~7) | ((g & 7) ^ mix(row & 7))));
          s[t] = H::mul(w, q[k], s[t]);
        }
      float best = -INFINITY;
#pragma unroll
      for (int k = 0; k < 32; k++) {
        float x = s[k >> 4][k & 15] * mult;
        if (!whole) x = first + 32 * (k >> 4) + 8 * (k >> 2 & 3) + 4 * hl + (k & 3) < hi ? x : -INFINITY;
        s[k >> 4][k & 15] = x;
        best = fmaxf(best, x);
      }
      best = max2(best);
      if (__any(best - m > kTop)) {
        const float raised = best - m > kTop ? best - kBias : m, shrink = __builtin_amdgcn_exp2f(m - raised);
        m = raised;
        l *= shrink;
#pragma unroll
        for (int e = 0; e < DT; e++) o[e] *= shrink;
      }
      u32x4_v p[4];
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const int at = 8 * j + 2 * k;
          p[j][k] = H::pack(__builtin_amdgcn_exp2f(s[at >> 4][at & 15] - m), __builtin_amdgcn_exp2f(s[at >> 4][(at & 15) + 1] - m));
          l += H::sum(p[j][k]);
        }
#pragma unroll
      for (int j = 0; j < 4; j++)
#pragma unroll
        for (int e = 0; e < DT; e++) {
          uint2 w[2];
#pragma unroll
          for (int z = 0; z < 2; z++) {
            const int row = 16 * j + 8 * z + 4 * hl + (lane >> 2 & 3), col = 32 * e + 16 * (lane >> 4 & 1) + 4 * (lane & 3);
            const int g = col / 8;
            w[z] = __builtin_bit_cast(uint2, read_column(values_at + row * VROW + 16 * ((g & ~7) | ((g & 7) ^ mix(row & 7))) + 2 * (col & 7)));
          }
          o[e] = H::mul((u32x4_v){w[0].x, w[0].y, w[1].x, w[1].y}, p[j], o[e]);
        }
    }
    l = sum2(l);
    const float f = poisoned ? NAN : l == 0.f ? 0.f : 1.f / l;
    if (live) {
      uint16_t *dst = a.out + ((int64_t)(q0 + f0 + mine) * a.heads + h) * D + 4 * hl;
#pragma unroll
      for (int e = 0; e < DT; e++)
#pragma unroll
        for (int k = 0; k < 4; k++)
          store4<BF16>(dst + 32 * e + 8 * k, (f32x4_v){o[e][4 * k], o[e][4 * k + 1], o[e][4 * k + 2], o[e][4 * k + 3]} * f);
    }
    __syncthreads();  // before the next unit's tiles
  }
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

std::atomic<uint64_t> g_raised[16];

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
  constexpr int id = 6 * (W == 512) + 3 * BF16;
  const size_t lds = (W == 512 ? 2 : 3) * kTile * 2 * (W + kRope) + s.rows * (2 * kTile + 16 + 32);
  constexpr size_t most = (W == 512 ? 2 : 3) * kTile * 2 * (W + kRope) + 64 * (2 * kTile + 16 + 32);
  auto go = [&](auto kernel, int which, int threads) {
    const int rc = dynamic_lds((const void *)kernel, id + which, most, "latent attend: LDS attribute");
    if (rc) return rc;
    hipLaunchKernelGGL(kernel, dim3((unsigned)s.max_workers), dim3(threads), lds, st, d);
    return sq_internal_launched("latent_attend_kernel");
  };
  const int rc = s.rows == 16 ? go(latent_attend_kernel<W, 1, 1, BF16>, 0, 256)
                 : s.rows == 32 ? go(latent_attend_kernel<W, 2, 1, BF16>, 1, 512)
                                : go(latent_attend_kernel<W, 2, 2, BF16>, 2, 512);
  if (rc) return rc;
  hipLaunchKernelGGL((latent_merge_kernel<W, BF16>), dim3((unsigned)s.max_merges, (unsigned)s.merge_rows), dim3(512), 0, st, d);
  return sq_internal_launched("latent_merge_kernel");
}

template <int D, bool BF16>
int launch_expanded(const ExpandedDev &d, hipStream_t st) {
  constexpr size_t lds = 2 * 64 * 2 * (2 * D + kRope);
  const int rc = dynamic_lds((const void *)expanded_attend_kernel<D, BF16>, 12 + 2 * (D == 128) + BF16, lds, "expanded attention: LDS attribute");
  if (rc) return rc;
  hipLaunchKernelGGL((expanded_attend_kernel<D, BF16>), dim3((unsigned)d.max_workers * d.heads), dim3(512), lds, st, d);
  return sq_internal_launched("expanded_attend_kernel");
}

}  // namespace

extern "C" {

int sq_latent_append(const sq_latent_cache *c, const sq_latent_append_args *a, const sq_rotary *r, const sq_rotary_rows *rows,
                     void *stream) {
  int rc = check_cache(c);
  if (rc) return rc;
  if (!a) return fail(SQ_EINVAL, "latent append: null arguments");
  if (a->tokens == 0) return 0;
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
    if (r->dim > kRope) return fail(SQ_ESHAPE, "latent append: the rotation turns more dims than a rope key has");
    d.r = *r;
  }
  if (rows && rows->tokens) {
    if (!r) return fail(SQ_EINVAL, "latent append: queries are turned by a rotary");
    rc = rotary::check_rows(r, rows);
    if (rc) return rc;
    if (rows->dtype != c->dtype) return fail(SQ_EINVAL, "latent append: queries have the cache's type");
    d.q = *rows;
    d.q_lanes = rows->heads;
    const int64_t more = rows->tokens * rows->heads * (r->dim / 16);
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
  hipLaunchKernelGGL(latent_gather_kernel, dim3((unsigned)blocks), dim3(256), sizeof(int64_t) * (size_t)a->batch, (hipStream_t)stream, *c, *a);
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
  if (!(a->scale > -3e38f && a->scale < 3e38f)) return fail(SQ_EINVAL, "latent attend: scale must be finite");
  const sq_kv_schedule &s = a->schedule;
  rc = sq_internal_check_schedule(&s, a->tokens, 1);
  if (rc) return rc;
  if (s.kv_heads != 1 || s.window || s.few_work || (s.rows != 16 && s.rows != 32 && s.rows != 64))
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
  if (a->dim != 64 && a->dim != 128) return fail(SQ_ESHAPE, "expanded attention: heads have 64 or 128 dims");
  if (a->dtype != SQ_BF16 && a->dtype != SQ_F16) return fail(SQ_EINVAL, "expanded attention: operands are bf16 or fp16");
  if (a->batch <= 0 || a->batch > SQ_KV_MAX_REQUESTS) return fail(SQ_EINVAL, "expanded attention: batch must be in [1, 4096]");
  if ((a->q_stride | a->q_head_stride | a->k_stride | a->k_head_stride | a->v_stride | a->v_head_stride | a->rope_stride) & 7 ||
      (((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->rope | (uintptr_t)a->out) & 15))
    return fail(SQ_EINVAL, "expanded attention: strides must be multiples of 8 and starts 16-byte aligned");
  if (a->q_stride < 0 || a->q_head_stride < 0 || a->k_stride < 0 || a->k_head_stride < 0 || a->v_stride < 0 ||
      a->v_head_stride < 0 || a->rope_stride < 0)
    return fail(SQ_EINVAL, "expanded attention: negative stride");
  if (!(a->scale > -3e38f && a->scale < 3e38f)) return fail(SQ_EINVAL, "expanded attention: scale must be finite");
  const sq_kv_schedule &s = a->schedule;
  const int rc = sq_internal_check_schedule(&s, a->tokens, a->batch);
  if (rc) return rc;
  if (s.kv_heads != s.q_heads || s.window || s.few_work || s.rows != 256)
    return fail(SQ_ESHAPE, "expanded attention: the schedule is for another kind of attention");
  const ExpandedDev d = {(const uint16_t *)a->q, (const uint16_t *)a->k, (const uint16_t *)a->v, (const uint16_t *)a->rope,
                         (uint16_t *)a->out, a->cu, a->starts, s.units, s.starts, a->tokens, a->rows, a->q_stride,
                         a->q_head_stride, a->k_stride, a->k_head_stride, a->v_stride, a->v_head_stride, a->rope_stride,
                         a->batch, s.q_heads, s.causal, s.max_units, s.max_workers, s.rows, a->scale};
  hipStream_t st = (hipStream_t)stream;
  const bool bf16 = a->dtype == SQ_BF16;
  if (a->dim == 64) return bf16 ? launch_expanded<64, true>(d, st) : launch_expanded<64, false>(d, st);
  return bf16 ? launch_expanded<128, true>(d, st) : launch_expanded<128, false>(d, st);
}

}  // extern "C"
