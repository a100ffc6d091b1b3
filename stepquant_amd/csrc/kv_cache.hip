// MI355X (gfx950) kernels for keys and values held in 8 bits in pages: block
// tables and slot maps from request lengths, the quantising write and its
// read-back, and attention over the pages.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <atomic>
#include <type_traits>
#include <utility>

#include "internal.h"
#include "stepquant_hip.h"

// every fused multiply-add is written out, so that codes round as defined
#pragma clang fp contract(off)

namespace {

typedef __bf16 bf16x2_v __attribute__((ext_vector_type(2)));
typedef _Float16 half2_v __attribute__((ext_vector_type(2)));
typedef _Float16 half8_v __attribute__((ext_vector_type(8)));
typedef float f32x2_v __attribute__((ext_vector_type(2)));
typedef float f32x4_v __attribute__((ext_vector_type(4)));
typedef uint32_t u32x4_v __attribute__((ext_vector_type(4)));

constexpr float kFloor = 8.673617379884035e-19f;  // 2^-60, the least peak of a block
constexpr float kNone = -3e38f;                   // a row's largest score before it has seen a key
constexpr float kLarge = 0x1p20f;                 // scores from here on (in log2) hold no fine fractions
constexpr int kTile = 64;                         // keys of one attention tile

__device__ __forceinline__ float bf_lo(uint32_t w) { return __uint_as_float(w << 16); }
__device__ __forceinline__ float bf_hi(uint32_t w) { return __uint_as_float(w & 0xffff0000u); }

// eight 16-bit elements as floats
__device__ __forceinline__ void widen8(u32x4_v w, int dtype, float x[8]) {
  if (dtype == SQ_BF16) {
#pragma unroll
    for (int i = 0; i < 4; i++) x[2 * i] = bf_lo(w[i]), x[2 * i + 1] = bf_hi(w[i]);
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t pair = w[i];  // (bit_cast of a vector's element takes the vector's first)
      const half2_v h = __builtin_bit_cast(half2_v, pair);
      x[2 * i] = (float)h[0], x[2 * i + 1] = (float)h[1];
    }
  }
}

__device__ __forceinline__ uint32_t bf16_bits(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
__device__ __forceinline__ uint32_t f16_bits(float x) { return __builtin_bit_cast(uint16_t, (_Float16)x); }

__device__ __forceinline__ int64_t load_index(const void *p, int dtype, int64_t i) {
  return dtype == SQ_I64 ? ((const int64_t *)p)[i] : (int64_t)((const int32_t *)p)[i];
}

// ------------------------------------------------------------ block tables
//
// Sums over the requests: the ends of their packed rows, of their new pages
// and of the page entries that they touch; a request is granted if its pages
// end within the free ones.  Every workgroup sums the requests for itself
// (they are few) and then serves its share of the tokens and pages, so a plan
// is one launch; the last workgroups lay out the attention layers' work.
//
// What bounds it is its chain of sums, each some 0.3 us with two barriers, and
// the first loads (0.25 MB are written for 16,384 tokens): 9.0 us for 256
// requests of one new token, 11.4 us for 48 prompts of up to 2731, commit 1.9.
// Loops stay rolled and sums take 32 bits: 9 KB of code in place of 51, whose
// fetching cost more than the branches (48 prompts 15.9 -> 13.2 us).

constexpr int kPlanThreads = 512;
constexpr int kMaxSlots = 4096;
constexpr int kPlanShare = 1024;  // tokens (and page entries) of one workgroup

struct PlanDev {
  sq_kv_tables t;
  sq_kv_plan_args p;
  int share_blocks;
};

// Sums of the threads before, and of all.  They stop at 2^31 - 1, which no size
// that fits reaches.  Every use calls one copy of the code.
constexpr uint32_t kMost = 0x7fffffffu;

struct Scan {
  uint32_t before, all;
};

template <int CTRL, int ROWS>
__device__ __forceinline__ uint32_t dpp(uint32_t x) {  // 0 where no lane is named
  return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, CTRL, ROWS, 0xf, false);
}

__device__ __forceinline__ uint32_t wave_max(uint32_t x) {  // lane 63 holds the wave's
  x = max(x, dpp<0x111, 0xf>(x));
  x = max(x, dpp<0x112, 0xf>(x));
  x = max(x, dpp<0x114, 0xf>(x));
  x = max(x, dpp<0x118, 0xf>(x));
  x = max(x, dpp<0x142, 0xa>(x));
  return max(x, dpp<0x143, 0xc>(x));
}

__device__ __attribute__((noinline)) Scan block_scan(uint32_t x) {
  __shared__ uint32_t waves[kPlanThreads / 64];
  const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
  // 16 lanes by shifts, then the ends of the rows of 16 over the rows behind
  uint32_t y = min(x + dpp<0x111, 0xf>(x), kMost);
  y = min(y + dpp<0x112, 0xf>(y), kMost);
  y = min(y + dpp<0x114, 0xf>(y), kMost);
  y = min(y + dpp<0x118, 0xf>(y), kMost);
  y = min(y + dpp<0x142, 0xa>(y), kMost);
  y = min(y + dpp<0x143, 0xc>(y), kMost);
  __syncthreads();
  if (lane == 63) waves[wave] = y;
  __syncthreads();
  const uint32_t left = __shfl_up((int)y, 1, 64);
  Scan r = {lane ? left : 0u, 0u};
#pragma unroll
  for (int w = 0; w < kPlanThreads / 64; w++) {
    const uint32_t n = waves[w];
    r.before = w < wave ? min(r.before + n, kMost) : r.before;
    r.all = min(r.all + n, kMost);
  }
  return r;
}

// First index whose entry exceeds x (n when none does).
__device__ __forceinline__ int upper_bound(const int32_t *a, int n, int x) {
  int lo = 0, hi = n;
  while (lo < hi) {
    const int mid = (lo + hi) >> 1;
    if (a[mid] > x) hi = mid;
    else lo = mid + 1;
  }
  return lo;
}

__device__ __forceinline__ uint32_t ring_at(int64_t i, int64_t capacity) {
  return (uint64_t)i >> 32 ? (uint32_t)(i % capacity) : (uint32_t)i % (uint32_t)capacity;
}

// What a workgroup knows of the requests, [batch] each, in LDS.
struct PlanLds {
  int32_t *end;    // end of the request's packed rows, at most `tokens`
  int32_t *old;    // tokens held; -1: not granted
  int32_t *tiles;  // end of its page entries (then: of its sets of query rows)
  int32_t *first;  // first of its new pages among those of the plan
  int32_t *row;
};

// One attention layer's units: sets of `rows` query rows with the tiles of
// keys that they see, the longest of a request first.
//
// Either every set is a worker of its own, and the device takes them as its
// slots come free: then the last ones to start, the short ones, decide how
// unevenly it ends.  Or the sets' tiles, one after the other, are dealt out in
// equal shares, one for each slot, and sets that lie across a border are cut
// there.  The second costs `cut_tiles` a worker (partial results to write, to
// read and to join) and is taken where it ends sooner by that count.
struct Set {  // query rows f0 to f0 + rows - 1 of request b, and the keys that they see
  int b, f0, rows, kv0, kv1, n;
};

__device__ __forceinline__ int set_rows(const sq_kv_plan_args &p, const PlanLds &L, int b) {
  return (b < p.batch ? L.end[b] : (int)p.tokens) - (b ? L.end[b - 1] : 0);
}

__device__ __forceinline__ Set find_set(const sq_kv_schedule &s, const sq_kv_plan_args &p, const PlanLds &L, int rows, int e) {
  const int G = s.q_heads / s.kv_heads;
  Set r;
  r.b = upper_bound(L.tiles, p.batch + 1, e);
  const int count = set_rows(p, L, r.b);
  r.f0 = (L.tiles[r.b] - 1 - e) * rows;  // the request's last rows first
  r.rows = min(rows, count * G - r.f0);
  r.kv0 = r.kv1 = r.n = 0;
  const int old = r.b < p.batch ? L.old[r.b] : -1;
  if (old >= 0) {
    r.kv1 = s.causal ? old + (r.f0 + r.rows - 1) / G + 1 : old + count;
    if (s.window > 0) r.kv0 = max(0, old + r.f0 / G - s.window + 1) & ~(kTile - 1);
    r.n = (r.kv1 - r.kv0 + kTile - 1) / kTile;
  }
  return r;
}

__device__ void plan_schedule(const sq_kv_schedule &s, const sq_kv_plan_args &p, const PlanLds &L) {
  __shared__ int32_t starts[kMaxSlots + 1];
  __shared__ uint32_t bounds[2];  // the most and the least tiles of a set
  const int tid = threadIdx.x, B = p.batch, G = s.q_heads / s.kv_heads;
  const int NB = B + 1;  // the last: packed rows past every request's
  uint32_t sum = 0;
  const int items = (NB + kPlanThreads - 1) / kPlanThreads;
  Scan scan;
  int rows = s.rows, min_tiles = s.min_tiles, cut_tiles = s.cut_tiles;
  if (s.few_work > 0) {
    // query rows times the tiles that they see, about: little work goes to sets of 32
#pragma unroll 1
    for (int i = 0; i < items; i++) {
      const int b = tid * items + i;
      if (b < B && L.old[b] >= 0) {
        const int count = set_rows(p, L, b);
        uint32_t keys = (uint32_t)L.old[b] + (s.causal ? count / 2 : count);
        if (s.window > 0) keys = min(keys, (uint32_t)s.window);
        sum = min(sum + (uint32_t)min((uint64_t)count * s.q_heads * (keys / kTile + 1), (uint64_t)kMost), kMost);
      }
    }
    scan = block_scan(sum);
    if (scan.all <= (uint32_t)s.few_work) rows = 32, min_tiles = s.few_min_tiles, cut_tiles = s.few_cut_tiles;
    sum = 0;
  }
#pragma unroll 1
  for (int i = 0; i < items; i++) {
    const int b = tid * items + i;
    if (b < NB) sum += (uint32_t)(set_rows(p, L, b) * G + rows - 1) / rows;
  }
  if (tid == 0) bounds[0] = 0, bounds[1] = kMost;
  scan = block_scan(sum);
  uint32_t at = scan.before;
#pragma unroll 1
  for (int i = 0; i < items; i++) {
    const int b = tid * items + i;
    if (b < NB) L.tiles[b] = (int32_t)(at += (uint32_t)(set_rows(p, L, b) * G + rows - 1) / rows);
  }
  __syncthreads();
  const int sets = (int)scan.all;
  uint32_t most = 0, least = kMost;
  sum = 0;
  Set own = {};  // the thread's last set: its only one where there are few
#pragma unroll 1
  for (int e = tid; e < sets; e += kPlanThreads) {
    own = find_set(s, p, L, rows, e);
    const uint32_t n = own.n;
    sum = min(sum + n, kMost);
    most = max(most, n);
    least = min(least, n);
  }
  most = wave_max(most), least = kMost - wave_max(kMost - least);
  if ((tid & 63) == 63) {
    atomicMax(&bounds[0], most);
    atomicMin(&bounds[1], least);
  }
  const uint32_t tiles = block_scan(sum).all;  // (its barriers stand behind the atomics, too)
  most = bounds[0], least = bounds[1];
  // worker w has the tiles from w * share on
  const uint32_t slots = max(1, s.slots / s.kv_heads), share = max((uint32_t)min_tiles, (tiles + slots - 1) / slots);
  // tiles until the last slot is done, either way
  const uint32_t whole = (uint32_t)sets <= slots ? most : max(most, (tiles + slots - 1) / slots + least);
  const bool dealt = share + cut_tiles < whole && tiles < kMost;
  const int workers = dealt ? (int)((tiles + share - 1) / share) : sets;
  if (dealt)
    for (int w = tid; w < workers; w += kPlanThreads) starts[w] = (int)kMost;
  uint32_t units = 0, merges = 0, before = 0;  // of the sets before; `before` counts their tiles
#pragma unroll 1
  for (int e0 = 0; e0 < sets; e0 += kPlanThreads) {
    const int e = e0 + tid;
    Set r = {};
    if (e < sets) r = sets <= kPlanThreads ? own : find_set(s, p, L, rows, e);
    uint32_t a = 0, u = e, m = 0;
    int w0 = 0, k = e < sets;
    if (dealt) {
      scan = block_scan(r.n);
      a = before + scan.before;
      before += scan.all;
      w0 = min(a / share, (uint32_t)workers - 1);
      if (r.n) k = (int)((a + r.n - 1) / share) - w0 + 1;
      // units and merges in one sum: fewer than 2^13 and 2^10 here
      scan = block_scan(k | (uint32_t)(k > 1) << 16);
      u = units + (scan.before & 0xffff), m = merges + (scan.before >> 16);
      units += scan.all & 0xffff, merges += scan.all >> 16;
    }
    const bool cut = k > 1;
    const uint32_t q = u - (e - m);  // units of cut sets before: all but one for each other set
    const int q0 = e < sets && r.b ? L.end[r.b - 1] : 0;
#pragma unroll 1
    for (int j = 0; j < k; j++) {
      if (u + j >= (uint32_t)s.max_units) break;
      int32_t *o = s.units + 8 * (int64_t)(u + j);
      const int t0 = j ? (int)((w0 + j) * share - a) : 0, t1 = j + 1 < k ? (int)((w0 + j + 1) * share - a) : r.n;
      o[0] = r.b < B ? L.row[r.b] : 0;
      o[1] = q0;
      o[2] = r.f0;
      o[3] = r.rows;
      o[4] = r.b < B ? L.old[r.b] : 0;
      o[5] = r.kv0 + t0 * kTile;
      o[6] = min(r.kv1, r.kv0 + t1 * kTile);
      o[7] = cut ? (int)q + j : -1;
      if (dealt) atomicMin(&starts[w0 + j], (int)u + j);
    }
    if (cut && m < (uint32_t)s.max_merges) {
      int32_t *o = s.merges + 8 * (int64_t)m;
      o[0] = q0;
      o[1] = r.f0;
      o[2] = r.rows;
      o[3] = q;
      o[4] = k;
    }
  }
  __syncthreads();
#pragma unroll 1
  for (int w = tid; w <= s.max_workers; w += kPlanThreads)
    s.starts[w] = w < workers ? dealt ? min((int)units, starts[w]) : w : dealt ? (int)units : sets;
  if (tid == 0) s.starts[s.max_workers + 1] = rows;
#pragma unroll 1
  for (int m = merges + tid; m < s.max_merges; m += kPlanThreads) s.merges[8 * (int64_t)m + 2] = 0;
}

__global__ __launch_bounds__(kPlanThreads) void kv_plan_kernel(PlanDev d) {
  extern __shared__ int32_t lds[];
  __shared__ uint32_t waves[2 * kPlanThreads / 64];
  const sq_kv_tables &t = d.t;
  const sq_kv_plan_args &p = d.p;
  const int tid = threadIdx.x, B = p.batch, P = t.page_tokens;
  PlanLds L;
  L.end = lds;
  L.old = L.end + B + 1;
  L.tiles = L.old + B + 1;
  L.first = L.tiles + B + 1;
  L.row = L.first + B + 1;
  const int items = (B + kPlanThreads - 1) / kPlanThreads, b0 = min(B, tid * items), b1 = min(B, b0 + items);
  const int64_t head = t.counters[0], tail = t.counters[1];
  const int64_t room = tail - head;
  const int most = (int)min((int64_t)p.max_count, p.tokens);  // no request with more new tokens finds room
  uint32_t sum = 0;
#pragma unroll 1
  for (int b = b0; b < b1; b++) {
    const int64_t r = load_index(p.rows, p.rows_dtype, b), n = load_index(p.counts, p.counts_dtype, b);
    const bool there = r >= 0 && r < t.requests;
    L.row[b] = there ? (int)r : -1;
    L.old[b] = there ? t.lens[r] : -1;
    // (its rows count all the same; past 2^30 the sums stop counting)
    const int count = (int)(n < 0 ? 0 : n > (1 << 30) ? 1 << 30 : n);
    L.first[b] = count;
    sum = min(sum + count, kMost);
  }
  Scan scan = block_scan(sum);
  uint32_t at = scan.before;
  sum = 0;
#pragma unroll 1
  for (int b = b0; b < b1; b++) {
    const uint32_t count = L.first[b];
    at = min(at + count, kMost);
    const int old = L.old[b];
    L.end[b] = (int)min((int64_t)at, p.tokens);
    // pages for the new tokens; -1: the request does not fit
    int need = -1;
    if (old >= 0 && count <= (uint32_t)most && at <= p.tokens && old <= (int)kMost - (int)count) {
      const uint32_t blocks = (old + count + P - 1) / P;
      if (blocks <= (uint32_t)t.width) need = blocks - ((uint32_t)old + P - 1) / P;
    }
    L.tiles[b] = need;
    sum = min(sum + max(need, 0), kMost);
  }
  scan = block_scan(sum);
  at = scan.before;
  uint32_t taken = 0;
  sum = 0;
#pragma unroll 1
  for (int b = b0; b < b1; b++) {
    const int need = L.tiles[b], old = L.old[b], count = L.first[b];
    const uint32_t first = at;
    at = min(at + max(need, 0), kMost);
    const bool ok = need == 0 || (need > 0 && at <= room);
    if (ok && need) taken = at;
    const int touched = ok && count ? ((uint32_t)old + count + P - 1) / P - old / P : 0;
    if (blockIdx.x == 0) {
      p.lens[b] = L.row[b] < 0 ? 0 : ok ? old + count : old;
      p.granted[b] = ok;
    }
    L.first[b] = ok ? (int)first : 0;
    L.old[b] = ok ? old : -1;
    L.tiles[b] = touched;
    sum += touched;
  }
  scan = block_scan(sum);
  at = scan.before;
#pragma unroll 1
  for (int b = b0; b < b1; b++) L.tiles[b] = (int)(at += L.tiles[b]);
  const int n_tiles = (int)scan.all;
  __syncthreads();
  if ((int)blockIdx.x >= d.share_blocks) {
    plan_schedule(p.schedules[blockIdx.x - d.share_blocks], p, L);
    return;
  }
  if (blockIdx.x == 0) {
    // the pages taken: up to those of the last request that needed and got one
#pragma unroll 1
    for (int k = 1; k < 64; k <<= 1) taken = max(taken, (uint32_t)__shfl_xor((int)taken, k, 64));
    __syncthreads();
    if ((tid & 63) == 0) waves[tid >> 6] = taken;
    __syncthreads();
    if (tid == 0) {
#pragma unroll 1
      for (int w = 0; w < kPlanThreads / 64; w++) taken = max(taken, waves[w]);
      p.counters[0] = head + taken;
      p.counters[1] = tail;
      p.cu[0] = 0;
    }
    for (int b = tid; b < B; b += kPlanThreads) p.cu[b + 1] = L.end[b];
  }
  const uint32_t h0 = ring_at(head, t.capacity);
  // the page of a request's block: its own, or the ring's entry that it gets
  auto page_of = [&](int b, int block) {
    const int had = (int)(((uint32_t)L.old[b] + P - 1) / P);
    uint32_t i = h0 + L.first[b] + (block - had);
    if (i >= (uint32_t)t.capacity) i -= t.capacity;
    return block < had ? t.table[(int64_t)L.row[b] * t.width + block] : t.free_pages[i];
  };
  const int from = blockIdx.x * kPlanShare, upto = from + kPlanShare;
#pragma unroll 1
  for (int i = from + tid; i < upto && i < p.tokens; i += kPlanThreads) {
    const int b = upper_bound(L.end, B, i);
    int64_t slot = -1;
    int pos = -1;
    if (b < B && L.old[b] >= 0) {
      pos = L.old[b] + i - (b ? L.end[b - 1] : 0);
      const int block = (uint32_t)pos / P;
      slot = (int64_t)page_of(b, block) * P + (pos - block * P);
    }
    p.slots[i] = slot;
    p.positions[i] = pos;
  }
#pragma unroll 1
  for (int i = from + tid; i < upto && i < p.max_tiles; i += kPlanThreads) {
    int page = 0, filled = 0, start = 0, token = 0;
    if (i < n_tiles) {
      const int b = upper_bound(L.tiles, B, i);
      const int old = L.old[b], base = b ? L.end[b - 1] : 0;
      const int block = (uint32_t)old / P + i - (b ? L.tiles[b - 1] : 0);
      page = page_of(b, block);
      if (block >= (int)(((uint32_t)old + P - 1) / P)) t.table[(int64_t)L.row[b] * t.width + block] = page;
      start = max(0, old - block * P);
      token = base + max(0, block * P - old);
      filled = min(P, old + L.end[b] - base - block * P);
    }
    p.pages[i] = page;
    p.filled[i] = filled;
    *(int2 *)(p.tiles + 2 * (int64_t)i) = make_int2(start, token);
  }
}

__global__ __launch_bounds__(256) void kv_commit_kernel(PlanDev d) {
  const int b = blockIdx.x * 256 + threadIdx.x;
  if (b == 0) d.t.counters[0] = d.p.counters[0];
  if (b >= d.p.batch) return;
  const int64_t r = load_index(d.p.rows, d.p.rows_dtype, b);
  if (r >= 0 && r < d.t.requests) d.t.lens[r] = d.p.lens[b];
}

// One workgroup: pages go back in the order of the rows and their blocks.
__global__ __launch_bounds__(kPlanThreads) void kv_release_kernel(sq_kv_tables t, const void *rows, int rows_dtype,
                                                                  int n) {
  extern __shared__ int32_t lds[];
  int32_t *end = lds, *row = lds + n;
  const int tid = threadIdx.x, items = (n + kPlanThreads - 1) / kPlanThreads;
  const int b0 = min(n, tid * items), b1 = min(n, b0 + items);
  const int64_t tail = t.counters[1];
  uint32_t sum = 0;
#pragma unroll 1
  for (int b = b0; b < b1; b++) {
    const int64_t r = load_index(rows, rows_dtype, b);
    const bool there = r >= 0 && r < t.requests;
    // the exchange leaves a row's pages to one of the entries that name it
    const int len = there ? atomicExch(&t.lens[r], 0) : 0;
    row[b] = there ? (int)r : 0;
    end[b] = len > 0 ? (int)min(((uint32_t)len + t.page_tokens - 1) / t.page_tokens, (uint32_t)t.width) : 0;
    sum = min(sum + end[b], kMost);
  }
  const Scan scan = block_scan(sum);
  uint32_t at = scan.before;
#pragma unroll 1
  for (int b = b0; b < b1; b++) end[b] = (int32_t)(at += end[b]);
  __syncthreads();
  // (more pages than there are: tables that were not filled here)
  const int64_t total = min((int64_t)scan.all, t.capacity);
  const uint32_t t0 = ring_at(tail, t.capacity);
  for (int i = tid; i < total; i += kPlanThreads) {
    const int b = upper_bound(end, n, i);
    int32_t *entry = t.table + (int64_t)row[b] * t.width + (i - (b ? end[b - 1] : 0));
    const uint32_t j = t0 + i;
    t.free_pages[j >= (uint32_t)t.capacity ? j - t.capacity : j] = *entry;
    *entry = 0;
  }
  if (tid == 0) t.counters[1] = tail + total;
}

// ------------------------------------------------------------ codes

// x / d rounded to nearest for a divisor of at most 11 significant bits, from
// its rounded reciprocal: one correction with the exact residual (as in the
// packed pages' fit; x and the quotient of normal size, which they are
// wherever the code is not 0).
__device__ __forceinline__ float quotient(float x, float d, float inv) {
  const float q = x * inv;
  return fmaf(fmaf(-q, d, x), inv, q);
}

// four values, each at most `top` in magnitude, as one word of codes
template <bool FP8>
__device__ __forceinline__ uint32_t code4(const float y[4]) {
  if (FP8) {
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return __builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], w, true);
  }
  // 1.5 * 2^23 + 128: the sum's low byte is rint(y) + 128
  uint32_t u[4];
#pragma unroll
  for (int i = 0; i < 4; i++) u[i] = __float_as_uint(y[i] + 12583040.f);
  const uint32_t a = __builtin_amdgcn_perm(u[1], u[0], 0x0c0c0400), b = __builtin_amdgcn_perm(u[3], u[2], 0x0c0c0400);
  return a | b << 16;
}

template <bool FP8>
__device__ __forceinline__ void decode4(uint32_t w, float x[4]) {
  if (FP8) {
    const auto a = __builtin_amdgcn_cvt_pk_f32_fp8(w, false), b = __builtin_amdgcn_cvt_pk_f32_fp8(w, true);
    x[0] = a[0], x[1] = a[1], x[2] = b[0], x[3] = b[1];
  } else {
#pragma unroll
    for (int i = 0; i < 4; i++) x[i] = (float)(int)(w >> 8 * i & 255) - 128.f;
  }
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// One workgroup per (page entry, head, keys or values): it finds the peak of
// its new values, brings the block's older codes to it where it grew, and
// writes the new codes.  A thread holds N groups of 8 adjacent dims between
// the two, so the new values are read once, 16 bytes a lane.  HBM bounds it:
// 16,384 tokens of 8 heads of 128 dims, 101 MB, in 20.2 us (5.0 TB/s); 64
// single tokens take 3.7 us, a launch and two loads one after the other.
template <bool FP8, int N>
__global__ __launch_bounds__(256) void kv_append_kernel(sq_kv_cache c, sq_kv_append_args a, int log_dim) {
  __shared__ uint32_t peaks[4];
  const int tid = threadIdx.x, tile = blockIdx.x, h = blockIdx.y, part = blockIdx.z;
  const int64_t page = a.pages[tile];
  const int start = a.tiles[2 * (int64_t)tile], token = a.tiles[2 * (int64_t)tile + 1], filled = a.filled[tile];
  if (page <= 0 || page >= c.num_pages) return;
  if (start < 0 || start >= filled || filled > c.page_tokens || token < 0 || token + (int64_t)filled - start > a.tokens)
    return;
  const float top = FP8 ? 448.f : 127.f;
  const uint16_t *src = (const uint16_t *)(part ? a.v : a.k) + h * (part ? a.v_head_stride : a.k_head_stride);
  const int64_t stride = part ? a.v_stride : a.k_stride;
  uint8_t *base = c.data + page * c.page_bytes + ((int64_t)(2 * h + part) * c.page_tokens << log_dim);
  const int64_t peaks_at = 2 * (int64_t)c.heads * c.page_tokens << log_dim;
  float *peak_at = (float *)(c.data + page * c.page_bytes + peaks_at) + 2 * h + part;
  const int from = start << (log_dim - 3), upto = filled << (log_dim - 3);
  u32x4_v x[N];
  uint32_t most = 0;  // magnitudes as bits: their order, and NaN above all
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int g = from + i * 256 + tid;
    if (g < upto) {
      const int e = g << 3, t = e >> log_dim;
      x[i] = *(const u32x4_v *)(src + (int64_t)(token + t - start) * stride + (e & ((1 << log_dim) - 1)));
#pragma unroll
      for (int k = 0; k < 4; k++) most = max(most, max(x[i][k] & 0x7fffu, x[i][k] >> 16 & 0x7fffu));
    }
  }
#pragma unroll
  for (int k = 1; k < 64; k <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, k, 64));
  if ((tid & 63) == 0) peaks[tid >> 6] = most;
  const float before = start ? *peak_at : kFloor;
  __syncthreads();
  most = max(max(peaks[0], peaks[1]), max(peaks[2], peaks[3]));
  const float fresh = a.dtype == SQ_BF16 ? bf_lo(most) : (float)__builtin_bit_cast(_Float16, (uint16_t)most);
  // the larger of the two, as magnitudes' bits, so that NaN stays
  const float peak = __uint_as_float(max(max(__float_as_uint(fresh), __float_as_uint(before) & 0x7fffffffu),
                                         __float_as_uint(kFloor)));
  const float inv = 1.f / peak;
  const bool good = finite(peak);
  if (tid == 0) *peak_at = peak;
  const uint32_t zero = FP8 ? 0u : 0x80808080u;
  if (peak != before) {
    // both peaks 2^-32 of their size where a code times one would pass 32 bits
    const float down = peak > 0x1p100f ? 0x1p-32f : 1.f, was = before * down, now = peak * down, inv_now = 1.f / now;
    for (int g = tid; g < from; g += 256) {
      uint2 w = *(const uint2 *)(base + 8 * (int64_t)g);
      float y[8];
      decode4<FP8>(w.x, y);
      decode4<FP8>(w.y, y + 4);
#pragma unroll
      for (int k = 0; k < 8; k++) y[k] = quotient(y[k] * was, now, inv_now);
      w.x = good ? code4<FP8>(y) : zero;
      w.y = good ? code4<FP8>(y + 4) : zero;
      *(uint2 *)(base + 8 * (int64_t)g) = w;
    }
  }
#pragma unroll
  for (int i = 0; i < N; i++) {
    const int g = from + i * 256 + tid;
    if (g < upto) {
      float y[8];
      widen8(x[i], a.dtype, y);
#pragma unroll
      for (int k = 0; k < 8; k++) y[k] = quotient(y[k], peak, inv) * top;
      *(uint2 *)(base + 8 * (int64_t)g) = make_uint2(good ? code4<FP8>(y) : zero, good ? code4<FP8>(y + 4) : zero);
    }
  }
}

// Codes times peak / top, 8 dims a lane; the same 16,384 tokens to bf16,
// 101 MB, in 17.3 us (5.8 TB/s).
template <bool FP8>
__global__ __launch_bounds__(256) void kv_decode_kernel(sq_kv_cache c, const int32_t *pages, const int32_t *filled,
                                                        void *k, void *v, int dtype, int log_dim) {
  const int tid = threadIdx.x, h = blockIdx.y, part = blockIdx.z;
  const int64_t n = blockIdx.x;
  const int64_t page = pages[n];
  const bool there = page > 0 && page < c.num_pages;
  const int held = there ? filled ? filled[n] : c.page_tokens : 0;
  const uint8_t *at = c.data + (there ? page : 0) * c.page_bytes;
  const uint8_t *base = at + ((int64_t)(2 * h + part) * c.page_tokens << log_dim);
  const int64_t peaks_at = 2 * (int64_t)c.heads * c.page_tokens << log_dim;
  const float scale = ((const float *)(at + peaks_at))[2 * h + part] / (FP8 ? 448.f : 127.f);
  void *out = part ? v : k;
  const int groups = c.page_tokens << (log_dim - 3);
  for (int g = tid; g < groups; g += 256) {
    const int t = g >> (log_dim - 3), d = (g << 3) & ((1 << log_dim) - 1);
    float x[8] = {};
    if (t < held) {
      const uint2 w = *(const uint2 *)(base + 8 * (int64_t)g);
      decode4<FP8>(w.x, x);
      decode4<FP8>(w.y, x + 4);
#pragma unroll
      for (int i = 0; i < 8; i++) x[i] *= scale;
    }
    const int64_t o = (((n * c.page_tokens + t) * c.heads + h) << log_dim) + d;
    if (dtype == SQ_F32) {
      *(float4 *)((float *)out + o) = make_float4(x[0], x[1], x[2], x[3]);
      *(float4 *)((float *)out + o + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
      u32x4_v w;
#pragma unroll
      for (int i = 0; i < 4; i++)
        w[i] = dtype == SQ_BF16 ? bf16_bits(x[2 * i]) | bf16_bits(x[2 * i + 1]) << 16
                                : f16_bits(x[2 * i]) | f16_bits(x[2 * i + 1]) << 16;
      *(u32x4_v *)((uint16_t *)out + o) = w;
    }
  }
}

// ------------------------------------------------------------ attention
//
// A unit's keys go by tiles of 64.  S^T = K Q^T and O^T = V^T P^T run as
// 16x16x32 half-precision products: a query row is a column, so a lane holds
// scores and outputs of one row only, and the rounded probabilities of one
// product are the operand of the next without leaving their registers.
// Codes of at most 8 bits are exact as halves, and so are queries: a row is
// brought near 2^14 by a power of two first, where bfloat16's 8 bits fit.  So
// scores are sums in 32 bits of exact products, times a block's peak; what is
// rounded are the probabilities, to 11 bits, and the outputs.  (bfloat16 would
// round them to 8.)  A half's exponents reach from 2^-24 to 2^15: the largest of a
// row stand near the upper end, so that small ones keep their bits.

struct AttendDev {
  sq_kv_cache c;
  const uint16_t *q;
  uint16_t *out;
  float *ws;
  const int32_t *table;
  const int32_t *units;
  const int32_t *merges;
  const int32_t *starts;
  int64_t requests, tokens, q_stride, q_head_stride;
  int32_t width, dtype, q_heads, kv_heads, causal, window, max_partials, max_units, max_workers, unit_rows;
  float scale;
};

__device__ __forceinline__ float reduce_max2(float x) {  // over the lanes l and l ^ 32
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
}

__device__ __forceinline__ float reduce_sum2(float x) {
  auto a = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(a[0]) + __uint_as_float(a[1]);
}

__device__ __forceinline__ float reduce_max4(float x) {  // over the lanes l, l ^ 16, l ^ 32, l ^ 48
  x = reduce_max2(x);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}

__device__ __forceinline__ float reduce_sum4(float x) {
  x = reduce_sum2(x);
  auto b = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// The unit of a row's weights: `below` the largest score, so that more of the
// small weights are halves.  Large scores as they are: the difference would be
// rounded, and the largest weight pass what a half holds.
__device__ __forceinline__ float weight_unit(float best, float below) {
  return fabsf(best) < kLarge ? best - below : best;
}

__device__ __forceinline__ uint32_t half2_bits(half2_v h) { return __builtin_bit_cast(uint32_t, h); }

// Two probabilities as the halves that enter the products, their sum added in
// 32 bits.  The sum is of the rounded ones, so that their rounding cancels
// where one key has most of a row (5e-5 in place of 1e-4 of an output there).
__device__ __forceinline__ uint32_t weigh2(float p0, float p1, float &sum) {
  const half2_v h = __builtin_convertvector((f32x2_v){p0, p1}, half2_v);
  sum = __builtin_amdgcn_fdot2(h, (half2_v){(_Float16)1.f, (_Float16)1.f}, sum, false);
  return half2_bits(h);
}

// two keys' codes (bytes 2 i and 2 i + 1 of w) as halves
template <bool FP8, int I>
__device__ __forceinline__ uint32_t key2(uint32_t w) {
  if (FP8) return half2_bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)w, 1.f, I));
  // 0x64uu is 1024 + u
  const uint32_t m = __builtin_amdgcn_perm(0x64646464u, w, I ? 0x04030402 : 0x04010400);
  return half2_bits(__builtin_bit_cast(half2_v, m) - (half2_v){(_Float16)1152.f, (_Float16)1152.f});
}

// One dim (byte E) of two tokens, or of eight, as halves; int8 codes come out
// 2^-10 of their size: a byte is the half u 2^-24, and one fused product
// makes it (u - 128) 2^-10.
template <bool FP8, int E>
__device__ __forceinline__ uint32_t value2(uint32_t w0, uint32_t w1) {
  if (FP8) {
    const uint32_t m = __builtin_amdgcn_perm(w1, w0, 0x0c0c0000 | (4 + E) << 8 | E);
    return half2_bits(__builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int)m, 1.f, false));
  }
  const half2_v mul = {(_Float16)16384.f, (_Float16)16384.f}, add = {(_Float16)-.125f, (_Float16)-.125f};
  const uint32_t m = __builtin_amdgcn_perm(w1, w0, 0x0c000c00 | (4 + E) << 16 | E);
  return half2_bits(__builtin_elementwise_fma(__builtin_bit_cast(half2_v, m), mul, add));
}

template <bool FP8, int E>
__device__ __forceinline__ half8_v value8(const uint32_t w[8]) {
  u32x4_v o;
#pragma unroll
  for (int i = 0; i < 4; i++) o[i] = value2<FP8, E>(w[2 * i], w[2 * i + 1]);
  return __builtin_bit_cast(half8_v, o);
}

// a code's share of the value that it stands for, beside its block's peak
template <bool FP8>
constexpr float kKeyUnit = FP8 ? 1.f / 448.f : 1.f / 127.f;
template <bool FP8>
constexpr float kValueUnit = FP8 ? 1.f / 448.f : 1024.f / 127.f;

// Outputs that are sums over keys, not yet divided by the sum of weights, are
// held 2^-40 of their size: as many of the largest values as a row can see stay
// within 32 bits, and the least peak's stay normal numbers.
constexpr float kRoom = 0x1p40f;

// The power of two that brings a bfloat16 row with this largest magnitude, in
// [2^e, 2^(e+1)), below 2^15, and its inverse.  Rows below 2^-100 come less far:
// still within a half's normal numbers, and the inverse times a scale within those
// of 32 bits.  Rows with an infinity or a NaN stay as they are.
__device__ __forceinline__ void row_shift(float most, float *shift, float *unit) {
  const int e = max((int)(__float_as_uint(most) >> 23) - 127, -100);
  *shift = e < 128 ? __uint_as_float((uint32_t)(127 + 14 - e) << 23) : 1.f;
  *unit = e < 128 ? __uint_as_float((uint32_t)(127 - 14 + e) << 23) : 1.f;
}

template <typename F, int... E>
__device__ __forceinline__ void each(F f, std::integer_sequence<int, E...>) {
  (f(std::integral_constant<int, E>{}), ...);
}

template <int N>
struct alignas(N) Bytes {  // a lane's N bytes of one token's values
  uint32_t w[N / 4];
  __device__ __forceinline__ uint32_t word(int i) const { return w[i]; }
};
template <>
struct Bytes<2> {
  uint16_t w;
  __device__ __forceinline__ uint32_t word(int) const { return w; }
};

// N values of one row's output as halves of its type
template <int N>
__device__ __forceinline__ void store_row(uint16_t *dst, bool bf16, const float *x) {
  uint32_t w[N / 2];
#pragma unroll
  for (int i = 0; i < N / 2; i++) {
    const f32x2_v y = {x[2 * i], x[2 * i + 1]};
    // both are computed: a branch for every pair costs more
    const uint32_t b = __builtin_bit_cast(uint32_t, __builtin_convertvector(y, bf16x2_v));
    const uint32_t h = half2_bits(__builtin_convertvector(y, half2_v));
    w[i] = bf16 ? b : h;
  }
  if constexpr (N == 2) *(uint32_t *)dst = w[0];
  else if constexpr (N == 4) *(uint2 *)dst = make_uint2(w[0], w[1]);
  else *(uint4 *)dst = make_uint4(w[0], w[1], w[2], w[3]);
}

typedef float f32x16_v __attribute__((ext_vector_type(16)));

// Units of up to 256 rows: 8 waves of 32 rows (of 256 dims: 128 rows at a time,
// each wave half of their outputs' dims).
// A tile is converted to halves once for the workgroup, into LDS, in the order
// in which the 32x32x16 products take it.
//
// Two waves share a SIMD, one of each half of the workgroup, and the halves
// run half a tile apart: while one issues its products (this tile's values,
// the next tile's keys: 32 of 32 cycles each at 128 dims), the other one's
// vector instructions (softmax, conversion of a later tile) have the SIMD.  A
// barrier ends each half.
//
// LDS bounds the products (each reads one operand there, 128 bytes a cycle for
// the four SIMDs, which is all that LDS gives; 64 rows a wave would halve that,
// and need twice the registers), and the vector instructions of the other half
// fill what is left.  A prompt of 8192 tokens, 32 heads over 8 of 128 dims (550
// GFLOP): 566 to 581 us, 950 to 970 TFLOP/s of the 1130 that a large library product
// reaches there; the products alone, without softmax and conversion, take 400 us.
// 256 dims 860 TFLOP/s, as tiles are converted for 128 rows, not 256; 64 dims 635
// (int8) and 665 (e4m3), as scores cost the same there and products half.  The
// halves half a tile apart took 128 dims from 827 to 670 us, peaks by way of LDS and
// masks without conditions (no scalar register spilled) to 579.  The order of
// products and LDS reads that the groups below ask for takes 3% off; wave priorities
// change nothing, nor do 8 operands ahead in place of 4.
//
// A row's sum is kept in units of 2^m, m kBias below its largest score, and its
// outputs in units of 2^(m + gap), such that the largest score and log2 of the
// block's value peak together make 2^kBias: so what enters the products as halves
// is a probability times its block's peak, whichever blocks the row's outputs come
// from.  (The gap by itself, as 32 bits do not hold it beside a score past 2^24.)
// Both are raised only when a half or a weight would pass 2^kTop; so halves hold all
// bits of a product down to 2^-24 of the row's largest and some down to 2^-34.
// Where a block's values are smaller than others by more than 2^kSmall, the sum
// takes its weights before they are halves; from the others it has all bits of
// weights down to 2^-20 of the largest.  (A prompt of 8192 tokens: 611 us with the
// largest half at 2^0 to 2^8, 615 so, 622 with 2^11 to 2^15: the narrower, the more
// tiles raise the units.)  m starts at a number below every score, so that no
// difference of it needs care.
constexpr float kBias = 10.f, kTop = 15.f, kSmall = 4.f;

template <int D, bool FP8>
__device__ __forceinline__ void attend_many(const AttendDev &a, uint4 *tiles) {
  constexpr int KS = D / 16, DT = D / 32;                   // k steps and dim tiles
  constexpr int KF = 65, KB = 2 * KS * KF, VB = 4 * DT * 64;  // uint4 of a step's keys, of a tile's keys and values
  // Of 256 dims, whose outputs would fill a wave's registers, two waves share 32
  // rows: each takes the scores of half of a tile's keys and the outputs of
  // half of the dims, and they pass each other their probabilities in LDS.
  constexpr bool PAIRS = D == 256;
  constexpr int ST = PAIRS ? 1 : 2;                         // a wave's groups of 32 keys of a tile
  constexpr int OT = PAIRS ? DT / 2 : DT;                   // a wave's dim tiles
  constexpr int WR = PAIRS ? 128 : 256;                     // rows of the workgroup at a time
  constexpr int KN = KS > 8 ? KS / 8 : 1;                   // 16-byte groups of keys of a thread
  const int tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, c = lane & 31, hl = lane >> 5;
  const int late = wave >> 2, side = PAIRS ? wave & 1 : 0, e0 = side * OT;
  const int h = blockIdx.x % a.kv_heads, worker = blockIdx.x / a.kv_heads, G = a.q_heads / a.kv_heads;
  const int unit0 = max(0, a.starts[worker]), unit1 = min(a.starts[worker + 1], a.max_units);
  for (int unit_at = unit0; unit_at < unit1; unit_at++) {
    const int32_t *u = a.units + 8 * (int64_t)unit_at;
    const int row = u[0], q0 = u[1], pos0 = u[4], kv0 = u[5], part = u[7];
    if (u[3] <= 0 || u[3] > a.unit_rows || q0 < 0 || u[2] < 0 || q0 + (int64_t)(u[2] + u[3] - 1) / G >= a.tokens)
      continue;
    const int end = row >= 0 && row < a.requests ? (int)min((int64_t)u[6], (int64_t)a.width * a.c.page_tokens) : 0;
    const int P = a.c.page_tokens, per = P / kTile, tile0 = kv0 / kTile;
    const int64_t peaks_at = 2 * (int64_t)a.c.heads * P * D + 8 * h;
    const int32_t *entries = a.table + (int64_t)row * a.width;
    uint4 *const kb = tiles, *const vb = tiles + 2 * KB;
    // the peaks of two tiles, and whether their pages exist
    float4 *const peaks = (float4 *)(vb + 2 * VB);
    // (pairs) probabilities of a wave, and its rows' units, then sums
    uint4 *const shared = (uint4 *)(peaks + 2), *const passed = shared + wave * 128, *const taken = shared + (wave ^ 1) * 128;
    float2 *const shared_m = (float2 *)(shared + 8 * 128);
    float2 *const passed_m = shared_m + wave * 32, *const taken_m = shared_m + (wave ^ 1) * 32;
    const int pages = (int)a.c.num_pages, first_key = 2 * h * P * D;
    const uint32_t page_bytes = (uint32_t)a.c.page_bytes;

    for (int turn = 0; turn < u[3]; turn += WR) {
      const int f0 = u[2] + turn, rows = min(u[3] - turn, WR);
      // (the unit's last rows may be of another turn)
      const int kv1 = a.causal ? min(end, pos0 + (f0 + rows - 1) / G + 1) : end;
      const int n = max(0, (kv1 - kv0 + kTile - 1) / kTile);
      const int first_row = 32 * (PAIRS ? wave >> 1 : wave), mine = first_row + c;
      const bool live = mine < rows;
      const int t = live ? (f0 + mine) / G : 0, head = h * G + (live ? f0 + mine - t * G : 0);
      half8_v qf[KS];
      float mult;
      auto read_queries = [&]() {
        const uint16_t *src = a.q + (int64_t)(q0 + t) * a.q_stride + head * a.q_head_stride + 8 * hl;
        u32x4_v w[KS];
#pragma unroll
        for (int s = 0; s < KS; s++) w[s] = live ? *(const u32x4_v *)(src + 16 * s) : (u32x4_v){0, 0, 0, 0};
        float unit = 1.f;
        if (a.dtype == SQ_BF16) {
          float most = 0, shift;
#pragma unroll
          for (int s = 0; s < KS; s++)
#pragma unroll
            for (int i = 0; i < 4; i++) most = fmaxf(most, fmaxf(fabsf(bf_lo(w[s][i])), fabsf(bf_hi(w[s][i]))));
          row_shift(reduce_max2(most), &shift, &unit);
#pragma unroll
          for (int s = 0; s < KS; s++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              w[s][i] = f16_bits(bf_lo(w[s][i]) * shift) | f16_bits(bf_hi(w[s][i]) * shift) << 16;
        }
        // scores keep their order when they are scaled: the sign goes to the query
        const uint32_t flip = a.scale < 0.f ? 0x80008000u : 0u;
#pragma unroll
        for (int s = 0; s < KS; s++) qf[s] = __builtin_bit_cast(half8_v, w[s] ^ flip);
        mult = fabsf(a.scale) * 1.4426950408889634f * unit * kKeyUnit<FP8>;
      };
      // what the row sees, and what every row of the wave sees whole
      const int hi = live && a.causal ? min(kv1, pos0 + t + 1) : kv1;
      const int lo = live && a.window > 0 ? pos0 + t - a.window + 1 : 0;
      const int all_hi = min(kv1, a.causal ? pos0 + (f0 + first_row) / G + 1 : kv1);
      const int all_lo = a.window > 0 ? pos0 + (f0 + max(1, min(rows, first_row + 32)) - 1) / G - a.window + 1 : 0;
      f32x16_v o[OT], s[ST];
      half8_v pf[2 * ST];
#pragma unroll
      for (int e = 0; e < OT; e++)
#pragma unroll
        for (int k = 0; k < 16; k++) o[e][k] = 0.f;
      float m = kNone, l = 0.f, gap = 0.f;
      float both = kNone, both_gap = 0.f;  // (pairs) m and gap of the outputs: the larger unit of the two waves'

      // The tiles in order; past the last one the last again, so that loads ahead
      // need no branch.  The lanes hold where the pages of 64 tiles lie (all ones:
      // a page that does not exist) and the tiles in them.
      int ahead = 0;
      uint32_t page_lo = 0, page_hi = 0, in_page = 0;
      bool known;
      const uint8_t *base;  // of the page of the tile
      auto next_tile = [&]() {
        if ((ahead & 63) == 0) {
          const int tile = tile0 + min(ahead + lane, n - 1), block = tile / per, page = entries[block];
          const uint64_t off = page > 0 && page < pages ? (uint64_t)(uint32_t)page * page_bytes : ~(uint64_t)0;
          page_lo = (uint32_t)off, page_hi = (uint32_t)(off >> 32), in_page = (tile - block * per) * (kTile * D);
        }
        const uint32_t hi = __builtin_amdgcn_readlane(page_hi, ahead & 63), lo = __builtin_amdgcn_readlane(page_lo, ahead & 63);
        known = hi != 0xffffffffu;
        base = a.c.data + (known ? (uint64_t)hi << 32 | lo : 0);
        const uint8_t *at = base + (uint32_t)(first_key + __builtin_amdgcn_readlane(in_page, ahead & 63));
        ahead++;
        return at;
      };
      u32x4_v ck[KN], ck0[KN];
      Bytes<D / 32> cv[4];
      auto load_keys = [&](u32x4_v *ck, const uint8_t *at) {
        if (KS >= 8 || wave < KS)
#pragma unroll
          for (int k = 0; k < KN; k++) ck[k] = *(const u32x4_v *)(at + 16 * (tid + 512 * k));
      };
      const int vtoken = 16 * (wave >> 1) + 8 * hl + 4 * (wave & 1);
      auto load_values = [&](const uint8_t *at) {
#pragma unroll
        for (int k = 0; k < 4; k++) cv[k] = *(const Bytes<D / 32> *)(at + (int64_t)P * D + (vtoken + k) * D + c * DT);
      };
      // keys: [32 tokens][16 dims][half of them][token] of eight dims; steps lie
      // 65 groups apart, so that a wave's writes, 8 of a token's, fall on
      // different banks
      auto put_keys = [&](const u32x4_v *ck, uint4 *dst) {
        if (KS >= 8 || wave < KS)
#pragma unroll
          for (int k = 0; k < KN; k++) {
            const int i = tid + 512 * k, token = i / KS, st = i % KS;
            uint4 *at = dst + ((token >> 5) * KS + st) * KF + (token & 31);
#pragma unroll
            for (int b = 0; b < 2; b++) {
              const uint32_t w0 = ck[k][2 * b], w1 = ck[k][2 * b + 1];
              at[32 * b] = make_uint4(key2<FP8, 0>(w0), key2<FP8, 1>(w0), key2<FP8, 0>(w1), key2<FP8, 1>(w1));
            }
          }
      };
      // values: [dim tile e][16 tokens][half][r] of the eight tokens of a
      // product's lane, for dim r D / 32 + e
      auto put_values = [&](uint4 *dst) {
        uint2 *at = (uint2 *)(dst + ((wave >> 1) * 64 + 32 * (wave & 1) + c)) + hl;
        auto one = [&](auto E) {
          constexpr int e = decltype(E)::value;
          uint32_t b[4];
#pragma unroll
          for (int k = 0; k < 4; k++) b[k] = cv[k].word(e / 4);
          at[512 * e] = make_uint2(value2<FP8, e & 3>(b[0], b[1]), value2<FP8, e & 3>(b[2], b[3]));
        };
        each(one, std::make_integer_sequence<int, DT>{});
      };
      // Outputs with one tile's values (with VALUES), then scores with another
      // one's keys; the operands are read DEEP products ahead.
      auto products = [&](auto VALUES, const uint4 *values, const uint4 *keys) {
        constexpr int NV = decltype(VALUES)::value ? 4 * OT : 0, N = NV + ST * KS, DEEP = 4;
        half8_v pv[4];
        if constexpr (!PAIRS) {
#pragma unroll
          for (int j = 0; j < 4; j++) pv[j] = pf[j];
        } else if constexpr (NV > 0) {
          // own probabilities and the other wave's, brought to one unit: units are
          // whole numbers here, so that the factors are powers of two
          const uint4 w0 = taken[lane], w1 = taken[64 + lane];
          const float2 theirs = taken_m[c];
          const float over = (theirs.x - m) + (theirs.y - gap);  // their unit above the own one
          const float high = over > 0.f ? theirs.x : m, high_gap = over > 0.f ? theirs.y : gap;
          const float rise = (high - both) + (high_gap - both_gap);
          pv[0] = pf[0], pv[1] = pf[1];
          pv[2] = __builtin_bit_cast(half8_v, w0), pv[3] = __builtin_bit_cast(half8_v, w1);
          if (__any(over != 0.f)) {
            auto scale = [&](float e0, float e1) {
              const _Float16 f0 = (_Float16)__builtin_amdgcn_exp2f(e0), f1 = (_Float16)__builtin_amdgcn_exp2f(e1);
              pv[0] *= f0, pv[1] *= f0, pv[2] *= f1, pv[3] *= f1;
            };
            scale(fmaxf(fminf(-over, 0.f), -14.f), fmaxf(fminf(over, 0.f), -14.f));
            // (in two factors where one would be too small for a half)
            if (__any(fabsf(over) > 14.f)) scale(fminf(14.f - over, 0.f), fminf(14.f + over, 0.f));
            // both go on with the larger unit, for weights and for outputs
            const float top = fmaxf(m, theirs.x);
            gap = over > 0.f ? theirs.y + (theirs.x - top) : gap + (m - top);
            l *= __builtin_amdgcn_exp2f(m - top);
            m = top;
          }
          if (__any(rise > 0.f)) {
            const float shrink = __builtin_amdgcn_exp2f(fminf(-rise, 0.f));
            if (rise > 0.f) both = high, both_gap = high_gap;
#pragma unroll
            for (int e = 0; e < OT; e++)
#pragma unroll
              for (int k = 0; k < 16; k++) o[e][k] *= shrink;
          }
        }
#pragma unroll
        for (int tt = 0; tt < ST; tt++)
#pragma unroll
          for (int k = 0; k < 16; k++) s[tt][k] = 0.f;
        uint4 w[DEEP];
        // (pairs: the wave's own half of the keys first)
        const uint4 *const near = PAIRS ? values + (4 * e0 + 2 * side) * 64 + lane : values + lane;
        const uint4 *const far = PAIRS ? values + (4 * e0 + 2 * (1 - side) - 2) * 64 + lane : near;
        const uint4 *const key = keys + side * (KS * KF) + lane;
        auto read = [&](int i) {
          if (i < NV) return (i / OT < 2 ? near : far)[(4 * (i % OT) + i / OT) * 64];
          return key[((i - NV) % ST * KS + (i - NV) / ST) * KF];
        };
#pragma unroll
        for (int i = 0; i < DEEP; i++) w[i] = read(i);
#pragma unroll
        for (int i = 0; i < N; i++) {
          const half8_v x = __builtin_bit_cast(half8_v, w[i % DEEP]);
          if (i < NV) o[i % OT] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, pv[i / OT], o[i % OT], 0, 0, 0);
          else
            s[(i - NV) % ST] = __builtin_amdgcn_mfma_f32_32x32x16_f16(x, qf[(i - NV) / ST], s[(i - NV) % ST], 0, 0, 0);
          if (i + DEEP < N) w[i % DEEP] = read(i + DEEP);
        }
        __builtin_amdgcn_sched_group_barrier(0x100, DEEP, 0);  // LDS reads
#pragma unroll
        for (int i = 0; i < N - DEEP; i++) {
          __builtin_amdgcn_sched_group_barrier(0x8, 1, 0);  // a product
          __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
        }
        __builtin_amdgcn_sched_group_barrier(0x8, DEEP, 0);
      };
      auto softmax = [&](int i) {
        const float4 peak = peaks[i & 1];
        const int first = kv0 + i * kTile;
        const bool known = __builtin_amdgcn_readfirstlane(__float_as_uint(peak.z)) != 0;
        bool some = true;
        if (!(known && first + kTile <= all_hi && first >= all_lo)) {  // some row does not see all of the tile
          const int mine = first + 32 * side + 4 * hl, above = known ? hi - mine : 0, below = lo - mine;
#pragma unroll
          for (int k = 0; k < 16 * ST; k++) {
            const int j = 32 * (k >> 4) + 8 * (k >> 2 & 3) + (k & 3);
            // all ones where below <= j < above; as conditions, 64 of them would
            // spill the loop's scalar registers
            int seen = ((j - above) & (below - 1 - j)) >> 31;
            asm("" : "+v"(seen));
            const float x = s[k >> 4][k & 15];
            s[k >> 4][k & 15] = __uint_as_float((__float_as_uint(x) & seen) | (0xff800000u & ~seen));
          }
          some = known && first < hi && first + kTile > lo;
        }
        float best = s[0][0];
#pragma unroll
        for (int k = 1; k < 16 * ST; k++) best = fmaxf(best, s[k >> 4][k & 15]);
        best = reduce_max2(best);
        // a tile that the row does not see takes no part in it, whatever its
        // peaks; a factor of 0 would make NaN of the scores that are masked
        float f = mult * peak.x;
        f = !some ? 1.f : f == 0.f ? 1e-37f : f;
        best *= f;
        // the halves are the probabilities times 2^size
        const float part = some ? __builtin_amdgcn_logf(peak.y) : 0.f;
        float size = part - gap, off = size - m;
        const float by = best - m;
        // (m of large scores, in units in which 2^20 passes kTop)
        if (__any(fmaxf(fmaxf(by, by + size), fmaxf(size * (-kTop / kSmall), fabsf(fmaxf(m, best)) * 0x1p-16f)) > kTop)) {
          const float unit = weight_unit(best, kBias), raised = fmaxf(m, PAIRS ? floorf(unit) : unit);
          const float was = gap + (m - raised), wanted = (best - raised) + (part - kBias);
          gap = fmaxf(was, PAIRS ? floorf(wanted) : wanted);
          const float shrink = __builtin_amdgcn_exp2f(was - gap);
          l *= __builtin_amdgcn_exp2f(m - raised);
          m = raised;
          if constexpr (!PAIRS) {
#pragma unroll
            for (int e = 0; e < OT; e++)
#pragma unroll
              for (int k = 0; k < 16; k++) o[e][k] *= shrink;
          }
          size = part - gap, off = size - m;
          float less = m;
          if (__any(fabsf(m) >= kLarge - kBias)) {
            // scores of which 32 bits hold no fine fractions: rounded before the difference,
            // as the maximum is, so that no weight exceeds what a half holds
#pragma unroll
            for (int k = 0; k < 16 * ST; k++) s[k >> 4][k & 15] = s[k >> 4][k & 15] * f - m;
            f = 1.f, off = size, less = 0.f;
          }
          if (__any(size < -kSmall)) {  // small values: as halves, some of their probabilities would be missing in the sum
#pragma unroll
            for (int k = 0; k < 16 * ST; k++) l += __builtin_amdgcn_exp2f(fmaf(s[k >> 4][k & 15], f, -less));
            size = -kNone;
          }
        }
        float sum = 0;
#pragma unroll
        for (int j = 0; j < 2 * ST; j++) {
          u32x4_v w;
#pragma unroll
          for (int k = 0; k < 4; k++) {
            float p[2];
#pragma unroll
            for (int b = 0; b < 2; b++) {
              const int at = 8 * j + 2 * k + b;
              p[b] = __builtin_amdgcn_exp2f(fmaf(s[at >> 4][at & 15], f, off));
            }
            w[k] = weigh2(p[0], p[1], sum);
          }
          pf[j] = __builtin_bit_cast(half8_v, w);
        }
        l = fmaf(sum, __builtin_amdgcn_exp2f(-size), l);
        if constexpr (PAIRS) {
          passed[lane] = __builtin_bit_cast(uint4, pf[0]);
          passed[64 + lane] = __builtin_bit_cast(uint4, pf[1]);
          if (hl == 0) passed_m[c] = make_float2(m, gap);
        }
      };

      float4 peak, peak0;
      const uint8_t *at = nullptr, *keys = nullptr;
      auto load_peak = [&]() {
        const float2 x = *(const float2 *)(base + peaks_at);
        peak = make_float4(x.x, x.y, known ? 1.f : 0.f, 0.f);
      };
      // the first tiles' loads go out before the queries', whose conversion they run under
      if (n > 0) {
        at = next_tile();
        load_keys(ck0, at);
        load_peak();
        peak0 = peak;
        load_values(at);
        keys = next_tile();
        load_keys(ck, keys);
        load_peak();
      }
      read_queries();
      if (n > 0) {
        // Step j of the loop needs values j and keys j + 1.  The early waves put
        // their share of them there in step j, the late ones, whose step j begins
        // half a step later, in step j - 1.
        put_keys(ck0, kb);
        if (tid == 0) peaks[0] = peak0;
        auto load = [&](const uint8_t *values, const uint8_t *keys) {
          load_values(values);
          load_keys(ck, keys);
          load_peak();
        };
        if (late) {
          put_values(vb);
          put_keys(ck, kb + KB);
          at = keys;
          keys = next_tile();
          load(at, keys);
        }
        __syncthreads();
        if (late) __syncthreads();
        products(std::false_type{}, vb, kb);
        __syncthreads();
        for (int i = 0; i < n; i++) {
          softmax(i);
          // (past the last tile: into buffers that nothing reads)
          put_values(vb + ((i + late) & 1) * VB);
          put_keys(ck, kb + ((i + late + 1) & 1) * KB);
          if (tid == 0) peaks[(i + 1) & 1] = peak;
          at = keys;
          keys = next_tile();
          load(at, keys);
          __syncthreads();
          __builtin_amdgcn_sched_barrier(0);
          products(std::true_type{}, vb + (i & 1) * VB, kb + ((i + 1) & 1) * KB);
          __builtin_amdgcn_sched_barrier(0);
          __syncthreads();
        }
        if (!late) __syncthreads();
        __syncthreads();  // the next turn writes where the last products read
      }
      l = reduce_sum2(l);
      if constexpr (PAIRS) {
        // the two waves' sums, brought to one maximum (their last products are done)
        if (hl == 0) passed_m[c] = make_float2(m, l);
        __syncthreads();
        const float2 theirs = taken_m[c];
        const float high = fmaxf(m, theirs.x);
        l = fmaf(l, __builtin_amdgcn_exp2f(m - high), theirs.y * __builtin_amdgcn_exp2f(theirs.x - high));
        m = high;
        gap = (both - high) + both_gap;
        __syncthreads();
      }
      // the outputs' unit beside the sum's, in two factors: 2^128 is in reach
      const float root = l == 0.f ? 0.f : __builtin_amdgcn_exp2f(.5f * gap), unit = root * kValueUnit<FP8>;
      if (part < 0) {
        // through LDS, by the wave alone, so that whole rows go out 16 bytes a lane
        constexpr int OD = 32 * OT, OW = OD * 2 + 8;  // a wave's dims of a row, and the bytes from row to row
        const float f = l == 0.f ? 0.f : root / l;
        uint8_t *rows_at = (uint8_t *)tiles + wave * (32 * OW);
#pragma unroll
        for (int k = 0; k < 16; k++) {
          float x[OT];
#pragma unroll
          for (int e = 0; e < OT; e++) x[e] = o[e][k] * unit * f;
          store_row<OT>((uint16_t *)(rows_at + c * OW) + (8 * (k >> 2) + 4 * hl + (k & 3)) * OT, a.dtype == SQ_BF16, x);
        }
        __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
        __builtin_amdgcn_wave_barrier();
        if constexpr (PAIRS) {
          // the wave's dims are every other group of four: 8 bytes a lane
          constexpr int LANES = OD / 4;
#pragma unroll
          for (int i = 0; i < 32 * LANES / 64; i++) {
            const int r = (64 * i + lane) / LANES, d = (64 * i + lane) % LANES, f = f0 + first_row + r;
            if (first_row + r < rows)
              *(uint2 *)(a.out + ((int64_t)(q0 + f / G) * a.q_heads + h * G + f % G) * D + 8 * d + e0) =
                  *(const uint2 *)(rows_at + r * OW + 8 * d);
          }
        } else {
          constexpr int LANES = OD / 8;
#pragma unroll
          for (int i = 0; i < 32 * LANES / 64; i++) {
            const int r = (64 * i + lane) / LANES, d = (64 * i + lane) % LANES, f = f0 + first_row + r;
            const uint2 *src = (const uint2 *)(rows_at + r * OW + 16 * d);  // (rows lie 8 bytes off a multiple of 16)
            const uint2 x0 = src[0], x1 = src[1];
            if (first_row + r < rows)
              *(uint4 *)(a.out + ((int64_t)(q0 + f / G) * a.q_heads + h * G + f % G) * D + 8 * d) =
                  make_uint4(x0.x, x0.y, x1.x, x1.y);
          }
        }
        __syncthreads();  // before the next unit's tiles
      } else {
        // as the registers hold them: a wave writes 64 OT floats in a row
        typedef float vec __attribute__((ext_vector_type(OT)));
        const int64_t slot = (int64_t)part * a.kv_heads + h;
        float *dst = a.ws + ((slot * (PAIRS ? 16 : 8) + turn / WR * 8 + wave) * (16 * 64) + lane) * OT;
#pragma unroll
        for (int k = 0; k < 16; k++) {
          vec x;
#pragma unroll
          for (int e = 0; e < OT; e++) x[e] = o[e][k] * unit * (root / kRoom);
          *(vec *)(dst + k * 64 * OT) = x;
        }
        if (live && hl == 0 && e0 == 0) {
          float *ml = a.ws + (int64_t)a.max_partials * a.kv_heads * a.unit_rows * D;
          ml += 2 * (slot * a.unit_rows + turn + mine);
          ml[0] = m;
          ml[1] = l;
        }
      }
    }
  }
}

template <int D, bool FP8>
__global__ __launch_bounds__(512, 2) void kv_attend_rows_kernel(AttendDev a) {
  extern __shared__ uint4 tiles[];
  attend_many<D, FP8>(a, tiles);
}

// 16 rows of a unit: the four waves take its tiles in turn and are joined at
// its end; keys and values go from memory to registers, in the order in which
// a product's lanes hold them (keys 16 bytes of a token, values a token's
// D / 16 bytes), so nothing passes LDS.  The next tile's keys are under way
// during a tile's softmax, and the next unit's first ones while the waves are
// joined.  Tiles of 256 dims are taken by halves, which keeps a lane within 256
// registers and two waves on a SIMD.
//
// HBM bounds it where there is enough to read: 256 requests of 4096 tokens (8
// heads of 128 dims, 2.16 GB) 356 us, 6.1 TB/s; 64 of up to 8192 (593 MB) 112
// us; one of 131,072 (270 MB) 44 us.  A short one (1000 tokens of 2 heads of 256
// dims) takes 8.4 to 9.8 us: loads of the schedule, the table, the pages and the
// partial results one after the other.  Values fetched a tile ahead as well
// cost 2 to 5% (registers), three workgroups on a CU 10 to 16%.
//
// EITHER: where the plan decides between units of 256 rows and of 32, which
// have the halves of a workgroup of 512 then.
template <int D>
constexpr int kJoin = 4 * 16 * (D + 4) + 128;  // floats of LDS

template <int D, bool FP8, bool EITHER>
__global__ __launch_bounds__(EITHER ? 512 : 256, 2) void kv_attend_kernel(AttendDev a) {
  extern __shared__ float floats[];
  if (EITHER && a.starts[a.max_workers + 1] != 32) {
    attend_many<D, FP8>(a, (uint4 *)floats);
    return;
  }
  float *const smem = floats + (EITHER ? (threadIdx.x >> 8) * kJoin<D> : 0);
  constexpr int KS = D / 32, DT = D / 16, LDO = D + 4;
  constexpr int NT = D == 256 ? 2 : 4, STEP = 16 * NT;  // 16-key groups and keys of a step
  const int tid = EITHER ? threadIdx.x & 255 : threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int lane = tid & 63, c = lane & 15, g = lane >> 4;
  // Units of 32 rows have two workgroups, which run side by side on one XCD (8
  // apart, blocks go to the 8 in turn) so that its L2 gives one of them the keys.
  const int unit_rows = EITHER ? 32 : a.unit_rows;
  const bool two = !EITHER && unit_rows == 32;
  const uint32_t id = two ? (blockIdx.x >> 4) * 8 + (blockIdx.x & 7) : blockIdx.x;
  const int at_row = EITHER ? 16 * (threadIdx.x >> 8) : two ? 2 * (blockIdx.x & 8) : 0;
  const int h = id % a.kv_heads, worker = id / a.kv_heads, G = a.q_heads / a.kv_heads;
  if (worker >= a.max_workers) return;
  const int unit0 = max(0, a.starts[worker]), unit1 = min(a.starts[worker + 1], a.max_units);
  if (unit0 >= unit1) return;
  const int P = a.c.page_tokens, per = P / STEP, log_per = 31 - __clz(per);
  const bool pow2 = (per & (per - 1)) == 0;
  const int64_t peaks_at = 2 * (int64_t)a.c.heads * P * D + 8 * h;
  auto entry_of = [&](int step) { return pow2 ? step >> log_per : step / per; };

  struct Unit {
    int row, q0, f0, rows, pos0, kv0, kv1, part, n;
  };
  auto read_unit = [&](int i) {
    const int32_t *u = a.units + 8 * (int64_t)i;
    Unit x = {u[0], u[1], u[2] + at_row, min(u[3] - at_row, 16), u[4], u[5], u[6], u[7], 0};
    if (x.rows <= 0 || u[3] > unit_rows || x.q0 < 0 || x.f0 < 0 ||
        x.q0 + (int64_t)(x.f0 + x.rows - 1) / G >= a.tokens)
      x.rows = 0;
    // a row of the table that does not exist holds no keys
    const bool held = x.rows > 0 && x.row >= 0 && x.row < a.requests;
    x.kv1 = held ? (int)min((int64_t)x.kv1, (int64_t)a.width * P) : 0;
    x.n = max(0, (x.kv1 - x.kv0 + STEP - 1) / STEP);
    return x;
  };

  Bytes<D / 16> vf[NT / 2][8];
  u32x4_v kf[NT][D / 64];
  int ids = 0, page = 0;
  const uint8_t *page_at = nullptr, *at = nullptr;
  // the lanes hold the pages of 64 of the wave's steps
  auto fetch_ids = [&](const Unit &u, int i) {
    const int mine = i + 4 * lane;
    ids = mine < u.n ? a.table[(int64_t)u.row * a.width + entry_of(u.kv0 / STEP + mine)] : 0;
  };
  auto open = [&](const Unit &u, int i) {  // step i of a unit: its page, and its keys on their way
    const int step = u.kv0 / STEP + i;
    const int p = __builtin_amdgcn_readlane(ids, (i >> 2) & 63);
    page = p > 0 && p < a.c.num_pages ? p : 0;
    page_at = a.c.data + page * a.c.page_bytes;
    at = page_at + ((int64_t)(2 * h) * P + (step - entry_of(step) * per) * STEP) * D;
#pragma unroll
    for (int t = 0; t < NT; t++)
#pragma unroll
      for (int s = 0; s < D / 64; s++) kf[t][s] = *(const u32x4_v *)(at + (16 * t + c) * D + 64 * s + 16 * g);
  };
  auto begin = [&](const Unit &u) {
    if (wave < u.n) {
      fetch_ids(u, wave);
      open(u, wave);
    }
  };

  Unit u = read_unit(unit0);
  begin(u);
  for (int unit_at = unit0; unit_at < unit1; unit_at++) {
    const Unit following = read_unit(min(unit_at + 1, unit1 - 1));
    // queries
    half8_v qf[KS];
    float mult, m = -INFINITY, l = 0.f;
    int hi, lo;
    f32x4_v o[DT];
    {
      const int f = u.f0 + c;
      const bool live = c < u.rows;
      const int t = live ? f / G : 0, head = h * G + (live ? f - t * G : 0);
      const uint16_t *src = a.q + (int64_t)(u.q0 + t) * a.q_stride + head * a.q_head_stride + 16 * g;
      u32x4_v w[D / 64][2];
#pragma unroll
      for (int s = 0; s < D / 64; s++)
#pragma unroll
        for (int k = 0; k < 2; k++) w[s][k] = live ? *(const u32x4_v *)(src + 64 * s + 8 * k) : (u32x4_v){0, 0, 0, 0};
      float unit = 1.f;
      if (a.dtype == SQ_BF16) {
        float most = 0;
#pragma unroll
        for (int s = 0; s < D / 64; s++)
#pragma unroll
          for (int k = 0; k < 2; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              most = fmaxf(most, fmaxf(fabsf(bf_lo(w[s][k][i])), fabsf(bf_hi(w[s][k][i]))));
        most = reduce_max4(most);
        float shift;
        row_shift(most, &shift, &unit);
#pragma unroll
        for (int s = 0; s < D / 64; s++)
#pragma unroll
          for (int k = 0; k < 2; k++)
#pragma unroll
            for (int i = 0; i < 4; i++)
              w[s][k][i] = f16_bits(bf_lo(w[s][k][i]) * shift) | f16_bits(bf_hi(w[s][k][i]) * shift) << 16;
      }
#pragma unroll
      for (int s = 0; s < KS; s++) qf[s] = __builtin_bit_cast(half8_v, w[s / 2][s & 1]);
      mult = a.scale * 1.4426950408889634f * unit * kKeyUnit<FP8>;
      hi = live && a.causal ? min(u.kv1, u.pos0 + t + 1) : u.kv1;
      lo = live && a.window > 0 ? u.pos0 + t - a.window + 1 : 0;
#pragma unroll
      for (int e = 0; e < DT; e++) o[e] = (f32x4_v){0, 0, 0, 0};
    }
    // steps that every row sees whole need no mask: below the first row's last
    // key and from the last row's first one on
    const int all_hi = min(u.kv1, a.causal ? u.pos0 + u.f0 / G + 1 : u.kv1);
    const int all_lo = a.window > 0 ? u.pos0 + (u.f0 + u.rows - 1) / G - a.window + 1 : 0;
    for (int i = wave; i < u.n; i += 4) {
      const float2 peak = *(const float2 *)(page_at + peaks_at);
      const int first = u.kv0 + i * STEP;
      const bool known = page != 0;
      {
        const uint8_t *vat = at + (int64_t)P * D;
#pragma unroll
        for (int s = 0; s < NT / 2; s++)
#pragma unroll
          for (int j = 0; j < 8; j++)
            vf[s][j] = *(const Bytes<D / 16> *)(vat + (32 * s + 16 * (j >> 2) + 4 * g + (j & 3)) * D + c * DT);
      }
      f32x4_v s[NT];
#pragma unroll
      for (int t = 0; t < NT; t++) {
        s[t] = (f32x4_v){0, 0, 0, 0};
#pragma unroll
        for (int k = 0; k < KS; k++) {
          u32x4_v w;
          const uint32_t w0 = kf[t][k / 2][2 * (k & 1)], w1 = kf[t][k / 2][2 * (k & 1) + 1];
          w[0] = key2<FP8, 0>(w0), w[1] = key2<FP8, 1>(w0), w[2] = key2<FP8, 0>(w1), w[3] = key2<FP8, 1>(w1);
          const half8_v kh = __builtin_bit_cast(half8_v, w);
          s[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kh, qf[k], s[t], 0, 0, 0);
        }
      }
      if (i + 4 < u.n) {
        if ((((i + 4) >> 2) & 63) == 0) fetch_ids(u, i + 4);
        open(u, i + 4);
      }
      const bool whole = known && first + STEP <= all_hi && first >= all_lo;
      half8_v pf[NT / 2];
      const float f = mult * peak.x;
      float best = -INFINITY;
#pragma unroll
      for (int t = 0; t < NT; t++)
#pragma unroll
        for (int k = 0; k < 4; k++) {
          float x = s[t][k] * f;
          if (!whole) {
            const int j = first + 16 * t + 4 * g + k;
            x = known && j < hi && j >= lo ? x : -INFINITY;
          }
          s[t][k] = x;
          best = fmaxf(best, x);
        }
      // Weights are in units of 2^m, 15 below the row's largest score: a half then
      // holds all bits of a weight down to 2^-29 of the row's largest, and some down
      // to 2^-39.
      best = fmaxf(weight_unit(reduce_max4(best), 15.f), m);
      const float base = best == -INFINITY ? 0.f : best;
      const float alpha = __builtin_amdgcn_exp2f(m - base);
      const bool keep = __all(m == best);
      m = best;
      float sum = 0;
      u32x4_v w[NT / 2];
#pragma unroll
      for (int t = 0; t < NT; t++) {
        float p[4];
#pragma unroll
        for (int k = 0; k < 4; k++) p[k] = __builtin_amdgcn_exp2f(s[t][k] - base);
#pragma unroll
        for (int k = 0; k < 2; k++) w[t >> 1][2 * (t & 1) + k] = weigh2(p[2 * k], p[2 * k + 1], sum);
      }
      l = fmaf(l, alpha, sum);
#pragma unroll
      for (int t = 0; t < NT / 2; t++) pf[t] = __builtin_bit_cast(half8_v, w[t]);
      // a row that sees none of the step takes nothing from it, whatever its peak
      const bool some = whole || (known && first < hi && first + STEP > lo);
      const float sv = some ? peak.y * (kValueUnit<FP8> / kRoom) : 0.f;
      auto value = [&](auto E) {
        constexpr int e = decltype(E)::value;
        half8_v v[NT / 2];
#pragma unroll
        for (int s2 = 0; s2 < NT / 2; s2++) {
          uint32_t w[8];
#pragma unroll
          for (int j = 0; j < 8; j++) w[j] = vf[s2][j].w[e / 4];
          v[s2] = value8<FP8, e & 3>(w);
        }
        f32x4_v x = {0, 0, 0, 0};
#pragma unroll
        for (int s2 = 0; s2 < NT / 2; s2++) x = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[s2], pf[s2], x, 0, 0, 0);
#pragma unroll
        for (int k = 0; k < 4; k++) {
          const float was = keep ? o[e][k] : o[e][k] * alpha;
          o[e][k] = fmaf(x[k], sv, was);
        }
      };
      each(value, std::make_integer_sequence<int, DT>{});
    }
    if (unit_at + 1 < unit1) begin(following);
    // the four waves' shares of each row, joined through LDS
    float *so = smem;                 // [4][16][LDO]
    float *sm = smem + 4 * 16 * LDO;  // [4][16] maxima, then sums
    const float sum = reduce_sum4(l);
    __syncthreads();  // (after the last unit's readers)
    if (g == 0) {
      sm[16 * wave + c] = m;
      sm[64 + 16 * wave + c] = sum;
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
      float *dst = so + (16 * wave + c) * LDO + (4 * g + k) * DT;
#pragma unroll
      for (int e = 0; e < DT; e += 4)
        *(f32x4_v *)(dst + e) = (f32x4_v){o[e][k], o[e + 1][k], o[e + 2][k], o[e + 3][k]};
    }
    __syncthreads();
    for (int i = tid; i < 16 * (D / 4); i += 256) {
      const int j = i / (D / 4), d = 4 * (i % (D / 4));
      if (j >= u.rows) break;
      float mm = fmaxf(fmaxf(sm[j], sm[16 + j]), fmaxf(sm[32 + j], sm[48 + j]));
      const float base = mm == -INFINITY ? 0.f : mm;
      float all = 0;
      f32x4_v x = {0, 0, 0, 0};
#pragma unroll
      for (int w = 0; w < 4; w++) {
        const float f = __builtin_amdgcn_exp2f(sm[16 * w + j] - base);
        all = fmaf(sm[64 + 16 * w + j], f, all);
        x += *(const f32x4_v *)(so + (16 * w + j) * LDO + d) * f;
      }
      const int f = u.f0 + j;
      if (u.part < 0) {
        x *= all == 0.f ? 0.f : kRoom / all;
        const int t = f / G, head = h * G + f - t * G;
        store_row<4>(a.out + ((int64_t)(u.q0 + t) * a.q_heads + head) * D + d, a.dtype == SQ_BF16, (const float *)&x);
      } else {
        const int64_t slot = ((int64_t)u.part * a.kv_heads + h) * unit_rows + at_row + j;
        *(f32x4_v *)(a.ws + slot * D + d) = x;
        if (d == 0) {
          float *ml = a.ws + (int64_t)a.max_partials * a.kv_heads * unit_rows * D + 2 * slot;
          ml[0] = mm;
          ml[1] = all;
        }
      }
    }
    u = following;
  }
}

// Joins the parts of query rows of units of up to 32, by their maxima: one
// workgroup per (merge, head) and row; LANES lanes read a part, GROUPS parts at
// a time.  3.9 to 5.0 us, most of them a launch's own; 6.7 us for 64 parts.
template <int D>
__device__ __forceinline__ void merge_few(const AttendDev &a, int unit_rows) {
  constexpr int LANES = D / 4, GROUPS = 512 / LANES, AHEAD = 4;
  __shared__ f32x4_v part_o[GROUPS][LANES];
  __shared__ float part_l[GROUPS], part_m[GROUPS];
  const int tid = threadIdx.x, h = blockIdx.x % a.kv_heads, j = blockIdx.y;
  const int32_t *u = a.merges + 8 * (int64_t)(blockIdx.x / a.kv_heads);
  const int q0 = u[0], f0 = u[1], rows = u[2], p0 = u[3], n = u[4], G = a.q_heads / a.kv_heads;
  if (j >= rows) return;
  const int lane = tid % LANES, grp = tid / LANES;
  const float *ml = a.ws + (int64_t)a.max_partials * a.kv_heads * unit_rows * D;
  const int64_t slot0 = ((int64_t)p0 * a.kv_heads + h) * unit_rows + j, step = (int64_t)a.kv_heads * unit_rows;
  // every group of lanes joins its parts as they come, then the groups
  f32x4_v x = {0, 0, 0, 0};
  float sum = 0, mm = -INFINITY;
#pragma unroll 1
  for (int i0 = grp; i0 < n; i0 += AHEAD * GROUPS) {
    float2 stat[AHEAD];
    f32x4_v y[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; k++) {  // (past the end the last part again, with no weight)
      const int64_t s = slot0 + min(i0 + k * GROUPS, n - 1) * step;
      stat[k] = *(const float2 *)(ml + 2 * s);
      y[k] = *(const f32x4_v *)(a.ws + s * D + 4 * lane);
    }
#pragma unroll
    for (int k = 0; k < AHEAD; k++) {
      if (i0 + k * GROUPS >= n) break;
      const float high = fmaxf(mm, stat[k].x), base = high == -INFINITY ? 0.f : high;
      const float was = __builtin_amdgcn_exp2f(mm - base), w = __builtin_amdgcn_exp2f(stat[k].x - base);
      mm = high;
      sum = fmaf(sum, was, stat[k].y * w);
      x = x * was + y[k] * w;
    }
  }
  part_o[grp][lane] = x;
  if (lane == 0) part_l[grp] = sum, part_m[grp] = mm;
  __syncthreads();
  if (grp) return;
  const int groups = min(GROUPS, n);
#pragma unroll 1
  for (int i = 1; i < groups; i++) mm = fmaxf(mm, part_m[i]);
  const float base = mm == -INFINITY ? 0.f : mm;
  sum = 0;
  x = (f32x4_v){0, 0, 0, 0};
#pragma unroll 1
  for (int i = 0; i < groups; i++) {
    const float w = __builtin_amdgcn_exp2f(part_m[i] - base);
    x += part_o[i][lane] * w;
    sum = fmaf(part_l[i], w, sum);
  }
  x *= sum == 0.f ? 0.f : kRoom / sum;
  const int t = (f0 + j) / G, head = h * G + f0 + j - t * G;
  store_row<4>(a.out + ((int64_t)(q0 + t) * a.q_heads + head) * D + 4 * lane, a.dtype == SQ_BF16, (const float *)&x);
}

// Joins the parts of units of up to 256 rows, in the order in which a wave's
// registers of kv_attend_rows_kernel went out: one workgroup per (merge, head)
// and wave; its two halves take the parts in turn, two at a time.  19.6 us for
// the parts of 4 chunks of 701 tokens, 16 heads over 2 of 256 dims (up to 67 MB, written
// the kernel before).
template <int D>
__device__ __forceinline__ void merge_many(const AttendDev &a) {
  constexpr int DT = D / 32, OT = D == 256 ? DT / 2 : DT, BLOCKS = D == 256 ? 16 : 8;
  typedef float vec __attribute__((ext_vector_type(OT)));
  __shared__ vec part_o[4][256];
  __shared__ float2 part_s[256];
  const int h = blockIdx.x % a.kv_heads, wave = blockIdx.y & 7, turn = blockIdx.y >> 3;
  const int32_t *u = a.merges + 8 * (int64_t)(blockIdx.x / a.kv_heads);
  const int q0 = u[0], f0 = u[1], rows = u[2], p0 = u[3], n = u[4], G = a.q_heads / a.kv_heads;
  const int tid = threadIdx.x & 255, half = threadIdx.x >> 8, k0 = tid >> 6;
  const int lane = tid & 63, c = lane & 31, hl = lane >> 5;
  const int e0 = D == 256 ? (wave & 1) * OT : 0;
  const int first = D == 256 ? 128 * turn + 32 * (wave >> 1) : 32 * wave, j = first + c;
  if (first >= rows) return;
  const float *ml = a.ws + (int64_t)a.max_partials * a.kv_heads * a.unit_rows * D + 2 * (int64_t)min(j, rows - 1);
  vec x[4];
#pragma unroll
  for (int i = 0; i < 4; i++) x[i] = (vec)(0.f);
  float sum = 0, mm = -INFINITY;
#pragma unroll 2
  for (int i = half; i < n; i += 2) {
    const int64_t slot = (int64_t)(p0 + i) * a.kv_heads + h;
    const float2 stat = *(const float2 *)(ml + 2 * slot * a.unit_rows);
    vec y[4];
#pragma unroll
    for (int k = 0; k < 4; k++)
      y[k] = *(const vec *)(a.ws + (((slot * BLOCKS + blockIdx.y) * 16 + k0 + 4 * k) * 64 + lane) * OT);
    const float high = fmaxf(mm, stat.x), base = high == -INFINITY ? 0.f : high;
    const float was = __builtin_amdgcn_exp2f(mm - base), w = __builtin_amdgcn_exp2f(stat.x - base);
    mm = high;
    sum = fmaf(sum, was, stat.y * w);
#pragma unroll
    for (int k = 0; k < 4; k++) x[k] = x[k] * was + y[k] * w;
  }
  if (half) {
#pragma unroll
    for (int k = 0; k < 4; k++) part_o[k][tid] = x[k];
    part_s[tid] = make_float2(mm, sum);
  }
  __syncthreads();
  if (half || j >= rows) return;
  const float2 other = part_s[tid];
  const float high = fmaxf(mm, other.x), base = high == -INFINITY ? 0.f : high;
  float mine = __builtin_amdgcn_exp2f(mm - base), theirs = __builtin_amdgcn_exp2f(other.x - base);
  sum = fmaf(sum, mine, other.y * theirs);
  const float f = sum == 0.f ? 0.f : kRoom / sum;
  mine *= f, theirs *= f;
  const int t = (f0 + j) / G, head = h * G + f0 + j - t * G;
  uint16_t *dst = a.out + ((int64_t)(q0 + t) * a.q_heads + head) * D + e0;
#pragma unroll
  for (int i = 0; i < 4; i++) {
    const int k = k0 + 4 * i;
    x[i] = x[i] * mine + part_o[i][tid] * theirs;
    store_row<OT>(dst + (8 * (k >> 2) + 4 * hl + (k & 3)) * DT, a.dtype == SQ_BF16, (const float *)&x[i]);
  }
}

template <int D>
__global__ __launch_bounds__(512) void kv_merge_kernel(AttendDev a) {
  merge_few<D>(a, a.unit_rows);
}

template <int D>
__global__ __launch_bounds__(512) void kv_merge_rows_kernel(AttendDev a) {
  merge_many<D>(a);
}

template <int D>
__global__ __launch_bounds__(512) void kv_merge_either_kernel(AttendDev a) {
  if (a.starts[a.max_workers + 1] == 32) merge_few<D>(a, 32);
  else if (blockIdx.y < (D == 256 ? 16 : 8)) merge_many<D>(a);
}

// ------------------------------------------------------------ host side

int fail(int code, const char *msg) { return sq_internal_fail(code, msg); }

bool index_type(int32_t dtype) { return dtype == SQ_I32 || dtype == SQ_I64; }

int check_cache(const sq_kv_cache *c) {
  if (!c || !c->data || ((uintptr_t)c->data & 15)) return fail(SQ_EINVAL, "kv cache: null or misaligned pages");
  if (c->dim != 64 && c->dim != 128 && c->dim != 256) return fail(SQ_ESHAPE, "kv cache: dim must be 64, 128 or 256");
  if (c->heads <= 0 || c->heads > 4096) return fail(SQ_ESHAPE, "kv cache: heads must be in [1, 4096]");
  if (c->page_tokens <= 0 || c->page_tokens % kTile || c->page_tokens * (int64_t)c->dim > 32768)
    return fail(SQ_ESHAPE, "kv cache: page_tokens must be a multiple of 64 with page_tokens * dim <= 32768");
  if (c->storage != SQ_KV_INT8 && c->storage != SQ_KV_FP8) return fail(SQ_ESTORAGE, "kv cache: unknown storage");
  if (c->num_pages <= 0 || c->num_pages > 0x7fffffff || c->page_bytes % 16 || c->page_bytes > 0x7fffffff ||
      c->page_bytes < (int64_t)c->heads * (2 * (int64_t)c->page_tokens * c->dim + 8))
    return fail(SQ_EINVAL, "kv cache: page count or page bytes");
  return 0;
}

int check_tables(const sq_kv_tables *t) {
  if (!t || !t->table || !t->lens || !t->free_pages || !t->counters) return fail(SQ_EINVAL, "kv tables: null pointer");
  if (t->requests <= 0 || t->requests > 0x7fffffff || t->width <= 0 || t->capacity <= 0 || t->capacity > 0x7fffffff)
    return fail(SQ_EINVAL, "kv tables: sizes must be positive 32-bit numbers");
  if (t->page_tokens <= 0) return fail(SQ_ESHAPE, "kv tables: page_tokens must be positive");
  return 0;
}

int check_schedule(const sq_kv_schedule *s, int64_t tokens, int64_t batch) {
  if (!s->units || !s->merges || !s->starts) return fail(SQ_EINVAL, "kv schedule: null pointer");
  if (s->kv_heads <= 0 || s->q_heads <= 0 || s->q_heads % s->kv_heads)
    return fail(SQ_ESHAPE, "kv schedule: q_heads must be a positive multiple of kv_heads");
  if (s->rows != 16 && s->rows != 32 && s->rows != 256) return fail(SQ_ESHAPE, "kv schedule: rows");
  if (s->window < 0 || (s->window > 0 && !s->causal))
    return fail(SQ_EINVAL, "kv schedule: a window is non-negative and needs causal attention");
  if (s->slots <= 0 || s->slots > kMaxSlots) return fail(SQ_EINVAL, "kv schedule: slots must be in [1, 4096]");
  if (s->min_tiles <= 0 || s->cut_tiles < 0 || s->merge_rows <= 0 || s->merge_rows > s->rows)
    return fail(SQ_EINVAL, "kv schedule: min_tiles, cut_tiles or merge_rows");
  const int64_t G = s->q_heads / s->kv_heads;
  if (tokens * G > 0x3fffffff) return fail(SQ_EINVAL, "kv schedule: tokens * heads of a group too large");
  if (s->few_work < 0 || (s->few_work > 0 && (s->rows != 256 || s->few_min_tiles <= 0 || s->few_cut_tiles < 0)))
    return fail(SQ_EINVAL, "kv schedule: few_work, few_min_tiles or few_cut_tiles");
  const int64_t least = s->few_work > 0 ? 32 : s->rows, sets = (tokens * G + least - 1) / least + batch + 1;
  const int64_t slots = s->slots / s->kv_heads > 1 ? s->slots / s->kv_heads : 1;
  const int64_t larger = sets > slots ? sets : slots, smaller = sets < slots ? sets : slots;
  if (s->max_workers < larger || s->max_units < sets + slots || s->max_merges < smaller ||
      s->max_partials < 2 * slots || s->max_units >= 1 << 24)
    return fail(SQ_EINVAL, "kv schedule: room for workers, units, merges or partials");
  // (a launch has fewer than 2^32 threads, 512 a workgroup)
  if ((int64_t)s->max_workers * s->kv_heads >= 1 << 23 || (int64_t)s->max_merges * s->kv_heads >= 1 << 23)
    return fail(SQ_EINVAL, "kv schedule: workers * heads too large");
  return 0;
}

int check_plan(const sq_kv_tables *t, const sq_kv_plan_args *p) {
  const int rc = check_tables(t);
  if (rc) return rc;
  if (!p || !p->rows || !p->counts || !p->cu || !p->slots || !p->positions || !p->lens || !p->granted || !p->pages ||
      !p->filled || !p->tiles || !p->counters)
    return fail(SQ_EINVAL, "kv plan: null pointer");
  if ((uintptr_t)p->tiles & 7) return fail(SQ_EINVAL, "kv plan: tiles must be 8-byte aligned");
  if (!index_type(p->rows_dtype) || !index_type(p->counts_dtype))
    return fail(SQ_EINVAL, "kv plan: rows and counts are int32 or int64");
  if (p->batch <= 0 || p->batch > SQ_KV_MAX_REQUESTS) return fail(SQ_EINVAL, "kv plan: batch must be in [1, 4096]");
  if (p->max_count < 0) return fail(SQ_EINVAL, "kv plan: negative max_count");
  if (p->tokens < 0 || p->tokens > 0x3fffffff) return fail(SQ_EINVAL, "kv plan: tokens must be in [0, 2^30)");
  int64_t tiles = p->tokens / t->page_tokens + 2 * (int64_t)p->batch;
  if (tiles > p->tokens) tiles = p->tokens;
  if (p->max_tiles < tiles) return fail(SQ_EINVAL, "kv plan: room for page entries");
  if (p->n_schedules < 0 || p->n_schedules > SQ_KV_MAX_SCHEDULES)
    return fail(SQ_EINVAL, "kv plan: number of schedules");
  for (int i = 0; i < p->n_schedules; i++) {
    const sq_kv_schedule &s = p->schedules[i];
    const int e = check_schedule(&s, p->tokens, p->batch);
    if (e) return e;
    const int64_t most = (int64_t)p->max_count * (s.q_heads / s.kv_heads);
    if (s.merge_rows < (most < s.rows ? most : s.rows)) return fail(SQ_EINVAL, "kv plan: merge_rows below max_count's");
  }
  return 0;
}

// Raises a kernel's limit of dynamic LDS to the most that it takes, once per
// kernel (each with an id of its own) and device.
std::atomic<uint64_t> g_raised[16];

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

int log2_of(int x) { return 31 - __builtin_clz((unsigned)x); }

template <int D, bool FP8>
int launch_attend(const AttendDev &d, const sq_kv_schedule &s, hipStream_t st) {
  const unsigned blocks = s.max_workers * s.kv_heads;
  auto go = [&](auto kernel, int id, unsigned grid, int threads, size_t lds) {
    const int rc = dynamic_lds((const void *)kernel, 2 * id + FP8, lds, "kv attend: LDS attribute");
    if (rc) return rc;
    hipLaunchKernelGGL(kernel, dim3(grid), dim3(threads), lds, st, d);
    return sq_internal_launched("kv_attend_kernel");
  };
  constexpr size_t joined = kJoin<D> * sizeof(float);
  // tiles, peaks, and what the pairs of waves share; the outputs' way out
  constexpr size_t staged = 2 * sizeof(uint4) * (2 * (D / 16) * 65 + 4 * (D / 32) * 64 + 1) + (D == 256 ? 8 * (2048 + 256) : 0);
  constexpr size_t rows_out = 256 * (D == 256 ? 264 : 2 * D + 8);
  constexpr size_t many = staged > rows_out ? staged : rows_out;
  // (ids of kernels with more than 64 KiB: one of each kind needs one of 256 dims, the many rows' one of 128)
  int rc;
  if (s.few_work > 0) rc = go(kv_attend_kernel<D, FP8, true>, 3 + D / 64, blocks, 512, many > 2 * joined ? many : 2 * joined);
  else if (s.rows == 256) rc = go(kv_attend_rows_kernel<D, FP8>, D == 256 ? 2 : 3, blocks, 512, many);
  else rc = go(kv_attend_kernel<D, FP8, false>, 1, s.rows == 32 ? (blocks + 7) / 8 * 16 : blocks, 256, joined);
  if (rc) return rc;
  const unsigned merges = s.max_merges * s.kv_heads;
  const unsigned waves = (unsigned)(s.merge_rows + 31) / 32 * (D == 256 ? 2 : 1);  // of a unit that have rows
  if (s.few_work > 0) hipLaunchKernelGGL(kv_merge_either_kernel<D>, dim3(merges, 32), dim3(512), 0, st, d);
  else if (s.rows == 256) hipLaunchKernelGGL(kv_merge_rows_kernel<D>, dim3(merges, waves), dim3(512), 0, st, d);
  else hipLaunchKernelGGL(kv_merge_kernel<D>, dim3(merges, (unsigned)s.merge_rows), dim3(512), 0, st, d);
  return sq_internal_launched("kv_merge_kernel");
}

}  // namespace

extern "C" {

int sq_kv_plan(const sq_kv_tables *t, const sq_kv_plan_args *p, void *stream) {
  const int rc = check_plan(t, p);
  if (rc) return rc;
  PlanDev d = {*t, *p, 0};
  const int64_t share = p->tokens > p->max_tiles ? p->tokens : p->max_tiles;
  d.share_blocks = (int)((share + kPlanShare - 1) / kPlanShare);
  if (d.share_blocks < 1) d.share_blocks = 1;
  const size_t lds = 5 * sizeof(int32_t) * (size_t)(p->batch + 1);
  const int e = dynamic_lds((const void *)kv_plan_kernel, 0, 5 * sizeof(int32_t) * (SQ_KV_MAX_REQUESTS + 1),
                            "kv plan: LDS attribute");
  if (e) return e;
  hipLaunchKernelGGL(kv_plan_kernel, dim3((unsigned)(d.share_blocks + p->n_schedules)), dim3(kPlanThreads), lds,
                     (hipStream_t)stream, d);
  return sq_internal_launched("kv_plan_kernel");
}

int sq_kv_commit(const sq_kv_tables *t, const sq_kv_plan_args *p, void *stream) {
  const int rc = check_plan(t, p);
  if (rc) return rc;
  PlanDev d = {*t, *p, 0};
  hipLaunchKernelGGL(kv_commit_kernel, dim3((unsigned)((p->batch + 255) / 256)), dim3(256), 0, (hipStream_t)stream, d);
  return sq_internal_launched("kv_commit_kernel");
}

int sq_kv_release(const sq_kv_tables *t, const void *rows, int32_t rows_dtype, int64_t n, void *stream) {
  const int rc = check_tables(t);
  if (rc) return rc;
  if (n == 0) return 0;
  if (!rows || !index_type(rows_dtype) || n < 0 || n > SQ_KV_MAX_REQUESTS)
    return fail(SQ_EINVAL, "kv release: rows must be int32 or int64, at most 4096 of them");
  hipLaunchKernelGGL(kv_release_kernel, dim3(1), dim3(kPlanThreads), 2 * sizeof(int32_t) * (size_t)n, (hipStream_t)stream,
                     *t, rows, rows_dtype, (int)n);
  return sq_internal_launched("kv_release_kernel");
}

int sq_kv_append(const sq_kv_cache *c, const sq_kv_append_args *a, void *stream) {
  const int rc = check_cache(c);
  if (rc) return rc;
  if (!a) return fail(SQ_EINVAL, "kv append: null arguments");
  if (a->max_tiles == 0) return 0;
  if (!a->k || !a->v || !a->pages || !a->filled || !a->tiles || a->max_tiles < 0)
    return fail(SQ_EINVAL, "kv append: null pointer");
  if (a->dtype != SQ_BF16 && a->dtype != SQ_F16) return fail(SQ_EINVAL, "kv append: keys and values are bf16 or fp16");
  if ((a->k_stride | a->k_head_stride | a->v_stride | a->v_head_stride) & 7 || (((uintptr_t)a->k | (uintptr_t)a->v) & 15))
    return fail(SQ_EINVAL, "kv append: strides must be multiples of 8 and starts 16-byte aligned");
  if (a->k_stride < 0 || a->k_head_stride < 0 || a->v_stride < 0 || a->v_head_stride < 0)
    return fail(SQ_EINVAL, "kv append: negative stride");
  const int n = c->page_tokens * c->dim / 2048;
  const dim3 grid((unsigned)a->max_tiles, (unsigned)c->heads, 2);
  auto go = [&](auto kernel) {
    hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, *c, *a, log2_of(c->dim));
    return sq_internal_launched("kv_append_kernel");
  };
  if (c->storage == SQ_KV_FP8)
    return n <= 2 ? go(kv_append_kernel<true, 2>) : n <= 4 ? go(kv_append_kernel<true, 4>)
           : n <= 8 ? go(kv_append_kernel<true, 8>) : go(kv_append_kernel<true, 16>);
  return n <= 2 ? go(kv_append_kernel<false, 2>) : n <= 4 ? go(kv_append_kernel<false, 4>)
         : n <= 8 ? go(kv_append_kernel<false, 8>) : go(kv_append_kernel<false, 16>);
}

int sq_kv_decode(const sq_kv_cache *c, const int32_t *pages, const int32_t *filled, int64_t n, void *k, void *v,
                 int32_t out_dtype, void *stream) {
  const int rc = check_cache(c);
  if (rc) return rc;
  if (n == 0) return 0;
  if (!pages || !k || !v || n < 0 || n >= 1 << 24) return fail(SQ_EINVAL, "kv decode: null pointer or page count");
  if (out_dtype != SQ_F32 && out_dtype != SQ_BF16 && out_dtype != SQ_F16)
    return fail(SQ_EINVAL, "kv decode: output dtype");
  if (((uintptr_t)k | (uintptr_t)v) & 15) return fail(SQ_EINVAL, "kv decode: outputs must be 16-byte aligned");
  const dim3 grid((unsigned)n, (unsigned)c->heads, 2);
  if (c->storage == SQ_KV_FP8)
    hipLaunchKernelGGL(kv_decode_kernel<true>, grid, dim3(256), 0, (hipStream_t)stream, *c, pages, filled, k, v, out_dtype,
                       log2_of(c->dim));
  else
    hipLaunchKernelGGL(kv_decode_kernel<false>, grid, dim3(256), 0, (hipStream_t)stream, *c, pages, filled, k, v, out_dtype,
                       log2_of(c->dim));
  return sq_internal_launched("kv_decode_kernel");
}

int sq_kv_attend(const sq_kv_cache *c, const sq_kv_attend_args *a, void *stream) {
  int rc = check_cache(c);
  if (rc) return rc;
  if (!a) return fail(SQ_EINVAL, "kv attend: null arguments");
  if (a->tokens == 0) return 0;
  if (!a->q || !a->out || !a->table || a->tokens < 0 || a->requests <= 0 || a->width <= 0)
    return fail(SQ_EINVAL, "kv attend: null pointer or size");
  if (a->dtype != SQ_BF16 && a->dtype != SQ_F16) return fail(SQ_EINVAL, "kv attend: queries are bf16 or fp16");
  if ((a->q_stride | a->q_head_stride) & 7 || ((uintptr_t)a->q & 15) || ((uintptr_t)a->out & 15))
    return fail(SQ_EINVAL, "kv attend: strides must be multiples of 8 and starts 16-byte aligned");
  if (a->q_stride < 0 || a->q_head_stride < 0) return fail(SQ_EINVAL, "kv attend: negative stride");
  if (!(a->scale > -3e38f && a->scale < 3e38f)) return fail(SQ_EINVAL, "kv attend: scale must be finite");
  rc = check_schedule(&a->schedule, a->tokens, 1);
  if (rc) return rc;
  if (a->schedule.kv_heads != c->heads)
    return fail(SQ_ESHAPE, "kv attend: the schedule is for another number of KV heads");
  if (!a->workspace || ((uintptr_t)a->workspace & 15))
    return fail(SQ_EINVAL, "kv attend: null or misaligned workspace");
  const sq_kv_schedule &s = a->schedule;
  const AttendDev d = {*c, (const uint16_t *)a->q, (uint16_t *)a->out, a->workspace, a->table, s.units, s.merges, s.starts,
                       a->requests, a->tokens, a->q_stride, a->q_head_stride, a->width, a->dtype, s.q_heads, s.kv_heads,
                       s.causal, s.window, s.max_partials, s.max_units, s.max_workers, s.rows, a->scale};
  const bool fp8 = c->storage == SQ_KV_FP8;
  hipStream_t st = (hipStream_t)stream;
  if (c->dim == 64) return fp8 ? launch_attend<64, true>(d, s, st) : launch_attend<64, false>(d, s, st);
  if (c->dim == 128) return fp8 ? launch_attend<128, true>(d, s, st) : launch_attend<128, false>(d, s, st);
  return fp8 ? launch_attend<256, true>(d, s, st) : launch_attend<256, false>(d, s, st);
}

}  // extern "C"
