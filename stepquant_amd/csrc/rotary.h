// Rotary positions in device code; not part of the library's C ABI.
//
// Pair i of a head's first `dim` dims turns by position * f_i.  A frequency is
// held as turns a position, a 64-bit fraction: its product with the position,
// modulo 2^64, is the fraction of a turn that is left, off by position * 2^-65 of a
// turn, with no table of angles and no longest position (position times frequency in
// 32-bit floats is off by 0.004 rad at position 2^17).  The upper 32 bits of
// the product, 2^-32 of a turn, become the angle, a float on an eighth of a turn either
// side: 1.2e-7 rad off at most.  Sine and cosine are Taylor polynomials there, off by at most
// 2.4e-7 with the angle's error.
//
// A thread takes 16 dims, 8 pairs: two 16-byte groups `dim / 2` apart in the
// half layout, two adjacent ones in the interleaved layout.
#ifndef STEPQUANT_ROTARY_H
#define STEPQUANT_ROTARY_H

#include <hip/hip_runtime.h>
#include <stdint.h>

#include "stepquant_hip.h"

namespace rotary {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
typedef _Float16 half2 __attribute__((ext_vector_type(2)));

__device__ __forceinline__ void turn(uint32_t u, float magnitude, float &c, float &s) {
  const uint32_t quarter = (u + 0x20000000u) >> 30;
  const float x = (float)(int32_t)(u - (quarter << 30)) * 0x1.921fb6p-30f, y = x * x;  // 2 pi 2^-32
  float sine = fmaf(y, 2.7557319e-6f, -1.9841270e-4f), cosine = fmaf(y, 2.4801587e-5f, -1.3888889e-3f);
  sine = fmaf(sine, y, 8.3333333e-3f), cosine = fmaf(cosine, y, 4.1666667e-2f);
  sine = fmaf(sine, y, -.16666667f), cosine = fmaf(cosine, y, -.5f);
  sine = fmaf(sine, x * y, x), cosine = fmaf(cosine, y, 1.f);
  const bool odd = quarter & 1;
  c = __uint_as_float(__float_as_uint(odd ? sine : cosine) ^ ((quarter + 1) & 2) << 30) * magnitude;
  s = __uint_as_float(__float_as_uint(odd ? cosine : sine) ^ (quarter & 2) << 30) * magnitude;
}

// cosines and sines of pairs 8 item to 8 item + 7 at a position
struct Angles {
  float c[8], s[8];
  __device__ __forceinline__ void at(const sq_rotary &r, int item, uint64_t position) {
#pragma unroll
    for (int i = 0; i < 8; i++) turn((uint32_t)(position * r.turns[8 * item + i] >> 32), r.magnitude, c[i], s[i]);
  }
};

// the two 8-element groups of 16-dim item `item`
__device__ __forceinline__ void groups(const sq_rotary &r, int item, int &a, int &b) {
  const bool apart = !r.interleaved && item < r.dim / 16;
  a = apart ? item : 2 * item;
  b = apart ? item + r.dim / 16 : 2 * item + 1;
}

__device__ __forceinline__ void rotate(bool interleaved, const Angles &t, float x[16]) {
  if (interleaved) {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float a = x[2 * i], b = x[2 * i + 1];
      x[2 * i] = fmaf(a, t.c[i], -(b * t.s[i]));
      x[2 * i + 1] = fmaf(a, t.s[i], b * t.c[i]);
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; i++) {
      const float a = x[i], b = x[8 + i];
      x[i] = fmaf(a, t.c[i], -(b * t.s[i]));
      x[8 + i] = fmaf(a, t.s[i], b * t.c[i]);
    }
  }
}

// eight elements as loaded, as floats, and back; 32-bit ones take two loads
template <int T>
struct Eight {
  u32x4 w[T == SQ_F32 ? 2 : 1];
  __device__ __forceinline__ void load(const void *p, int64_t at) {
    if constexpr (T == SQ_F32) {
      w[0] = *(const u32x4 *)((const float *)p + at);
      w[1] = *(const u32x4 *)((const float *)p + at + 4);
    } else {
      w[0] = *(const u32x4 *)((const uint16_t *)p + at);
    }
  }
  __device__ __forceinline__ void store(void *p, int64_t at) const {
    if constexpr (T == SQ_F32) {
      *(u32x4 *)((float *)p + at) = w[0];
      *(u32x4 *)((float *)p + at + 4) = w[1];
    } else {
      *(u32x4 *)((uint16_t *)p + at) = w[0];
    }
  }
  __device__ __forceinline__ void widen(float *x) const {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const uint32_t word = w[0][i];
      if constexpr (T == SQ_F32) {
        x[i] = __uint_as_float(word), x[4 + i] = __uint_as_float(w[T == SQ_F32][i]);
      } else if constexpr (T == SQ_BF16) {
        x[2 * i] = __uint_as_float(word << 16), x[2 * i + 1] = __uint_as_float(word & 0xffff0000u);
      } else {
        const half2 h = __builtin_bit_cast(half2, word);
        x[2 * i] = (float)h[0], x[2 * i + 1] = (float)h[1];
      }
    }
  }
  __device__ __forceinline__ void narrow(const float *x) {
#pragma unroll
    for (int i = 0; i < 4; i++) {
      const f32x2 y = {x[2 * i], x[2 * i + 1]};
      if constexpr (T == SQ_F32) w[0][i] = __float_as_uint(x[i]), w[T == SQ_F32][i] = __float_as_uint(x[4 + i]);
      else if constexpr (T == SQ_BF16) w[0][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(y, bf16x2));
      else w[0][i] = __builtin_bit_cast(uint32_t, __builtin_convertvector(y, half2));
    }
  }
};

__device__ __forceinline__ int64_t position_of(const void *p, int dtype, int64_t i) {
  return dtype == SQ_I64 ? ((const int64_t *)p)[i] : (int64_t)((const int32_t *)p)[i];
}

// Items of 16 dims of a head that threads of its own kernel take: those that turn and, unless rows
// are turned in place, those that are copied, so that these have as many loads under way
// (11,000 tokens of 16 heads of 256 dims, 64 of them turned: 40.7 us; 49.6 where threads that
// turn copy what is left).  Beside appends they do, whose kernels have room for fewer
// waves (those tokens with their keys 51.7 us, 55.8 with threads that copy).
__host__ __device__ __forceinline__ int row_items(const sq_rotary &r, const sq_rotary_rows &a, bool copiers) {
  return copiers && a.x != a.out ? (a.head_dim + 15) / 16 : r.dim / 16;
}

// Thread `id` of the rows' `lanes * row_items` threads a token (lanes * PER >= heads):
// 16 dims of PER heads, whose angles it computes once, and without COPIERS its share of
// the dims that do not turn.
template <int T, int PER, bool COPIERS = false>
__device__ __forceinline__ void rotate_rows_typed(const sq_rotary &r, const sq_rotary_rows &a, int lanes, uint32_t id) {
  const uint32_t items = row_items(r, a, COPIERS), threads = lanes * items;
  const uint32_t token = id / threads, rest = id - token * threads, lane = rest / items, item = rest - lane * items;
  if (token >= a.tokens) return;
  const bool turns = !COPIERS || item < (uint32_t)r.dim / 16;
  const int64_t position = turns ? position_of(a.positions, a.positions_dtype, token) : -1;
  int ga, gb;
  groups(r, item, ga, gb);
  const bool two = !COPIERS || 8 * gb < a.head_dim;  // (heads have whole groups of 8 dims)
  const int64_t from = token * a.x_stride, to = token * a.out_stride;
  Eight<T> xa[PER], xb[PER];
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int h = lane + k * lanes;
    if (h < a.heads) {
      xa[k].load(a.x, from + h * a.x_head_stride + 8 * ga);
      if (two) xb[k].load(a.x, from + h * a.x_head_stride + 8 * gb);
    }
  }
  Angles t;
  if (position >= 0) t.at(r, item, position);
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int h = lane + k * lanes;
    if (h >= a.heads) break;
    if (position >= 0) {
      float x[16];
      xa[k].widen(x), xb[k].widen(x + 8);
      rotate(r.interleaved, t, x);
      xa[k].narrow(x), xb[k].narrow(x + 8);
    }
    xa[k].store(a.out, to + h * a.out_head_stride + 8 * ga);
    if (two) xb[k].store(a.out, to + h * a.out_head_stride + 8 * gb);
  }
  if (COPIERS || a.x == a.out) return;
  const int n = a.head_dim / 8;
#pragma unroll
  for (int k = 0; k < PER; k++) {
    const int h = lane + k * lanes;
    if (h >= a.heads) break;
#pragma unroll 4
    for (int g = 2 * items + item; g < n; g += items) {
      Eight<T> x;
      x.load(a.x, from + h * a.x_head_stride + 8 * g);
      x.store(a.out, to + h * a.out_head_stride + 8 * g);
    }
  }
}

template <int PER>
__device__ __forceinline__ void rotate_rows(const sq_rotary &r, const sq_rotary_rows &a, int lanes, uint32_t id) {
  if (a.dtype == SQ_BF16) rotate_rows_typed<SQ_BF16, PER>(r, a, lanes, id);
  else if (a.dtype == SQ_F16) rotate_rows_typed<SQ_F16, PER>(r, a, lanes, id);
  else rotate_rows_typed<SQ_F32, PER>(r, a, lanes, id);
}

// Heads of a thread.  Four share their angles where there are enough items of 16 dims to fill the
// GPU all the same: 2^17 of 128 dims take 3.9 us so and 3.7 one by one, 2^18
// 5.7 and 6.5, 2^20 12.0 and 16.4, 2^22 50 and 59 (5.4 TB/s; a copy reaches 5), in 16 bits.  Rows
// of 32 bits follow the same rule: 2^18 items 9.2 us with the host's share, 2^20 27, 2^22 103 (5.2 TB/s).
inline int heads_per_thread(const sq_rotary *r, const sq_rotary_rows *a) {
  return a->tokens * a->heads * row_items(*r, *a, true) >= (int64_t)1 << 18 ? 4 : 1;
}
// threads that a token's heads are dealt out to, PER heads each
inline int head_lanes(int heads, int per) { return (heads + per - 1) / per; }

// Host checks; 0, or the error that sq_last_error() then tells.
__attribute__((visibility("hidden"))) int check(const sq_rotary *r);
__attribute__((visibility("hidden"))) int check_rows(const sq_rotary *r, const sq_rotary_rows *a);

}  // namespace rotary

#endif
