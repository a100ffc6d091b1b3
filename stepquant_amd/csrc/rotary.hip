// MI355X (gfx950) kernel of rotary positions.
#include "rotary.h"

#include "internal.h"

namespace {

// HBM bounds it where there is enough to turn (16,384 tokens of 32 heads of 128 dims: 50 us,
// 5.4 TB/s); a decode step's rows take less than the launch (64 tokens: 2.8 us in a graph).
template <int T, int PER>
__global__ __launch_bounds__(256) void rotary_kernel(sq_rotary r, sq_rotary_rows a, int lanes) {
  rotary::rotate_rows_typed<T, PER, true>(r, a, lanes, blockIdx.x * 256 + threadIdx.x);
}

int fail(int code, const char *msg) { return sq_internal_fail(code, msg); }

}  // namespace

namespace rotary {

int check(const sq_rotary *r) {
  if (!r || !r->turns || ((uintptr_t)r->turns & 7)) return fail(SQ_EINVAL, "rotary: null or misaligned frequencies");
  if (r->dim <= 0 || r->dim % 16 || r->dim > 1024) return fail(SQ_ESHAPE, "rotary: dim must be a multiple of 16, at most 1024");
  if (!(r->magnitude > -3e38f && r->magnitude < 3e38f)) return fail(SQ_EINVAL, "rotary: magnitude must be finite");
  return 0;
}

int check_rows(const sq_rotary *r, const sq_rotary_rows *a) {
  if (!a || !a->x || !a->out || !a->positions || a->tokens < 0) return fail(SQ_EINVAL, "rotary: null pointer or size");
  if (a->dtype != SQ_F32 && a->dtype != SQ_BF16 && a->dtype != SQ_F16) return fail(SQ_EINVAL, "rotary: rows are fp32, bf16 or fp16");
  if (a->positions_dtype != SQ_I32 && a->positions_dtype != SQ_I64) return fail(SQ_EINVAL, "rotary: positions are int32 or int64");
  if (a->heads <= 0 || a->heads > 65536 || a->head_dim < r->dim || a->head_dim % 8 || a->head_dim > 65536)
    return fail(SQ_ESHAPE, "rotary: heads, or head_dim below the rotated dims or no multiple of 8");
  const int64_t whole = a->dtype == SQ_F32 ? 3 : 7;
  if ((a->x_stride | a->x_head_stride | a->out_stride | a->out_head_stride) & whole || (((uintptr_t)a->x | (uintptr_t)a->out) & 15))
    return fail(SQ_EINVAL, "rotary: strides must be whole 16 bytes and starts 16-byte aligned");
  if (a->x_stride < 0 || a->x_head_stride < 0 || a->out_stride < 0 || a->out_head_stride < 0)
    return fail(SQ_EINVAL, "rotary: negative stride");
  if (a->x == a->out && ((a->tokens > 1 && a->x_stride != a->out_stride) || (a->heads > 1 && a->x_head_stride != a->out_head_stride)))
    return fail(SQ_EINVAL, "rotary: rows that are turned in place have one layout");
  return 0;
}

}  // namespace rotary

extern "C" int sq_rotary_apply(const sq_rotary *r, const sq_rotary_rows *rows, void *stream) {
  int rc = rotary::check(r);
  if (rc) return rc;
  if (rows && rows->tokens == 0) return 0;
  rc = rotary::check_rows(r, rows);
  if (rc) return rc;
  sq_rotary_rows a = *rows;
  const int64_t items = rotary::row_items(*r, a, true);
  const bool many = rotary::heads_per_thread(r, rows) > 1;
  const int lanes = rotary::head_lanes(a.heads, rotary::heads_per_thread(r, rows));
  const int64_t threads = lanes * items, size = a.dtype == SQ_F32 ? 4 : 2;
  // (a launch has fewer than 2^32 threads)
  const int64_t most = ((int64_t)1 << 31) / threads;
  for (int64_t left = rows->tokens; left > 0; left -= most) {
    a.tokens = left < most ? left : most;
    const dim3 grid((unsigned)((a.tokens * threads + 255) / 256));
    auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, grid, dim3(256), 0, (hipStream_t)stream, *r, a, lanes); };
    if (a.dtype == SQ_BF16) many ? go(rotary_kernel<SQ_BF16, 4>) : go(rotary_kernel<SQ_BF16, 1>);
    else if (a.dtype == SQ_F16) many ? go(rotary_kernel<SQ_F16, 4>) : go(rotary_kernel<SQ_F16, 1>);
    else many ? go(rotary_kernel<SQ_F32, 4>) : go(rotary_kernel<SQ_F32, 1>);
    rc = sq_internal_launched("rotary_kernel");
    if (rc) return rc;
    a.x = (const char *)a.x + a.tokens * a.x_stride * size;
    a.out = (char *)a.out + a.tokens * a.out_stride * size;
    a.positions = (const char *)a.positions + a.tokens * (a.positions_dtype == SQ_I64 ? 8 : 4);
  }
  return 0;
}
