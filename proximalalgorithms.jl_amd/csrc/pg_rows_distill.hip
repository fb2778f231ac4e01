// Distillation from a teacher's top logits: the entry point (kernels: pg_rows_distill.h, one translation unit per element type).
#include "pg_rows_distill.h"

namespace pgrows {
namespace {
__global__ void store_zero(double* out, void* value, int f64) {
  if (f64) store_value<double>(0.0, out, value);
  else store_value<float>(0.0, out, value);
}

}  // namespace
}  // namespace pgrows

extern "C" {

int32_t pg_rows_abi_version(void) { return PG_ROWS_ABI_VERSION; }

pg_status pg_distill_value_and_gradient(pg_ctx* c, const pg_distill* d, int32_t dtype, const void* scores, int64_t ld, void* grad,
                                        int64_t grad_ld, void* value, double* f_out) {
  using namespace pgrows;
  PG_REQUIRE(c != nullptr && d != nullptr, "null argument");
  PG_REQUIRE(dtype_ok(dtype), "bad dtype");
  PG_REQUIRE(d->rows >= 0 && d->classes >= 0 && d->top >= 0, "negative size");
  PG_REQUIRE(d->classes <= MAX_CLASSES, "at most 2^24 classes");
  PG_REQUIRE(d->top <= MAX_TOP, "top must be at most 1024");
  PG_REQUIRE(d->temperature > 0.0 && std::isfinite(d->temperature), "temperature must be positive and finite");
  PG_REQUIRE(d->lam >= 0.0 && d->label_lam >= 0.0 && std::isfinite(d->lam) && std::isfinite(d->label_lam), "lam and label_lam must be nonnegative and finite");
  const bool any = d->rows > 0 && d->classes > 0;
  if (any) {
    PG_REQUIRE(scores != nullptr && grad != nullptr, "null rows");
    PG_REQUIRE((ld >= d->classes && grad_ld >= d->classes) || d->rows == 1, "rows overlap: ld below the number of classes");
    PG_REQUIRE(scores != grad || ld == grad_ld || d->rows == 1, "a gradient in the scores' own buffer needs the scores' ld");
    PG_REQUIRE(((uintptr_t)scores | (uintptr_t)grad) % dtype_size(dtype) == 0, "scores or gradient not aligned to their element");
    if (d->top > 0) {
      PG_REQUIRE(d->teacher != nullptr && d->index != nullptr, "null teacher");
      PG_REQUIRE(dtype_ok(d->teacher_dtype), "bad teacher_dtype");
      PG_REQUIRE(d->index_bits == 32 || d->index_bits == 64, "index_bits must be 32 or 64");
    }
    PG_REQUIRE(d->teacher_lse == nullptr || d->lse_dtype == PG_F32 || d->lse_dtype == PG_F64, "bad lse_dtype");
    PG_REQUIRE(d->weights == nullptr || d->weights_dtype == PG_F32 || d->weights_dtype == PG_F64, "bad weights_dtype");
    PG_REQUIRE(d->labels == nullptr || d->label_bits == 32 || d->label_bits == 64, "label_bits must be 32 or 64");
  }
  DeviceScope dev(c->device);
  PG_TRY(dev.st);
  PG_TRY(refuse_foreign_capture(c));
  double* out = f_out != nullptr ? c->dscal + PG_S_MISC : nullptr;
  if (!any) {
    store_zero<<<1, 1, 0, c->stream>>>(out, value, dtype == PG_F64);
    PG_LAUNCH_CHECK();
  } else {
    DArgs a{};
    a.x = scores, a.g = grad, a.t = d->teacher, a.idx = d->index, a.lse = d->teacher_lse, a.w = d->weights, a.lab = d->labels;
    a.ldx = ld, a.ldg = grad_ld, a.ldt = d->teacher_ld, a.ldi = d->index_ld;
    a.V = (int)d->classes, a.K = (int)d->top;
    a.tdt = d->teacher_dtype, a.ibits = d->index_bits, a.lsedt = d->lse_dtype, a.wdt = d->weights_dtype, a.labbits = d->label_bits;
    a.invT = 1.0 / d->temperature, a.lam = d->lam, a.lab_lam = d->label_lam;
    a.squares = d->temperature == 2.0 ? 1 : (d->temperature == 4.0 ? 2 : 0);
    a.partials = c->red_partials, a.counter = c->row_tickets, a.out = out, a.value = value;
    PG_TRY(dtype == PG_F32 ? distill_f32(c, a, d->rows) : dtype == PG_F64 ? distill_f64(c, a, d->rows)
           : dtype == PG_BF16 ? distill_bf16(c, a, d->rows) : distill_f16(c, a, d->rows));
  }
  if (f_out == nullptr) return PG_OK;
  PG_TRY(pg_read_scalars(c, PG_S_MISC, 1));
  *f_out = c->hscal[PG_S_MISC];
  return PG_OK;
}

}  // extern "C"
