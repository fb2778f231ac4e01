#include "pg_rows_distill.h"

pg_status pgrows::distill_bf16(pg_ctx* c, const DArgs& a, int64_t rows) { return run_t<__bf16>(c, a, rows); }
