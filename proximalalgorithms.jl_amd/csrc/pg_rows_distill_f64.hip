#include "pg_rows_distill.h"

pg_status pgrows::distill_f64(pg_ctx* c, const DArgs& a, int64_t rows) { return run_t<double>(c, a, rows); }
