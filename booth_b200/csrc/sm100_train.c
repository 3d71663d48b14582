/* sm100_train.c -- the training operators: layer normalisation and its gradient.
 *
 * Like the workloads in sm100_ops.c each call checks its arguments on the host,
 * enqueues its kernels on the device's stream and returns. Nothing is allocated
 * and nothing is waited for, so the calls can be captured into a graph; device
 * memory beyond the operands is a workspace the caller passes in, so two graphs, or
 * two streams that the caller orders, share one only where the caller says so. */
#define _POSIX_C_SOURCE 200809L
#include <limits.h>
#include <stdio.h>
#include <string.h>

#include "sm100_internal.h"

static int bad_arg(sm100_dev_t *dev, const char *what)
{
    if (dev) snprintf(dev->err, sizeof dev->err, "%s", what);
    fprintf(stderr, "sm100_rt: %s\n", what);
    return SM100_ERR_ARG;
}

/* Position of an element type in the kernel tables; -1: not a type of these operators. */
static int type_index(int t) { return t == SM100_F32 ? 0 : t == SM100_BF16 ? 1 : t == SM100_F16 ? 2 : -1; }
static unsigned type_bytes(int t) { return t == SM100_F32 ? 4u : t == SM100_BF16 || t == SM100_F16 ? 2u : 0u; }

/* A [rows, cols] operand with rows `ld` elements apart: non-NULL, aligned to its
 * element, the pitch no shorter than a row and the whole below 2^62 bytes. */
static int matrix_ok(sm100_ptr_t p, unsigned esz, long long rows, long long cols, long long ld)
{
    if (!p || (p & (esz - 1)) || ld < cols) return 0;
    return rows <= 1 || ld <= (1ll << 59) / rows;
}

/* ---- layer normalisation ---- */

/* Kernel of a (value type, parameter type) pair, in the order of the names in sm100_shim.c; -1: no such pair. */
static int ln_pair(int dtype, int wdtype)
{
    if (dtype == SM100_F32) return wdtype == SM100_F32 ? 0 : -1;
    if (dtype == SM100_BF16) return wdtype == SM100_BF16 ? 1 : wdtype == SM100_F32 ? 2 : -1;
    if (dtype == SM100_F16) return wdtype == SM100_F16 ? 3 : wdtype == SM100_F32 ? 4 : -1;
    return -1;
}

enum { LN_V8, LN_V16, LN_V32, LN_S8, LN_S16, LN_LOOP };

typedef struct { int form, group; unsigned block, grid; } ln_shape_t;

/* How rows are dealt to threads. Eight values a thread for narrow rows, and for
 * rows so few that each has an SM to itself (more threads shorten the one row);
 * sixteen otherwise, which halves what the reductions and the barriers cost per
 * value; thirty-two for vector rows too wide for 512 threads at sixteen; else the
 * form that walks the row. Blocks stay: as many as an SM holds (`threads`), each
 * taking every grid-th row. */
static ln_shape_t ln_shape(const sm100_dev_t *dev, long long rows, int cols, int vec, int threads)
{
    ln_shape_t s;
    int cpt = cols <= 1024 || (cols <= 4096 && rows < 2ll * dev->sm_count) ? 8 : cols <= 8192 ? 16 : cols <= 16384 && vec ? 32 : 0;
    s.form = cpt == 8 ? (vec ? LN_V8 : LN_S8) : cpt == 16 ? (vec ? LN_V16 : LN_S16) : cpt == 32 ? LN_V32 : LN_LOOP;
    if (!cpt) {
        s.group = 512;
        s.block = 512;
    } else {
        int g = (cols + cpt - 1) / cpt;
        if (g <= 32) { int p = 1; while (p < g) p *= 2; g = p; }
        else g = (g + 31) / 32 * 32;
        s.group = g;
        s.block = g <= 32 ? 128u : (unsigned)g;
    }
    const long long per_block = s.group <= 32 ? (long long)s.block / s.group : 1;
    long long want = (rows + per_block - 1) / per_block, per_sm = threads / (int)s.block;
    if (per_sm < 1) per_sm = 1;
    if (want > dev->sm_count * per_sm) want = dev->sm_count * per_sm;
    s.grid = (unsigned)(want < 1 ? 1 : want);
    return s;
}

int booth_sm100_layernorm(sm100_dev_t *dev, sm100_ptr_t y, sm100_ptr_t x, sm100_ptr_t w, sm100_ptr_t b,
                          sm100_ptr_t mean, sm100_ptr_t rstd, long long rows, int cols,
                          long long ldx, long long ldy, float eps, int dtype, int wdtype)
{
    int rc = sm100_enter(dev);
    if (rc != SM100_OK) return rc;
    const int pair = ln_pair(dtype, wdtype);
    if (pair < 0) return bad_arg(dev, "booth_sm100_layernorm: types are f32 with f32 parameters, or bf16 or f16 with parameters of the same type or f32");
    if (rows < 0 || cols < 1 || !(eps >= 0.0f)) return bad_arg(dev, "booth_sm100_layernorm: need rows >= 0, cols >= 1, eps >= 0");
    if (rows == 0) return SM100_OK;
    const unsigned e = type_bytes(dtype), we = type_bytes(wdtype);
    if (!matrix_ok(x, e, rows, cols, ldx) || !matrix_ok(y, e, rows, cols, ldy) || (w & (we - 1)) || (b & (we - 1)) || ((mean | rstd) & 3) ||
        (x == y && ldx != ldy))
        return bad_arg(dev, "booth_sm100_layernorm: x and y non-NULL, every operand aligned to its element, pitches >= cols (equal ones when y is x)");
    const int vec = !(((x | y | w | b) & 15) || cols % (int)(16 / e) || ldx % (16 / e) || ldy % (16 / e));
    const ln_shape_t s = ln_shape(dev, rows, cols, vec, 1024);
    int group = s.group;
    void *args[] = { &y, &x, &w, &b, &mean, &rstd, &rows, &cols, &ldx, &ldy, &eps, &group };
    return sm100_launch_k_overlapped(dev, SM100_K_LN_FWD + pair * SM100_LN_FORMS + s.form, s.grid, s.block, 0, args);
}

/* Partial rows of the parameters' gradients: one a block, or one a row range in the walking form. */
#define LN_LOOP_PARTS 64
#define LN_BWD_THREADS 512

size_t booth_sm100_layernorm_backward_workspace(sm100_dev_t *dev, long long rows, int cols, int dtype, int wdtype)
{
    if (!dev || rows < 0 || cols < 1 || ln_pair(dtype, wdtype) < 0) {
        bad_arg(dev, "booth_sm100_layernorm_backward_workspace: bad argument");
        return 0;
    }
    size_t parts = LN_LOOP_PARTS;
    for (int vec = 0; vec < 2; vec++) {
        const ln_shape_t s = ln_shape(dev, rows, cols, vec, LN_BWD_THREADS);
        if (s.form != LN_LOOP && s.grid > parts) parts = s.grid;
    }
    return parts * 2 * (size_t)cols * sizeof(float);
}

int booth_sm100_layernorm_backward(sm100_dev_t *dev, sm100_ptr_t dx, sm100_ptr_t dw, sm100_ptr_t db,
                                   sm100_ptr_t dy, sm100_ptr_t x, sm100_ptr_t w, sm100_ptr_t mean, sm100_ptr_t rstd,
                                   long long rows, int cols, long long lddx, long long lddy, long long ldx,
                                   int dtype, int wdtype, sm100_ptr_t ws, size_t ws_bytes)
{
    int rc = sm100_enter(dev);
    if (rc != SM100_OK) return rc;
    const int pair = ln_pair(dtype, wdtype);
    if (pair < 0) return bad_arg(dev, "booth_sm100_layernorm_backward: types are f32 with f32 parameters, or bf16 or f16 with parameters of the same type or f32");
    if (rows < 0 || cols < 1) return bad_arg(dev, "booth_sm100_layernorm_backward: need rows >= 0, cols >= 1");
    const unsigned e = type_bytes(dtype), we = type_bytes(wdtype);
    const int params = dw || db;
    if (rows > 0 && (!matrix_ok(dy, e, rows, cols, lddy) || !matrix_ok(x, e, rows, cols, ldx) || (dx && !matrix_ok(dx, e, rows, cols, lddx)) ||
                     !mean || !rstd || ((mean | rstd) & 3) || (w & (we - 1)) || (dx && (dx == dy || dx == x))))
        return bad_arg(dev, "booth_sm100_layernorm_backward: dy, x, mean and rstd non-NULL, every operand aligned to its element, "
                            "pitches >= cols, dx apart from dy and x");
    if ((dw | db) & (we - 1)) return bad_arg(dev, "booth_sm100_layernorm_backward: dw and db must be aligned to their element");
    if (params && (!ws || (ws & 15) || ws_bytes < booth_sm100_layernorm_backward_workspace(dev, rows, cols, dtype, wdtype)))
        return bad_arg(dev, "booth_sm100_layernorm_backward: workspace missing, not 16-byte aligned or too small");
    int parts = 0;
    if (rows > 0 && (dx || params)) {
        const int vec = !(((x | dy | dx | w) & 15) || cols % (int)(16 / e) || ldx % (16 / e) || lddy % (16 / e) || (dx && lddx % (16 / e)));
        const ln_shape_t s = ln_shape(dev, rows, cols, vec, LN_BWD_THREADS);
        int group = s.group;
        sm100_ptr_t partial = params ? ws : 0;
        void *args[] = { &dx, &partial, &dy, &x, &w, &mean, &rstd, &rows, &cols, &lddx, &lddy, &ldx, &group };
        parts = (int)s.grid;
        if (s.form != LN_LOOP || dx) {
            rc = sm100_launch_k_overlapped(dev, SM100_K_LN_BWD + pair * SM100_LN_FORMS + s.form, s.grid, s.block, 0, args);
            if (rc != SM100_OK) return rc;
        }
        if (s.form == LN_LOOP && params) {
            parts = rows < LN_LOOP_PARTS ? (int)rows : LN_LOOP_PARTS;
            void *ca[] = { &partial, &dy, &x, &mean, &rstd, &rows, &cols, &lddy, &ldx };
            rc = sm100_launch_k3_overlapped(dev, SM100_K_LN_COLUMNS + type_index(dtype), (unsigned)(((long long)cols + 255) / 256), (unsigned)parts, 1, 256, 1, 1, 0, ca);
            if (rc != SM100_OK) return rc;
        }
    }
    if (params) {
        void *pa[] = { &dw, &db, &ws, &parts, &cols };
        rc = sm100_launch_k3_overlapped(dev, SM100_K_LN_PARAM_GRAD + type_index(wdtype), (unsigned)(((long long)cols + 31) / 32), 2, 1, 256, 1, 1, 0, pa);
    }
    return rc;
}
