/* sm100_train.c -- the training operators: layer normalisation and its gradient,
 * Newton-Schulz orthogonalisation and the Muon update.
 *
 * Like the workloads in sm100_ops.c each call checks its arguments on the host,
 * enqueues its kernels on the device's stream and returns. Nothing is allocated
 * and nothing is waited for, so the calls can be captured into a graph; device
 * memory beyond the operands is a workspace the caller passes in, so two graphs, or
 * two streams that the caller orders, share one only where the caller says so. */
#define _POSIX_C_SOURCE 200809L
#include <limits.h>
#include <math.h>
#include <stdio.h>
#include <string.h>

#include "sm100_internal.h"
#include "kernels/orth_params.cuh"

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

/* Columns are counted in 32 bits, and the last step past them has to fit as well. */
#define LN_MAX_COLS (1 << 30)

/* Kernel of a (value type, parameter type) pair, in the order of the names in sm100_shim.c; -1: no such pair. */
static int ln_pair(int dtype, int wdtype)
{
    if (dtype == SM100_F32) return wdtype == SM100_F32 ? 0 : -1;
    if (dtype == SM100_BF16) return wdtype == SM100_BF16 ? 1 : wdtype == SM100_F32 ? 2 : -1;
    if (dtype == SM100_F16) return wdtype == SM100_F16 ? 3 : wdtype == SM100_F32 ? 4 : -1;
    return -1;
}

/* A form of the kernels: its place among the names, the values a thread has, the most threads a row may have, what
 * the SM's registers hold of its threads, whether the parameters are kept in shared memory, and the bytes of a value
 * it is for (0: any). */
typedef struct { int at, vec, cpt, most; unsigned resident; int kept, bytes; } ln_form_t;

/* Rows so few that each has an SM to itself get eight values a thread: more threads
 * shorten the one row. Else as many values as the registers bear, thirty-two forward and
 * sixteen backward, which spreads what a row costs each thread beside its values; rows too wide for
 * these take the forms that keep parameters or row in shared memory. */
static const ln_form_t ln_forward[] = { { 0, 1, 8, 512, 1024, 0, 0 }, { 1, 1, 32, 256, 512, 0, 0 }, { 2, 1, 16, 640, 640, 1, 0 }, { 3, 1, 32, 512, 512, 1, 0 },
                                        { 4, 0, 8, 512, 768, 0, 0 }, { 5, 0, 16, 512, 640, 0, 0 }, { 6, 0, 32, 512, 512, 1, 0 } };
static const ln_form_t ln_backward[] = { { 0, 1, 8, 512, 768, 0, 0 }, { 1, 1, 16, 256, 512, 0, 0 }, { 2, 1, 20, 512, 512, 1, 4 }, { 2, 1, 16, 640, 640, 1, 2 },
                                         { 3, 1, 32, 512, 512, 1, 0 },
                                         { 4, 0, 8, 512, 768, 0, 0 }, { 5, 0, 16, 512, 512, 0, 0 }, { 6, 0, 32, 512, 512, 1, 0 } };
#define LN_COUNT(a) ((int)(sizeof(a) / sizeof((a)[0])))
#define LN_LOOP 7

/* Shared memory for rings: what an SM has less the blocks' own few KB. */
#define LN_RING_SM (204u << 10)

typedef struct { int form, loop, group, depth; unsigned block, grid, ring; } ln_shape_t;

/* How rows are dealt to threads: the form, the group of threads a row has, and blocks
 * that stay, each taking every grid-th row: as many as an SM holds by registers, and by
 * rings of up to four rows each. */
static ln_shape_t ln_shape(const sm100_dev_t *dev, long long rows, int cols, unsigned esz, int vec, int backward)
{
    ln_shape_t s;
    const ln_form_t *forms = backward ? ln_backward : ln_forward, *f = NULL;
    const int n = backward ? LN_COUNT(ln_backward) : LN_COUNT(ln_forward), few = rows < 2ll * dev->sm_count;
    for (int i = 0; i < n && !f; i++)
        if (forms[i].vec == vec && (!forms[i].bytes || forms[i].bytes == (int)esz) && (forms[i].cpt > 8 || few || (!vec && cols <= 64)) && cols <= forms[i].cpt * forms[i].most) f = &forms[i];
    s.loop = !f;
    s.form = f ? f->at : LN_LOOP;
    s.depth = 1;
    s.ring = 0;
    s.group = 512;
    s.block = 512;
    if (f) {
        int g = (cols + f->cpt - 1) / f->cpt;
        if (g <= 32) { int p = vec ? 1 : 8; while (p < g) p *= 2; g = p; }
        else g = (g + 31) / 32 * 32;
        s.group = g;
        s.block = g <= 32 ? 128u : (unsigned)g;
    }
    const long long per_block = s.group <= 32 ? (long long)s.block / s.group : 1;
    unsigned per_sm = (f ? f->resident : 1024u) / s.block;
    if (per_sm < 1) per_sm = 1;
    if (f) {
        const unsigned arrays = backward ? 2u : 1u, slot = ((unsigned)(f->cpt * s.group) * esz + 15u) / 16u * 16u + 16u;
        const unsigned row = vec ? s.block * (unsigned)f->cpt * esz * arrays : (unsigned)per_block * slot * arrays;
        const unsigned kept = f->kept ? s.block * (unsigned)f->cpt * (backward ? 4u : 8u) : 0u;
        s.depth = 4;
        while (s.depth > 2 && per_sm * ((unsigned)s.depth * row + kept) > LN_RING_SM) s.depth--;
        while (per_sm > 1 && per_sm * ((unsigned)s.depth * row + kept) > LN_RING_SM) per_sm--;
        if ((unsigned)s.depth * row + kept > LN_RING_SM) s.depth = 1;
        s.ring = (unsigned)s.depth * row + kept;
    }
    long long want = (rows + per_block - 1) / per_block;
    if (want > (long long)dev->sm_count * per_sm) want = (long long)dev->sm_count * per_sm;
    s.grid = (unsigned)(want < 1 ? 1 : want);
    return s;
}

static int ln_ready(sm100_dev_t *dev)
{
    if (dev->ln_smem_set) return SM100_OK;
    for (int pair = 0; pair < 5; pair++)
        for (int backward = 0; backward < 2; backward++)
            for (int i = 0; i < LN_LOOP; i++) {
                const int k = (backward ? SM100_K_LN_BWD + pair * SM100_LN_BWD_FORMS : SM100_K_LN_FWD + pair * SM100_LN_FWD_FORMS) + i;
                CUresult cr = dev->api->FuncSetAttribute(dev->k[k], CU_FUNC_ATTRIBUTE_MAX_DYNAMIC_SHARED_SIZE_BYTES, (int)LN_RING_SM);
                if (cr != CUDA_SUCCESS) return sm100_fail(dev, "raising the layer normalisation kernels' shared memory limit", cr);
            }
    dev->ln_smem_set = 1;
    return SM100_OK;
}

int booth_sm100_layernorm(sm100_dev_t *dev, sm100_ptr_t y, sm100_ptr_t x, sm100_ptr_t w, sm100_ptr_t b,
                          sm100_ptr_t mean, sm100_ptr_t rstd, long long rows, int cols,
                          long long ldx, long long ldy, float eps, int dtype, int wdtype)
{
    int rc = sm100_enter(dev);
    if (rc != SM100_OK) return rc;
    const int pair = ln_pair(dtype, wdtype);
    if (pair < 0) return bad_arg(dev, "booth_sm100_layernorm: types are f32 with f32 parameters, or bf16 or f16 with parameters of the same type or f32");
    if (rows < 0 || cols < 1 || cols > LN_MAX_COLS || !(eps >= 0.0f)) return bad_arg(dev, "booth_sm100_layernorm: need rows >= 0, 1 to 2^30 columns, eps >= 0");
    if (rows == 0) return SM100_OK;
    const unsigned e = type_bytes(dtype), we = type_bytes(wdtype);
    if (!matrix_ok(x, e, rows, cols, ldx) || !matrix_ok(y, e, rows, cols, ldy) || (w & (we - 1)) || (b & (we - 1)) || ((mean | rstd) & 3) ||
        (x == y && ldx != ldy) || (mean && mean == rstd))
        return bad_arg(dev, "booth_sm100_layernorm: x and y non-NULL, every operand aligned to its element, pitches >= cols (equal ones when y is x), "
                            "mean apart from rstd");
    const int vec = !(((x | y | w | b) & 15) || cols % (int)(16 / e) || ldx % (16 / e) || ldy % (16 / e));
    if ((rc = ln_ready(dev)) != SM100_OK) return rc;
    const ln_shape_t s = ln_shape(dev, rows, cols, e, vec, 0);
    int group = s.group, depth = s.depth;
    void *args[] = { &y, &x, &w, &b, &mean, &rstd, &rows, &cols, &ldx, &ldy, &eps, &group, &depth };
    return sm100_launch_k_overlapped(dev, SM100_K_LN_FWD + pair * SM100_LN_FWD_FORMS + s.form, s.grid, s.block, s.ring, args);
}

/* Partial rows of the parameters' gradients: one a block, or one a row range in the walking form. */
#define LN_LOOP_PARTS 64

size_t booth_sm100_layernorm_backward_workspace(sm100_dev_t *dev, long long rows, int cols, int dtype, int wdtype)
{
    if (!dev || rows < 0 || cols < 1 || cols > LN_MAX_COLS || ln_pair(dtype, wdtype) < 0) {
        bad_arg(dev, "booth_sm100_layernorm_backward_workspace: bad argument");
        return 0;
    }
    size_t parts = LN_LOOP_PARTS;
    for (int vec = 0; vec < 2; vec++) {
        const ln_shape_t s = ln_shape(dev, rows, cols, type_bytes(dtype), vec, 1);
        if (!s.loop && s.grid > parts) parts = s.grid;
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
    if (rows < 0 || cols < 1 || cols > LN_MAX_COLS) return bad_arg(dev, "booth_sm100_layernorm_backward: need rows >= 0, 1 to 2^30 columns");
    const unsigned e = type_bytes(dtype), we = type_bytes(wdtype);
    const int params = dw || db;
    if (rows > 0 && (!matrix_ok(dy, e, rows, cols, lddy) || !matrix_ok(x, e, rows, cols, ldx) || (dx && !matrix_ok(dx, e, rows, cols, lddx)) ||
                     !mean || !rstd || ((mean | rstd) & 3) || (w & (we - 1)) || (dx && (dx == dy || dx == x))))
        return bad_arg(dev, "booth_sm100_layernorm_backward: dy, x, mean and rstd non-NULL, every operand aligned to its element, "
                            "pitches >= cols, dx apart from dy and x");
    if (((dw | db) & (we - 1)) || (params && dw == db)) return bad_arg(dev, "booth_sm100_layernorm_backward: dw and db must be aligned to their element and apart");
    if (params && (!ws || (ws & 15) || ws_bytes < booth_sm100_layernorm_backward_workspace(dev, rows, cols, dtype, wdtype)))
        return bad_arg(dev, "booth_sm100_layernorm_backward: workspace missing, not 16-byte aligned or too small");
    int parts = 0;
    if (rows > 0 && (dx || params)) {
        const int vec = !(((x | dy | dx | w) & 15) || cols % (int)(16 / e) || ldx % (16 / e) || lddy % (16 / e) || (dx && lddx % (16 / e)));
        if ((rc = ln_ready(dev)) != SM100_OK) return rc;
        const ln_shape_t s = ln_shape(dev, rows, cols, e, vec, 1);
        int group = s.group, depth = s.depth;
        sm100_ptr_t partial = params ? ws : 0;
        void *args[] = { &dx, &partial, &dy, &x, &w, &mean, &rstd, &rows, &cols, &lddx, &lddy, &ldx, &group, &depth };
        parts = (int)s.grid;
        if (!s.loop || dx) {
            rc = sm100_launch_k_overlapped(dev, SM100_K_LN_BWD + pair * SM100_LN_BWD_FORMS + s.form, s.grid, s.block, s.ring, args);
            if (rc != SM100_OK) return rc;
        }
        if (s.loop && params) {
            parts = rows < LN_LOOP_PARTS ? (int)rows : LN_LOOP_PARTS;
            void *ca[] = { &partial, &dy, &x, &mean, &rstd, &rows, &cols, &lddy, &ldx };
            rc = sm100_launch_k3_overlapped(dev, SM100_K_LN_COLUMNS + type_index(dtype), (unsigned)(((long long)cols + 255) / 256), (unsigned)parts, 1, 256, 1, 1, 0, ca);
            if (rc != SM100_OK) return rc;
        }
    }
    if (params) {
        void *pa[] = { &dw, &db, &ws, &parts, &cols };
        /* the more threads a block the fewer partial rows each adds, as long as all blocks run at once:
         * 592 rows of 1024 columns 2 us faster with 1024 threads, 148 of 10000 7.6 against 13.3 us with 512 */
        const unsigned blocks = (unsigned)(((long long)cols + 31) / 32), threads = 2 * blocks <= (unsigned)dev->sm_count ? 1024u : 512u;
        rc = sm100_launch_k3_overlapped(dev, SM100_K_LN_PARAM_GRAD + type_index(wdtype), blocks, 2, 1, threads, 1, 1, 0, pa);
    }
    return rc;
}

/* ---- orthogonalisation and Muon ---- */

#define ORTH_MAX_SIDE (1 << 20)
#define ORTH_SMEM (1024u + 6u * 32768u + 8u * 4096u)    /* 6 x 32 KB or 3 x 64 KB of operand stages, 4 KB for each epilogue warp, and 1 KB to align them */

static size_t up(size_t v, size_t a) { return (v + a - 1) / a * a; }

/* Where things lie in the workspace: the norms' partial sums, then fp16 planes, then the
 * sums of tiles whose K is shared (128 KB a CTA). X is short x long, S and Q short x
 * short; rows of a plane are a multiple of 64 elements apart. X exists twice, the products
 * read one copy and write the other. One-plane results (bf16) keep lo planes of X only. */
typedef struct orth_layout {
    long long s, l, x_pitch, a_pitch;
    int parts;
    size_t x_hi[2], x_lo[2], s_hi, s_lo, q_hi, q_lo, sums, bytes;
} orth_layout_t;

static int orth_layout(const sm100_dev_t *dev, orth_layout_t *o, int batch, int rows, int cols, int two_planes)
{
    if (batch < 1 || batch > 65535 || rows < 1 || cols < 1 || rows > ORTH_MAX_SIDE || cols > ORTH_MAX_SIDE) return 0;
    o->s = rows < cols ? rows : cols;
    o->l = rows < cols ? cols : rows;
    o->x_pitch = (long long)up((size_t)o->l, 64);
    o->a_pitch = (long long)up((size_t)o->s, 64);
    /* the norm: a few thousand elements a block, some four blocks an SM over the batch */
    long long parts = ((long long)rows * cols + 4095) / 4096, most = 592 / batch > 8 ? 592 / batch : 8;
    o->parts = (int)(parts < most ? parts : most);
    const size_t x = up((size_t)batch * o->s * o->x_pitch * 2, 128), a = up((size_t)batch * o->s * o->a_pitch * 2, 128);
    size_t at = up((size_t)batch * o->parts * sizeof(double), 128);
    for (int i = 0; i < 2; i++) { o->x_hi[i] = at; at += x; o->x_lo[i] = at; at += x; }
    o->s_hi = at; at += a;
    o->s_lo = at; if (two_planes) at += a;
    o->q_hi = at; at += a;
    o->q_lo = at; if (two_planes) at += a;
    /* sums of shared tiles: 16, 64 or 128 KB a CTA by tile side, eight parts a tile at most (four pairs), all at once on the GPU */
    size_t sums = 0;
    for (int side = 64; side <= 256; side *= 2) {
        const long long ctas = 8ll * batch * ((o->l + side - 1) / side) * ((o->s + side - 1) / side);
        const size_t need = (size_t)(ctas < dev->sm_count ? ctas : dev->sm_count) * (side == 64 ? 16384u : side == 128 ? 65536u : 131072u);
        if (need > sums) sums = need;
    }
    o->sums = at; at += sums;
    o->bytes = at;
    const long long t = (o->l + 63) / 64;
    return t * ((o->s + 63) / 64) <= INT_MAX / batch;
}

size_t booth_sm100_orthogonalise_workspace(sm100_dev_t *dev, int batch, int rows, int cols, int dtype)
{
    orth_layout_t o;
    if (!dev || type_index(dtype) < 0 || !orth_layout(dev, &o, batch, rows, cols, dtype != SM100_BF16)) {
        bad_arg(dev, "booth_sm100_orthogonalise_workspace: bad argument");
        return 0;
    }
    return o.bytes;
}

/* Map of one plane: batch matrices of rows x cols, rows `pitch` apart, in boxes of 64 x 64
 * (128 bytes a row, 128-byte swizzle). What lies outside a matrix reads as zero. */
static int plane_map(sm100_dev_t *dev, CUtensorMap *map, CUdeviceptr p, long long rows, long long cols, long long pitch, int batch)
{
    cuuint64_t dims[3] = { (cuuint64_t)cols, (cuuint64_t)rows, (cuuint64_t)batch };
    cuuint64_t strides[2] = { (cuuint64_t)pitch * 2, (cuuint64_t)pitch * rows * 2 };
    cuuint32_t box[3] = { 64, 64, 1 }, step[3] = { 1, 1, 1 };
    CUresult cr = dev->api->TensorMapEncodeTiled(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 3, (void *)(size_t)p, dims, strides, box, step,
                                                 CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                                                 CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return cr == CUDA_SUCCESS ? SM100_OK : sm100_fail(dev, "cuTensorMapEncodeTiled", cr);
}

/* cuTensorMapEncodeTiled wants its maps on 64-byte boundaries. */
typedef struct { CUtensorMap hi __attribute__((aligned(64))), lo __attribute__((aligned(64))); } plane_maps_t;

/* How many clusters of `ctas` CTAs of the product kernels the GPU holds at once (asked of
 * the driver once; else what the SMs hold, less one in seven for clusters that have
 * to fit inside a group of SMs). Only a measure for the choice below: no cluster waits for another. */
static int orth_clusters(sm100_dev_t *dev, int ctas)
{
    if (dev->orth_clusters[ctas]) return dev->orth_clusters[ctas];
    int n = dev->sm_count / ctas;
    if (ctas > 2) n = n * 6 / 7;
    if (dev->api->OccupancyMaxActiveClusters) {
        CUlaunchAttribute attr;
        memset(&attr, 0, sizeof attr);
        attr.id = CU_LAUNCH_ATTRIBUTE_CLUSTER_DIMENSION;
        attr.value.clusterDim.x = (unsigned)ctas; attr.value.clusterDim.y = 1; attr.value.clusterDim.z = 1;
        CUlaunchConfig cfg;
        memset(&cfg, 0, sizeof cfg);
        cfg.gridDimX = (unsigned)ctas * 64u; cfg.gridDimY = 1; cfg.gridDimZ = 1;
        cfg.blockDimX = 384; cfg.blockDimY = 1; cfg.blockDimZ = 1;
        cfg.sharedMemBytes = ORTH_SMEM;
        cfg.hStream = dev->stream;
        cfg.attrs = &attr; cfg.numAttrs = 1;
        int got = 0;
        if (dev->api->OccupancyMaxActiveClusters(&got, dev->k[SM100_K_ORTH_PRODUCT + 4], &cfg) == CUDA_SUCCESS && got > 0) n = got;
    }
    dev->orth_clusters[ctas] = n > 0 ? n : 1;
    return dev->orth_clusters[ctas];
}

typedef struct { int side, split; long long tiles; double us; } orth_plan_t;

/* One product with a given tile side: the parts its K is cut into and how long it takes,
 * in microseconds measured in a chain of products (one plane, two planes). A product costs
 * `base`, a K block of 64 `block` (64-tiles slow one another down in L2: .001 more for every CTA), a
 * further wave its K blocks or, if that is longer, its epilogue; parts meet at `meet`. A
 * 1000 x 1000 x 1000 product in two planes comes to 17, 12 (two parts) and 15 us by side, 2048 cubed to 95, 53 and 34.
 * The choice is worth: 1024 x 4096 f32 322 us, 334 with the larger `base` and `meet` of an epilogue through shared
 * memory; 2048 x 8192 bf16 624 against 648; 768 x 768 bf16 132 against 128 the other way.
 * K is shared only while everything runs at once. */
static orth_plan_t orth_product_plan(sm100_dev_t *dev, int side, long long rows, long long cols, long long K, int batch, int sym, int two_planes)
{
    static const struct { double base[2], block[2], epilogue, meet; } cost[3] = {
        { { 3.3, 3.9 }, { 0.22, 0.26 }, 1.5, 1.0 }, { { 4.0, 4.5 }, { 0.30, 0.75 }, 2.5, 1.5 }, { { 6.0, 7.0 }, { 0.32, 0.85 }, 4.5, 2.5 } };
    const int f = side == 64 ? 0 : side == 128 ? 1 : 2, ctas = side == 256 ? 2 : 1;
    const long long m = (rows + side - 1) / side, n = (cols + side - 1) / side, chunks = (K + 127) / 128;
    orth_plan_t best = { side, 1, batch * (sym ? m * (m + 1) / 2 : m * n), 0.0 };
    for (int s = 1; s * ctas <= 8 && s <= chunks; s++) {
        const long long slots = orth_clusters(dev, s * ctas), waves = (best.tiles + slots - 1) / slots;
        if (s > 1 && (waves > 1 || s * ctas * best.tiles > dev->sm_count)) break;
        const double running = (double)(best.tiles < slots ? best.tiles : slots) * s;
        const double blocks = 2.0 * ((chunks + s - 1) / s) * (cost[f].block[two_planes] + (f == 0 ? 0.001 * running : 0.0));
        const double us = cost[f].base[two_planes] + blocks + (waves - 1) * fmax(blocks, cost[f].epilogue) + (s > 1 ? cost[f].meet : 0.0);
        if (s == 1 || us < best.us) { best.us = us; best.split = s; }
    }
    return best;
}

/* Forms of a step's three products, chosen together: rows of a product may span two tiles of the triangle that the
 * product before it stored, not more (see the kernel), so small tiles for S and Q keep the update from large ones. */
static void orth_plan(sm100_dev_t *dev, const orth_layout_t *o, int batch, int poly, int two_planes, orth_plan_t plan[3])
{
    orth_plan_t g[3], q[3], u[3];
    double best = 0.0;
    for (int f = 0; f < 3; f++) {
        g[f] = orth_product_plan(dev, 64 << f, o->s, o->s, o->l, batch, 1, two_planes);
        q[f] = orth_product_plan(dev, 64 << f, o->s, o->s, o->s, batch, 1, two_planes);
        u[f] = orth_product_plan(dev, 64 << f, o->s, o->l, o->s, batch, 0, two_planes);
    }
    for (int i = 0; i < 3; i++)
        for (int j = 0; j < 3; j++)
            for (int k = 0; k < 3; k++) {
                if (poly ? j > i + 1 || k > j + 1 : j != i || k > i + 1) continue;
                const double us = g[i].us + (poly ? q[j].us : 0.0) + u[k].us;
                if (best == 0.0 || us < best) { best = us; plan[0] = g[i]; plan[1] = q[j]; plan[2] = u[k]; }
            }
}

static int orth_launch(sm100_dev_t *dev, const orth_plan_t *plan, const plane_maps_t *a, const plane_maps_t *b, const plane_maps_t *out,
                       orth_product_t *p, int two_planes)
{
    const int ctas = (plan->side == 256 ? 2 : 1) * plan->split, form = plan->side == 64 ? 0 : plan->side == 128 ? 2 : 4;
    /* a shared tile's cluster takes that one tile: the parts meet a fixed number of times */
    const long long slots = orth_clusters(dev, ctas), groups = plan->split > 1 || plan->tiles < slots ? plan->tiles : slots;
    p->split = plan->split;
    void *args[] = { (void *)&a->hi, (void *)&a->lo, (void *)&b->hi, (void *)&b->lo, (void *)&out->hi, (void *)&out->lo, p };
    const int rc = sm100_launch_k_cluster(dev, SM100_K_ORTH_PRODUCT + form + (two_planes ? 1 : 0), (unsigned)(groups * ctas), (unsigned)ctas, 384, ORTH_SMEM, args);
    p->silent = 0;
    if (p->mode <= ORTH_POLY) p->tri = plan->side;      /* how the product that reads this one finds its triangle */
    return rc;
}

static int orth_status_ready(sm100_dev_t *dev)
{
    if (!dev->orth_smem_set) {
        for (int i = 0; i < 6; i++) {
            CUresult cr = dev->api->FuncSetAttribute(dev->k[SM100_K_ORTH_PRODUCT + i], CU_FUNC_ATTRIBUTE_MAX_DYNAMIC_SHARED_SIZE_BYTES, (int)ORTH_SMEM);
            if (cr != CUDA_SUCCESS) return sm100_fail(dev, "raising the product kernels' shared memory limit", cr);
        }
        dev->orth_smem_set = 1;
    }
    dev->orth_pending = 1;
    return SM100_OK;
}

/* src -> normalise -> ns->steps x (gram, polynomial, update); the last update goes to w. */
static int newton_schulz(sm100_dev_t *dev, orth_source_t *src, const orth_product_t *last, int batch, int two_planes,
                         const booth_newton_schulz_t *ns, float factor, sm100_ptr_t ws, const orth_layout_t *o)
{
    int rc = orth_status_ready(dev);
    if (rc != SM100_OK) return rc;
    /* the maps first: whatever can fail fails before the momentum changes */
    plane_maps_t x[2], sm, qm;
    for (int i = 0; i < 2; i++) {
        if ((rc = plane_map(dev, &x[i].hi, ws + o->x_hi[i], o->s, o->l, o->x_pitch, batch)) != SM100_OK) return rc;
        if ((rc = plane_map(dev, &x[i].lo, ws + o->x_lo[i], o->s, o->l, o->x_pitch, batch)) != SM100_OK) return rc;
    }
    if ((rc = plane_map(dev, &sm.hi, ws + o->s_hi, o->s, o->s, o->a_pitch, batch)) != SM100_OK) return rc;
    if ((rc = plane_map(dev, &qm.hi, ws + o->q_hi, o->s, o->s, o->a_pitch, batch)) != SM100_OK) return rc;
    sm.lo = sm.hi; qm.lo = qm.hi;       /* not read or written by the one-plane kernels */
    if (two_planes) {
        if ((rc = plane_map(dev, &sm.lo, ws + o->s_lo, o->s, o->s, o->a_pitch, batch)) != SM100_OK) return rc;
        if ((rc = plane_map(dev, &qm.lo, ws + o->q_lo, o->s, o->s, o->a_pitch, batch)) != SM100_OK) return rc;
    }
    const int tall = src->rows > src->cols;
    CUdeviceptr partial = ws;
    int parts = o->parts;
    void *na[] = { src, &partial };
    rc = sm100_launch_k3_overlapped(dev, SM100_K_ORTH_NORM, (unsigned)parts, (unsigned)batch, 1, 256, 1, 1, 0, na);
    if (rc != SM100_OK) return rc;
    CUdeviceptr hi = ws + o->x_hi[0], lo = ws + o->x_lo[0];
    float eps = ns->eps;
    long long pitch = o->x_pitch, plane = o->x_pitch * o->s;
    int t = tall;
    void *sa[] = { src, &partial, &parts, &eps, &hi, &lo, &pitch, &plane, &t };
    rc = sm100_launch_k3_overlapped(dev, SM100_K_ORTH_SPLIT, (unsigned)((src->cols + 63) / 64), (unsigned)((src->rows + 63) / 64), (unsigned)batch,
                                    256, 1, 1, 0, sa);
    if (rc != SM100_OK) return rc;
    /* a I + b A + c A A = c (A + beta I)^2 + gamma I; without the square, b A + a I. X is held times 2^14, S times
     * 2^12 (|A| < 4 and |beta| <= 4), Q times what its largest value over singular values below 2 allows. */
    const double a = ns->a, b = ns->b, c = ns->c, xs = 16384.0, ss = 4096.0;
    const double beta = c != 0.0 ? b / (2.0 * c) : 0.0, gamma = c != 0.0 ? a - b * b / (4.0 * c) : a;
    double most = fmax(fabs(a), fabs(a + 4.0 * b + 16.0 * c));
    if (beta < 0.0) most = fmax(most, fabs(gamma));         /* the polynomial's value at its vertex */
    double qs = 16384.0;
    while (qs * most > 60000.0) qs *= 0.5;

    orth_plan_t plan[3];
    orth_plan(dev, o, batch, c != 0.0, two_planes, plan);
    orth_product_t q = *last;
    q.batch = batch;
    q.sums = ws + o->sums;
    q.status = dev->scratch + SM100_SCRATCH_ORTH_STATUS;
    q.told = (unsigned long long)(size_t)dev->orth_told;        /* page-locked memory has one address for both sides */
    q.wait_ns = (unsigned long long)dev->gemm_wait_ms * 1000000ull;
    const int steps = ns->steps & ~BOOTH_NS_TEST_SILENT_PRODUCER;
    q.silent = (ns->steps & BOOTH_NS_TEST_SILENT_PRODUCER) != 0;        /* the first product's producers issue nothing */
    for (int i = 0; i < steps; i++) {
        const int from = i & 1, to = from ^ 1, end = i == steps - 1;
        q.rows = q.cols = (int)o->s;
        q.mode = ORTH_GRAM; q.K = (int)o->l; q.lo = two_planes;
        q.out_hi = ws + (c == 0.0 ? o->q_hi : o->s_hi); q.out_lo = ws + (c == 0.0 ? o->q_lo : o->s_lo);
        q.out_pitch = o->a_pitch; q.out_plane = o->a_pitch * o->s;
        if (c == 0.0) {
            q.alpha = (float)(b * qs / (xs * xs)); q.diag = (float)(a * qs);
            if ((rc = orth_launch(dev, &plan[0], &x[from], &x[from], &qm, &q, two_planes)) != SM100_OK) return rc;
        } else {
            q.alpha = (float)(ss / (xs * xs)); q.diag = (float)(beta * ss);
            if ((rc = orth_launch(dev, &plan[0], &x[from], &x[from], &sm, &q, two_planes)) != SM100_OK) return rc;
            q.mode = ORTH_POLY; q.K = (int)o->s;
            q.out_hi = ws + o->q_hi; q.out_lo = ws + o->q_lo;
            q.alpha = (float)(c * qs / (ss * ss)); q.diag = (float)(gamma * qs);
            if ((rc = orth_launch(dev, &plan[1], &sm, &sm, &qm, &q, two_planes)) != SM100_OK) return rc;
        }
        q.mode = end ? ORTH_RESULT : ORTH_UPDATE; q.K = (int)o->s; q.lo = 1;
        q.cols = (int)o->l;
        q.out_hi = ws + o->x_hi[to]; q.out_lo = ws + o->x_lo[to];
        q.out_pitch = o->x_pitch; q.out_plane = o->x_pitch * o->s;
        q.alpha = (float)(end ? factor / (qs * xs) : 1.0 / qs); q.diag = 0.0f;
        if ((rc = orth_launch(dev, &plan[2], &qm, &x[from], &x[to], &q, two_planes)) != SM100_OK) return rc;
    }
    return SM100_OK;
}

static const booth_newton_schulz_t ns_default = { 5, 3.4445f, -4.7750f, 2.0315f, 1e-7f };

static int ns_ok(const booth_newton_schulz_t *ns)
{
    const int steps = ns->steps & ~BOOTH_NS_TEST_SILENT_PRODUCER;
    return steps >= 1 && steps <= 64 && isfinite(ns->a) && isfinite(ns->b) && isfinite(ns->c) && isfinite(ns->eps) && ns->eps > 0.0f &&
           (ns->c == 0.0f || fabsf(ns->b) <= 8.0f * fabsf(ns->c));
}

/* batch matrices: the pitch no shorter than a row, the last element within 2^59 elements of the first. */
static int matrices_ok(sm100_ptr_t p, int dtype, int batch, int rows, int cols, long long ld, long long stride)
{
    if (!matrix_ok(p, type_bytes(dtype), rows, cols, ld) || stride < 0) return 0;
    return batch <= 1 || (stride >= cols && stride <= (1ll << 59) / batch);
}

/* Whether the rows of all matrices lie apart, as what is written must: one matrix behind the other, side by side, or in any
 * other way in which no row of the matrix k further on begins inside a row of this one, or the other way round. */
static int apart(int batch, int rows, int cols, long long ld, long long stride)
{
    if (batch <= 1 || stride >= (rows - 1) * ld + cols || ld >= (batch - 1) * stride + cols) return 1;
    for (long long k = 1; k < batch; k++) {
        const long long row = k * stride / ld, in = k * stride - row * ld;
        if (row >= rows) break;
        if (in < cols || (row + 1 < rows && ld - in < cols)) return 0;
    }
    return 1;
}

/* Whether groups of four elements of every row are aligned to their size. */
static int four_ok(sm100_ptr_t p, int dtype, int batch, int cols, long long ld, long long stride)
{
    return !(p & (4 * type_bytes(dtype) - 1)) && cols % 4 == 0 && ld % 4 == 0 && (batch == 1 || stride % 4 == 0);
}

int booth_sm100_orthogonalise(sm100_dev_t *dev, sm100_ptr_t out, sm100_ptr_t in, int batch, int rows, int cols,
                              long long ld_in, long long stride_in, long long ld_out, long long stride_out,
                              int dtype, const booth_newton_schulz_t *ns, sm100_ptr_t ws, size_t ws_bytes)
{
    int rc = sm100_enter(dev);
    if (rc != SM100_OK) return rc;
    orth_layout_t o;
    if (!ns) ns = &ns_default;
    if (type_index(dtype) < 0) return bad_arg(dev, "booth_sm100_orthogonalise: the type is f32, bf16 or f16");
    if (!ns_ok(ns)) return bad_arg(dev, "booth_sm100_orthogonalise: need 1 to 64 steps, finite coefficients with c = 0 or |b| <= 8 |c|, and eps > 0");
    if (!orth_layout(dev, &o, batch, rows, cols, dtype != SM100_BF16) || !matrices_ok(in, dtype, batch, rows, cols, ld_in, stride_in) ||
        !matrices_ok(out, dtype, batch, rows, cols, ld_out, stride_out) || !apart(batch, rows, cols, ld_out, stride_out) ||
        (in == out && (ld_in != ld_out || (batch > 1 && stride_in != stride_out))))
        return bad_arg(dev, "booth_sm100_orthogonalise: need 1 to 65535 matrices of 1 to 2^20 rows and columns, operands non-NULL and aligned to "
                            "their element, pitches >= cols, strides >= cols (equal ones when out is in), matrices of out apart from one another");
    if (!ws || (ws & 127) || ws_bytes < o.bytes)
        return bad_arg(dev, "booth_sm100_orthogonalise: workspace missing, not 128-byte aligned or too small");
    orth_source_t src;
    memset(&src, 0, sizeof src);
    src.g = in; src.ld_g = ld_in; src.stride_g = stride_in; src.type_g = type_index(dtype);
    src.rows = rows; src.cols = cols;
    src.vec = four_ok(in, dtype, batch, cols, ld_in, stride_in);
    src.flat = ld_in == cols;
    orth_product_t last;
    memset(&last, 0, sizeof last);
    last.w = out; last.ld_w = ld_out; last.stride_w = stride_out; last.type_w = type_index(dtype);
    last.tall = rows > cols;
    last.vec_w = four_ok(out, dtype, batch, cols, ld_out, stride_out);
    return newton_schulz(dev, &src, &last, batch, dtype != SM100_BF16, ns, 1.0f, ws, &o);
}

int booth_sm100_muon_step(sm100_dev_t *dev, sm100_ptr_t w, sm100_ptr_t m, sm100_ptr_t g, int batch, int rows, int cols,
                          const booth_muon_t *p, const booth_newton_schulz_t *ns, sm100_ptr_t ws, size_t ws_bytes)
{
    int rc = sm100_enter(dev);
    if (rc != SM100_OK) return rc;
    orth_layout_t o;
    if (!ns) ns = &ns_default;
    if (!p || type_index(p->wdtype) < 0 || type_index(p->mdtype) < 0 || type_index(p->gdtype) < 0)
        return bad_arg(dev, "booth_sm100_muon_step: the types are f32, bf16 or f16");
    if (!ns_ok(ns)) return bad_arg(dev, "booth_sm100_muon_step: need 1 to 64 steps, finite coefficients with c = 0 or |b| <= 8 |c|, and eps > 0");
    if (!isfinite(p->lr) || !isfinite(p->scale) || !isfinite(p->weight_decay) || !(p->momentum >= 0.0f && p->momentum <= 1.0f))
        return bad_arg(dev, "booth_sm100_muon_step: need a finite learning rate, scale and weight decay, and momentum in [0, 1]");
    const int two_planes = p->wdtype != SM100_BF16;
    if (!orth_layout(dev, &o, batch, rows, cols, two_planes) || !matrices_ok(w, p->wdtype, batch, rows, cols, p->ld_w, p->stride_w) ||
        !matrices_ok(m, p->mdtype, batch, rows, cols, p->ld_m, p->stride_m) || !apart(batch, rows, cols, p->ld_w, p->stride_w) ||
        !apart(batch, rows, cols, p->ld_m, p->stride_m) || !matrices_ok(g, p->gdtype, batch, rows, cols, p->ld_g, p->stride_g) ||
        w == m || w == g || m == g)
        return bad_arg(dev, "booth_sm100_muon_step: need 1 to 65535 matrices of 1 to 2^20 rows and columns; w, m and g non-NULL, apart from one "
                            "another and aligned to their element; pitches >= cols, strides >= cols, matrices of w and of m apart");
    if (!ws || (ws & 127) || ws_bytes < o.bytes)
        return bad_arg(dev, "booth_sm100_muon_step: workspace missing, not 128-byte aligned or too small");
    orth_source_t src;
    memset(&src, 0, sizeof src);
    src.g = g; src.ld_g = p->ld_g; src.stride_g = p->stride_g; src.type_g = type_index(p->gdtype);
    src.m = m; src.ld_m = p->ld_m; src.stride_m = p->stride_m; src.type_m = type_index(p->mdtype);
    src.rows = rows; src.cols = cols;
    src.nesterov = p->nesterov != 0; src.mu = p->momentum;
    src.vec = four_ok(g, p->gdtype, batch, cols, p->ld_g, p->stride_g) && four_ok(m, p->mdtype, batch, cols, p->ld_m, p->stride_m);
    src.flat = p->ld_g == cols && p->ld_m == cols;
    orth_product_t last;
    memset(&last, 0, sizeof last);
    last.w = w; last.ld_w = p->ld_w; last.stride_w = p->stride_w; last.type_w = type_index(p->wdtype);
    last.tall = rows > cols;
    last.vec_w = four_ok(w, p->wdtype, batch, cols, p->ld_w, p->stride_w);
    last.keep = (float)(1.0 - (double)p->lr * p->weight_decay);
    return newton_schulz(dev, &src, &last, batch, two_planes, ns, (float)(-(double)p->lr * p->scale), ws, &o);
}
