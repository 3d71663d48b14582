// layernorm.cu -- layer normalisation of the rows of a matrix, and its gradient.
//
// Forward, per row of `cols` values:
//     mean = sum x / cols,  var = sum (x - mean)^2 / cols,  rstd = 1 / sqrt(var + eps)
//     y = (x - mean) rstd w + b
// Backward, with xhat = (x - mean) rstd, p = mean(w dy), q = mean(w dy xhat):
//     dx = rstd (w dy - p - xhat q);   dw = sum over rows of dy xhat;   db = sum over rows of dy
//
// Both read every value once and write every result once, so HBM bounds them. A
// row belongs to one group of threads: 1 to 32 lanes of a warp for narrow rows, a whole
// block for wider ones, 8 or 16 values a thread. The mean is taken first and the variance
// from the differences (the row is on chip, a second pass costs no memory), with the
// differences' own mean as a correction, so a row far from zero loses nothing.
//
// Blocks stay and walk over the rows. Vector forms keep the next few rows on their way
// with cp.async into a ring in shared memory, in which every thread has places of its
// own for what it alone reads, so the ring needs no barrier; with the next row held in
// registers instead, 16 KB an SM were in flight and 16384 x 4096 bf16 took 116 us forward
// and 128 backward.
//
// The backward pass walks the rows once for all three results: each thread adds dy
// and dy xhat of its own columns into registers over all the rows its block sees,
// the block writes one partial row, and layernorm_param_grad adds the partial
// rows in index order. No atomics: results repeat bit for bit.
//
// Sums, statistics and products are fp32 (the last sum over the blocks double);
// values are rounded to the tensor's type once, when they are stored.
//
// Forms: v8, v16, vw read 16-byte vectors (row starts and parameters 16-byte
// aligned, cols a multiple of the vector), vw up to 1024 threads a row with the parameters
// from cache; s8, s16 read single elements, neighbouring threads on neighbouring
// columns, for any alignment; loop goes through the row several times from
// cache, for rows no block can hold.
#include "common.cuh"
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace ln {

__device__ __forceinline__ float to_f32(float v) { return v; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 v) { return __bfloat162float(v); }
__device__ __forceinline__ float to_f32(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T from_f32(float v);
template <> __device__ __forceinline__ float from_f32<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_f32<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_f32<__half>(float v) { return __float2half_rn(v); }

// E values read or written by one access: 16 bytes, or one element (E = 1).
template <typename T, int E> struct __align__(E * sizeof(T)) Chunk { T v[E]; };

template <typename T, int E> __device__ __forceinline__ void load_params(const T *p, long long col, float (&out)[E])
{
    if constexpr (E * sizeof(T) > 16) {         // fp32 parameters beside 16-bit values: two 16-byte loads
        const Chunk<T, E / 2> a = *reinterpret_cast<const Chunk<T, E / 2> *>(p + col);
        const Chunk<T, E / 2> b = *reinterpret_cast<const Chunk<T, E / 2> *>(p + col + E / 2);
#pragma unroll
        for (int e = 0; e < E / 2; e++) { out[e] = to_f32(a.v[e]); out[E / 2 + e] = to_f32(b.v[e]); }
    } else {
        const Chunk<T, E> a = *reinterpret_cast<const Chunk<T, E> *>(p + col);
#pragma unroll
        for (int e = 0; e < E; e++) out[e] = to_f32(a.v[e]);
    }
}

// The threads that share a row: `size` of them, thread `t`; `rows` groups in the
// block. Up to 32 threads a group is part of a warp (a power of two), above that
// it is the whole block.
struct Group {
    int size, t, index, per_block;
    unsigned turn;
    __device__ __forceinline__ Group(int size_) : size(size_), turn(0)
    {
        const int tid = (int)threadIdx.x;
        if (size > 32) { t = tid; index = 0; per_block = 1; }
        else { t = tid & (size - 1); index = tid / size; per_block = (int)blockDim.x / size; }
    }
    // Sums of a and b over the group, the same bits in every thread. Called by all threads of
    // the block in step. `sh` holds 2 x 32 values; the halves alternate, so one barrier a call is enough.
    __device__ __forceinline__ float2 sum2(float a, float b, float2 (*sh)[32])
    {
        const int top = size < 32 ? size : 32;
        for (int o = top >> 1; o > 0; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            b += __shfl_xor_sync(0xffffffffu, b, o);
        }
        if (size > 32) {
            const int warps = size >> 5, lane = t & 31;
            float2 *s = sh[turn & 1];
            turn++;
            if (lane == 0) s[t >> 5] = make_float2(a, b);
            __syncthreads();
            const float2 v = lane < warps ? s[lane] : make_float2(0.f, 0.f);
            a = v.x; b = v.y;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                a += __shfl_xor_sync(0xffffffffu, a, o);
                b += __shfl_xor_sync(0xffffffffu, b, o);
            }
        }
        return make_float2(a, b);
    }
};

template <typename T, int E, int NCH>
__device__ __forceinline__ void load_row(Chunk<T, E> (&c)[NCH], const T *row, const Group &g, int cols, bool live)
{
#pragma unroll
    for (int j = 0; j < NCH; j++) {
        const int col = (j * g.size + g.t) * E;
        if (live && col < cols) c[j] = *reinterpret_cast<const Chunk<T, E> *>(row + col);
        else {
#pragma unroll
            for (int e = 0; e < E; e++) c[j].v[e] = from_f32<T>(0.f);
        }
    }
}

// The ring: `depth` rows ahead of A arrays; chunk j of array a of a stage at ((stage A + a) NCH + j) blockDim 16 bytes,
// 16 bytes a thread. Every row position commits one group, with or without copies, so that the count of groups
// tells which row has landed.
template <int A, int NCH> struct Ring {
    uint32_t base, row_bytes;
    int depth, stage;
    __device__ __forceinline__ Ring(int depth_) : depth(depth_), stage(0)
    {
        extern __shared__ uint4 ln_ring[];
        base = (uint32_t)__cvta_generic_to_shared(ln_ring) + threadIdx.x * 16u;
        row_bytes = blockDim.x * 16u;
    }
    __device__ __forceinline__ uint32_t at(int a, int j) const { return base + (uint32_t)((stage * A + a) * NCH + j) * row_bytes; }
    template <typename T, int E> __device__ __forceinline__ void fetch(int a, const T *row, const Group &g, int cols, bool live) const
    {
#pragma unroll
        for (int j = 0; j < NCH; j++) {
            const int col = (j * g.size + g.t) * E;
            if (live && col < cols) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(at(a, j)), "l"(row + col) : "memory");
        }
    }
    __device__ __forceinline__ void commit() const { asm volatile("cp.async.commit_group;" ::: "memory"); }
    __device__ __forceinline__ void next() { stage = stage + 1 == depth ? 0 : stage + 1; }
    // This thread's oldest outstanding row has landed.
    __device__ __forceinline__ void wait() const
    {
        if (depth == 4) asm volatile("cp.async.wait_group 3;" ::: "memory");
        else if (depth == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
        else if (depth == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    template <typename T, int E> __device__ __forceinline__ Chunk<T, E> get(int a, int j, bool live) const
    {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (live) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at(a, j)) : "memory");
        return *reinterpret_cast<const Chunk<T, E> *>(&v);
    }
};

// Mean and 1/deviation of a row held as NCH chunks.
template <typename T, int E, int NCH>
__device__ __forceinline__ void row_stats(const Chunk<T, E> (&c)[NCH], Group &g, int cols, float eps, float2 (*sh)[32], float &mean, float &rstd)
{
    float s = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; j++)
#pragma unroll
        for (int e = 0; e < E; e++) s += to_f32(c[j].v[e]);      // columns past the end hold zero
    const float m = g.sum2(s, 0.f, sh).x / (float)cols;
    float d1 = 0.f, d2 = 0.f;
#pragma unroll
    for (int j = 0; j < NCH; j++)
        if ((j * g.size + g.t) * E < cols) {
#pragma unroll
            for (int e = 0; e < E; e++) { const float d = to_f32(c[j].v[e]) - m; d1 += d; d2 = fmaf(d, d, d2); }
        }
    const float2 t = g.sum2(d1, d2, sh);
    const float dm = t.x / (float)cols;                          // what rounding left in m
    mean = m + dm;
    rstd = __frsqrt_rn(fmaxf(t.y / (float)cols - dm * dm, 0.f) + eps);
    if (!(t.y == t.y)) rstd = t.y;                               // fmaxf drops a NaN; the row keeps it
}

template <typename T, typename W, bool VEC, int CPT, bool HOLD>
__device__ __forceinline__ void forward(T *__restrict__ y, const T *__restrict__ x, const W *__restrict__ w, const W *__restrict__ b,
                                        float *__restrict__ mean_out, float *__restrict__ rstd_out, long long rows, int cols,
                                        long long ldx, long long ldy, float eps, int group, int depth)
{
    constexpr int E = VEC ? 16 / (int)sizeof(T) : 1, NCH = CPT / E;
    __shared__ float2 sh[2][32];
    Group g(group);
    float pw[HOLD ? NCH : 1][E], pb[HOLD ? NCH : 1][E];         // the parameters of this thread's columns
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const long long step = (long long)gridDim.x * g.per_block;
    long long base = (long long)blockIdx.x * g.per_block;
    Ring<1, VEC ? NCH : 1> ring(depth);
    Chunk<T, E> cur[NCH], nxt[VEC ? 1 : NCH];
    if constexpr (VEC) {
        for (int d = 0; d < depth; d++) {
            const long long row = base + g.index + d * step;
            ring.template fetch<T, E>(0, x + row * ldx, g, cols, row < rows);
            ring.commit();
            ring.next();
        }
    } else {
        load_row<T, E, NCH>(cur, x + (base + g.index) * ldx, g, cols, base + g.index < rows);
    }
    const auto params = [&](int j, float (&qw)[E], float (&qb)[E]) {
        const int col = (j * g.size + g.t) * E;
#pragma unroll
        for (int e = 0; e < E; e++) { qw[e] = 1.f; qb[e] = 0.f; }
        if (col < cols) {
            if (w) load_params<W, E>(w, col, qw);
            if (b) load_params<W, E>(b, col, qb);
        }
    };
    if constexpr (HOLD) {
#pragma unroll
        for (int j = 0; j < NCH; j++) params(j, pw[j], pb[j]);
    }
    for (; base < rows; base += step) {
        const long long row = base + g.index;
        if constexpr (VEC) {
            ring.wait();
#pragma unroll
            for (int j = 0; j < NCH; j++) cur[j] = ring.template get<T, E>(0, j, row < rows && (j * g.size + g.t) * E < cols);
        } else {
            load_row<T, E, NCH>(nxt, x + (row + step) * ldx, g, cols, row + step < rows);
        }
        float mean, rstd;
        row_stats<T, E, NCH>(cur, g, cols, eps, sh, mean, rstd);
        if constexpr (VEC) {                    // the row is in registers: its places may fill again
            const long long ahead = row + depth * step;
            ring.template fetch<T, E>(0, x + ahead * ldx, g, cols, ahead < rows);
            ring.commit();
            ring.next();
        }
        if (row < rows) {
            if (g.t == 0) {
                if (mean_out) mean_out[row] = mean;
                if (rstd_out) rstd_out[row] = rstd;
            }
            T *out = y + row * ldy;
#pragma unroll
            for (int j = 0; j < NCH; j++) {
                const int col = (j * g.size + g.t) * E;
                if (col < cols) {
                    Chunk<T, E> o;
                    if constexpr (HOLD) {
#pragma unroll
                        for (int e = 0; e < E; e++) o.v[e] = from_f32<T>(fmaf((to_f32(cur[j].v[e]) - mean) * rstd, pw[j][e], pb[j][e]));
                    } else {
                        float qw[E], qb[E];
                        params(j, qw, qb);
#pragma unroll
                        for (int e = 0; e < E; e++) o.v[e] = from_f32<T>(fmaf((to_f32(cur[j].v[e]) - mean) * rstd, qw[e], qb[e]));
                    }
                    *reinterpret_cast<Chunk<T, E> *>(out + col) = o;
                }
            }
        }
        if constexpr (!VEC) {
#pragma unroll
            for (int j = 0; j < NCH; j++) cur[j] = nxt[j];
        }
    }
}

// Rows of any length: three passes over the row, the second and third from cache.
template <typename T, typename W>
__device__ __forceinline__ void forward_loop(T *y, const T *x, const W *__restrict__ w, const W *__restrict__ b, float *__restrict__ mean_out,
                                             float *__restrict__ rstd_out, long long rows, int cols, long long ldx, long long ldy, float eps)
{
    __shared__ float2 sh[2][32];
    Group g((int)blockDim.x);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *src = x + row * ldx;
        T *out = y + row * ldy;
        float s = 0.f;
        for (int c = g.t; c < cols; c += g.size) s += to_f32(src[c]);
        const float m = g.sum2(s, 0.f, sh).x / (float)cols;
        float d1 = 0.f, d2 = 0.f;
        for (int c = g.t; c < cols; c += g.size) { const float d = to_f32(src[c]) - m; d1 += d; d2 = fmaf(d, d, d2); }
        const float2 t = g.sum2(d1, d2, sh);
        const float dm = t.x / (float)cols, mean = m + dm;
        float rstd = __frsqrt_rn(fmaxf(t.y / (float)cols - dm * dm, 0.f) + eps);
        if (!(t.y == t.y)) rstd = t.y;
        if (g.t == 0) {
            if (mean_out) mean_out[row] = mean;
            if (rstd_out) rstd_out[row] = rstd;
        }
        for (int c = g.t; c < cols; c += g.size)
            out[c] = from_f32<T>(fmaf((to_f32(src[c]) - mean) * rstd, w ? to_f32(w[c]) : 1.f, b ? to_f32(b[c]) : 0.f));
    }
}

// Adds dy and dy xhat of each thread's columns over the rows of its block (partial,
// when asked for: [block][2][cols]) and writes dx (when asked for). A vector row is read from its ring places twice,
// for the two sums and for dx, and its places are filled again right behind the second read.
template <typename T, typename W, bool VEC, int CPT, bool HOLD>
__device__ __forceinline__ void backward(T *__restrict__ dx, float *__restrict__ partial, const T *__restrict__ dy, const T *__restrict__ x,
                                         const W *__restrict__ w, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                                         long long rows, int cols, long long lddx, long long lddy, long long ldx, int group, int depth)
{
    constexpr int E = VEC ? 16 / (int)sizeof(T) : 1, NCH = CPT / E;
    __shared__ float2 sh[2][32];
    __shared__ float part[2][256];              // narrow rows: the block's groups add up here
    Group g(group);
    float pw[HOLD ? NCH : 1][E], aw[NCH][E], ab[NCH][E];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const float inv = 1.f / (float)cols;
    const long long step = (long long)gridDim.x * g.per_block;
    long long base = (long long)blockIdx.x * g.per_block;
    Ring<2, VEC ? NCH : 1> ring(depth);
    Chunk<T, E> sx[VEC ? 1 : NCH], sd[VEC ? 1 : NCH], nx[VEC ? 1 : NCH], nd[VEC ? 1 : NCH];
    if constexpr (VEC) {
        for (int d = 0; d < depth; d++) {
            const long long row = base + g.index + d * step;
            ring.template fetch<T, E>(0, x + row * ldx, g, cols, row < rows);
            ring.template fetch<T, E>(1, dy + row * lddy, g, cols, row < rows);
            ring.commit();
            ring.next();
        }
    } else {
        load_row<T, E, NCH>(sx, x + (base + g.index) * ldx, g, cols, base + g.index < rows);
        load_row<T, E, NCH>(sd, dy + (base + g.index) * lddy, g, cols, base + g.index < rows);
    }
    const auto weight = [&](int j, float (&q)[E]) {
        const int col = (j * g.size + g.t) * E;
#pragma unroll
        for (int e = 0; e < E; e++) q[e] = 1.f;
        if (w && col < cols) load_params<W, E>(w, col, q);
    };
#pragma unroll
    for (int j = 0; j < NCH; j++) {
#pragma unroll
        for (int e = 0; e < E; e++) { aw[j][e] = 0.f; ab[j][e] = 0.f; }
        if constexpr (HOLD) weight(j, pw[j]);
    }
    float cm = 0.f, cr = 0.f;
    if (base + g.index < rows) { cm = mean_in[base + g.index]; cr = rstd_in[base + g.index]; }
    for (; base < rows; base += step) {
        const long long row = base + g.index, next = row + step;
        float nm = 0.f, nr = 0.f;
        if (next < rows) { nm = mean_in[next]; nr = rstd_in[next]; }
        if constexpr (VEC) ring.wait();
        else {
            load_row<T, E, NCH>(nx, x + next * ldx, g, cols, next < rows);
            load_row<T, E, NCH>(nd, dy + next * lddy, g, cols, next < rows);
        }
        float s1 = 0.f, s2 = 0.f;
        // rows past the last have dy = 0 (and mean = rstd = 0): they add nothing
#pragma unroll
        for (int j = 0; j < NCH; j++) {
            if ((j * g.size + g.t) * E < cols) {
                float qw[E];
                if constexpr (!HOLD) weight(j, qw);
                Chunk<T, E> cx, cd;
                if constexpr (VEC) { cx = ring.template get<T, E>(0, j, row < rows); cd = ring.template get<T, E>(1, j, row < rows); }
                else { cx = sx[j]; cd = sd[j]; }
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const float d = to_f32(cd.v[e]), xh = (to_f32(cx.v[e]) - cm) * cr;
                    const float wd = d * (HOLD ? pw[HOLD ? j : 0][e] : qw[e]);
                    s1 += wd;
                    s2 = fmaf(wd, xh, s2);
                    ab[j][e] += d;
                    aw[j][e] = fmaf(d, xh, aw[j][e]);
                }
            }
        }
        const float2 t = g.sum2(s1, s2, sh);
        if (dx && row < rows) {
            const float p = t.x * inv, q = t.y * inv;
            T *out = dx + row * lddx;
#pragma unroll
            for (int j = 0; j < NCH; j++) {
                const int col = (j * g.size + g.t) * E;
                if (col < cols) {
                    float qw[E];
                    if constexpr (!HOLD) weight(j, qw);
                    Chunk<T, E> cx, cd, o;
                    if constexpr (VEC) { cx = ring.template get<T, E>(0, j, true); cd = ring.template get<T, E>(1, j, true); }
                    else { cx = sx[j]; cd = sd[j]; }
#pragma unroll
                    for (int e = 0; e < E; e++) {
                        const float xh = (to_f32(cx.v[e]) - cm) * cr;
                        const float wd = to_f32(cd.v[e]) * (HOLD ? pw[HOLD ? j : 0][e] : qw[e]);
                        o.v[e] = from_f32<T>(cr * (wd - p - xh * q));
                    }
                    *reinterpret_cast<Chunk<T, E> *>(out + col) = o;
                }
            }
        }
        cm = nm; cr = nr;
        if constexpr (VEC) {
            const long long ahead = row + depth * step;
            ring.template fetch<T, E>(0, x + ahead * ldx, g, cols, ahead < rows);
            ring.template fetch<T, E>(1, dy + ahead * lddy, g, cols, ahead < rows);
            ring.commit();
            ring.next();
        } else {
#pragma unroll
            for (int j = 0; j < NCH; j++) { sx[j] = nx[j]; sd[j] = nd[j]; }
        }
    }
    if (!partial) return;
    float *pw_out = partial + (size_t)blockIdx.x * 2 * cols, *pb_out = pw_out + cols;
    if (g.size > 32) {
#pragma unroll
        for (int j = 0; j < NCH; j++)
#pragma unroll
            for (int e = 0; e < E; e++) {
                const int col = (j * g.size + g.t) * E + e;
                if (col < cols) { pw_out[col] = aw[j][e]; pb_out[col] = ab[j][e]; }
            }
        return;
    }
    // narrow rows (cols <= 256): first over the groups of a warp, then over the warps in turn
    for (int o = 16; o >= g.size; o >>= 1)
#pragma unroll
        for (int j = 0; j < NCH; j++)
#pragma unroll
            for (int e = 0; e < E; e++) {
                aw[j][e] += __shfl_xor_sync(0xffffffffu, aw[j][e], o);
                ab[j][e] += __shfl_xor_sync(0xffffffffu, ab[j][e], o);
            }
    const int warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31;
    for (int k = 0; k < ((int)blockDim.x >> 5); k++) {
        if (warp == k && lane < g.size) {
#pragma unroll
            for (int j = 0; j < NCH; j++)
#pragma unroll
                for (int e = 0; e < E; e++) {
                    const int col = (j * g.size + g.t) * E + e;
                    if (col < cols && col < 256) {
                        part[0][col] = k ? part[0][col] + aw[j][e] : aw[j][e];
                        part[1][col] = k ? part[1][col] + ab[j][e] : ab[j][e];
                    }
                }
        }
        __syncthreads();
    }
    for (int c = (int)threadIdx.x; c < cols && c < 256; c += (int)blockDim.x) { pw_out[c] = part[0][c]; pb_out[c] = part[1][c]; }
}

template <typename T, typename W>
__device__ __forceinline__ void backward_loop(T *__restrict__ dx, const T *__restrict__ dy, const T *__restrict__ x, const W *__restrict__ w,
                                              const float *__restrict__ mean_in, const float *__restrict__ rstd_in, long long rows, int cols,
                                              long long lddx, long long lddy, long long ldx)
{
    __shared__ float2 sh[2][32];
    Group g((int)blockDim.x);
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const float inv = 1.f / (float)cols;
    for (long long row = blockIdx.x; row < rows; row += gridDim.x) {
        const T *sx = x + row * ldx, *sd = dy + row * lddy;
        T *out = dx + row * lddx;
        const float m = mean_in[row], r = rstd_in[row];
        float s1 = 0.f, s2 = 0.f;
        for (int c = g.t; c < cols; c += g.size) {
            const float wd = to_f32(sd[c]) * (w ? to_f32(w[c]) : 1.f);
            s1 += wd;
            s2 = fmaf(wd, (to_f32(sx[c]) - m) * r, s2);
        }
        const float2 t = g.sum2(s1, s2, sh);
        const float p = t.x * inv, q = t.y * inv;
        for (int c = g.t; c < cols; c += g.size) {
            const float wd = to_f32(sd[c]) * (w ? to_f32(w[c]) : 1.f);
            out[c] = from_f32<T>(r * (wd - p - (to_f32(sx[c]) - m) * r * q));
        }
    }
}

// The column sums of the loop form: block (i, j) adds columns 256 i.. over rows j, j + gridDim.y, ...
template <typename T>
__device__ __forceinline__ void backward_columns(float *__restrict__ partial, const T *__restrict__ dy, const T *__restrict__ x,
                                                 const float *__restrict__ mean_in, const float *__restrict__ rstd_in, long long rows, int cols,
                                                 long long lddy, long long ldx)
{
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int c = (int)(blockIdx.x * 256 + threadIdx.x);
    if (c >= cols) return;
    float aw = 0.f, ab = 0.f;
    for (long long row = blockIdx.y; row < rows; row += gridDim.y) {
        const float d = to_f32(dy[row * lddy + c]);
        ab += d;
        aw = fmaf(d, (to_f32(x[row * ldx + c]) - mean_in[row]) * rstd_in[row], aw);
    }
    float *out = partial + (size_t)blockIdx.y * 2 * cols;
    out[c] = aw;
    out[cols + c] = ab;
}

// dw and db: column sums of the `parts` partial rows, 32 columns a block, 32
// threads on each column, in double and in a fixed order. blockIdx.y 0: dw, 1: db.
template <typename W>
__device__ __forceinline__ void param_grad(W *__restrict__ dw, W *__restrict__ db, const float *__restrict__ partial, int parts, int cols)
{
    __shared__ double sh[32][33];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    W *out = blockIdx.y ? db : dw;
    if (!out) return;
    const int lane = (int)threadIdx.x & 31, ty = (int)threadIdx.x >> 5, c = (int)blockIdx.x * 32 + lane;
    double s = 0.0;
    if (c < cols) {
        const float *p = partial + (size_t)blockIdx.y * cols + c;
#pragma unroll 8
        for (int i = ty; i < parts; i += 32) s += (double)__ldcg(p + (size_t)i * 2 * cols);
    }
    sh[ty][lane] = s;
    __syncthreads();
    // warp ty adds column ty of the block
    s = sh[lane][ty];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
    const int mine = (int)blockIdx.x * 32 + ty;
    if (lane == 0 && mine < cols) out[mine] = from_f32<W>((float)s);
}

}  // namespace ln

#define LN_FORM(name, T, W, form, VEC, CPT, HOLD, THREADS)                                                                                \
    extern "C" __global__ void __launch_bounds__(THREADS)                                                                                \
    layernorm_##name##_##form(T *y, const T *x, const W *w, const W *b, float *mean, float *rstd, long long rows, int cols,              \
                              long long ldx, long long ldy, float eps, int group, int depth)                                             \
    { ln::forward<T, W, VEC, CPT, HOLD>(y, x, w, b, mean, rstd, rows, cols, ldx, ldy, eps, group, depth); }                              \
    extern "C" __global__ void __launch_bounds__(THREADS)                                                                                \
    layernorm_bwd_##name##_##form(T *dx, float *partial, const T *dy, const T *x, const W *w, const float *mean, const float *rstd,      \
                                  long long rows, int cols, long long lddx, long long lddy, long long ldx, int group, int depth)         \
    { ln::backward<T, W, VEC, CPT, HOLD>(dx, partial, dy, x, w, mean, rstd, rows, cols, lddx, lddy, ldx, group, depth); }

#define LN_KERNELS(name, T, W)                                                                                                           \
    LN_FORM(name, T, W, v8, true, 8, true, 512)                                                                                          \
    LN_FORM(name, T, W, v16, true, 16, true, 512)                                                                                        \
    LN_FORM(name, T, W, vw, true, 16, false, 1024)                                                                                       \
    LN_FORM(name, T, W, s8, false, 8, true, 512)                                                                                         \
    LN_FORM(name, T, W, s16, false, 16, true, 512)                                                                                       \
    extern "C" __global__ void __launch_bounds__(512)                                                                                    \
    layernorm_##name##_loop(T *y, const T *x, const W *w, const W *b, float *mean, float *rstd, long long rows, int cols,                \
                            long long ldx, long long ldy, float eps, int group, int depth)                                               \
    { (void)group; (void)depth; ln::forward_loop<T, W>(y, x, w, b, mean, rstd, rows, cols, ldx, ldy, eps); }                             \
    extern "C" __global__ void __launch_bounds__(512)                                                                                    \
    layernorm_bwd_##name##_loop(T *dx, float *partial, const T *dy, const T *x, const W *w, const float *mean, const float *rstd,        \
                                long long rows, int cols, long long lddx, long long lddy, long long ldx, int group, int depth)           \
    { (void)group; (void)partial; (void)depth; ln::backward_loop<T, W>(dx, dy, x, w, mean, rstd, rows, cols, lddx, lddy, ldx); }

LN_KERNELS(f32, float, float)
LN_KERNELS(bf16, __nv_bfloat16, __nv_bfloat16)
LN_KERNELS(bf16_f32, __nv_bfloat16, float)
LN_KERNELS(f16, __half, __half)
LN_KERNELS(f16_f32, __half, float)

#define LN_COLUMNS(name, T)                                                                                                              \
    extern "C" __global__ void __launch_bounds__(256)                                                                                    \
    layernorm_bwd_columns_##name(float *partial, const T *dy, const T *x, const float *mean, const float *rstd, long long rows,          \
                                 int cols, long long lddy, long long ldx)                                                                \
    { ln::backward_columns<T>(partial, dy, x, mean, rstd, rows, cols, lddy, ldx); }                                                      \
    extern "C" __global__ void __launch_bounds__(1024)                                                                                    \
    layernorm_param_grad_##name(T *dw, T *db, const float *partial, int parts, int cols)                                                 \
    { ln::param_grad<T>(dw, db, partial, parts, cols); }
LN_COLUMNS(f32, float)
LN_COLUMNS(bf16, __nv_bfloat16)
LN_COLUMNS(f16, __half)
