// layernorm.cu -- layer normalisation of the rows of a matrix, and its gradient.
//
// Forward, per row of `cols` values:
//     mean = sum x / cols,  var = sum (x - mean)^2 / cols,  rstd = 1 / sqrt(var + eps)
//     y = (x - mean) rstd w + b
// Backward, with xhat = (x - mean) rstd, p = mean(w dy), q = mean(w dy xhat):
//     dx = rstd (w dy - p - xhat q);   dw = sum over rows of dy xhat;   db = sum over rows of dy
//
// Both read every value once and write every result once, so HBM bounds them: 16384 x 4096 bf16 takes 51 us forward
// and 80 us backward, 81 and 77 % of what the copy rate allows; calls back to back overlap at their ends and take 47 and 74, 87
// and 83 % (8192 x 4096 f32: 49 and 71; 65536 x 1024 bf16: 51
// and 71; unaligned 32768 x 1001 bf16: 46 and 80, 43 and 38 %, bound by instructions). A row belongs to one
// group of threads: 1 to 32 lanes of a warp for narrow rows, a whole block for wider ones, 8 to 32 values a thread: a
// row costs a thread some 150 instructions beside its values, which with 8 values were most of them. The mean
// is taken first and the variance from the differences (the row is on chip, a second pass costs no memory), with
// the differences' own mean as a correction, so a row far from zero loses nothing.
//
// Blocks stay and walk over the rows. The next few rows are on their way with cp.async
// into a ring in shared memory. In vector forms every thread has places of its
// own for what it alone reads, so the ring needs no barrier. (With the next row held in
// registers instead, 16 KB an SM were in flight and 16384 x 4096 bf16 took 116 us forward
// and 128 backward.) Rows of any other alignment come in 16-byte units all the same and are read
// value by value. A spill in the walk is dear, with the SM's memory given to the ring no cache is left
// for it: the forms are cut, and distances between a thread's values kept opaque, so that there is none forward and 16 bytes at
// most backward (sx, loop and the vx of f32).
//
// The backward pass walks the rows once for all three results: each thread adds dy
// and dy xhat of its own columns into registers over all the rows its block sees,
// the block writes one partial row, and layernorm_param_grad adds the partial
// rows in index order. No atomics: results repeat bit for bit.
//
// Sums, statistics and products are fp32 (the last sum over the blocks double);
// values are rounded to the tensor's type once, when they are stored.
//
// Forms: v8, v16, v32, vw, vx read 16-byte vectors (row starts and parameters 16-byte
// aligned, cols a multiple of the vector), with 8, 16 or 32 values a thread; vw (16 values, 20 of f32 backward) and
// vx (32) are for rows too wide for these and keep the parameters in shared memory, vx also reads the row a second
// time from the ring instead of keeping it. s8, s16, sx read single elements, neighbouring threads on neighbouring
// columns, for any alignment. loop goes through the row several times from
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

// Two fp32 values in a register pair: the packed forms do two operations an instruction, each rounded as by itself.
struct Pair { uint64_t v; };
__device__ __forceinline__ Pair pair(float a, float b)
{
    Pair p;
    asm("mov.b64 %0, {%1, %2};" : "=l"(p.v) : "f"(a), "f"(b));
    return p;
}
__device__ __forceinline__ float2 split(Pair p)
{
    float2 f;
    asm("mov.b64 {%0, %1}, %2;" : "=f"(f.x), "=f"(f.y) : "l"(p.v));
    return f;
}
__device__ __forceinline__ Pair add(Pair a, Pair b) { Pair r; asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ Pair mul(Pair a, Pair b) { Pair r; asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r.v) : "l"(a.v), "l"(b.v)); return r; }
__device__ __forceinline__ Pair fma(Pair a, Pair b, Pair c) { Pair r; asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r.v) : "l"(a.v), "l"(b.v), "l"(c.v)); return r; }
// Two neighbouring values of a chunk, to and from their type.
__device__ __forceinline__ Pair widen(const float *v) { return pair(v[0], v[1]); }
__device__ __forceinline__ Pair widen(const __nv_bfloat16 *v)
{
    const uint32_t w = *reinterpret_cast<const uint32_t *>(v);
    return pair(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
}
__device__ __forceinline__ Pair widen(const __half *v)
{
    const float2 f = __half22float2(*reinterpret_cast<const __half2 *>(v));
    return pair(f.x, f.y);
}
__device__ __forceinline__ void narrow(float *v, Pair p) { const float2 f = split(p); v[0] = f.x; v[1] = f.y; }
__device__ __forceinline__ void narrow(__nv_bfloat16 *v, Pair p) { const float2 f = split(p); *reinterpret_cast<__nv_bfloat162 *>(v) = __floats2bfloat162_rn(f.x, f.y); }
__device__ __forceinline__ void narrow(__half *v, Pair p) { const float2 f = split(p); *reinterpret_cast<__half2 *>(v) = __floats2half2_rn(f.x, f.y); }

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
    // Sums over the group, the same bits in every thread. Called by all threads of the block in step. `sh` holds
    // 2 x 32 values; the halves alternate, so one barrier a call is enough.
    __device__ __forceinline__ float2 sum2(float a, float b, float2 (*sh)[32])
    {
        if (size < 32) {
            for (int o = size >> 1; o > 0; o >>= 1) {
                a += __shfl_xor_sync(0xffffffffu, a, o);
                b += __shfl_xor_sync(0xffffffffu, b, o);
            }
            return make_float2(a, b);
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            a += __shfl_xor_sync(0xffffffffu, a, o);
            b += __shfl_xor_sync(0xffffffffu, b, o);
        }
        if (size > 32) {
            float2 *s = sh[turn & 1];
            turn++;
            if ((t & 31) == 0) s[t >> 5] = make_float2(a, b);
            __syncthreads();
            const int warps = size >> 5;
            if (warps <= 8) {           // a few broadcast reads are shorter than a second tree
                a = b = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < warps) { const float2 v = s[i]; a += v.x; b += v.y; }
            } else {
                const float2 v = (t & 31) < warps ? s[t & 31] : make_float2(0.f, 0.f);
                a = v.x; b = v.y;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) {
                    a += __shfl_xor_sync(0xffffffffu, a, o);
                    b += __shfl_xor_sync(0xffffffffu, b, o);
                }
            }
        }
        return make_float2(a, b);
    }
    __device__ __forceinline__ float sum(float a, float2 (*sh)[32])
    {
        if (size < 32) {
            for (int o = size >> 1; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
            return a;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
        if (size > 32) {
            float *s = reinterpret_cast<float *>(sh[turn & 1]);
            turn++;
            if ((t & 31) == 0) s[t >> 5] = a;
            __syncthreads();
            const int warps = size >> 5;
            if (warps <= 8) {
                a = 0.f;
#pragma unroll
                for (int i = 0; i < 8; i++)
                    if (i < warps) a += s[i];
            } else {
                a = (t & 31) < warps ? s[t & 31] : 0.f;
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) a += __shfl_xor_sync(0xffffffffu, a, o);
            }
        }
        return a;
    }
};

// The values of NCH chunks of E as pairs; a lone value a chunk (E = 1) pairs with the next chunk's.
template <typename T, int E, int NCH> __device__ __forceinline__ void widen_all(const Chunk<T, E> (&c)[NCH], Pair (&v)[NCH * E / 2])
{
    if constexpr (E == 1) {
#pragma unroll
        for (int i = 0; i < NCH / 2; i++) v[i] = pair(to_f32(c[2 * i].v[0]), to_f32(c[2 * i + 1].v[0]));
    } else {
#pragma unroll
        for (int j = 0; j < NCH; j++)
#pragma unroll
            for (int i = 0; i < E / 2; i++) v[j * E / 2 + i] = widen(&c[j].v[2 * i]);
    }
}

// A distance in bytes. OPAQUE: its multiples are added up where they are used and not held in registers from row to
// row, which many values a thread leave no room for (up to 440 bytes of spills).
template <bool OPAQUE> __device__ __forceinline__ uint32_t stride(uint32_t by)
{
    if constexpr (OPAQUE) asm volatile("mov.u32 %0, %0;" : "+r"(by));
    return by;
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
    // Where this thread's first chunk of array a lies; its others follow `step()` bytes apart.
    __device__ __forceinline__ uint32_t first(int a) const { return base + (uint32_t)((stage * A + a) * NCH) * row_bytes; }
    __device__ __forceinline__ uint32_t step() const { return stride<(NCH > 4)>(row_bytes); }
    // `valid`: this thread's chunks in the row
    template <typename T, int E> __device__ __forceinline__ void fetch(int a, const T *row, const Group &g, int valid, bool live) const
    {
        uint32_t to = first(a);
        const uint32_t by = step(), far = stride<(NCH > 4)>((uint32_t)g.size * 16u);
        const char *from = reinterpret_cast<const char *>(row + g.t * E);
#pragma unroll
        for (int j = 0; j < NCH; j++) {
            if (live && j < valid) asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to), "l"(from) : "memory");
            to += by;
            from += far;
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
    // The chunk at `at`, zero unless `live`.
    template <typename T, int E> static __device__ __forceinline__ Chunk<T, E> get(uint32_t at, bool live)
    {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (live) asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(at) : "memory");
        return *reinterpret_cast<const Chunk<T, E> *>(&v);
    }
};

// The ring for rows of any alignment: a row has a slot in which its bytes lie as they do in memory modulo 16. Whole
// 16-byte units come with cp.async; of the values at its two ends each thread brings at most one of either (a group has
// eight threads at least), 16-bit ones through a register, written to the slot at the next step. What one thread
// brings others read, so a row is ready behind a barrier of its group, and its slot is free behind the next one. A slot
// is as long as all values of a group's threads, zero behind the row, so that reading takes no comparisons.
template <typename T, int A> struct Slots {
    uint32_t base, pitch, groups, held[A][2], low[A], by_row[A];
    uint16_t edge[A][2];
    int depth, stage;
    template <bool USED> __device__ __forceinline__ void init(int depth_, int cpt, const Group &g)
    {
        extern __shared__ uint4 ln_ring[];
        depth = depth_;
        stage = 0;
        pitch = ((uint32_t)(cpt * g.size) * (uint32_t)sizeof(T) + 15u) / 16u * 16u + 16u;
        groups = (uint32_t)g.per_block;
        base = (uint32_t)__cvta_generic_to_shared(ln_ring) + (uint32_t)g.index * pitch;
        if constexpr (USED) {
            for (uint32_t u = threadIdx.x; u < (uint32_t)(depth * A) * groups * pitch / 16u; u += blockDim.x) ln_ring[u] = make_uint4(0, 0, 0, 0);
            __syncthreads();
        }
#pragma unroll
        for (int a = 0; a < A; a++) { held[a][0] = held[a][1] = 0; edge[a][0] = edge[a][1] = 0; }
    }
    // Array a: its first row and the distance of its rows, modulo 2^32 bytes.
    __device__ __forceinline__ void source(int a, const T *p, long long ld)
    {
        low[a] = (uint32_t)reinterpret_cast<uintptr_t>(p);
        by_row[a] = (uint32_t)ld * (uint32_t)sizeof(T);
    }
    __device__ __forceinline__ uint32_t slot(int a) const { return base + (uint32_t)(stage * A + a) * groups * pitch; }
    __device__ __forceinline__ void fetch(int a, const T *row, const Group &g, int cols, bool live)
    {
        if (!live) return;
        const uint32_t head = (uint32_t)reinterpret_cast<uintptr_t>(row) & 15u, bytes = (uint32_t)cols * (uint32_t)sizeof(T), to = slot(a) + head;
        const uint32_t gap = (16u - head) & 15u, lead = gap < bytes ? gap : bytes, units = (bytes - lead) / 16u, tail = (bytes - lead) & 15u;
        const uint32_t at = (uint32_t)g.t * (uint32_t)sizeof(T);
        const char *const from = reinterpret_cast<const char *>(row);
        if (at < 16u) {
            // an earlier row may have ended up to 15 bytes further on
            if (head + bytes + at < pitch) {
                if constexpr (sizeof(T) == 2) asm volatile("st.shared.u16 [%0], %1;" ::"r"(to + bytes + at), "h"((uint16_t)0) : "memory");
                else asm volatile("st.shared.u32 [%0], %1;" ::"r"(to + bytes + at), "r"(0) : "memory");
            }
#pragma unroll
            for (int e = 0; e < 2; e++) {
                const uint32_t o = e ? bytes - tail + at : at;
                if (at < (e ? tail : lead)) {
                    if constexpr (sizeof(T) == 2) {
                        held[a][e] = to + o;
                        edge[a][e] = *reinterpret_cast<const uint16_t *>(from + o);
                    } else {
                        asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" ::"r"(to + o), "l"(from + o) : "memory");
                    }
                }
            }
        }
        const char *src = from + lead + (uint32_t)g.t * 16u;
        uint32_t dst = to + lead + (uint32_t)g.t * 16u;
        for (uint32_t u = (uint32_t)g.t; u < units; u += (uint32_t)g.size) {
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
            src += (uint32_t)g.size * 16u;
            dst += (uint32_t)g.size * 16u;
        }
    }
    __device__ __forceinline__ void commit() const { asm volatile("cp.async.commit_group;" ::: "memory"); }
    __device__ __forceinline__ void next() { stage = stage + 1 == depth ? 0 : stage + 1; }
    __device__ __forceinline__ void settle()
    {
        if constexpr (sizeof(T) == 2)
#pragma unroll
        for (int a = 0; a < A; a++)
#pragma unroll
            for (int e = 0; e < 2; e++)
                if (held[a][e]) {
                    asm volatile("st.shared.u16 [%0], %1;" ::"r"(held[a][e]), "h"(edge[a][e]) : "memory");
                    held[a][e] = 0;
                }
    }
    static __device__ __forceinline__ void meet(const Group &g) { if (g.size > 32) __syncthreads(); else __syncwarp(); }
    // The oldest outstanding row is there for the whole group.
    __device__ __forceinline__ void wait(const Group &g)
    {
        settle();
        if (depth == 4) asm volatile("cp.async.wait_group 3;" ::: "memory");
        else if (depth == 3) asm volatile("cp.async.wait_group 2;" ::: "memory");
        else if (depth == 2) asm volatile("cp.async.wait_group 1;" ::: "memory");
        else asm volatile("cp.async.wait_group 0;" ::: "memory");
        meet(g);
    }
    // Where this thread's first value of row `row` lies; its others follow `step()` bytes apart.
    __device__ __forceinline__ uint32_t first(int a, long long row, const Group &g) const
    {
        return slot(a) + ((low[a] + (uint32_t)row * by_row[a]) & 15u) + (uint32_t)g.t * (uint32_t)sizeof(T);
    }
    template <bool OPAQUE> static __device__ __forceinline__ uint32_t step(const Group &g) { return stride<OPAQUE>((uint32_t)g.size * (uint32_t)sizeof(T)); }
    static __device__ __forceinline__ void put(char *&to, uint32_t by, float2 v, int left)
    {
        if (left > 0) *reinterpret_cast<T *>(to) = from_f32<T>(v.x);
        if (left > 1) *reinterpret_cast<T *>(to + by) = from_f32<T>(v.y);
        to += 2u * by;
    }
    static __device__ __forceinline__ float value(uint32_t at)
    {
        if constexpr (sizeof(T) == 4) {
            float v;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(at) : "memory");
            return v;
        } else {
            uint16_t v;
            asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(at) : "memory");
            return to_f32(*reinterpret_cast<const T *>(&v));
        }
    }
    static __device__ __forceinline__ Pair values(uint32_t &at, uint32_t by)
    {
        const float a = value(at), b = value(at + by);
        at += 2u * by;
        return pair(a, b);
    }
    template <int N> __device__ __forceinline__ void get_all(int a, long long row, const Group &g, Pair (&v)[N]) const
    {
        uint32_t at = first(a, row, g);
        const uint32_t by = step<(N > 8)>(g);
#pragma unroll
        for (int i = 0; i < N; i++) v[i] = values(at, by);
    }
};

// Parameters of wide rows, in fp32 in shared memory behind the ring: each thread has those of its own columns in places
// of its own, as with the ring. Array n of a chunk j; 16 bytes a thread (E = 1: 4).
struct Kept {
    uint32_t base, step;
    __device__ __forceinline__ Kept(uint32_t ring_bytes)
    {
        extern __shared__ uint4 ln_ring[];
        base = (uint32_t)__cvta_generic_to_shared(ln_ring) + ring_bytes;
        step = blockDim.x;
    }
    template <int E, int NCH> __device__ __forceinline__ uint32_t at(int n, int j, int k) const
    {
        return E == 1 ? base + ((uint32_t)(n * NCH + j) * step + threadIdx.x) * 4u : base + ((uint32_t)((n * NCH + j) * (E / 4 < 1 ? 1 : E / 4) + k) * step + threadIdx.x) * 16u;
    }
    template <int E, int NCH> __device__ __forceinline__ void put(int n, int j, const float (&q)[E]) const
    {
        if constexpr (E == 1) asm volatile("st.shared.f32 [%0], %1;" ::"r"(at<E, NCH>(n, j, 0)), "f"(q[0]) : "memory");
        else {
#pragma unroll
            for (int k = 0; k < E / 4; k++)
                asm volatile("st.shared.v4.f32 [%0], {%1, %2, %3, %4};" ::"r"(at<E, NCH>(n, j, k)), "f"(q[4 * k]), "f"(q[4 * k + 1]), "f"(q[4 * k + 2]), "f"(q[4 * k + 3]) : "memory");
        }
    }
    template <int E, int NCH> __device__ __forceinline__ void get(int n, int j, float (&q)[E]) const
    {
        if constexpr (E == 1) asm volatile("ld.shared.f32 %0, [%1];" : "=f"(q[0]) : "r"(at<E, NCH>(n, j, 0)) : "memory");
        else {
#pragma unroll
            for (int k = 0; k < E / 4; k++)
                asm volatile("ld.shared.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(q[4 * k]), "=f"(q[4 * k + 1]), "=f"(q[4 * k + 2]), "=f"(q[4 * k + 3]) : "r"(at<E, NCH>(n, j, k)) : "memory");
        }
    }
};

// How many of a thread's chunks of E values lie in the row (whole or not at all: cols is a multiple of E).
template <int E> __device__ __forceinline__ int valid_of(const Group &g, int cols)
{
    return g.t * E < cols ? (cols / E - g.t + g.size - 1) / g.size : 0;
}

// The mean that a caller gets, from the sum's m and the mean dm of the rounded differences x - m. Values of one binade all lose the
// same low bits of m in that subtraction, so dm is good to half a step of the values and no better: it corrects m where
// the row lies far from zero beside its spread (there x - m is exact, or rounded by less than a step of m), and spoils
// it where m is small (bf16 rows of 1024 with means below 1e-2: 1.1e-4 of the mean against 3.5e-7 for m alone). An
// infinity leaves no dm, and m is the mean. (y takes the same rounded differences and is right with dm either way.)
__device__ __forceinline__ float mean_of(float m, float dm, float var) { return m * m > var && fabsf(dm) < INFINITY ? m + dm : m; }

// Rounding may leave a variance below zero; a NaN (of a row that holds one, or whose sums overflow) stays one.
__device__ __forceinline__ float rstd_of(float var, float eps) { return __frsqrt_rn((var > 0.f ? var : var == var ? 0.f : var) + eps); }

// v: a row's values in, their differences from `m` out (zero outside the row). Their mean is `dm`; `mean` as above.
template <int E, int N>
__device__ __forceinline__ void row_stats(Pair (&v)[N], Group &g, int valid, float inv, float eps, float2 (*sh)[32], float &mean, float &dm, float &rstd)
{
    Pair s = pair(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; i++) s = add(s, v[i]);                // columns past the end hold zero
    float2 f = split(s);
    const float m = g.sum(f.x + f.y, sh) * inv;
    const Pair nm = pair(-m, -m);
    Pair d1 = pair(0.f, 0.f), d2 = pair(0.f, 0.f);
#pragma unroll
    for (int i = 0; i < N; i++) {
        v[i] = add(v[i], nm);
        if constexpr (E == 1) {
            const float2 x = split(v[i]);
            v[i] = pair(2 * i < valid ? x.x : 0.f, 2 * i + 1 < valid ? x.y : 0.f);
        } else {
            if (2 * i / (E < 2 ? 2 : E) >= valid) v[i] = pair(0.f, 0.f);
        }
        d1 = add(d1, v[i]);
        d2 = fma(v[i], v[i], d2);
    }
    const float2 a = split(d1), b = split(d2);
    const float2 t = g.sum2(a.x + a.y, b.x + b.y, sh);
    dm = t.x * inv;
    const float var = t.y * inv - dm * dm;
    mean = mean_of(m, dm, var);
    rstd = rstd_of(var, eps);
}

template <typename T, typename W, bool VEC, int CPT, bool HOLD>
__device__ __forceinline__ void forward(T *__restrict__ y, const T *__restrict__ x, const W *__restrict__ w, const W *__restrict__ b,
                                        float *__restrict__ mean_out, float *__restrict__ rstd_out, long long rows, int cols,
                                        long long ldx, long long ldy, float eps, int group, int depth)
{
    constexpr int E = VEC ? 16 / (int)sizeof(T) : 1, NCH = CPT / E;
    __shared__ float2 sh[2][32];
    Group g(group);
    Pair pw[HOLD ? CPT / 2 : 1], pb[HOLD ? CPT / 2 : 1];           // the parameters of this thread's columns
    const float inv = 1.f / (float)cols;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const long long step = (long long)gridDim.x * g.per_block;
    long long base = (long long)blockIdx.x * g.per_block;
    Ring<1, VEC ? NCH : 1> ring(depth);
    Slots<T, 1> slots;
    slots.template init<!VEC>(depth, CPT, g);
    slots.source(0, x, ldx);
    const int valid = valid_of<E>(g, cols);
    for (int d = 0; d < depth; d++) {
        const long long row = base + g.index + d * step;
        if constexpr (VEC) {
            ring.template fetch<T, E>(0, x + row * ldx, g, valid, row < rows);
            ring.commit();
            ring.next();
        } else {
            slots.settle();
            slots.fetch(0, x + row * ldx, g, cols, row < rows);
            slots.commit();
            slots.next();
        }
    }
    // parameters of chunk j's columns
    const auto params = [&](int j, float (&qw)[E], float (&qb)[E]) {
        const int col = (j * g.size + g.t) * E;
#pragma unroll
        for (int e = 0; e < E; e++) { qw[e] = 1.f; qb[e] = 0.f; }
        if (col < cols) {
            if (w) load_params<W, E>(w, col, qw);
            if (b) load_params<W, E>(b, col, qb);
        }
    };
    const Kept kept(VEC ? (uint32_t)(depth * NCH) * blockDim.x * 16u : (uint32_t)depth * slots.groups * slots.pitch);
    if constexpr (!HOLD) {
#pragma unroll
        for (int j = 0; j < NCH; j++) {
            float qw[E], qb[E];
            params(j, qw, qb);
            kept.template put<E, NCH>(0, j, qw);
            kept.template put<E, NCH>(1, j, qb);
        }
    }
    if constexpr (HOLD) {
        float qw[NCH][E], qb[NCH][E];
#pragma unroll
        for (int j = 0; j < NCH; j++) params(j, qw[j], qb[j]);
#pragma unroll
        for (int i = 0; i < CPT / 2; i++) {
            pw[i] = pair(qw[2 * i / E][2 * i % E], qw[(2 * i + 1) / E][(2 * i + 1) % E]);
            pb[i] = pair(qb[2 * i / E][2 * i % E], qb[(2 * i + 1) / E][(2 * i + 1) % E]);
        }
    }
    for (; base < rows; base += step) {
        const long long row = base + g.index;
        Pair v[CPT / 2];
        if constexpr (VEC) {
            ring.wait();
            Chunk<T, E> cur[NCH];
            uint32_t at = ring.first(0);
            const uint32_t by = ring.step();
#pragma unroll
            for (int j = 0; j < NCH; j++) {
                cur[j] = ring.template get<T, E>(at, row < rows && j < valid);
                at += by;
            }
            widen_all<T, E, NCH>(cur, v);
        } else {
            slots.wait(g);
            slots.get_all(0, row, g, v);
        }
        float mean, dm, rstd;
        row_stats<E, CPT / 2>(v, g, valid, inv, eps, sh, mean, dm, rstd);
        const long long ahead = row + depth * step;          // the row is in registers: its places may fill again
        if constexpr (VEC) {
            ring.template fetch<T, E>(0, x + ahead * ldx, g, valid, ahead < rows);
            ring.commit();
            ring.next();
        } else {
            if (g.size <= 32) __syncwarp();
            slots.fetch(0, x + ahead * ldx, g, cols, ahead < rows);
            slots.commit();
            slots.next();
        }
        if (row < rows) {
            if (g.t == 0) {
                if (mean_out) mean_out[row] = mean;
                if (rstd_out) rstd_out[row] = rstd;
            }
            T *out = y + row * ldy;
            const Pair r2 = pair(rstd, rstd), shift = pair(-dm * rstd, -dm * rstd);
#pragma unroll
            for (int i = 0; i < CPT / 2; i++) v[i] = fma(v[i], r2, shift);
            if constexpr (E == 1) {
                char *to = reinterpret_cast<char *>(out + g.t);
                const uint32_t by = slots.template step<!HOLD>(g);
#pragma unroll
                for (int i = 0; i < CPT / 2; i++) {
                    if constexpr (!HOLD) {
                        float qw[2][E], qb[2][E];
#pragma unroll
                        for (int h = 0; h < 2; h++) {
                            kept.template get<E, NCH>(0, 2 * i + h, qw[h]);
                            kept.template get<E, NCH>(1, 2 * i + h, qb[h]);
                        }
                        v[i] = fma(v[i], pair(qw[0][0], qw[1][0]), pair(qb[0][0], qb[1][0]));
                    } else {
                        v[i] = fma(v[i], pw[i], pb[i]);
                    }
                    const float2 f = split(v[i]);
                    slots.put(to, by, f, valid - 2 * i);
                }
            } else {
                char *to = reinterpret_cast<char *>(out + g.t * E);
                const uint32_t far = stride<(NCH > 4)>((uint32_t)g.size * 16u);
#pragma unroll
                for (int j = 0; j < NCH; j++) {
                    if (j < valid) {
                        Chunk<T, E> o;
                        float qw[E], qb[E];
                        if constexpr (!HOLD) { kept.template get<E, NCH>(0, j, qw); kept.template get<E, NCH>(1, j, qb); }
#pragma unroll
                        for (int i = 0; i < E / 2; i++) {
                            const int n = j * E / 2 + i;
                            if constexpr (HOLD) narrow(&o.v[2 * i], fma(v[n], pw[n], pb[n]));
                            else narrow(&o.v[2 * i], fma(v[n], pair(qw[2 * i], qw[2 * i + 1]), pair(qb[2 * i], qb[2 * i + 1])));
                        }
                        *reinterpret_cast<Chunk<T, E> *>(to) = o;
                    }
                    to += far;
                }
            }
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
        const float m = g.sum(s, sh) / (float)cols;
        float d1 = 0.f, d2 = 0.f;
        for (int c = g.t; c < cols; c += g.size) { const float d = to_f32(src[c]) - m; d1 += d; d2 = fmaf(d, d, d2); }
        const float2 t = g.sum2(d1, d2, sh);
        const float dm = t.x / (float)cols, mean = m + dm, var = t.y / (float)cols - dm * dm;
        const float rstd = rstd_of(var, eps);
        if (g.t == 0) {
            if (mean_out) mean_out[row] = mean_of(m, dm, var);
            if (rstd_out) rstd_out[row] = rstd;
        }
        for (int c = g.t; c < cols; c += g.size)
            out[c] = from_f32<T>(fmaf((to_f32(src[c]) - mean) * rstd, w ? to_f32(w[c]) : 1.f, b ? to_f32(b[c]) : 0.f));
    }
}

// Adds dy and dy xhat of each thread's columns over the rows of its block (partial,
// when asked for: [block][2][cols]) and writes dx (when asked for).
template <typename T, typename W, bool VEC, int CPT, bool HOLD, bool KEEP_ROW>
__device__ __forceinline__ void backward(T *__restrict__ dx, float *__restrict__ partial, const T *__restrict__ dy, const T *__restrict__ x,
                                         const W *__restrict__ w, const float *__restrict__ mean_in, const float *__restrict__ rstd_in,
                                         long long rows, int cols, long long lddx, long long lddy, long long ldx, int group, int depth)
{
    constexpr int E = VEC ? 16 / (int)sizeof(T) : 1, NCH = CPT / E, N = CPT / 2;
    __shared__ float2 sh[2][32];
    __shared__ float part[2][512];              // narrow rows: the block's groups add up here
    Group g(group);
    Pair pw[HOLD ? N : 1], aw[N], ab[N];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const float inv = 1.f / (float)cols;
    const long long step = (long long)gridDim.x * g.per_block;
    long long base = (long long)blockIdx.x * g.per_block;
    Ring<2, VEC ? NCH : 1> ring(depth);
    Slots<T, 2> slots;
    slots.template init<!VEC>(depth, CPT, g);
    slots.source(0, x, ldx);
    slots.source(1, dy, lddy);
    const int valid = valid_of<E>(g, cols);
    for (int d = 0; d < depth; d++) {
        const long long row = base + g.index + d * step;
        if constexpr (VEC) {
            ring.template fetch<T, E>(0, x + row * ldx, g, valid, row < rows);
            ring.template fetch<T, E>(1, dy + row * lddy, g, valid, row < rows);
            ring.commit();
            ring.next();
        } else {
            slots.settle();
            slots.fetch(0, x + row * ldx, g, cols, row < rows);
            slots.fetch(1, dy + row * lddy, g, cols, row < rows);
            slots.commit();
            slots.next();
        }
    }
    const auto weight = [&](int j, float (&q)[E]) {
        const int col = (j * g.size + g.t) * E;
#pragma unroll
        for (int e = 0; e < E; e++) q[e] = 1.f;
        if (w && col < cols) load_params<W, E>(w, col, q);
    };
    const Kept kept(VEC ? (uint32_t)(depth * 2 * NCH) * blockDim.x * 16u : (uint32_t)(depth * 2) * slots.groups * slots.pitch);
    if constexpr (!HOLD) {
#pragma unroll
        for (int j = 0; j < NCH; j++) {
            float q[E];
            weight(j, q);
            kept.template put<E, NCH>(0, j, q);
        }
    }
    if constexpr (HOLD) {
        float q[NCH][E];
#pragma unroll
        for (int j = 0; j < NCH; j++) weight(j, q[j]);
#pragma unroll
        for (int i = 0; i < N; i++) pw[i] = pair(q[2 * i / E][2 * i % E], q[(2 * i + 1) / E][(2 * i + 1) % E]);
    }
#pragma unroll
    for (int i = 0; i < N; i++) aw[i] = ab[i] = pair(0.f, 0.f);
    float cm = 0.f, cr = 0.f;
    if (base + g.index < rows) { cm = mean_in[base + g.index]; cr = rstd_in[base + g.index]; }
    for (; base < rows; base += step) {
        const long long row = base + g.index, next = row + step;
        float nm = 0.f, nr = 0.f;
        if (next < rows) { nm = mean_in[next]; nr = rstd_in[next]; }
        if constexpr (VEC) ring.wait();
        else slots.wait(g);
        // xhat and w dy of this thread's columns, kept for dx (KEEP_ROW) or formed again from the ring. Outside the row and
        // past the last row dy is zero: such places add nothing (and past the last row mean = rstd = 0).
        constexpr int KEEP = KEEP_ROW ? N : E == 1 ? 1 : E / 2;
        Pair xh[KEEP], wd[KEEP];
        const Pair nmean = pair(-cm, -cm), r2 = pair(cr, cr);
        Pair s1 = pair(0.f, 0.f), s2 = pair(0.f, 0.f);
        if constexpr (VEC) {
            uint32_t xa = ring.first(0), da = ring.first(1);
            const uint32_t by = ring.step();
#pragma unroll
            for (int j = 0; j < NCH; j++) {
                const bool live = row < rows && j < valid;
                const Chunk<T, E> xc = ring.template get<T, E>(xa, live), dc = ring.template get<T, E>(da, live);
                xa += by;
                da += by;
                float q[E];
                if constexpr (!HOLD) kept.template get<E, NCH>(0, j, q);
#pragma unroll
                for (int i = 0; i < E / 2; i++) {
                    const int n = j * E / 2 + i, k = KEEP_ROW ? n : i;
                    const Pair d = widen(&dc.v[2 * i]);
                    xh[k] = mul(add(widen(&xc.v[2 * i]), nmean), r2);
                    ab[n] = add(ab[n], d);
                    aw[n] = fma(d, xh[k], aw[n]);
                    if constexpr (HOLD) wd[k] = mul(d, pw[n]);
                    else wd[k] = mul(d, pair(q[2 * i], q[2 * i + 1]));
                    s1 = add(s1, wd[k]);
                    s2 = fma(wd[k], xh[k], s2);
                }
            }
        } else {
            uint32_t xa = slots.first(0, row, g), da = slots.first(1, row, g);
            const uint32_t by = slots.template step<!HOLD>(g);
            if constexpr (KEEP_ROW) {
                slots.get_all(0, row, g, xh);
                slots.get_all(1, row, g, wd);
            }
            if (row >= rows) {                  // a group past the end: its slot holds an earlier row
#pragma unroll
                for (int k = 0; k < KEEP; k++) xh[k] = wd[k] = pair(0.f, 0.f);
            }
#pragma unroll
            for (int n = 0; n < N; n++) {
                const int k = KEEP_ROW ? n : 0;
                if constexpr (!KEEP_ROW) {
                    xh[0] = slots.values(xa, by);
                    wd[0] = slots.values(da, by);
                }
                const Pair d = wd[k];
                xh[k] = mul(add(xh[k], nmean), r2);
                ab[n] = add(ab[n], d);
                aw[n] = fma(d, xh[k], aw[n]);
                if constexpr (HOLD) wd[k] = mul(d, pw[n]);
                else {
                    float q0[E], q1[E];
                    kept.template get<E, NCH>(0, 2 * n, q0);
                    kept.template get<E, NCH>(0, 2 * n + 1, q1);
                    wd[k] = mul(d, pair(q0[0], q1[0]));
                }
                s1 = add(s1, wd[k]);
                s2 = fma(wd[k], xh[k], s2);
            }
        }
        const float2 f1 = split(s1), f2 = split(s2);
        const float2 t = g.sum2(f1.x + f1.y, f2.x + f2.y, sh);
        const auto refill = [&]() {             // the row has been read: its places may fill again
            const long long ahead = row + depth * step;
            if constexpr (VEC) {
                ring.template fetch<T, E>(0, x + ahead * ldx, g, valid, ahead < rows);
                ring.template fetch<T, E>(1, dy + ahead * lddy, g, valid, ahead < rows);
                ring.commit();
                ring.next();
            } else {
                if (!KEEP_ROW) Slots<T, 2>::meet(g);          // the sums' barrier lies behind the first reading only
                else if (g.size <= 32) __syncwarp();
                slots.fetch(0, x + ahead * ldx, g, cols, ahead < rows);
                slots.fetch(1, dy + ahead * lddy, g, cols, ahead < rows);
                slots.commit();
                slots.next();
            }
        };
        if constexpr (KEEP_ROW) refill();
        if (dx && row < rows) {
            const float p = t.x * inv, q = t.y * inv;
            const Pair np = pair(-p, -p), nq = pair(-q, -q);
            T *out = dx + row * lddx;
            if constexpr (E == 1) {
                char *to = reinterpret_cast<char *>(out + g.t);
                uint32_t xa = slots.first(0, row, g), da = slots.first(1, row, g);
                const uint32_t by = slots.template step<!HOLD>(g);
#pragma unroll
                for (int i = 0; i < N; i++) {
                    const int k = KEEP_ROW ? i : 0;
                    if constexpr (!KEEP_ROW) {
                        float q0[E], q1[E];
                        kept.template get<E, NCH>(0, 2 * i, q0);
                        kept.template get<E, NCH>(0, 2 * i + 1, q1);
                        xh[0] = mul(add(slots.values(xa, by), nmean), r2);
                        wd[0] = mul(slots.values(da, by), pair(q0[0], q1[0]));
                    }
                    const float2 f = split(mul(r2, fma(xh[k], nq, add(wd[k], np))));
                    slots.put(to, by, f, valid - 2 * i);
                }
            } else {
                char *to = reinterpret_cast<char *>(out + g.t * E);
                uint32_t xa = ring.first(0), da = ring.first(1);
                const uint32_t by = ring.step(), far = stride<(NCH > 4)>((uint32_t)g.size * 16u);
#pragma unroll
                for (int j = 0; j < NCH; j++) {
                    if (j < valid) {
                        Chunk<T, E> o;
                        if constexpr (!KEEP_ROW) {
                            const Chunk<T, E> xc = ring.template get<T, E>(xa, true), dc = ring.template get<T, E>(da, true);
                            float u[E];
                            kept.template get<E, NCH>(0, j, u);
#pragma unroll
                            for (int i = 0; i < E / 2; i++) {
                                xh[i] = mul(add(widen(&xc.v[2 * i]), nmean), r2);
                                wd[i] = mul(widen(&dc.v[2 * i]), pair(u[2 * i], u[2 * i + 1]));
                            }
                        }
#pragma unroll
                        for (int i = 0; i < E / 2; i++) {
                            const int k = KEEP_ROW ? j * E / 2 + i : i;
                            narrow(&o.v[2 * i], mul(r2, fma(xh[k], nq, add(wd[k], np))));
                        }
                        *reinterpret_cast<Chunk<T, E> *>(to) = o;
                    }
                    to += far;
                    xa += by;
                    da += by;
                }
            }
        }
        if constexpr (!KEEP_ROW) refill();
        cm = nm; cr = nr;
    }
    if (!partial) return;
    float *pw_out = partial + (size_t)blockIdx.x * 2 * cols, *pb_out = pw_out + cols;
    float sw[CPT], sb[CPT];
#pragma unroll
    for (int i = 0; i < N; i++) {
        const float2 a = split(aw[i]), b = split(ab[i]);
        sw[2 * i] = a.x; sw[2 * i + 1] = a.y; sb[2 * i] = b.x; sb[2 * i + 1] = b.y;
    }
    if (g.size > 32) {
        if constexpr (VEC) {                    // 16 bytes a store: single values E apart cost a 32-byte sector each
#pragma unroll
            for (int n = 0; n < CPT; n += 4) {
                const int col = (n / E * g.size + g.t) * E + n % E;
                if (col < cols) {
                    *reinterpret_cast<float4 *>(pw_out + col) = make_float4(sw[n], sw[n + 1], sw[n + 2], sw[n + 3]);
                    *reinterpret_cast<float4 *>(pb_out + col) = make_float4(sb[n], sb[n + 1], sb[n + 2], sb[n + 3]);
                }
            }
        } else {
#pragma unroll
            for (int n = 0; n < CPT; n++) {
                const int col = n * g.size + g.t;
                if (col < cols) { pw_out[col] = sw[n]; pb_out[col] = sb[n]; }
            }
        }
        return;
    }
    // narrow rows (cols <= 512): first over the groups of a warp, then over the warps in turn
    for (int o = 16; o >= g.size; o >>= 1)
#pragma unroll
        for (int n = 0; n < CPT; n++) {
            sw[n] += __shfl_xor_sync(0xffffffffu, sw[n], o);
            sb[n] += __shfl_xor_sync(0xffffffffu, sb[n], o);
        }
    const int warp = (int)threadIdx.x >> 5, lane = (int)threadIdx.x & 31;
    for (int k = 0; k < ((int)blockDim.x >> 5); k++) {
        if (warp == k && lane < g.size) {
#pragma unroll
            for (int n = 0; n < CPT; n++) {
                const int col = (n / E * g.size + g.t) * E + n % E;
                if (col < cols && col < 512) {
                    part[0][col] = k ? part[0][col] + sw[n] : sw[n];
                    part[1][col] = k ? part[1][col] + sb[n] : sb[n];
                }
            }
        }
        __syncthreads();
    }
    for (int c = (int)threadIdx.x; c < cols && c < 512; c += (int)blockDim.x) { pw_out[c] = part[0][c]; pb_out[c] = part[1][c]; }
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

// dw and db: column sums of the `parts` partial rows, in double and in a fixed order. A block has 32 columns; a warp
// reads four partial rows at a time, four columns a lane; blockIdx.y 0: dw, 1: db.
template <typename W>
__device__ __forceinline__ void param_grad(W *__restrict__ dw, W *__restrict__ db, const float *__restrict__ partial, int parts, int cols)
{
    __shared__ double sh[32][33];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    W *out = blockIdx.y ? db : dw;
    if (!out) return;
    const int lane = (int)threadIdx.x & 31, ty = (int)threadIdx.x >> 5, warps = (int)blockDim.x >> 5;
    const int c0 = (int)blockIdx.x * 32, c = c0 + 4 * (lane & 7);
    const float *p = partial + (size_t)blockIdx.y * cols;
    double s[4] = { 0.0, 0.0, 0.0, 0.0 };
    if (cols % 4 == 0) {                        // the partial rows start on 16 bytes
        if (c < cols) {
#pragma unroll 4
            for (int i = 4 * ty + (lane >> 3); i < parts; i += 4 * warps) {
                const float4 v = __ldcg(reinterpret_cast<const float4 *>(p + (size_t)i * 2 * cols + c));
                s[0] += (double)v.x; s[1] += (double)v.y; s[2] += (double)v.z; s[3] += (double)v.w;
            }
        }
    } else {
#pragma unroll 4
        for (int i = 4 * ty + (lane >> 3); i < parts; i += 4 * warps)
#pragma unroll
            for (int e = 0; e < 4; e++)
                if (c + e < cols) s[e] += (double)__ldcg(p + (size_t)i * 2 * cols + c + e);
    }
#pragma unroll
    for (int e = 0; e < 4; e++) {
        s[e] += __shfl_xor_sync(0xffffffffu, s[e], 8);
        s[e] += __shfl_xor_sync(0xffffffffu, s[e], 16);
        if (lane < 8) sh[ty][4 * lane + e] = s[e];
    }
    __syncthreads();
    for (int n = ty; n < 32; n += warps) {
        double v = lane < warps ? sh[lane][n] : 0.0;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        if (lane == 0 && c0 + n < cols) out[c0 + n] = from_f32<W>((float)v);
    }
}

}  // namespace ln

#define LN_FORWARD(name, T, W, form, VEC, CPT, HOLD, THREADS, BLOCKS)                                                                     \
    extern "C" __global__ void __launch_bounds__(THREADS, BLOCKS)                                                                        \
    layernorm_##name##_##form(T *y, const T *x, const W *w, const W *b, float *mean, float *rstd, long long rows, int cols,              \
                              long long ldx, long long ldy, float eps, int group, int depth)                                             \
    { ln::forward<T, W, VEC, CPT, HOLD>(y, x, w, b, mean, rstd, rows, cols, ldx, ldy, eps, group, depth); }
#define LN_BACKWARD(name, T, W, form, VEC, CPT, HOLD, KEEP, THREADS)                                                                     \
    extern "C" __global__ void __launch_bounds__(THREADS)                                                                                \
    layernorm_bwd_##name##_##form(T *dx, float *partial, const T *dy, const T *x, const W *w, const float *mean, const float *rstd,      \
                                  long long rows, int cols, long long lddx, long long lddy, long long ldx, int group, int depth)         \
    { ln::backward<T, W, VEC, CPT, HOLD, KEEP>(dx, partial, dy, x, w, mean, rstd, rows, cols, lddx, lddy, ldx, group, depth); }

#define LN_KERNELS(name, T, W)                                                                                                           \
    LN_FORWARD(name, T, W, v8, true, 8, true, 512, 2)                                                                                    \
    LN_FORWARD(name, T, W, v32, true, 32, true, 256, 2)                                                                                  \
    LN_FORWARD(name, T, W, vw, true, 16, false, 640, 1)                                                                                  \
    LN_FORWARD(name, T, W, vx, true, 32, false, 512, 1)                                                                                  \
    LN_FORWARD(name, T, W, s8, false, 8, true, 512, 1)                                                                                   \
    LN_FORWARD(name, T, W, s16, false, 16, true, 512, 1)                                                                                 \
    LN_FORWARD(name, T, W, sx, false, 32, false, 512, 1)                                                                                 \
    LN_BACKWARD(name, T, W, v8, true, 8, true, true, 512)                                                                                \
    LN_BACKWARD(name, T, W, v16, true, 16, true, true, 256)                                                                              \
    LN_BACKWARD(name, T, W, vw, true, (sizeof(T) == 4 ? 20 : 16), false, true, (sizeof(T) == 4 ? 512 : 640))                                                                              \
    LN_BACKWARD(name, T, W, vx, true, 32, false, false, 512)                                                                             \
    LN_BACKWARD(name, T, W, s8, false, 8, true, true, 512)                                                                               \
    LN_BACKWARD(name, T, W, s16, false, 16, true, true, 512)                                                                             \
    LN_BACKWARD(name, T, W, sx, false, 32, false, false, 512)                                                                            \
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
    extern "C" __global__ void __launch_bounds__(1024)                                                                                   \
    layernorm_param_grad_##name(T *dw, T *db, const float *partial, int parts, int cols)                                                 \
    { ln::param_grad<T>(dw, db, partial, parts, cols); }
LN_COLUMNS(f32, float)
LN_COLUMNS(bf16, __nv_bfloat16)
LN_COLUMNS(f16, __half)
