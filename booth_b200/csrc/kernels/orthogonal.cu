// orthogonal.cu -- Newton-Schulz orthogonalisation of a matrix on the tensor cores.
//
//     X = G / (|G|_F + eps);   steps times:  A = X X^t,  X = (a I + b A + c A A) X
//
// drives the singular values of X towards one (the Muon optimiser's update). X is
// s x l with s <= l: a tall G is transposed on the way in and on the way out. With the
// square completed, beta = b / 2c and gamma = a - b^2 / 4c, a step is three plain products,
//     S = X X^t + beta I,   Q = c S S + gamma I,   X = Q X
// whose epilogues add at most a constant to the diagonal and read nothing. (The form P = b A + c A A,
// X = a X + P X reads A and X again, tile by tile, in the epilogue; that took 1.5 to 2 us
// per 32 columns of a tile and bound every product with K below 2000.) With c = 0: Q = b A + a I at once.
//
// All three run on fp16 operands with fp32 accumulation (tcgen05 kind::f16), which hold 11
// bits where bf16 holds 8 at the same rate. X is kept times 2^14, S times 2^12 and Q times a
// power of two that its coefficients allow: singular values stay below 2, so the scaled entries
// fit fp16, and small entries stay above its subnormal range.
//
// Precision, by the type of the result:
//   two planes (f32, f16 results): every operand is hi + lo = fp16(x) + fp16(x - hi), 22
//     bits, and a product is lo.hi + hi.lo + hi.hi. The tensor core adds with truncation, so a
//     long sum drifts: K is cut into chunks of 128 (64-tiles: two sums of 128 each), of 64 where the large diagonal of S or Q comes
//     in, whose sums are added round-to-nearest in registers. The result's error is 0.3 to 1.3 times
//     that of fp32 products, at sides of about 100 up to 1.6 times (96 x 96 2.0e-6 of the norm, 4096 x 4096 1.6e-6).
//   one plane (bf16 results): products use the hi parts only, a third of the work. X
//     still has a lo plane, and Q X adds Q_hi X_lo for the K blocks around the diagonal, where a X
//     comes from: the iteration multiplies what small singular values lose by up to
//     a^steps = 485, so with X rounded to 11 bits each step matrices of low rank came out 2 to 4 %
//     off, with the lo blocks 2e-3 to 4e-3, 1.7e-3 of which is the rounding to bf16.
//
// S and Q are symmetric: only tiles on and below the diagonal are computed and stored.
// Where a product needs a block above the diagonal it loads the mirrored block and has the
// tensor core take it transposed (an operand may have either index contiguous), so nothing
// is stored twice.
//
// Launches per call: orth_norm (sums of squares; Muon: also the momentum), orth_split (planes of
// the normalised, possibly transposed matrix), then steps x 3 products. A product kernel
// keeps one CTA or CTA pair per SM (pair) and walks over the tiles of all matrices of
// the batch; the roles inside are those of the fp32 GEMM: warp 0 TMA, warp 1 MMA, warps 4-11
// drain tensor memory, apply the epilogue and store.
//   256: 256 x 256 tile per two CTAs, tcgen05.mma.cta_group::2
//   128: 128 x 128 tile per CTA
//   64:  64 x 64 tile per CTA, for products so small that they are all latency
// With few tiles the K of a tile is shared by up to four pairs or eight CTAs of a cluster.
#include "common.cuh"
#include "orth_params.cuh"
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

namespace orth {

using gemm::WaitCtl;
using gemm::mbar_wait;
using gemm::smem_u32;

constexpr float X_SCALE = 16384.f;       // 2^14

// Elements of a type known at run time: first the bits, then the values. (Load and conversion under one branch on the
// type would wait for each load before the next is issued.)
__device__ __forceinline__ uint32_t bits1(const void *p, int type, long long i)
{
    return type == ORTH_F32 ? static_cast<const uint32_t *>(p)[i] : static_cast<const uint16_t *>(p)[i];
}
__device__ __forceinline__ float value1(uint32_t x, int type)
{
    return type == ORTH_F32 ? __uint_as_float(x) : type == ORTH_BF16 ? __uint_as_float(x << 16) : __half2float(__ushort_as_half((unsigned short)x));
}
__device__ __forceinline__ void store1(void *p, int type, long long i, float v)
{
    if (type == ORTH_F32) static_cast<float *>(p)[i] = v;
    else if (type == ORTH_BF16) static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half *>(p)[i] = __float2half_rn(v);
}
// The value that a store to this type and a load back would give.
__device__ __forceinline__ float rounded(float v, int type)
{
    return type == ORTH_F32 ? v : type == ORTH_BF16 ? __bfloat162float(__float2bfloat16_rn(v)) : __half2float(__float2half_rn(v));
}
__device__ __forceinline__ float4 rounded4(float4 v, int type) { return make_float4(rounded(v.x, type), rounded(v.y, type), rounded(v.z, type), rounded(v.w, type)); }
// Four neighbouring elements; p + i is aligned to four elements.
__device__ __forceinline__ uint4 bits4(const void *p, int type, long long i)
{
    if (type == ORTH_F32) return *reinterpret_cast<const uint4 *>(static_cast<const float *>(p) + i);
    const uint2 r = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + i);
    return make_uint4(r.x, r.y, 0, 0);
}
__device__ __forceinline__ float4 values4(uint4 r, int type)
{
    if (type == ORTH_F32) return make_float4(__uint_as_float(r.x), __uint_as_float(r.y), __uint_as_float(r.z), __uint_as_float(r.w));
    if (type == ORTH_BF16)
        return make_float4(__uint_as_float(r.x << 16), __uint_as_float(r.x & 0xffff0000u), __uint_as_float(r.y << 16), __uint_as_float(r.y & 0xffff0000u));
    const float2 a = __half22float2(*reinterpret_cast<const __half2 *>(&r.x)), b = __half22float2(*reinterpret_cast<const __half2 *>(&r.y));
    return make_float4(a.x, a.y, b.x, b.y);
}
__device__ __forceinline__ void store4(void *p, int type, long long i, float4 v)
{
    if (type == ORTH_F32) { *reinterpret_cast<float4 *>(static_cast<float *>(p) + i) = v; return; }
    uint2 r;
    if (type == ORTH_BF16) {
        const __nv_bfloat162 a = __floats2bfloat162_rn(v.x, v.y), b = __floats2bfloat162_rn(v.z, v.w);
        r.x = *reinterpret_cast<const uint32_t *>(&a); r.y = *reinterpret_cast<const uint32_t *>(&b);
    } else {
        const __half2 a = __floats2half2_rn(v.x, v.y), b = __floats2half2_rn(v.z, v.w);
        r.x = *reinterpret_cast<const uint32_t *>(&a); r.y = *reinterpret_cast<const uint32_t *>(&b);
    }
    *reinterpret_cast<uint2 *>(static_cast<uint16_t *>(p) + i) = r;
}

using Source = orth_source_t;
using Product = orth_product_t;

__device__ __forceinline__ float lerp(float m, float g, float mu) { return fmaf(mu, m, (1.f - mu) * g); }
// What is orthogonalised, from the gradient and the stored momentum.
__device__ __forceinline__ float update_of(float m, float g, const Source &s) { return s.nesterov ? lerp(m, g, s.mu) : m; }

__device__ __forceinline__ float4 update4(float4 m, float4 g, const Source &s)
{
    return make_float4(update_of(m.x, g.x, s), update_of(m.y, g.y, s), update_of(m.z, g.z, s), update_of(m.w, g.w, s));
}

}  // namespace orth

// Sum of squares of each matrix, in double (squares of any finite value fit), one
// partial per block: block (i, k) takes every gridDim.x-th piece of matrix k. Muon: the
// momentum is brought up to date on the way and the stored, rounded value is used.
extern "C" __global__ void __launch_bounds__(256)
orth_norm(const __grid_constant__ orth::Source s, double *__restrict__ partial)
{
    using namespace orth;
    __shared__ double sh[8];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int k = (int)blockIdx.y, W = s.vec ? 4 : 1;
    // matrices without gaps are walked as one row, the others a row a block at a time
    const long long rows = s.flat ? 1 : s.rows, cols = s.flat ? (long long)s.rows * s.cols : s.cols;
    const long long r0 = s.flat ? 0 : blockIdx.x, r_step = s.flat ? 1 : gridDim.x;
    const long long c0 = (long long)((s.flat ? blockIdx.x * 256u : 0u) + threadIdx.x) * W, c_step = (s.flat ? gridDim.x : 1u) * 256ll * W;
    double sum = 0.0;
    for (long long r = r0; r < rows; r += r_step) {
        const long long at_g = k * s.stride_g + r * s.ld_g, at_m = k * s.stride_m + r * s.ld_m;
        // several loads ahead of the stores to m, which the compiler has to keep in order
        constexpr int N = 4;
        for (long long c = c0; c < cols; c += N * c_step) {
            if (s.vec) {
                uint4 g[N], m[N];
#pragma unroll
                for (int n = 0; n < N; n++) {
                    g[n] = m[n] = make_uint4(0, 0, 0, 0);
                    if (c + n * c_step < cols) {
                        g[n] = bits4(s.g, s.type_g, at_g + c + n * c_step);
                        if (s.m) m[n] = bits4(s.m, s.type_m, at_m + c + n * c_step);
                    }
                }
#pragma unroll
                for (int n = 0; n < N; n++) {
                    float4 u = values4(g[n], s.type_g);
                    if (s.m && c + n * c_step < cols) {
                        float4 x = values4(m[n], s.type_m);
                        x = rounded4(make_float4(lerp(x.x, u.x, s.mu), lerp(x.y, u.y, s.mu), lerp(x.z, u.z, s.mu), lerp(x.w, u.w, s.mu)), s.type_m);
                        store4(s.m, s.type_m, at_m + c + n * c_step, x);
                        u = update4(x, u, s);
                    }
                    sum += ((double)u.x * u.x + (double)u.y * u.y) + ((double)u.z * u.z + (double)u.w * u.w);
                }
            } else {
                uint32_t g[N], m[N];
#pragma unroll
                for (int n = 0; n < N; n++) {
                    g[n] = m[n] = 0;
                    if (c + n * c_step < cols) {
                        g[n] = bits1(s.g, s.type_g, at_g + c + n * c_step);
                        if (s.m) m[n] = bits1(s.m, s.type_m, at_m + c + n * c_step);
                    }
                }
#pragma unroll
                for (int n = 0; n < N; n++) {
                    float u = value1(g[n], s.type_g);
                    if (s.m && c + n * c_step < cols) {
                        const float x = rounded(lerp(value1(m[n], s.type_m), u, s.mu), s.type_m);
                        store1(s.m, s.type_m, at_m + c + n * c_step, x);
                        u = update_of(x, u, s);
                    }
                    sum += (double)u * u;
                }
            }
        }
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int i = 1; i < 8; i++) sum += sh[i];
        partial[(size_t)k * gridDim.x + blockIdx.x] = sum;
    }
}

// hi and lo planes of 2^14 u / (|u| + eps), s x l with rows `pitch` apart, transposed
// when the matrix is tall. A 64 x 64 tile of u a block; grid (column tiles, row tiles,
// matrices). A tall tile goes through shared memory, any other straight to its place.
extern "C" __global__ void __launch_bounds__(256)
orth_split(const __grid_constant__ orth::Source s, const double *__restrict__ partial, int parts, float eps, __half *__restrict__ hi,
           __half *__restrict__ lo, long long pitch, long long plane, int tall)
{
    using namespace orth;
    __shared__ float tile[64][65];
    __shared__ float s_scale;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int k = (int)blockIdx.z, r0 = (int)blockIdx.y * 64, c0 = (int)blockIdx.x * 64;
    const int tx = (int)threadIdx.x & 15, ty = (int)threadIdx.x >> 4;
    uint4 g[4], m[4];
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const int r = r0 + ty + 16 * p, c = c0 + 4 * tx;
        const long long at_g = k * s.stride_g + r * s.ld_g + c, at_m = k * s.stride_m + r * s.ld_m + c;
        g[p] = m[p] = make_uint4(0, 0, 0, 0);
        if (r >= s.rows) continue;
        if (s.vec) {
            if (c < s.cols) {
                g[p] = bits4(s.g, s.type_g, at_g);
                if (s.m) m[p] = bits4(s.m, s.type_m, at_m);
            }
        } else {
            uint32_t x[4], y[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[e] = c + e < s.cols ? bits1(s.g, s.type_g, at_g + e) : 0;
                y[e] = s.m && c + e < s.cols ? bits1(s.m, s.type_m, at_m + e) : 0;
            }
            g[p] = s.type_g == ORTH_F32 ? make_uint4(x[0], x[1], x[2], x[3]) : make_uint4(x[0] | x[1] << 16, x[2] | x[3] << 16, 0, 0);
            m[p] = s.type_m == ORTH_F32 ? make_uint4(y[0], y[1], y[2], y[3]) : make_uint4(y[0] | y[1] << 16, y[2] | y[3] << 16, 0, 0);
        }
    }
    if (threadIdx.x < 32) {
        double sum = 0.0;
        for (int i = (int)threadIdx.x; i < parts; i += 32) sum += partial[(size_t)k * parts + i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (threadIdx.x == 0) s_scale = (float)fmin((double)X_SCALE / (sqrt(sum) + (double)eps), 3.4e38);
    }
    float4 v[4];
#pragma unroll
    for (int p = 0; p < 4; p++) {
        v[p] = values4(g[p], s.type_g);
        if (s.m) v[p] = update4(values4(m[p], s.type_m), v[p], s);
    }
    if (tall) {
#pragma unroll
        for (int p = 0; p < 4; p++) {
            float *t = &tile[ty + 16 * p][4 * tx];
            t[0] = v[p].x; t[1] = v[p].y; t[2] = v[p].z; t[3] = v[p].w;
        }
    }
    __syncthreads();
    const float f = s_scale;
    __half *ph = hi + k * plane, *pl = lo + k * plane;
#pragma unroll
    for (int p = 0; p < 4; p++) {
        // row (of the plane) a, four columns from b; the pitch is a multiple of 64, so a whole group is in the plane
        const int a = ty + 16 * p, b = 4 * tx;
        const int row = (tall ? c0 : r0) + a, col = (tall ? r0 : c0) + b;
        if (tall) v[p] = make_float4(tile[b][a], tile[b + 1][a], tile[b + 2][a], tile[b + 3][a]);
        if (row < (tall ? s.cols : s.rows) && col < (tall ? s.rows : s.cols)) {
            const float x[4] = { f * v[p].x, f * v[p].y, f * v[p].z, f * v[p].w };
            __half h[4], l[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                h[e] = __float2half_rn(x[e]);
                l[e] = __float2half_rn(x[e] - __half2float(h[e]));
            }
            *reinterpret_cast<uint2 *>(ph + row * pitch + col) = *reinterpret_cast<const uint2 *>(h);
            *reinterpret_cast<uint2 *>(pl + row * pitch + col) = *reinterpret_cast<const uint2 *>(l);
        }
    }
}

namespace orth {

// The completion is counted on `bar`, for a pair on the leader's barrier. One elected lane issues.
template <bool PAIR>
__device__ __forceinline__ void load_box(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z)
{
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                     "@e cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n\t}"
                     ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
    else
        asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t"
                     "@e cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];\n\t}"
                     ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}

// fp16 x fp16 -> fp32; bits 15 and 16: the first or second operand's tile has its rows (columns), not K, contiguous.
__device__ __forceinline__ uint32_t instr_desc(int m, int n, bool a_t, bool b_t)
{
    return (1u << 4) | ((uint32_t)a_t << 15) | ((uint32_t)b_t << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// Shared-memory descriptor of an operand: 64 x 64 boxes, 128 bytes a box row, 128-byte swizzle, 8 rows 1024 bytes. K
// contiguous (`t` false): rows of the operand, the boxes one below the other. Else rows of K, each with 64
// rows of the operand; the next 64 lie 8192 bytes on. The address is the low word's low half, so a tile further on
// is a 32-bit addition; the high word never changes.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, bool t) { return ((addr & 0x3FFFFu) >> 4) | (t ? (8192u >> 4) << 16 : 0u); }
__device__ __forceinline__ uint64_t desc(uint32_t lo)
{
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "r"(lo), "n"((1024u >> 4) | (1u << 14) | (2u << 29)));
    return d;
}

// The control warps run their loops with all lanes in step, so that addresses and descriptors stay in uniform
// registers; one elected lane issues. (In a branch of a single lane every descriptor went through general
// registers, and the issuer took 650 clocks for the four one-plane products of a K block, which take 512.)
template <bool PAIR>
__device__ __forceinline__ void umma(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                     "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
}
// 32 halves of a row, whole 32-byte sectors at a time.
__device__ __forceinline__ void put_row(char *to, const uint32_t (&v)[16])
{
#pragma unroll
    for (int i = 0; i < 2; i++)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(to + 32 * i), "r"(v[8 * i]), "r"(v[8 * i + 1]), "r"(v[8 * i + 2]), "r"(v[8 * i + 3]),
                     "r"(v[8 * i + 4]), "r"(v[8 * i + 5]), "r"(v[8 * i + 6]), "r"(v[8 * i + 7]) : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const float *v)
{
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], "
                 "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
                 "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31};"
                 ::"f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]),
                   "f"(v[8]), "f"(v[9]), "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15]),
                   "f"(v[16]), "f"(v[17]), "f"(v[18]), "f"(v[19]), "f"(v[20]), "f"(v[21]), "f"(v[22]), "f"(v[23]),
                   "f"(v[24]), "f"(v[25]), "f"(v[26]), "f"(v[27]), "f"(v[28]), "f"(v[29]), "f"(v[30]), "f"(v[31]),
                   "r"(taddr) : "memory");
}
// Arrives on the barrier at this offset, for a pair in both of its CTAs (cluster ranks first, first + 1), once the
// products issued so far are complete.
template <bool PAIR> __device__ __forceinline__ void commit(uint32_t bar, uint32_t first)
{
    if constexpr (PAIR)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"((uint16_t)(3u << first)) : "memory");
    else gemm::umma_commit(bar);
}
__device__ __forceinline__ bool elected()
{
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e != 0;
}
__device__ __forceinline__ void expect_tx(uint32_t bar, uint32_t bytes)
{
    asm volatile("{\n\t.reg .pred e;\n\telect.sync _|e, 0xffffffff;\n\t@e mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;\n\t}"
                 ::"r"(bar), "r"(bytes) : "memory");
}
// Bounded wait of a whole warp.
__device__ __forceinline__ bool warp_wait(uint32_t bar, uint32_t parity, const WaitCtl &w, int code)
{
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, w, code));
}

// Tile number -> matrix, tile row and tile column. Tiles that run at the same time should share
// operand panels through L2: eight tile rows at a time, column by column; symmetric products
// number the tiles on and below the diagonal that way.
struct Tiles {
    int tm, tn, each;
    bool sym;
    __device__ __forceinline__ Tiles(const Product &p, int side)
    {
        tm = (p.rows + side - 1) / side; tn = (p.cols + side - 1) / side;
        sym = p.mode <= ORTH_POLY;
        each = sym ? tm * (tm + 1) / 2 : tm * tn;
    }
    __device__ __forceinline__ void at(int item, int &k, int &i, int &j) const
    {
        k = item / each;
        int t = item - k * each;
        if (!sym) { gemm::pair_tile_coords(t, tm, tn, i, j); return; }
        int r0 = 0, h;
        for (;; r0 += 8) {                      // the group of eight rows: r0 .. r0 + h - 1
            h = min(tm - r0, 8);
            const int n = h * r0 + h * (h + 1) / 2;
            if (t < n) break;
            t -= n;
        }
        if (t < h * (r0 + 1)) { j = t / h; i = r0 + t % h; return; }
        t -= h * (r0 + 1);
        for (j = r0 + 1, h--; t >= h; j++, h--) t -= h;
        i = j + t;
    }
};

__device__ __forceinline__ void sts(uint32_t a, uint4 v) { asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory"); }
__device__ __forceinline__ uint4 lds(uint32_t a)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void tma_store(const CUtensorMap *map, uint32_t src, int x, int y, int z)
{
    asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];"
                 ::"l"(map), "r"(src), "r"(x), "r"(y), "r"(z) : "memory");
    asm volatile("cp.async.bulk.commit_group;" ::: "memory");
}

// 64-tiles go out by TMA in boxes of 64 x 64 of a plane, which clips them at the matrix's edges: a lane puts its
// packed halves of row r, from 16-byte unit u0 on, into the box in the map's 128-byte swizzle.
template <int N>
__device__ __forceinline__ void put_box(uint32_t box, const uint32_t (&packed)[N], int r, int u0)
{
#pragma unroll
    for (int u = 0; u < N / 4; u++)
        sts(box + (uint32_t)(r * 128 + (((u0 + u) ^ r) & 7) * 16), make_uint4(packed[4 * u], packed[4 * u + 1], packed[4 * u + 2], packed[4 * u + 3]));
}
template <int THREADS> __device__ __forceinline__ void team_sync(int bar) { asm volatile("bar.sync %0, %1;" ::"r"(bar), "n"(THREADS) : "memory"); }
// Whether all warps of the team say so.
template <int THREADS> __device__ __forceinline__ bool all_ok(int bar, bool ok)
{
    uint32_t all;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.b32 p, %1, 0;\n\tbarrier.red.and.pred q, %2, %3, p;\n\tselp.u32 %0, 1, 0, q;\n\t}"
                 : "=r"(all) : "r"((uint32_t)ok), "r"(bar), "n"(THREADS) : "memory");
    return all != 0;
}

// Whether a wait has run out in a product of this handle that nobody has asked about yet, this call's earlier ones among
// them: its planes are incomplete, and the caller's matrix is left as it is. Asked once a tile, behind its sums, where the answer
// is on its way while they are read back.
__device__ __forceinline__ int gave_up(const Product &p)
{
    int v = 0;
    if (p.mode == ORTH_RESULT) asm volatile("ld.relaxed.gpu.global.b32 %0, [%1];" : "=r"(v) : "l"(p.status) : "memory");
    return v;
}

// Brings the weights a warp's rows will read into L2 while the products run.
__device__ __forceinline__ void prefetch_result(const Product &p, int lane, int k, int row0, int col0, int cols)
{
    const int bytes = p.type_w == ORTH_F32 ? 4 : 2;
    const char *const w = static_cast<const char *>(p.w) + k * p.stride_w * bytes;
    if (p.tall) {       // a column of the tile is a run of 32 elements of the caller's row
        for (int c = lane; c < cols && col0 + c < p.cols; c += 32)
            if (row0 < p.rows) asm volatile("prefetch.global.L2 [%0];" ::"l"(w + ((col0 + c) * p.ld_w + row0) * bytes));
    } else if (row0 + lane < p.rows) {
        for (int c = 0; c < cols && col0 + c < p.cols; c += 128 / bytes)
            asm volatile("prefetch.global.L2 [%0];" ::"l"(w + ((row0 + lane) * p.ld_w + col0 + c) * bytes));
    }
}

// One warp's 32 rows x 32 columns of the caller's matrix: N / 32 of its weights from part `n0` on, as bits, and the result, a
// row a lane in v. A tall matrix has a column of the piece as a contiguous run of its row: neighbouring lanes hold
// neighbouring rows. Else the piece goes through 4 KB of the warp's own shared memory, so that accesses run
// along the rows: eight rows of eight lanes' groups of four elements, or a column a lane.
template <int N, bool WIDE>
__device__ __forceinline__ void fetch_weights_of(const Product &p, uint32_t (&w)[N], int n0, int lane, int k, int row0, int col0)
{
    constexpr int type = WIDE ? ORTH_F32 : ORTH_BF16;       // as bits, 16-bit types are alike
    if (p.tall) {
        const long long o = k * p.stride_w + col0 * p.ld_w + row0 + lane;
#pragma unroll
        for (int j = 0; j < N; j++)
            if (row0 + lane < p.rows && col0 + n0 + j < p.cols) w[j] = bits1(p.w, type, o + (n0 + j) * p.ld_w);
    } else if (p.vec_w) {
        const int r0 = n0 + (lane >> 3), c = col0 + 4 * (lane & 7);
        const long long o = k * p.stride_w + (row0 + r0) * p.ld_w + c;
#pragma unroll
        for (int q = 0; q < N / 4; q++)
            if (row0 + r0 + 4 * q < p.rows && c < p.cols) {
                const uint4 x = bits4(p.w, type, o + 4 * q * p.ld_w);
                w[4 * q] = x.x; w[4 * q + 1] = x.y; w[4 * q + 2] = x.z; w[4 * q + 3] = x.w;
            }
    } else {
        const long long o = k * p.stride_w + row0 * p.ld_w + col0 + lane;
#pragma unroll
        for (int q = 0; q < N; q++)
            if (row0 + n0 + q < p.rows && col0 + lane < p.cols) w[q] = bits1(p.w, type, o + (n0 + q) * p.ld_w);
    }
}
template <int N>
__device__ __forceinline__ void fetch_weights(const Product &p, uint32_t (&w)[N], int n0, int lane, int k, int row0, int col0)
{
#pragma unroll
    for (int j = 0; j < N; j++) w[j] = 0;
    if (p.keep == 0.f) return;
    if (p.type_w == ORTH_F32) fetch_weights_of<N, true>(p, w, n0, lane, k, row0, col0);
    else fetch_weights_of<N, false>(p, w, n0, lane, k, row0, col0);
}
// The result's part `n0`.. with those weights. put_result comes first where the matrix is not tall.
__device__ __forceinline__ void put_result(const float (&v)[32], uint32_t buf, int lane)
{
    __syncwarp();
#pragma unroll
    for (int u = 0; u < 8; u++)
        sts(buf + (uint32_t)(lane * 128 + ((u ^ lane) & 7) * 16),
            make_uint4(__float_as_uint(v[4 * u]), __float_as_uint(v[4 * u + 1]), __float_as_uint(v[4 * u + 2]), __float_as_uint(v[4 * u + 3])));
    __syncwarp();
}
template <int N, int N0, int TYPE>
__device__ __forceinline__ void store_result_as(const Product &p, const float (&v)[32], const uint32_t (&w)[N], uint32_t buf, int lane, int k, int row0, int col0)
{
    if (p.tall) {
        const long long o = k * p.stride_w + col0 * p.ld_w + row0 + lane;
#pragma unroll
        for (int j = 0; j < N; j++)
            if (row0 + lane < p.rows && col0 + N0 + j < p.cols) store1(p.w, TYPE, o + (N0 + j) * p.ld_w, fmaf(p.keep, value1(w[j], TYPE), v[N0 + j]));
    } else if (p.vec_w) {
        const int u = lane & 7, r0 = N0 + (lane >> 3), c = col0 + 4 * u;
        const long long o = k * p.stride_w + (row0 + r0) * p.ld_w + c;
#pragma unroll
        for (int q = 0; q < N / 4; q++)
            if (row0 + r0 + 4 * q < p.rows && c < p.cols) {
                const int r = r0 + 4 * q;
                const uint4 x = lds(buf + (uint32_t)(r * 128 + ((u ^ r) & 7) * 16));
                const float4 y = values4(make_uint4(w[4 * q], w[4 * q + 1], w[4 * q + 2], w[4 * q + 3]), TYPE);
                store4(p.w, TYPE, o + 4 * q * p.ld_w, make_float4(fmaf(p.keep, y.x, __uint_as_float(x.x)), fmaf(p.keep, y.y, __uint_as_float(x.y)),
                                                                     fmaf(p.keep, y.z, __uint_as_float(x.z)), fmaf(p.keep, y.w, __uint_as_float(x.w))));
            }
    } else {
        const long long o = k * p.stride_w + row0 * p.ld_w + col0 + lane;
#pragma unroll
        for (int q = 0; q < N; q++) {
            const int r = N0 + q;
            float x;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(buf + (uint32_t)(r * 128 + (((lane >> 2) ^ r) & 7) * 16 + (lane & 3) * 4)) : "memory");
            if (row0 + r < p.rows && col0 + lane < p.cols) store1(p.w, TYPE, o + r * p.ld_w, fmaf(p.keep, value1(w[q], TYPE), x));
        }
    }
}

template <int N, int N0>
__device__ __forceinline__ void store_result(const Product &p, const float (&v)[32], const uint32_t (&w)[N], uint32_t buf, int lane, int k, int row0, int col0)
{
    if (p.type_w == ORTH_F32) store_result_as<N, N0, ORTH_F32>(p, v, w, buf, lane, k, row0, col0);
    else if (p.type_w == ORTH_BF16) store_result_as<N, N0, ORTH_BF16>(p, v, w, buf, lane, k, row0, col0);
    else store_result_as<N, N0, ORTH_F16>(p, v, w, buf, lane, k, row0, col0);
}

// A lane's part of row r of a 64 x 64 quarter in fp32, from 16-byte unit u0 on.
template <int N> __device__ __forceinline__ void put_quarter(uint32_t quarter, const uint32_t (&x)[N], int r, int u0)
{
#pragma unroll
    for (int u = 0; u < N / 4; u++)
        sts(quarter + (uint32_t)(r * 256 + ((u0 + u) ^ (r & 7)) * 16), make_uint4(x[4 * u], x[4 * u + 1], x[4 * u + 2], x[4 * u + 3]));
}

// A 64 x 64 tile of the result, rows of 65 floats in shared memory, into the caller's matrix by 256 threads, along its
// rows; loads ahead of stores.
__device__ __forceinline__ void store_result_64(const Product &p, uint32_t tile, int tid, int k, int row0, int col0)
{
    const auto at = [&](int r, int c) {
        float x;
        asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(tile + (uint32_t)(r * 65 + c) * 4) : "memory");
        return x;
    };
    if (p.vec_w && !p.tall) {
        const int c = 4 * (tid & 15);
        uint4 w[4];
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const int r = (tid >> 4) + 16 * n;
            w[n] = make_uint4(0, 0, 0, 0);
            if (p.keep != 0.f && row0 + r < p.rows && col0 + c < p.cols) w[n] = bits4(p.w, p.type_w, k * p.stride_w + (row0 + r) * p.ld_w + col0 + c);
        }
#pragma unroll
        for (int n = 0; n < 4; n++) {
            const int r = (tid >> 4) + 16 * n;
            const float4 y = values4(w[n], p.type_w);
            if (row0 + r < p.rows && col0 + c < p.cols)
                store4(p.w, p.type_w, k * p.stride_w + (row0 + r) * p.ld_w + col0 + c,
                       make_float4(fmaf(p.keep, y.x, at(r, c)), fmaf(p.keep, y.y, at(r, c + 1)), fmaf(p.keep, y.z, at(r, c + 2)), fmaf(p.keep, y.w, at(r, c + 3))));
        }
        return;
    }
    // an element a thread, neighbouring threads along the caller's row
    uint32_t w[16];
#pragma unroll
    for (int n = 0; n < 16; n++) {
        const int x = tid & 63, y = (tid >> 6) + 4 * n, r = p.tall ? x : y, c = p.tall ? y : x;
        const long long o = k * p.stride_w + (p.tall ? (col0 + c) * p.ld_w + row0 + r : (row0 + r) * p.ld_w + col0 + c);
        w[n] = p.keep != 0.f && row0 + r < p.rows && col0 + c < p.cols ? bits1(p.w, p.type_w, o) : 0;
    }
#pragma unroll
    for (int n = 0; n < 16; n++) {
        const int x = tid & 63, y = (tid >> 6) + 4 * n, r = p.tall ? x : y, c = p.tall ? y : x;
        const long long o = k * p.stride_w + (p.tall ? (col0 + c) * p.ld_w + row0 + r : (row0 + r) * p.ld_w + col0 + c);
        if (row0 + r < p.rows && col0 + c < p.cols) store1(p.w, p.type_w, o, fmaf(p.keep, value1(w[n], p.type_w), at(r, c)));
    }
}

// Shared memory: operand stages; behind them 32 KB in which results are staged. 64-tiles: 48 KB in which the quarters of
// the product meet, and a box each for hi and lo.
constexpr uint32_t OPERAND_BYTES = 196608, OPERAND_BYTES_64 = 163840, QUARTERS_64 = 49152;

// Two planes: where the accumulator is drained, after every `run` K blocks (64-tiles, whose small products and halves of K blocks
// have sums of their own: 4; else 2) and after every one on the tile's diagonal.
__device__ __forceinline__ bool chunk_ends(int kb, int run, int diag0, int diag, bool sym)
{
    return (kb & (run - 1)) == run - 1 || (sym && kb >= diag0 && kb < diag0 + diag);
}

// 384 threads; grid: any number of CTAs (pairs), each takes every grid-th tile. p.split > 1: a
// cluster of that many CTAs (pairs) shares one tile, each takes a range of K, and the sums meet in the
// workspace, every split-th 32 columns of the tile with each owner; the grid is then one cluster a tile. Few tiles
// leave most of the GPU idle: the 10 tiles of a 1000 x 1000 symmetric product with K = 2049 took 33 us
// on 36 single CTAs. (Through distributed shared memory instead of L2 the meeting alone took 10 us.)
template <int PLANES, int SIDE>
__device__ __forceinline__ void product(const CUtensorMap &a_hi, const CUtensorMap &a_lo, const CUtensorMap &b_hi, const CUtensorMap &b_lo,
                                        const CUtensorMap &o_hi, const CUtensorMap &o_lo, const Product &p)
{
    using namespace gemm;
    constexpr bool PAIR = SIDE == 256;
    constexpr int BK = 64, ROWS = SIDE == 64 ? 64 : 128;            // K block; rows of an operand that one CTA holds
    constexpr uint32_t TILE = ROWS * BK * 2;                        // one operand plane of one CTA
    constexpr uint32_t STAGE = 2 * PLANES * TILE;
    constexpr int STAGES = (SIDE == 64 ? OPERAND_BYTES_64 : OPERAND_BYTES) / STAGE;
    constexpr int HALF = SIDE / 2;                                  // columns per epilogue warp
    // Rows and columns of one tensor instruction. 64-tiles in two planes take hi and lo, which lie one below the
    // other, as one operand of 128: the four quarters of a 128 x 128 product are hi.hi, hi.lo, lo.hi and lo.lo (which
    // costs nothing here and is taken along), four instructions a K block instead of twelve (an instruction takes some 90 clocks however small it is).
    constexpr int MMA = SIDE == 64 ? 64 * PLANES : SIDE;
    // 64-tiles in two planes have two sums, one of the first and one of the second half of each K block: an instruction drops of
    // each of its products what lies 25 bits below the sum it adds to, and half as many instructions make half the sum. Small
    // matrices need that, they have no long sums in which such losses would even out: 128 x 128 was 2.4 times as far off as with fp32
    // products and is 1.2 times, 256 x 256 1.5 and is 0.8, for 1 to 2 us a call. (A sum drained after every half block was no
    // more exact and took 12 to 27 us.)
    constexpr bool FINE = SIDE == 64 && PLANES == 2;
    constexpr uint32_t TMEM_COLS = (FINE ? 4 : 2) * MMA;            // two accumulators
    const WaitCtl status = { p.status, p.wait_ns };

    extern __shared__ uint8_t smem_orth[];
    __shared__ __align__(8) uint64_t bars[2 * STAGES + 4];
    __shared__ uint32_t s_tmem;

    constexpr int CTAS = PAIR ? 2 : 1;
    const uint32_t cta = cluster_ctarank(), rank = PAIR ? cta & 1u : 0u, first = cta - rank;    // first: the pair's leader
    const bool leader = rank == 0;
    const int split = p.split, part = (int)cta / CTAS;
    const uint32_t smem0 = (smem_u32(smem_orth) + 1023u) & ~1023u;
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[STAGES]);
    const uint32_t acc_full0 = smem_u32(&bars[2 * STAGES]), acc_empty0 = smem_u32(&bars[2 * STAGES + 2]);
    const int warp = __shfl_sync(0xffffffffu, (int)threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    const int C = (int)(gridDim.x / (unsigned)(CTAS * split)), cl = (int)(blockIdx.x / (unsigned)(CTAS * split));
    const Tiles tiles(p, SIDE);
    const int items = tiles.each * p.batch;
    // K blocks of this pair: [kb0, kb1), an even number but for the last
    const int all_kb = (p.K + BK - 1) / BK, all_ck = (all_kb + 1) / 2;
    const int kb0 = 2 * (all_ck * part / split), kb1 = min(all_kb, 2 * (all_ck * (part + 1) / split));
    // Which operand blocks come transposed. X as the second operand of Q X has its columns contiguous. Of a
    // symmetric operand the block at K block kb is above the stored triangle when kb's tile lies beyond the tile
    // of the rows. (Rows that span two of the triangle's tiles take the rule of the upper one: for the
    // lower one that differs only inside its own diagonal tile, which is stored whole.)
    const bool a_sym = p.mode != ORTH_GRAM, b_sym = p.mode == ORTH_POLY, b_cols = p.mode >= ORTH_UPDATE;
    const int tri_kb = p.tri / BK;
    // first K block that comes transposed, of rows that begin at tile index x of SIDE
    const auto turn = [&](int x, bool sym) { return sym ? (x * (SIDE / BK) / tri_kb + 1) * tri_kb : 0x7fffffff; };
    // One plane, Q X: ahead of the K blocks, those on the tile's diagonal with the lo plane of X.
    constexpr int DIAG = SIDE / BK, RUN = SIDE == 64 ? 4 : 2;
    const auto lo_from = [&](int x) { return max(x * DIAG, kb0); };
    const auto lo_count = [&](int x) { return PLANES == 1 && b_cols ? max(0, min(x * DIAG + DIAG, kb1) - lo_from(x)) : 0; };

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int b = 0; b < 2; b++) { mbar_init(acc_full0 + 8 * b, 1); mbar_init(acc_empty0 + 8 * b, PAIR ? 16 : 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 32) {        // the descriptors, while the kernel before still runs
        asm volatile("prefetch.tensormap [%0];" ::"l"(&a_hi) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&b_hi) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&b_lo) : "memory");
        if constexpr (PLANES == 2) asm volatile("prefetch.tensormap [%0];" ::"l"(&a_lo) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&o_hi) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&o_lo) : "memory");
    }
    __syncwarp();
    if (warp == 1) {
        if constexpr (PAIR) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(TMEM_COLS) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem = s_tmem;
    asm volatile("griddepcontrol.wait;" ::: "memory");              // everything above touched only this CTA (pair)
    asm volatile("griddepcontrol.launch_dependents;");
    // 384 threads start with 168 registers each; the epilogue's two warpgroups take what the control warpgroup gives up
    if (warp < 4) {
      asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
      if (warp == 0) {
        {
            uint32_t st = smem0, full = full0, empty = empty0, ph = 1;      // stage and its barriers
            bool ok = true;
            for (int item = cl; ok && !p.silent && item < items; item += C) {
                int k, i, j;
                tiles.at(item, k, i, j);
                const int m0 = i * SIDE + (int)rank * 128, n0 = j * SIDE + (int)rank * 128;
                const int a_turn = turn(i, a_sym), b_turn = b_cols ? 0 : turn(j, b_sym);
                int lo = lo_count(i);
                for (int kb = lo ? lo_from(i) : kb0; kb < kb1;) {
                    if (!warp_wait(empty, ph, status, 1)) { ok = false; break; }
                    if (leader) expect_tx(full, CTAS * STAGE);
                    const uint32_t bar = PAIR ? map_to_cta(full, first) : full;
                    const CUtensorMap *const b1 = lo ? &b_lo : &b_hi;
                    const bool a_t = kb >= a_turn, b_t = kb >= b_turn;
#pragma unroll
                    for (int h = 0; h < ROWS / 64; h++) {           // 64 rows of an operand at a time
                        const uint32_t d = st + (uint32_t)h * 8192u;
                        const int ax = a_t ? m0 + 64 * h : kb * BK, ay = a_t ? kb * BK : m0 + 64 * h;
                        const int bx = b_t ? n0 + 64 * h : kb * BK, by = b_t ? kb * BK : n0 + 64 * h;
                        load_box<PAIR>(d, &a_hi, bar, ax, ay, k);
                        load_box<PAIR>(d + PLANES * TILE, b1, bar, bx, by, k);
                        if constexpr (PLANES == 2) {
                            load_box<PAIR>(d + TILE, &a_lo, bar, ax, ay, k);
                            load_box<PAIR>(d + 3 * TILE, &b_lo, bar, bx, by, k);
                        }
                    }
                    st += STAGE; full += 8; empty += 8;
                    if (full == full0 + 8 * STAGES) { st = smem0; full = full0; empty = empty0; ph ^= 1u; }
                    kb = lo && --lo == 0 ? kb0 : kb + 1;
                }
            }
        }
        __syncwarp();
      } else if (warp == 1) {
        if (leader) {
            uint32_t s_lo = desc_lo(smem0, false), full = full0, empty = empty0, ph = 0;
            uint32_t g = 0, buf = 0;
            bool ok = true;
            for (int item = cl; ok && item < items; item += C) {
                int k, i, j;
                tiles.at(item, k, i, j);
                const int a_turn = turn(i, a_sym), b_turn = b_cols ? 0 : turn(j, b_sym);
                int lo = lo_count(i);
                uint32_t acc = 0;
                for (int kb = lo ? lo_from(i) : kb0; kb < kb1;) {
                    if (acc == 0) {                                 // a chunk begins
                        buf = g & 1u;
                        ok = warp_wait(acc_empty0 + 8 * buf, ((g >> 1) & 1u) ^ 1u, status, 4);
                        if (!ok) break;
                        g++;
                    }
                    const uint32_t tacc = tmem + buf * (TMEM_COLS / 2);
                    ok = warp_wait(full, ph, status, 2);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const bool a_t = kb >= a_turn, b_t = kb >= b_turn;
                    const uint32_t idesc = instr_desc(MMA, MMA, a_t, b_t);
                    const uint32_t at = a_t ? (8192u >> 4) << 16 : 0u, bt = b_t ? (8192u >> 4) << 16 : 0u;
                    const uint32_t ah = s_lo | at, bh = (s_lo + (PLANES * TILE >> 4)) | bt;
                    // sixteen of K further: 32 bytes along a row, or sixteen rows
                    const uint32_t ak = a_t ? 2048 >> 4 : 32 >> 4, bk = b_t ? 2048 >> 4 : 32 >> 4;
                    // two planes: the small products first. The tensor core truncates what it adds to a sum
                    // to the sum's last bit, so adds to a sum that is still small cost less.
                    const uint32_t al = ah + (TILE >> 4), bl = bh + (TILE >> 4);
                    const int next = lo && --lo == 0 ? kb0 : kb + 1;
                    const bool ends = next == kb1 || (PLANES == 2 && chunk_ends(kb, RUN, i * DIAG, DIAG, a_sym));
                    if (elected()) {
                        if constexpr (PLANES == 2 && SIDE != 64) {
#pragma unroll
                            for (int kk = 0; kk < BK / 16; kk++) {
                                umma<PAIR>(tacc, desc(al + kk * ak), desc(bh + kk * bk), idesc, kk ? 1u : acc);
                                umma<PAIR>(tacc, desc(ah + kk * ak), desc(bl + kk * bk), idesc, 1u);
                            }
                        }
#pragma unroll
                        for (int kk = 0; kk < BK / 16; kk++)
                            umma<PAIR>(FINE ? tacc + (uint32_t)(kk / 2 * MMA) : tacc, desc(ah + kk * ak), desc(bh + kk * bk), idesc,
                                       (PLANES == 2 && SIDE != 64) || (FINE ? kk & 1 : kk) ? 1u : acc);
                        commit<PAIR>(empty, first);
                        if (ends) commit<PAIR>(acc_full0 + 8 * buf, first);
                    }
                    __syncwarp();
                    acc = ends ? 0u : 1u;
                    kb = next;
                    s_lo += STAGE >> 4; full += 8; empty += 8;
                    if (full == full0 + 8 * STAGES) { s_lo = desc_lo(smem0, false); full = full0; empty = empty0; ph ^= 1u; }
                }
            }
        }
        __syncwarp();
      }
      if (split > 1) cluster_sync_all();                            // the meeting of the epilogue warps
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int e = warp - 4, q = warp & 3, h = e >> 2;
        const uint32_t acc_empty = PAIR ? map_to_cta(acc_empty0, first) : acc_empty0;
        const uint32_t staging = smem0 + OPERAND_BYTES;
        const bool issuer = e == 0 && lane == 0;      // of the 64-tiles' stores
        uint32_t g = 0;
        bool ok = true;
        if constexpr (SIDE == 64) {
            // The quarters of the product meet in shared memory; then each warp has 32 rows x 16 columns of the tile.
            const uint32_t quarters = smem0 + OPERAND_BYTES_64, box = quarters + QUARTERS_64;
            const int r = (e & 1) * 32 + lane, c16 = e >> 1;
            for (int item = cl; ok && item < items; item += C) {
                int k, i, j;
                tiles.at(item, k, i, j);
                if (p.mode == ORTH_RESULT && p.keep != 0.f && part == 0) prefetch_result(p, lane, k, i * 64 + (e & 1) * 32, j * 64 + c16 * 16, 16);
                if constexpr (PLANES == 1) {
                    // 64 rows: 16 lanes of each quarter of tensor memory; this warp's half of the columns
                    const uint32_t buf = g & 1u;
                    ok = warp_wait(acc_full0 + 8 * buf, (g >> 1) & 1u, status, 3);
                    g++;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    uint32_t x[32];
                    tmem_ld32(tmem + ((uint32_t)(q * 32) << 16) + buf * (uint32_t)MMA + (uint32_t)(h * 32), x);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(acc_empty + 8 * buf);
                    if (lane < 16) put_quarter(quarters, x, q * 16 + lane, h * 8);
                } else {
                    // Rows of hi (q 0, 1) or lo, columns of hi or lo. Warps of hi rows have the columns of one of them (h); of the
                    // lo rows each has half the columns of both, lo.hi and the small lo.lo, which it adds up.
                    const uint32_t mine = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(q < 2 ? h * 64 : h * 32), more = q < 2 ? 32u : 64u;
                    float acc[64];
#pragma unroll
                    for (int c = 0; c < 64; c++) acc[c] = 0.f;
                    for (int kb = kb0; kb < kb1; kb++) {
                        if (kb + 1 < kb1 && !chunk_ends(kb, RUN, i * DIAG, DIAG, a_sym)) continue;
                        const uint32_t buf = g & 1u;
                        ok = ok && warp_wait(acc_full0 + 8 * buf, (g >> 1) & 1u, status, 3);
                        if (!ok) break;
                        g++;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                        for (int half = 0; half < 2; half++) {
                            uint32_t x[2][32];
                            tmem_ld32(mine + buf * (TMEM_COLS / 2) + (uint32_t)(half * MMA), x[0]);
                            tmem_ld32(mine + buf * (TMEM_COLS / 2) + (uint32_t)(half * MMA) + more, x[1]);
                            asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                            for (int c = 0; c < 32; c++) acc[c] = __fadd_rn(acc[c], __uint_as_float(x[0][c]));
                            if (q < 2) {
#pragma unroll
                                for (int c = 0; c < 32; c++) acc[32 + c] = __fadd_rn(acc[32 + c], __uint_as_float(x[1][c]));
                            } else {
#pragma unroll
                                for (int c = 0; c < 32; c++) acc[c] = __fadd_rn(acc[c], __uint_as_float(x[1][c]));
                            }
                        }
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(acc_empty + 8 * buf);
                    }
                    uint32_t x[2][32];
#pragma unroll
                    for (int c = 0; c < 32; c++) { x[0][c] = __float_as_uint(acc[c]); x[1][c] = __float_as_uint(acc[32 + c]); }
                    put_quarter(quarters + (q < 2 ? h : 2) * 16384u, x[0], (q & 1) * 32 + lane, q < 2 ? 0 : h * 8);
                    if (q < 2) put_quarter(quarters + h * 16384u, x[1], (q & 1) * 32 + lane, 8);
                }
                const int stop = gave_up(p);
                ok = all_ok<256>(1, ok);
                float v[16];
#pragma unroll
                for (int u = 0; u < 4; u++) {
                    const uint32_t at = quarters + (uint32_t)(r * 256 + ((c16 * 4 + u) ^ (r & 7)) * 16);
                    uint4 x = lds(at);
                    v[4 * u] = __uint_as_float(x.x); v[4 * u + 1] = __uint_as_float(x.y); v[4 * u + 2] = __uint_as_float(x.z); v[4 * u + 3] = __uint_as_float(x.w);
                    if constexpr (PLANES == 2) {
                        const uint4 y = lds(at + 16384u), z = lds(at + 32768u);
                        v[4 * u] += __uint_as_float(y.x) + __uint_as_float(z.x); v[4 * u + 1] += __uint_as_float(y.y) + __uint_as_float(z.y);
                        v[4 * u + 2] += __uint_as_float(y.z) + __uint_as_float(z.z); v[4 * u + 3] += __uint_as_float(y.w) + __uint_as_float(z.w);
                    }
                }
                if (split > 1) {        // part 0 has the tile; the others' sums: [part][warp][4 columns][lane][4]
                    float *const to = p.sums + ((size_t)(cl * split + part) * 8 + e) * 512 + lane * 4;
                    if (part != 0) {
#pragma unroll
                        for (int u = 0; u < 4; u++) __stcg(reinterpret_cast<float4 *>(to + u * 128), make_float4(v[4 * u], v[4 * u + 1], v[4 * u + 2], v[4 * u + 3]));
                    }
                    cluster_sync_all();
                    if (part != 0) continue;
                    for (int from = 1; from < split; from++) {
#pragma unroll
                        for (int u = 0; u < 4; u++) {
                            const float4 x = __ldcg(reinterpret_cast<const float4 *>(to + (size_t)from * 4096 + u * 128));
                            v[4 * u] += x.x; v[4 * u + 1] += x.y; v[4 * u + 2] += x.z; v[4 * u + 3] += x.w;
                        }
                    }
                }
#pragma unroll
                for (int c = 0; c < 16; c++) v[c] *= p.alpha;
                if (!ok) break;
                if (p.mode == ORTH_RESULT) {
                    team_sync<256>(1);          // every warp has read the quarters
#pragma unroll
                    for (int c = 0; c < 16; c++)
                        asm volatile("st.shared.f32 [%0], %1;" ::"r"(quarters + (uint32_t)(r * 65 + c16 * 16 + c) * 4), "f"(v[c]) : "memory");
                    team_sync<256>(1);
                    if (!__any_sync(0xffffffffu, stop)) store_result_64(p, quarters, (int)threadIdx.x - 128, k, i * 64, j * 64);
                    team_sync<256>(1);
                    continue;
                }
                if (tiles.sym && i == j) {
#pragma unroll
                    for (int c = 0; c < 16; c++) v[c] += r == c16 * 16 + c ? p.diag : 0.f;
                }
                uint32_t hi[8], lo[8];
#pragma unroll
                for (int c = 0; c < 8; c++) {
                    const __half2 x = __floats2half2_rn(v[2 * c], v[2 * c + 1]);
                    const float2 f = __half22float2(x);
                    const __half2 y = __floats2half2_rn(v[2 * c] - f.x, v[2 * c + 1] - f.y);
                    hi[c] = *reinterpret_cast<const uint32_t *>(&x);
                    lo[c] = *reinterpret_cast<const uint32_t *>(&y);
                }
                if (issuer) asm volatile("cp.async.bulk.wait_group.read 0;" ::: "memory");      // the boxes' last content has left
                team_sync<256>(1);
                put_box(box, hi, r, c16 * 2);
                if (p.lo) put_box(box + 8192u, lo, r, c16 * 2);
                asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                team_sync<256>(1);
                if (issuer) {
                    tma_store(&o_hi, box, j * 64, i * 64, k);
                    if (p.lo) tma_store(&o_lo, box + 8192u, j * 64, i * 64, k);
                }
            }
        } else {
        for (int item = cl; ok && item < items; item += C) {
            int k, i, j;
            tiles.at(item, k, i, j);
            const int row0 = i * SIDE + (int)rank * 128 + q * 32, col0 = j * SIDE + h * HALF;
            if (p.mode == ORTH_RESULT && p.keep != 0.f) prefetch_result(p, lane, k, row0, col0, HALF);
            const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(h * HALF);
            uint32_t buf = g & 1u;
            // the first piece of 32 columns this part owns. One plane: its weights a piece ahead; two planes, where the sums
            // need the registers: half of them at a time, when they are needed.
            constexpr int PIECES = HALF / 32;
            const int piece0 = h * PIECES, own0 = (part + 8 * split - piece0) % split;
            uint32_t w[PLANES == 1 ? 32 : 1];
            const auto weights = [&](int cc) {
                if (p.mode == ORTH_RESULT && cc < PIECES) fetch_weights(p, w, 0, lane, k, row0, col0 + cc * 32);
            };
            if constexpr (PLANES == 1) {
                weights(own0);
                ok = __all_sync(0xffffffffu, mbar_wait(acc_full0 + 8 * buf, (g >> 1) & 1u, status, 3));
                g++;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            } else {
                // the chunks' sums in registers; the total goes back to tensor memory in place of the last chunk, so
                // that the epilogue below holds 32 columns at a time (with all of them in registers it
                // spilled, and beside 225 KB of shared memory there is no first-level cache to spill to)
                float acc[HALF];
#pragma unroll
                for (int c = 0; c < HALF; c++) acc[c] = 0.f;
                for (int kb = kb0; kb < kb1; kb++) {
                    if (kb + 1 < kb1 && !chunk_ends(kb, RUN, i * DIAG, DIAG, a_sym)) continue;
                    buf = g & 1u;
                    ok = __all_sync(0xffffffffu, ok && mbar_wait(acc_full0 + 8 * buf, (g >> 1) & 1u, status, 3));
                    if (!ok) break;
                    g++;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (int cc = 0; cc < HALF / 16; cc++) {
                        uint32_t r[16];
                        tmem_ld16(lanes + buf * (uint32_t)SIDE + (uint32_t)(cc * 16), r);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int c = 0; c < 16; c++) acc[cc * 16 + c] = __fadd_rn(acc[cc * 16 + c], __uint_as_float(r[c]));
                    }
                    if (kb + 1 == kb1) {
#pragma unroll
                        for (int cc = 0; cc < HALF / 32; cc++) tmem_st32(lanes + buf * (uint32_t)SIDE + (uint32_t)(cc * 32), acc + cc * 32);
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    } else {
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(acc_empty + 8 * buf);
                    }
                }
            }
            const int stop = gave_up(p);
            // where this warp's sums lie when parts meet: [part][CTA][warp][4 columns][lane][4]
            constexpr size_t WARP_SUMS = 32 * HALF, part_step = (size_t)CTAS * 8 * WARP_SUMS;
            const size_t sums_at = (((size_t)cl * split * CTAS + rank) * 8 + e) * WARP_SUMS + lane * 4;
            if (split > 1) {
#pragma unroll 1
                for (int cc = 0; ok && cc < HALF / 32; cc++) {
                    if ((piece0 + cc) % split == part) continue;
                    uint32_t r[32];
                    tmem_ld32(lanes + buf * (uint32_t)SIDE + (uint32_t)(cc * 32), r);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    float *const to = p.sums + sums_at + part * part_step + cc * 1024;
#pragma unroll
                    for (int u = 0; u < 8; u++)
                        __stcg(reinterpret_cast<float4 *>(to + u * 128), make_float4(__uint_as_float(r[4 * u]), __uint_as_float(r[4 * u + 1]),
                                                                                   __uint_as_float(r[4 * u + 2]), __uint_as_float(r[4 * u + 3])));
                }
                cluster_sync_all();
            }
            // Planes are stored from registers: a piece is 64 bytes of a row. (Through 64 x 64 boxes in shared memory and TMA it took
            // as long, with two barriers a box; and the code, a piece long, is fetched once instead of unrolled: the first
            // pass over it costs a microsecond of each product.)
#pragma unroll 1
            for (int cc = own0; ok && cc < PIECES; cc += split) {
                const int col = col0 + cc * 32;
                if (row0 >= p.rows || col >= p.cols) break;
                uint32_t r[32];
                tmem_ld32(lanes + buf * (uint32_t)SIDE + (uint32_t)(cc * 32), r);
                asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                float v[32];
#pragma unroll
                for (int c = 0; c < 32; c++) v[c] = __uint_as_float(r[c]);
                // the other parts' sums, two at a time so that their loads wait together, always from the next part on
                for (int n = 1; n < split; n += 2) {
                    const int from[2] = { part + n < split ? part + n : part + n - split, part + n + 1 < split ? part + n + 1 : part + n + 1 - split };
                    float4 x[2][8];
#pragma unroll
                    for (int o = 0; o < 2; o++) {
                        const float *const at = p.sums + sums_at + from[o] * part_step + cc * 1024;
#pragma unroll
                        for (int u = 0; u < 8; u++)
                            x[o][u] = n + o < split ? __ldcg(reinterpret_cast<const float4 *>(at + u * 128)) : make_float4(0.f, 0.f, 0.f, 0.f);
                    }
#pragma unroll
                    for (int u = 0; u < 8; u++) {
                        v[4 * u] += x[0][u].x + x[1][u].x; v[4 * u + 1] += x[0][u].y + x[1][u].y;
                        v[4 * u + 2] += x[0][u].z + x[1][u].z; v[4 * u + 3] += x[0][u].w + x[1][u].w;
                    }
                }
#pragma unroll
                for (int c = 0; c < 32; c++) v[c] *= p.alpha;
                if (p.mode == ORTH_RESULT) {
                    const uint32_t own = staging + (uint32_t)e * 4096u;
                    if (!p.tall) put_result(v, own, lane);
                    if constexpr (PLANES == 1) {
                        if (!__any_sync(0xffffffffu, stop)) store_result<32, 0>(p, v, w, own, lane, k, row0, col);
                        weights(cc + split);
                    } else if (!__any_sync(0xffffffffu, stop)) {
                        uint32_t x[16];
                        fetch_weights(p, x, 0, lane, k, row0, col);
                        store_result<16, 0>(p, v, x, own, lane, k, row0, col);
                        fetch_weights(p, x, 16, lane, k, row0, col);
                        store_result<16, 16>(p, v, x, own, lane, k, row0, col);
                    }
                    continue;
                }
                if (tiles.sym && i == j) {
#pragma unroll
                    for (int c = 0; c < 32; c++) v[c] += row0 + lane == col + c ? p.diag : 0.f;
                }
                const bool live = row0 + lane < p.rows;
                const long long at = (k * p.out_plane + (row0 + lane) * p.out_pitch + col) * 2;
                uint32_t y[16];
#pragma unroll
                for (int c = 0; c < 16; c++) {
                    const __half2 x = __floats2half2_rn(v[2 * c], v[2 * c + 1]);
                    const float2 f = __half22float2(x);
                    y[c] = *reinterpret_cast<const uint32_t *>(&x);
                    v[2 * c] -= f.x; v[2 * c + 1] -= f.y;
                }
                if (live) put_row(static_cast<char *>(p.out_hi) + at, y);
                if (p.lo) {
#pragma unroll
                    for (int c = 0; c < 16; c++) {
                        const __half2 x = __floats2half2_rn(v[2 * c], v[2 * c + 1]);
                        y[c] = *reinterpret_cast<const uint32_t *>(&x);
                    }
                    if (live) put_row(static_cast<char *>(p.out_lo) + at, y);
                }
                __syncwarp();
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc_empty + 8 * buf);
        }
        }
        if (issuer) asm volatile("cp.async.bulk.wait_group 0;" ::: "memory");
        if (!ok) {      // a wait ran out: the host hears of it; copies that may still be in flight land before the shared memory is released
            if (lane == 0) {
                __threadfence_system();         // behind the status word
                asm volatile("st.relaxed.sys.global.b32 [%0], %1;" ::"l"(p.told), "r"(1) : "memory");
            }
            for (int n = 0; n < 64; n++) __nanosleep(4000);
        }
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if constexpr (PAIR) cluster_sync_all();         // nobody frees or exits while the peer may still signal or read
    if (warp == 1) {
        if constexpr (PAIR) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
        else asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(TMEM_COLS) : "memory");
    }
}

}  // namespace orth

// launched in clusters of split CTAs, the 256 forms of 2 x split
#define ORTH_PRODUCT(name, PLANES, SIDE)                                                                                             \
    extern "C" __global__ void __launch_bounds__(384, 1)                                                                             \
    name(const __grid_constant__ CUtensorMap a_hi, const __grid_constant__ CUtensorMap a_lo, const __grid_constant__ CUtensorMap b_hi, \
         const __grid_constant__ CUtensorMap b_lo, const __grid_constant__ CUtensorMap o_hi, const __grid_constant__ CUtensorMap o_lo, \
         const __grid_constant__ orth::Product p)                                                                                    \
    { orth::product<PLANES, SIDE>(a_hi, a_lo, b_hi, b_lo, o_hi, o_lo, p); }
ORTH_PRODUCT(orth_product_1_64, 1, 64)
ORTH_PRODUCT(orth_product_2_64, 2, 64)
ORTH_PRODUCT(orth_product_1_128, 1, 128)
ORTH_PRODUCT(orth_product_2_128, 2, 128)
ORTH_PRODUCT(orth_product_1_256, 1, 256)
ORTH_PRODUCT(orth_product_2_256, 2, 256)
