// orthogonal.cu -- Newton-Schulz orthogonalisation of a matrix on the tensor cores.
//
//     X = G / (|G|_F + eps);   steps times:  A = X X^t,  P = b A + c A A,  X = a X + P X
//
// drives the singular values of X towards one (the Muon optimiser's update). X is
// s x l with s <= l: a tall G is transposed on the way in and on the way out. All
// three products run on fp16 operands with fp32 accumulation (tcgen05 kind::f16),
// which hold 11 bits where bf16 holds 8 at the same rate. X and A are kept times 2^14
// and P times a power of two that its coefficients allow: singular values stay
// below 2, so the scaled entries fit fp16, and small entries stay above its
// subnormal range.
//
// Precision, by the type of the result:
//   two planes (f32, f16 results): every operand is hi + lo = fp16(x) + fp16(x - hi), 22
//     bits, and a product is lo.hi + hi.lo + hi.hi; K is cut into chunks of 128 whose sums
//     leave the tensor core (it adds with truncation, so a long sum drifts) and are
//     added round-to-nearest in registers. As exact as an fp32 iteration or better.
//   one plane (bf16 results): products use the hi parts only, a third of the work. X
//     still keeps hi + lo for the term a X: the iteration multiplies what small singular
//     values lose by up to a^steps = 485, so rounding X to 11 bits each step showed as 2 to
//     4 % on matrices of low rank, while rounding only the products' operands leaves 1e-3.
//
// A and P are symmetric: only tiles on and below the diagonal are computed and stored.
// Where a product needs a block above the diagonal it loads the mirrored block and has the
// tensor core take it transposed (an operand may have either index contiguous), so nothing
// is stored twice: with 2-byte transposed stores the epilogue of a 1024 x 1024
// product took 12 of its 27 us.
//
// Launches per call: orth_norm (sums of squares; Muon: also the momentum), orth_split (planes of
// the normalised, possibly transposed matrix), then steps x 3 products. A product kernel
// keeps one CTA or CTA pair per SM (pair) and walks over the tiles of all matrices of
// the batch; the roles inside are those of the fp32 GEMM: warp 0 TMA, warp 1 MMA, warps 4-11
// drain tensor memory and apply the epilogue.
//   pair:   256 x 256 tile per two CTAs, tcgen05.mma.cta_group::2
//   single: 128 x 128 tile per CTA, for matrices with too few tiles of the other size
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

__device__ __forceinline__ float load1(const void *p, int type, long long i)
{
    if (type == ORTH_F32) return static_cast<const float *>(p)[i];
    if (type == ORTH_BF16) return __bfloat162float(static_cast<const __nv_bfloat16 *>(p)[i]);
    return __half2float(static_cast<const __half *>(p)[i]);
}
__device__ __forceinline__ void store1(void *p, int type, long long i, float v)
{
    if (type == ORTH_F32) static_cast<float *>(p)[i] = v;
    else if (type == ORTH_BF16) static_cast<__nv_bfloat16 *>(p)[i] = __float2bfloat16_rn(v);
    else static_cast<__half *>(p)[i] = __float2half_rn(v);
}
// Four neighbouring elements; p + i is aligned to four elements.
__device__ __forceinline__ float4 load4(const void *p, int type, long long i)
{
    if (type == ORTH_F32) return *reinterpret_cast<const float4 *>(static_cast<const float *>(p) + i);
    const uint2 r = *reinterpret_cast<const uint2 *>(static_cast<const uint16_t *>(p) + i);
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

__device__ __forceinline__ float4 source4(const Source &s, int k, int r, int c)
{
    const float4 g = load4(s.g, s.type_g, k * s.stride_g + r * s.ld_g + c);
    if (!s.m) return g;
    const float4 m = load4(s.m, s.type_m, k * s.stride_m + r * s.ld_m + c);
    return make_float4(update_of(m.x, g.x, s), update_of(m.y, g.y, s), update_of(m.z, g.z, s), update_of(m.w, g.w, s));
}
__device__ __forceinline__ float source1(const Source &s, int k, int r, int c)
{
    const float g = load1(s.g, s.type_g, k * s.stride_g + r * s.ld_g + c);
    return s.m ? update_of(load1(s.m, s.type_m, k * s.stride_m + r * s.ld_m + c), g, s) : g;
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
    const int k = (int)blockIdx.y;
    const int w = s.vec ? 4 : 1, per_row = s.cols / w;
    const long long total = (long long)s.rows * per_row;
    double sum = 0.0;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < total; i += (long long)gridDim.x * 256) {
        const int r = (int)(i / per_row), c = (int)(i - (long long)r * per_row) * w;
        if (s.vec) {
            float4 u = load4(s.g, s.type_g, k * s.stride_g + r * s.ld_g + c);
            if (s.m) {
                const long long at = k * s.stride_m + r * s.ld_m + c;
                float4 m = load4(s.m, s.type_m, at);
                m = make_float4(lerp(m.x, u.x, s.mu), lerp(m.y, u.y, s.mu), lerp(m.z, u.z, s.mu), lerp(m.w, u.w, s.mu));
                store4(s.m, s.type_m, at, m);
                u = source4(s, k, r, c);
            }
            sum += ((double)u.x * u.x + (double)u.y * u.y) + ((double)u.z * u.z + (double)u.w * u.w);
        } else {
            float u = load1(s.g, s.type_g, k * s.stride_g + r * s.ld_g + c);
            if (s.m) {
                const long long at = k * s.stride_m + r * s.ld_m + c;
                store1(s.m, s.type_m, at, lerp(load1(s.m, s.type_m, at), u, s.mu));
                u = source1(s, k, r, c);
            }
            sum += (double)u * u;
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
// when the matrix is tall. One 64 x 64 tile of u a block through shared memory; grid
// (column tiles, row tiles, matrices).
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
    if (threadIdx.x < 32) {
        double sum = 0.0;
        for (int i = (int)threadIdx.x; i < parts; i += 32) sum += partial[(size_t)k * parts + i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (threadIdx.x == 0) s_scale = (float)fmin((double)X_SCALE / (sqrt(sum) + (double)eps), 3.4e38);
    }
    const int tx = (int)threadIdx.x & 15, ty = (int)threadIdx.x >> 4;
#pragma unroll
    for (int p = 0; p < 4; p++) {
        const int r = r0 + ty + 16 * p, c = c0 + 4 * tx;
        float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
        if (r < s.rows) {
            if (s.vec && c < s.cols) v = source4(s, k, r, c);
            else {
                if (c + 0 < s.cols) v.x = source1(s, k, r, c);
                if (c + 1 < s.cols) v.y = source1(s, k, r, c + 1);
                if (c + 2 < s.cols) v.z = source1(s, k, r, c + 2);
                if (c + 3 < s.cols) v.w = source1(s, k, r, c + 3);
            }
        }
        float *t = &tile[ty + 16 * p][4 * tx];
        t[0] = v.x; t[1] = v.y; t[2] = v.z; t[3] = v.w;
    }
    __syncthreads();
    const float f = s_scale;
    __half *ph = hi + k * plane, *pl = lo + k * plane;
#pragma unroll
    for (int p = 0; p < 4; p++) {
        // row (of the plane) a, four columns from b; the pitch is a multiple of 64, so a whole group is in the plane
        const int a = ty + 16 * p, b = 4 * tx;
        const int row = (tall ? c0 : r0) + a, col = (tall ? r0 : c0) + b;
        if (row < (tall ? s.cols : s.rows) && col < (tall ? s.rows : s.cols)) {
            __half h[4], l[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float v = f * (tall ? tile[b + e][a] : tile[a][b + e]);
                h[e] = __float2half_rn(v);
                l[e] = __float2half_rn(v - __half2float(h[e]));
            }
            *reinterpret_cast<uint2 *>(ph + row * pitch + col) = *reinterpret_cast<const uint2 *>(h);
            *reinterpret_cast<uint2 *>(pl + row * pitch + col) = *reinterpret_cast<const uint2 *>(l);
        }
    }
}

namespace orth {

__device__ __forceinline__ void tma_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z)
{
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}
__device__ __forceinline__ void tma_3d_pair(uint32_t dst, const CUtensorMap *map, uint32_t bar, int x, int y, int z)
{
    asm volatile("cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
                 ::"r"(dst), "l"(map), "r"(bar), "r"(x), "r"(y), "r"(z) : "memory");
}

// fp16 x fp16 -> fp32; bits 15 and 16: the first or second operand's tile has its rows (columns), not K, contiguous.
__device__ __forceinline__ uint32_t instr_desc(int m, int n, bool a_t, bool b_t)
{
    return (1u << 4) | ((uint32_t)a_t << 15) | ((uint32_t)b_t << 16) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}
// A tile of two 64 x 64 boxes, 128 bytes a box row, 128-byte swizzle, 8 rows 1024 bytes. K
// contiguous (`t` false): rows of the operand, the boxes one below the other. Else rows of K, each with 64
// rows of the operand; the next 64 lie 8192 bytes on.
__device__ __forceinline__ uint64_t tile_desc(uint32_t addr, bool t)
{
    return gemm::smem_desc(addr) | (t ? (uint64_t)(8192u >> 4) << 16 : 0ull);
}
// Sixteen of K further: 32 bytes along a row, or sixteen rows.
__device__ __forceinline__ uint64_t k_advance(int kk, bool t) { return (uint64_t)(kk * (t ? 2048 >> 4 : 32 >> 4)); }

template <bool PAIR>
__device__ __forceinline__ void umma(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t accumulate)
{
    if constexpr (PAIR)
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
    else
        asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\ttcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                     ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(accumulate) : "memory");
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
template <bool PAIR> __device__ __forceinline__ void commit(uint32_t bar)
{
    if constexpr (PAIR) gemm::umma_commit_pair(bar); else gemm::umma_commit(bar);
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

// One warp's 32 x 32 piece of the product, a row a lane in v, goes out through 4 KB of shared
// memory of the warp's own, so that global accesses run along rows: a piece's row is 64 bytes of a plane
// (two sectors), where a store straight from the registers touched 32 lines at once.
// Shared layout: 16-byte units, swizzled so that neither the lane-a-row nor the along-the-row access conflicts.
struct Stage {
    uint32_t base;
    int lane;
    // 16-byte unit u of row r: planes (hi, then lo 2048 bytes on) have 4 units a row, fp32 pieces 8
    __device__ __forceinline__ uint32_t half_at(int r, int u) const { return base + (uint32_t)(r * 64 + ((u ^ (r >> 1)) & 3) * 16); }
    __device__ __forceinline__ uint32_t f32_at(int r, int u) const { return base + (uint32_t)(r * 128 + ((u ^ r) & 7) * 16); }
};
__device__ __forceinline__ void sts(uint32_t a, uint4 v) { asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory"); }
__device__ __forceinline__ uint4 lds(uint32_t a)
{
    uint4 v;
    asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}

// The piece of `in` (A or X) at rows row0.., columns col0.., read along rows into registers; zero outside the matrix.
struct Piece { uint4 hi[4], lo[4]; };
__device__ __forceinline__ void fetch(const Product &p, Piece &x, int k, int row0, int col0, int lane)
{
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const int r = row0 + q * 8 + (lane >> 2), c = col0 + (lane & 3) * 8;
        x.hi[q] = x.lo[q] = make_uint4(0, 0, 0, 0);
        if (r < p.rows && c < p.cols) {
            const long long at = k * p.plane + r * p.pitch + c;
            x.hi[q] = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const __half *>(p.in_hi) + at));
            if (p.in_lo) x.lo[q] = __ldcg(reinterpret_cast<const uint4 *>(static_cast<const __half *>(p.in_lo) + at));
        }
    }
}

__device__ __forceinline__ void put(const Piece &in, const Stage &st)
{
#pragma unroll
    for (int q = 0; q < 4; q++) {
        const uint32_t a = st.half_at(q * 8 + (st.lane >> 2), st.lane & 3);
        sts(a, in.hi[q]);
        sts(a + 2048, in.lo[q]);
    }
}

// v (32 columns of this lane's row of the accumulator) -> epilogue -> memory. The piece of `in` is in the stage.
__device__ __forceinline__ void emit(const Product &p, float (&v)[32], const Stage &st, int k, int row0, int col0)
{
    const int lane = st.lane, row = row0 + lane;
#pragma unroll
    for (int j = 0; j < 32; j++) v[j] *= p.alpha;
    if (p.mode != ORTH_GRAM) {
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const uint32_t a = st.half_at(lane, q);
            const uint4 h = lds(a), l = lds(a + 2048);
            const __half2 *h2 = reinterpret_cast<const __half2 *>(&h), *l2 = reinterpret_cast<const __half2 *>(&l);
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const float2 x = __half22float2(h2[e]), y = __half22float2(l2[e]);
                v[8 * q + 2 * e] = fmaf(p.beta, x.x + y.x, v[8 * q + 2 * e]);
                v[8 * q + 2 * e + 1] = fmaf(p.beta, x.y + y.y, v[8 * q + 2 * e + 1]);
            }
        }
        __syncwarp();
    }
    if (p.mode != ORTH_RESULT) {
        // planes: the pitch is a multiple of 64 columns, so a unit of eight that begins inside the matrix lies inside the plane
#pragma unroll
        for (int q = 0; q < 4; q++) {
            __half2 h[4], l[4];
#pragma unroll
            for (int e = 0; e < 4; e++) {
                h[e] = __floats2half2_rn(v[8 * q + 2 * e], v[8 * q + 2 * e + 1]);
                const float2 f = __half22float2(h[e]);
                l[e] = __floats2half2_rn(v[8 * q + 2 * e] - f.x, v[8 * q + 2 * e + 1] - f.y);
            }
            const uint32_t a = st.half_at(lane, q);
            sts(a, *reinterpret_cast<const uint4 *>(h));
            sts(a + 2048, *reinterpret_cast<const uint4 *>(l));
        }
        __syncwarp();
#pragma unroll
        for (int q = 0; q < 4; q++) {
            const int r = q * 8 + (lane >> 2), u = lane & 3;
            if (row0 + r < p.rows && col0 + u * 8 < p.cols) {
                const long long at = k * p.plane + (row0 + r) * p.pitch + col0 + u * 8;
                const uint32_t a = st.half_at(r, u);
                *reinterpret_cast<uint4 *>(static_cast<__half *>(p.out_hi) + at) = lds(a);
                if (p.out_lo) *reinterpret_cast<uint4 *>(static_cast<__half *>(p.out_lo) + at) = lds(a + 2048);
            }
        }
        __syncwarp();
        return;
    }
    if (p.tall) {
        // neighbouring lanes hold neighbouring rows: a column is a contiguous run of the caller's row. Loads ahead of stores.
#pragma unroll
        for (int j0 = 0; j0 < 32; j0 += 8) {
            const long long o = k * p.stride_w + (long long)(col0 + j0) * p.ld_w + row;
            if (p.keep != 0.f) {
                float w[8];
#pragma unroll
                for (int j = 0; j < 8; j++) w[j] = row < p.rows && col0 + j0 + j < p.cols ? load1(p.w, p.type_w, o + j * p.ld_w) : 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) v[j0 + j] = fmaf(p.keep, w[j], v[j0 + j]);
            }
#pragma unroll
            for (int j = 0; j < 8; j++)
                if (row < p.rows && col0 + j0 + j < p.cols) store1(p.w, p.type_w, o + j * p.ld_w, v[j0 + j]);
        }
        return;
    }
#pragma unroll
    for (int u = 0; u < 8; u++)
        sts(st.f32_at(lane, u), make_uint4(__float_as_uint(v[4 * u]), __float_as_uint(v[4 * u + 1]), __float_as_uint(v[4 * u + 2]), __float_as_uint(v[4 * u + 3])));
    __syncwarp();
    if (p.vec_w) {
        const int u = lane & 7, r0 = lane >> 3, c = col0 + 4 * u;
#pragma unroll 1
        for (int q0 = 0; q0 < 8; q0 += 4) {
            const long long o = k * p.stride_w + (row0 + r0 + 4 * q0) * p.ld_w + c;
            float4 w[4];
#pragma unroll
            for (int q = 0; q < 4; q++) {
                w[q] = make_float4(0.f, 0.f, 0.f, 0.f);
                if (p.keep != 0.f && row0 + r0 + 4 * (q0 + q) < p.rows && c < p.cols) w[q] = load4(p.w, p.type_w, o + 4 * q * p.ld_w);
            }
#pragma unroll
            for (int q = 0; q < 4; q++)
                if (row0 + r0 + 4 * (q0 + q) < p.rows && c < p.cols) {
                    const uint4 x = lds(st.f32_at(r0 + 4 * (q0 + q), u));
                    store4(p.w, p.type_w, o + 4 * q * p.ld_w, make_float4(fmaf(p.keep, w[q].x, __uint_as_float(x.x)), fmaf(p.keep, w[q].y, __uint_as_float(x.y)),
                                                                         fmaf(p.keep, w[q].z, __uint_as_float(x.z)), fmaf(p.keep, w[q].w, __uint_as_float(x.w))));
                }
        }
    } else {
        // a column a lane, eight rows at a time
        const int c = col0 + lane;
#pragma unroll 1
        for (int q0 = 0; q0 < 32; q0 += 8) {
            const long long o = k * p.stride_w + (row0 + q0) * p.ld_w + c;
            float w[8];
#pragma unroll
            for (int q = 0; q < 8; q++) w[q] = p.keep != 0.f && row0 + q0 + q < p.rows && c < p.cols ? load1(p.w, p.type_w, o + q * p.ld_w) : 0.f;
#pragma unroll
            for (int q = 0; q < 8; q++) {
                float x;
                asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(st.f32_at(q0 + q, lane >> 2) + (uint32_t)(lane & 3) * 4) : "memory");
                if (row0 + q0 + q < p.rows && c < p.cols) store1(p.w, p.type_w, o + q * p.ld_w, fmaf(p.keep, w[q], x));
            }
        }
    }
    __syncwarp();
}

// 384 threads; grid: any number of CTAs (pairs), each takes every grid-th tile.
template <int PLANES, bool PAIR>
__device__ __forceinline__ void product(const CUtensorMap &a_hi, const CUtensorMap &a_lo, const CUtensorMap &b_hi, const CUtensorMap &b_lo, const Product &p)
{
    using namespace gemm;
    constexpr int BK = 64, SIDE = PAIR ? 256 : 128;                 // K block; tile side
    constexpr uint32_t TILE = 128 * BK * 2;                         // one operand plane of one CTA: 16 KB
    constexpr uint32_t STAGE = 2 * PLANES * TILE;
    constexpr int STAGES = 6 / PLANES;
    constexpr int CHUNK_KB = PLANES == 2 ? 2 : 1 << 30;             // K blocks per accumulation in tensor memory
    constexpr int HALF = SIDE / 2;                                  // columns per epilogue warp
    constexpr uint32_t TMEM_COLS = 2 * SIDE;                        // two accumulators
    const WaitCtl status = { p.status, p.wait_ns };

    extern __shared__ uint8_t smem_orth[];
    __shared__ __align__(8) uint64_t bars[2 * STAGES + 4];
    __shared__ uint32_t s_tmem;

    const uint32_t rank = PAIR ? cluster_ctarank() : 0;
    const bool leader = rank == 0;
    const uint32_t smem0 = (smem_u32(smem_orth) + 1023u) & ~1023u;
    const uint32_t full0 = smem_u32(&bars[0]), empty0 = smem_u32(&bars[STAGES]);
    const uint32_t acc_full0 = smem_u32(&bars[2 * STAGES]), acc_empty0 = smem_u32(&bars[2 * STAGES + 2]);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int C = (int)(PAIR ? gridDim.x >> 1 : gridDim.x), cl = (int)(PAIR ? blockIdx.x >> 1 : blockIdx.x);
    const Tiles tiles(p, SIDE);
    const int items = tiles.each * p.batch;
    const int nkb = (p.K + BK - 1) / BK;
    // Which operand blocks come transposed. X as the second operand of P X has its columns contiguous. Of a
    // symmetric operand the block at K block kb is above the stored triangle when kb's tile lies beyond the tile
    // of the rows. (A pair whose triangle was stored in 128-tiles takes the rule of its upper half: for the
    // lower half that differs only inside its own diagonal tile, which is stored whole.)
    const bool a_sym = p.mode != ORTH_GRAM, b_sym = p.mode == ORTH_POLY, b_cols = p.mode >= ORTH_UPDATE;
    const int tri_shift = p.tri == 256 ? 8 : 7;

    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; s++) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
        for (int b = 0; b < 2; b++) { mbar_init(acc_full0 + 8 * b, 1); mbar_init(acc_empty0 + 8 * b, PAIR ? 16 : 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (threadIdx.x == 32) {        // the descriptors, while the kernel before still runs
        asm volatile("prefetch.tensormap [%0];" ::"l"(&a_hi) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&b_hi) : "memory");
        if constexpr (PLANES == 2) {
            asm volatile("prefetch.tensormap [%0];" ::"l"(&a_lo) : "memory");
            asm volatile("prefetch.tensormap [%0];" ::"l"(&b_lo) : "memory");
        }
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
        if (lane == 0) {
            uint32_t it = 0;
            bool ok = true;
            for (int item = cl; ok && item < items; item += C) {
                int k, i, j;
                tiles.at(item, k, i, j);
                const int m0 = i * SIDE + (int)rank * 128, n0 = j * SIDE + (int)rank * 128;
                const int ti = (i * SIDE) >> tri_shift, tj = (j * SIDE) >> tri_shift;
                for (int kb = 0; kb < nkb; kb++, it++) {
                    const uint32_t s = it % STAGES, ph = (it / STAGES) & 1u;
                    if (!mbar_wait(empty0 + 8 * s, ph ^ 1u, status, 1)) { ok = false; break; }
                    const uint32_t st = smem0 + s * STAGE;
                    uint32_t bar = full0 + 8 * s;
                    if (leader) mbar_expect_tx(bar, (PAIR ? 2 : 1) * STAGE);
                    if constexpr (PAIR) bar = map_to_cta(bar, 0);
                    const int tk = (kb * BK) >> tri_shift;
                    const bool a_t = a_sym && tk > ti, b_t = b_cols || (b_sym && tk > tj);
#pragma unroll
                    for (int h = 0; h < 2; h++) {                   // 64 rows of an operand at a time
                        const uint32_t d = st + (uint32_t)h * (TILE / 2);
                        const int ax = a_t ? m0 + 64 * h : kb * BK, ay = a_t ? kb * BK : m0 + 64 * h;
                        const int bx = b_t ? n0 + 64 * h : kb * BK, by = b_t ? kb * BK : n0 + 64 * h;
                        if constexpr (PAIR) {
                            tma_3d_pair(d, &a_hi, bar, ax, ay, k);
                            tma_3d_pair(d + PLANES * TILE, &b_hi, bar, bx, by, k);
                            if constexpr (PLANES == 2) {
                                tma_3d_pair(d + TILE, &a_lo, bar, ax, ay, k);
                                tma_3d_pair(d + 3 * TILE, &b_lo, bar, bx, by, k);
                            }
                        } else {
                            tma_3d(d, &a_hi, bar, ax, ay, k);
                            tma_3d(d + PLANES * TILE, &b_hi, bar, bx, by, k);
                            if constexpr (PLANES == 2) {
                                tma_3d(d + TILE, &a_lo, bar, ax, ay, k);
                                tma_3d(d + 3 * TILE, &b_lo, bar, bx, by, k);
                            }
                        }
                    }
                }
            }
        }
        __syncwarp();
      } else if (warp == 1) {
        if (leader && lane == 0) {
            uint32_t it = 0, g = 0;
            bool ok = true;
            for (int item = cl; ok && item < items; item += C) {
                int k, i, j;
                tiles.at(item, k, i, j);
                const int ti = (i * SIDE) >> tri_shift, tj = (j * SIDE) >> tri_shift;
                for (int kb = 0; kb < nkb && ok; g++) {
                    const uint32_t buf = g & 1u;
                    ok = mbar_wait(acc_empty0 + 8 * buf, ((g >> 1) & 1u) ^ 1u, status, 4);
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t tacc = tmem + buf * (uint32_t)SIDE;
                    const int kb_end = PLANES == 2 ? min(kb + CHUNK_KB, nkb) : nkb;
                    uint32_t acc = 0;
                    for (; kb < kb_end; kb++, it++) {
                        const uint32_t s = it % STAGES, ph = (it / STAGES) & 1u;
                        ok = mbar_wait(full0 + 8 * s, ph, status, 2);
                        if (!ok) break;
                        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                        const uint32_t st = smem0 + s * STAGE;
                        const int tk = (kb * BK) >> tri_shift;
                        const bool a_t = a_sym && tk > ti, b_t = b_cols || (b_sym && tk > tj);
                        const uint32_t idesc = instr_desc(SIDE, SIDE, a_t, b_t), bt = st + PLANES * TILE;
                        const uint64_t ah = tile_desc(st, a_t), al = tile_desc(st + TILE, a_t), bh = tile_desc(bt, b_t), bl = tile_desc(bt + TILE, b_t);
                        // two planes: the small products first. The tensor core truncates what it adds to a sum
                        // to the sum's last bit, so adds to a sum that is still small cost less.
                        if constexpr (PLANES == 2) {
#pragma unroll
                            for (int kk = 0; kk < BK / 16; kk++) {
                                umma<PAIR>(tacc, al + k_advance(kk, a_t), bh + k_advance(kk, b_t), idesc, acc);
                                umma<PAIR>(tacc, ah + k_advance(kk, a_t), bl + k_advance(kk, b_t), idesc, 1u);
                                acc = 1;
                            }
                        }
#pragma unroll
                        for (int kk = 0; kk < BK / 16; kk++) {
                            umma<PAIR>(tacc, ah + k_advance(kk, a_t), bh + k_advance(kk, b_t), idesc, acc);
                            acc = 1;
                        }
                        commit<PAIR>(empty0 + 8 * s);
                    }
                    if (ok) commit<PAIR>(acc_full0 + 8 * buf);
                }
            }
        }
        __syncwarp();
      }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 208;");
        const int q = warp & 3, h = (warp - 4) >> 2;
        const uint32_t acc_empty = PAIR ? map_to_cta(acc_empty0, 0) : acc_empty0;
        const Stage stage = { smem0 + STAGES * STAGE + (uint32_t)(warp - 4) * 4096u, lane };
        uint32_t g = 0;
        bool ok = true;
        for (int item = cl; ok && item < items; item += C) {
            int k, i, j;
            tiles.at(item, k, i, j);
            const int row0 = i * SIDE + (int)rank * 128 + q * 32, col0 = j * SIDE + h * HALF;
            Piece in;
            if (p.mode != ORTH_GRAM) fetch(p, in, k, row0, col0, lane);       // lands while the products run
            const uint32_t lanes = tmem + ((uint32_t)(q * 32) << 16) + (uint32_t)(h * HALF);
            uint32_t buf = g & 1u;
            if constexpr (PLANES == 1) {
                ok = __all_sync(0xffffffffu, mbar_wait(acc_full0 + 8 * buf, (g >> 1) & 1u, status, 3));
                if (!ok) break;
                g++;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            } else {
                // the chunks' sums in registers; the total goes back to tensor memory in place of the last chunk, so
                // that the epilogue below holds 32 columns at a time (with all of them in registers it
                // spilled, and beside 225 KB of shared memory there is no first-level cache to spill to)
                float acc[HALF];
#pragma unroll
                for (int e = 0; e < HALF; e++) acc[e] = 0.f;
                for (int kb = 0; kb < nkb; kb += CHUNK_KB, g++) {
                    buf = g & 1u;
                    ok = __all_sync(0xffffffffu, ok && mbar_wait(acc_full0 + 8 * buf, (g >> 1) & 1u, status, 3));
                    if (!ok) break;
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
#pragma unroll
                    for (int cc = 0; cc < HALF / 16; cc++) {
                        uint32_t r[16];
                        tmem_ld16(lanes + buf * (uint32_t)SIDE + (uint32_t)(cc * 16), r);
                        asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                        for (int e = 0; e < 16; e++) acc[cc * 16 + e] = __fadd_rn(acc[cc * 16 + e], __uint_as_float(r[e]));
                    }
                    if (kb + CHUNK_KB >= nkb) {
#pragma unroll
                        for (int cc = 0; cc < HALF / 32; cc++) tmem_st32(lanes + buf * (uint32_t)SIDE + (uint32_t)(cc * 32), acc + cc * 32);
                        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
                    } else {
                        asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                        __syncwarp();
                        if (lane == 0) mbar_arrive_cluster(acc_empty + 8 * buf);
                    }
                }
                if (!ok) break;
            }
#pragma unroll 1
            for (int cc = 0; cc < HALF / 32; cc++) {
                if (row0 >= p.rows || col0 + cc * 32 >= p.cols) break;
                if (p.mode != ORTH_GRAM) {
                    put(in, stage);
                    if (cc + 1 < HALF / 32) fetch(p, in, k, row0, col0 + (cc + 1) * 32, lane);
                }
                float v[32];
                {
                    uint32_t r[32];
                    tmem_ld32(lanes + buf * (uint32_t)SIDE + (uint32_t)(cc * 32), r);
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
                    for (int e = 0; e < 32; e++) v[e] = __uint_as_float(r[e]);
                }
                emit(p, v, stage, k, row0, col0 + cc * 32);
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) mbar_arrive_cluster(acc_empty + 8 * buf);
        }
        if (!ok) {      // a wait ran out: copies that may still be in flight land before the shared memory is released
            for (int i = 0; i < 64; i++) __nanosleep(4000);
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

#define ORTH_PRODUCT(name, PLANES, PAIR, CLUSTER)                                                                                    \
    extern "C" __global__ void CLUSTER __launch_bounds__(384, 1)                                                                     \
    name(const __grid_constant__ CUtensorMap a_hi, const __grid_constant__ CUtensorMap a_lo, const __grid_constant__ CUtensorMap b_hi, \
         const __grid_constant__ CUtensorMap b_lo, const __grid_constant__ orth::Product p)                                           \
    { orth::product<PLANES, PAIR>(a_hi, a_lo, b_hi, b_lo, p); }
ORTH_PRODUCT(orth_product_1_single, 1, false, )
ORTH_PRODUCT(orth_product_2_single, 2, false, )
ORTH_PRODUCT(orth_product_1_pair, 1, true, __cluster_dims__(2, 1, 1))
ORTH_PRODUCT(orth_product_2_pair, 2, true, __cluster_dims__(2, 1, 1))
