// orth_params.cuh -- parameter blocks of the orthogonalisation kernels, shared by the
// kernels (orthogonal.cu) and the C host code that fills them (sm100_train.c): plain C
// layout, device addresses as typed pointers on the device and integers on the host.
#ifndef ORTH_PARAMS_CUH
#define ORTH_PARAMS_CUH
#ifdef __CUDACC__
#define ORTH_PTR(T) T *
#else
#define ORTH_PTR(T) unsigned long long
#endif

/* Element types inside the kernels. */
#define ORTH_F32  0
#define ORTH_BF16 1
#define ORTH_F16  2

/* The matrices a call reads: the gradient and, for Muon, the momentum beside it
 * (m = 0: none). Element (r, c) of matrix k lies at k * stride + r * ld + c. */
typedef struct orth_source {
    ORTH_PTR(const void) g;
    ORTH_PTR(void) m;
    long long ld_g, stride_g, ld_m, stride_m;
    int type_g, type_m, rows, cols, nesterov;
    int vec;                                            /* groups of four elements are aligned in g and m */
    int flat;                                           /* no gaps between rows in g and m */
    float mu;
} orth_source_t;

/* What a product kernel computes. */
#define ORTH_GRAM   0       /* S = X X^t + diag I */
#define ORTH_POLY   1       /* Q = alpha S S + diag I */
#define ORTH_UPDATE 2       /* X = Q X */
#define ORTH_RESULT 3       /* the same into the caller's matrix: w = keep w + value */

typedef struct orth_product {
    int mode, rows, cols, K, batch;                     /* of the product: rows x cols, square for GRAM and POLY */
    float alpha, diag;                                  /* out = alpha * accumulator, + diag where row = column */
    int tri;                                            /* tile side of the stored triangle of the symmetric operand */
    int split;                                          /* parts of K, one CTA (pair) of a cluster each */
    int lo;                                             /* whether out has a lo plane */
    ORTH_PTR(void) out_hi;                              /* the planes of out, rows out_pitch and matrices out_plane halves apart */
    ORTH_PTR(void) out_lo;
    long long out_pitch, out_plane;
    /* RESULT: element (r, c) of matrix k at k * stride_w + r * ld_w + c; transposed when tall */
    int type_w, tall, vec_w;
    float keep;                                         /* 0: w is not read */
    ORTH_PTR(void) w;
    long long ld_w, stride_w;
    ORTH_PTR(float) sums;                               /* where the parts of a tile meet */
    ORTH_PTR(int) status;                               /* the code of the first wait that ran out */
    ORTH_PTR(int) told;                                 /* in the host's memory: set when one has, for calls the host does not see */
    unsigned long long wait_ns;
    int silent;                                         /* the tests' way to see a wait run out: nothing is loaded */
} orth_product_t;
#endif
