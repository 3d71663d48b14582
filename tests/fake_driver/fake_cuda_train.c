/* fake_cuda_train.c -- fake_cuda.c with what the training operators' host tests need beside it: tensor maps of
 * three dimensions, a line for each product launch with its parameter block, and FAKE_CUDA_ORTH_STATUS=<code>, which
 * stores that code in the status word of every product kernel, the way the real kernel does when one of its
 * bounded waits runs out. Copies that the host waits for are logged. */
#define cuTensorMapEncodeTiled base_cuTensorMapEncodeTiled
#define cuLaunchKernelEx base_cuLaunchKernelEx
#define cuStreamSynchronize base_cuStreamSynchronize
#define cuMemcpyDtoH_v2 base_cuMemcpyDtoH_v2
#include "fake_cuda.c"
#undef cuTensorMapEncodeTiled
#undef cuLaunchKernelEx
#undef cuStreamSynchronize
#undef cuMemcpyDtoH_v2
#include "orth_params.cuh"

/* The words of the latest product, which FAKE_CUDA_ORTH_REPLAY=<code> sets when the stream is next waited for: a
 * captured call replayed behind the library's back. */
static int *orth_status, *orth_told;

CUresult cuStreamSynchronize(CUstream s)
{
    const char *code = getenv("FAKE_CUDA_ORTH_REPLAY");
    if (code && orth_status) { *orth_status = atoi(code); *orth_told = 1; unsetenv("FAKE_CUDA_ORTH_REPLAY"); }
    return base_cuStreamSynchronize(s);
}

CUresult cuMemcpyDtoH_v2(void *d, CUdeviceptr s, size_t n)
{
    logf_line("d2h_now\n");
    return base_cuMemcpyDtoH_v2(d, s, n);
}

CUresult cuTensorMapEncodeTiled(CUtensorMap *map, CUtensorMapDataType t, cuuint32_t rank, void *base, const cuuint64_t *dims,
                                const cuuint64_t *strides, const cuuint32_t *box, const cuuint32_t *estr,
                                CUtensorMapInterleave il, CUtensorMapSwizzle sw, CUtensorMapL2promotion l2,
                                CUtensorMapFloatOOBfill fill)
{
    char line[192];
    if (rank != 3) return base_cuTensorMapEncodeTiled(map, t, rank, base, dims, strides, box, estr, il, sw, l2, fill);
    memset(map, 0, sizeof *map);
    if (((size_t)map & 63) || ((size_t)base & 15) || (strides[0] & 15) || (strides[1] & 15)) return CUDA_ERROR_INVALID_VALUE;
    snprintf(line, sizeof line, "tensormap3 dims %llu %llu %llu strides %llu %llu box %u %u %u\n", (unsigned long long)dims[0],
             (unsigned long long)dims[1], (unsigned long long)dims[2], (unsigned long long)strides[0], (unsigned long long)strides[1],
             box[0], box[1], box[2]);
    logf_line(line);
    return CUDA_SUCCESS;
}

CUresult cuLaunchKernelEx(const CUlaunchConfig *c, CUfunction f, void **params, void **extra)
{
    if (strncmp(((fake_func_t *)f)->name, "orth_product", 12) == 0) {
        const orth_product_t *p = (const orth_product_t *)params[6];
        const char *code = getenv("FAKE_CUDA_ORTH_STATUS");
        char line[224];
        orth_status = (int *)(size_t)p->status;
        orth_told = (int *)(size_t)p->told;
        if (code) *orth_status = atoi(code);
        snprintf(line, sizeof line, "product mode %d rows %d cols %d K %d batch %d alpha %.9g diag %.9g keep %.9g tall %d vec %d silent %d\n",
                 p->mode, p->rows, p->cols, p->K, p->batch, p->alpha, p->diag, p->keep, p->tall, p->vec_w, p->silent);
        logf_line(line);
    }
    return base_cuLaunchKernelEx(c, f, params, extra);
}
