// GEMM of 8-bit floating point operands with one fp32 scale per block of 128 along K, on the CUDA cores:
//   C <- epi(alpha * sum_b sa[i, b] sb[b, j] (A[i, b] @ B[b, j]) + beta * C + bias[j])
// Takes any strides and any K, including 0.  It serves the layouts that the tensor-core kernels do not (an operand
// without a contiguous direction) and shows what they compute; it is bound by its fp32 fused multiply-adds.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>

#include "accb_internal.h"

namespace accb {
namespace {

constexpr int kTile = 64;       // rows and columns of C per block
constexpr int kStep = 32;       // K elements staged at a time (divides the scale block)

struct Params {
    int64_t m, n, k;
    int64_t as0, as1, bs0, bs1, cs0, cs1;
    int64_t sas0, sas1, sbs0, sbs1;
    int a_shift, b_shift;       // log2 of the rows of A / columns of B that share a scale
    int a_e5m2, b_e5m2;
    float alpha, beta;
    int relu;
    int64_t tiles_n;
};

__device__ __forceinline__ float fp8_to_float(uint8_t v, bool e5m2)
{
    return __half2float(__half(__nv_cvt_fp8_to_halfraw(v, e5m2 ? __NV_E5M2 : __NV_E4M3)));
}

template <typename TC>
__global__ void __launch_bounds__(256)
gemm_fp8_simt_kernel(const uint8_t* __restrict__ A, const uint8_t* __restrict__ B, TC* __restrict__ C,
                     const float* __restrict__ sa, const float* __restrict__ sb, const float* __restrict__ bias, const Params p)
{
    pdl_enter();
    __shared__ float as[kStep][kTile + 1], bs[kStep][kTile + 1];
    const int64_t row0 = (int64_t)(blockIdx.x / p.tiles_n) * kTile, col0 = (int64_t)(blockIdx.x % p.tiles_n) * kTile;
    const int tr = threadIdx.x / 16, tc = threadIdx.x % 16;
    float acc[4][4] = {};
    for (int64_t b = 0; b * ACCB_FP8_BLOCK < p.k; ++b) {
        float part[4][4] = {};
        const int64_t k_end = min((b + 1) * ACCB_FP8_BLOCK, p.k);
        for (int64_t k0 = b * ACCB_FP8_BLOCK; k0 < k_end; k0 += kStep) {
            __syncthreads();
            for (int e = threadIdx.x; e < kTile * kStep; e += 256) {
                // the faster index runs along the operand's smaller stride
                const int ar = p.as1 <= p.as0 ? e / kStep : e % kTile, ak = p.as1 <= p.as0 ? e % kStep : e / kTile;
                const int bc = p.bs0 <= p.bs1 ? e / kStep : e % kTile, bk = p.bs0 <= p.bs1 ? e % kStep : e / kTile;
                as[ak][ar] = (row0 + ar < p.m && k0 + ak < k_end) ? fp8_to_float(A[(row0 + ar) * p.as0 + (k0 + ak) * p.as1], p.a_e5m2) : 0.0f;
                bs[bk][bc] = (col0 + bc < p.n && k0 + bk < k_end) ? fp8_to_float(B[(k0 + bk) * p.bs0 + (col0 + bc) * p.bs1], p.b_e5m2) : 0.0f;
            }
            __syncthreads();
#pragma unroll 8
            for (int k = 0; k < kStep; ++k) {
                float x[4], y[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) { x[i] = as[k][tr * 4 + i]; y[i] = bs[k][tc + 16 * i]; }
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int j = 0; j < 4; ++j) part[i][j] = fmaf(x[i], y[j], part[i][j]);
            }
        }
        float ra[4], rb[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t r = row0 + tr * 4 + i, c = col0 + tc + 16 * i;
            ra[i] = r < p.m ? sa[(r >> p.a_shift) * p.sas0 + b * p.sas1] : 0.0f;
            rb[i] = c < p.n ? sb[b * p.sbs0 + (c >> p.b_shift) * p.sbs1] : 0.0f;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(part[i][j], ra[i] * rb[j], acc[i][j]);
    }
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int64_t r = row0 + tr * 4 + i, c = col0 + tc + 16 * j;
            if (r >= p.m || c >= p.n) continue;
            TC* d = C + r * p.cs0 + c * p.cs1;
            float v = acc[i][j] * p.alpha;
            if (p.beta != 0.0f) v = fmaf(p.beta, (float)*d, v);
            if (bias) v += bias[c];
            if (p.relu) v = v < 0.0f ? 0.0f : v;
            *d = (TC)v;
        }
}

}  // namespace

int launch_gemm_fp8_simt(const GemmFp8Launch& g, const char** err)
{
    const accb_gemm_desc& d = g.d;
    Params p;
    p.m = d.m; p.n = d.n; p.k = d.k;
    p.as0 = d.a_stride[0]; p.as1 = d.a_stride[1]; p.bs0 = d.b_stride[0]; p.bs1 = d.b_stride[1];
    p.cs0 = d.c_stride[0]; p.cs1 = d.c_stride[1];
    p.sas0 = g.s.a_stride[0]; p.sas1 = g.s.a_stride[1]; p.sbs0 = g.s.b_stride[0]; p.sbs1 = g.s.b_stride[1];
    p.a_shift = g.s.a_block == 1 ? 0 : 7; p.b_shift = g.s.b_block == 1 ? 0 : 7;
    p.a_e5m2 = d.a_type == ACCB_E5M2; p.b_e5m2 = d.b_type == ACCB_E5M2;
    p.alpha = d.alpha; p.beta = d.beta; p.relu = d.epilogue == ACCB_EPI_RELU;
    p.tiles_n = (d.n + kTile - 1) / kTile;
    const int64_t tiles = (d.m + kTile - 1) / kTile * p.tiles_n;
    if (tiles > 0x7fffffff) { *err = "too many tiles for this kernel's grid"; return ACCB_ERR_ARG; }
    const uint8_t* a = (const uint8_t*)g.a;
    const uint8_t* b = (const uint8_t*)g.b;
    const dim3 grid((unsigned)tiles), block(256);
    cudaError_t e;
    if (d.c_type == ACCB_F32) e = launch_pdl(gemm_fp8_simt_kernel<float>, grid, block, g.stream, a, b, (float*)g.c, g.a_scales, g.b_scales, g.bias, p);
    else if (d.c_type == ACCB_F16) e = launch_pdl(gemm_fp8_simt_kernel<__half>, grid, block, g.stream, a, b, (__half*)g.c, g.a_scales, g.b_scales, g.bias, p);
    else e = launch_pdl(gemm_fp8_simt_kernel<__nv_bfloat16>, grid, block, g.stream, a, b, (__nv_bfloat16*)g.c, g.a_scales, g.b_scales, g.bias, p);
    if (e != cudaSuccess) { *err = cudaGetErrorString(e); return ACCB_ERR_CUDA; }
    note_launches(1);
    return 1;
}

}  // namespace accb
