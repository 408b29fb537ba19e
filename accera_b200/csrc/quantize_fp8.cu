// Quantisation to 8-bit floating point, one fp32 scale for each group of 1 x 128 or 128 x 128 values.
//
//   s = 2^e, e the smallest integer with max|group| <= top * 2^e   (top = 448 for e4m3, 57344 for e5m2)
//   q = x / s, rounded once to the nearest 8-bit value, ties to even
//
// With top = 1.75 * 2^h (h = 8 or 15) and max|group| = m * 2^k, 1 <= m < 2, the exponent is k - h where m <= 1.75 and
// k - h + 1 otherwise: an integer addition on the bits of the maximum carries exactly then.  x / s is a product with the
// power of two 1 / s, hence exact in fp32 (down to values that round to zero anyway), so no rounding happens before the
// one to 8 bits, and the kernels agree with the formula bit for bit.
//
// The bound is HBM: each value is read once and written once as a byte; all arithmetic is on registers.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "accb_internal.h"

namespace accb {
namespace {

struct Params {
    int64_t rows, cols;
    int64_t xs0, xs1;
    int64_t qs;
    int64_t ss0, ss1;
    int64_t col_blocks;
    int h;                       // exponent of the largest 8-bit value: 8 or 15
};

constexpr int kGroup = ACCB_FP8_BLOCK;

// e of the group from max|x| over its finite values (fp32 bits), as fp32 bits of s and of 1 / s
__device__ __forceinline__ void group_scale(float amax, int h, float& s, float& inv)
{
    const uint32_t b = __float_as_uint(amax);
    int e = (int)((b + 0x1fffffu) >> 23) - 127 - h;          // m > 1.75 carries into the exponent
    e = max(-126, min(127, e));                               // zeros and tiny maxima: s stays a normal number
    if (b == 0) e = 0;
    s = __uint_as_float((uint32_t)(e + 127) << 23);
    // 1 / 2^127 is below the normal numbers; no maximum asks for it (e <= 120)
    inv = __uint_as_float((uint32_t)(127 - e) << 23);
}

__device__ __forceinline__ float finite_abs(float x)
{
    const float a = fabsf(x);
    return a <= 3.402823466e38f ? a : 0.0f;                   // infinities and NaN do not count
}

// x * inv, with an infinite x turned into NaN (the conversion would clamp it to the largest value)
__device__ __forceinline__ float scaled(float x, float inv) { const float y = x * inv; return fmaf(y, 0.0f, y); }

template <bool E5M2>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    uint16_t r;
    if constexpr (E5M2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// 16 bytes of x as they were loaded: kept packed until the scale is known, which halves the registers that wait for it
template <typename T> struct alignas(16) Vec16 { T v[16 / sizeof(T)]; };

// where the second pass converts again what the first has converted, the compiler must not keep the first's fp32 values
template <typename T> __device__ __forceinline__ void forget(Vec16<T>& w)
{
    uint4& u = reinterpret_cast<uint4&>(w);
    asm volatile("" : "+r"(u.x), "+r"(u.y), "+r"(u.z), "+r"(u.w));
}

// Groups along the rows of x.  TILE = false: a group is 128 neighbours of a row, taken by 128 * sizeof(T) / 16 threads
// with one 16-byte load each; a block takes kRowUnits * (threads / group) groups.  TILE = true: a block takes one square tile.
constexpr int kRowThreads = 256;

template <typename T, bool E5M2, bool TILE, bool VEC>
__global__ void __launch_bounds__(kRowThreads)
quantize_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scales, const Params p)
{
    pdl_enter();
    constexpr int E = 16 / (int)sizeof(T);                    // values a thread holds of one group
    constexpr int kPer = kGroup / E;                          // threads that share a group's row: 16 or 32
    constexpr int kSets = kRowThreads / kPer;                 // rows (TILE) or groups a block takes at once
    constexpr int kUnits = TILE ? kGroup / kSets : 4;
    __shared__ float warp_max[kRowThreads / 32];
    const int set = threadIdx.x / kPer, part = threadIdx.x % kPer;
    Vec16<T> v[kUnits];
    int64_t row[kUnits], col[kUnits];
    bool in[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        if constexpr (TILE) {
            row[u] = (int64_t)(blockIdx.x / p.col_blocks) * kGroup + u * kSets + set;
            col[u] = (int64_t)(blockIdx.x % p.col_blocks) * kGroup + part * E;
        } else {
            const int64_t g = ((int64_t)blockIdx.x * kUnits + u) * kSets + set;
            row[u] = g / p.col_blocks;
            col[u] = (g - row[u] * p.col_blocks) * kGroup + part * E;
        }
        in[u] = row[u] < p.rows && col[u] < p.cols;
        v[u] = Vec16<T>();
        if constexpr (VEC) {
            if (in[u]) v[u] = *reinterpret_cast<const Vec16<T>*>(x + row[u] * p.xs0 + col[u]);
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (in[u] && col[u] + e < p.cols) v[u].v[e] = x[row[u] * p.xs0 + (col[u] + e) * p.xs1];
        }
    }
    float amax[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        amax[u] = 0.0f;
#pragma unroll
        for (int e = 0; e < E; ++e) amax[u] = fmaxf(amax[u], finite_abs((float)v[u].v[e]));
        forget(v[u]);
    }
    if constexpr (TILE) {
        float m = 0.0f;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) m = fmaxf(m, amax[u]);
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = m;
        __syncthreads();
        m = warp_max[0];
#pragma unroll
        for (int w = 1; w < kRowThreads / 32; ++w) m = fmaxf(m, warp_max[w]);
#pragma unroll
        for (int u = 0; u < kUnits; ++u) amax[u] = m;
    } else {
#pragma unroll
        for (int o = kPer / 2; o; o >>= 1)
#pragma unroll
            for (int u = 0; u < kUnits; ++u) amax[u] = fmaxf(amax[u], __shfl_xor_sync(0xffffffffu, amax[u], o));
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        float s, inv;
        group_scale(amax[u], p.h, s, inv);
        if (TILE ? (u == 0 && threadIdx.x == 0) : (part == 0 && in[u]))
            scales[(TILE ? (int64_t)(blockIdx.x / p.col_blocks) : row[u]) * p.ss0 + (col[u] / kGroup) * p.ss1] = s;
        if (!in[u]) continue;
        uint32_t w[E / 4];
#pragma unroll
        for (int e = 0; e < E; e += 4)
            w[e / 4] = pack2<E5M2>(scaled((float)v[u].v[e], inv), scaled((float)v[u].v[e + 1], inv)) |
                       pack2<E5M2>(scaled((float)v[u].v[e + 2], inv), scaled((float)v[u].v[e + 3], inv)) << 16;
        uint8_t* dst = q + row[u] * p.qs + col[u];
        if constexpr (VEC) {
            if constexpr (E == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint32_t*>(dst) = w[0];
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) if (col[u] + e < p.cols) dst[e] = (uint8_t)(w[e / 4] >> (8 * (e % 4)));
        }
    }
}

// x contiguous along its rows' index (a transposed view): a block takes 128 columns of the view (which lie a pitch apart in
// memory) times a strip of its rows (contiguous), 64 rows or, for square tiles, 128.  A thread loads 16 bytes (E
// rows) of four neighbouring columns, so that it can store four bytes of a result row at a time to shared
// memory, from where rows of 128 bytes leave.
template <typename T, bool E5M2, bool TILE, bool VEC>
__global__ void __launch_bounds__(256)
quantize_across_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scales, const Params p, int64_t row_blocks,
                       int q_vec)
{
    pdl_enter();
    constexpr int E = 16 / (int)sizeof(T);
    constexpr int kStrip = 256 / 32 * E;                      // rows of the view that one set of loads covers: 64 or 32
    constexpr int kSets = TILE ? kGroup / kStrip : 1;
    constexpr int kRows = kSets * kStrip;
    constexpr int kPitch = kGroup + 4;
    __shared__ uint32_t bytes[kRows * kPitch / 4];
    __shared__ float col_max[8][kRows];
    const int64_t row0 = (int64_t)(blockIdx.x % row_blocks) * kRows, col_block = blockIdx.x / row_blocks, col0 = col_block * kGroup;
    const int octet = threadIdx.x % 8, quad = threadIdx.x / 8;                // which E rows, which four columns
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    Vec16<T> v[kSets][4];
#pragma unroll
    for (int z = 0; z < kSets; ++z)
#pragma unroll
        for (int c = 0; c < 4; ++c) {
            const int64_t r = row0 + z * kStrip + octet * E, k = col0 + quad * 4 + c;
            if constexpr (VEC) {
                if (k < p.cols && r < p.rows) v[z][c] = *reinterpret_cast<const Vec16<T>*>(x + k * p.xs1 + r);
                else v[z][c] = Vec16<T>();
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) v[z][c].v[e] = (k < p.cols && r + e < p.rows) ? x[k * p.xs1 + r + e] : (T)0.0f;
            }
        }
    // maxima of each row over its four columns here, over the warp's sixteen, over the block's 128
#pragma unroll
    for (int z = 0; z < kSets; ++z)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            float m = 0.0f;
#pragma unroll
            for (int c = 0; c < 4; ++c) m = fmaxf(m, finite_abs((float)v[z][c].v[e]));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
            if (lane < 8) col_max[warp][z * kStrip + octet * E + e] = m;
        }
#pragma unroll
    for (int z = 0; z < kSets; ++z)
#pragma unroll
        for (int c = 0; c < 4; ++c) forget(v[z][c]);
    __syncthreads();
    float tile_max = 0.0f;
    if constexpr (TILE) {
        float m = 0.0f;
        for (int i = lane; i < 8 * kRows; i += 32) m = fmaxf(m, col_max[i / kRows][i % kRows]);
#pragma unroll
        for (int o = 16; o; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        tile_max = m;
    }
#pragma unroll
    for (int z = 0; z < kSets; ++z)
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const int r = z * kStrip + octet * E + e;
            float m = tile_max;
            if constexpr (!TILE) {
                m = col_max[0][r];
#pragma unroll
                for (int w = 1; w < 8; ++w) m = fmaxf(m, col_max[w][r]);
            }
            float s, inv;
            group_scale(m, p.h, s, inv);
            if (TILE ? threadIdx.x == 0 && z == 0 && e == 0 : quad == 0 && row0 + r < p.rows)
                scales[(TILE ? (int64_t)(blockIdx.x % row_blocks) : row0 + r) * p.ss0 + col_block * p.ss1] = s;
            bytes[r * (kPitch / 4) + quad] = pack2<E5M2>(scaled((float)v[z][0].v[e], inv), scaled((float)v[z][1].v[e], inv)) |
                                             pack2<E5M2>(scaled((float)v[z][2].v[e], inv), scaled((float)v[z][3].v[e], inv)) << 16;
        }
    __syncthreads();
    const int64_t width = p.cols - col0 < kGroup ? p.cols - col0 : kGroup;
    if (q_vec && width == kGroup) {
        for (int i = threadIdx.x; i < kRows * 8; i += 256) {
            const int r = i / 8, part = i % 8;
            if (row0 + r >= p.rows) break;
            const uint32_t* b = bytes + r * (kPitch / 4) + part * 4;
            *reinterpret_cast<uint4*>(q + (row0 + r) * p.qs + col0 + part * 16) = make_uint4(b[0], b[1], b[2], b[3]);
        }
    } else {
        for (int i = threadIdx.x; i < kRows * kGroup; i += 256) {
            const int r = i / kGroup, c = i % kGroup;
            if (row0 + r < p.rows && c < width) q[(row0 + r) * p.qs + col0 + c] = (uint8_t)(bytes[r * (kPitch / 4) + c / 4] >> (8 * (c % 4)));
        }
    }
}

template <typename T, bool E5M2, bool TILE>
cudaError_t launch(const accb_quantize_fp8_desc& d, const void* xv, void* qv, float* scales, cudaStream_t stream)
{
    const T* x = (const T*)xv;
    uint8_t* q = (uint8_t*)qv;
    constexpr int E = 16 / (int)sizeof(T);
    Params p;
    p.rows = d.rows; p.cols = d.cols;
    p.xs0 = d.x_stride[0]; p.xs1 = d.x_stride[1];
    p.qs = d.q_stride;
    p.ss0 = d.scale_stride[0]; p.ss1 = d.scale_stride[1];
    p.col_blocks = (d.cols + kGroup - 1) / kGroup;
    p.h = E5M2 ? 15 : 8;
    const bool x_base = (reinterpret_cast<uintptr_t>(x) & 15) == 0;
    // contiguous along the view's rows index and not along its columns: the transposing kernel.  A single row of 16-byte
    // aligned neighbours counts as contiguous along the columns.
    const bool across = p.xs0 == 1 && p.xs1 != 1 && d.rows > 1;
    if (across) {
        constexpr int kRows = TILE ? kGroup : 256 / 32 * E;
        const int64_t row_blocks = (d.rows + kRows - 1) / kRows;
        const int64_t blocks = row_blocks * p.col_blocks;
        if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
        const bool vec = x_base && p.xs1 % E == 0 && d.rows % E == 0;
        const int q_vec = (reinterpret_cast<uintptr_t>(q) & 15) == 0 && p.qs % 16 == 0;
        return vec ? launch_pdl(quantize_across_kernel<T, E5M2, TILE, true>, dim3((unsigned)blocks), dim3(256), stream, x, q, scales, p, row_blocks, q_vec)
                   : launch_pdl(quantize_across_kernel<T, E5M2, TILE, false>, dim3((unsigned)blocks), dim3(256), stream, x, q, scales, p, row_blocks, q_vec);
    }
    constexpr int kSets = kRowThreads / (kGroup / E);
    const int64_t row_blocks = (d.rows + kGroup - 1) / kGroup;
    const int64_t blocks = TILE ? row_blocks * p.col_blocks : (d.rows * p.col_blocks + 4 * kSets - 1) / (4 * kSets);
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const bool vec = x_base && p.xs1 == 1 && (p.xs0 % E == 0 || d.rows == 1) && d.cols % E == 0 &&
                     (reinterpret_cast<uintptr_t>(q) % E) == 0 && (p.qs % E == 0 || d.rows == 1);
    return vec ? launch_pdl(quantize_rows_kernel<T, E5M2, TILE, true>, dim3((unsigned)blocks), dim3(kRowThreads), stream, x, q, scales, p)
               : launch_pdl(quantize_rows_kernel<T, E5M2, TILE, false>, dim3((unsigned)blocks), dim3(kRowThreads), stream, x, q, scales, p);
}

template <typename T>
cudaError_t by_kind(const accb_quantize_fp8_desc& d, const void* x, void* q, float* scales, cudaStream_t stream)
{
    const bool tile = d.block_rows != 1;
    if (d.q_type == ACCB_E5M2) return tile ? launch<T, true, true>(d, x, q, scales, stream) : launch<T, true, false>(d, x, q, scales, stream);
    return tile ? launch<T, false, true>(d, x, q, scales, stream) : launch<T, false, false>(d, x, q, scales, stream);
}

}  // namespace

int launch_quantize_fp8(const accb_quantize_fp8_desc& d, const void* x, void* q, float* scales, cudaStream_t stream, const char** err)
{
    cudaError_t e;
    if (d.x_type == ACCB_F32) e = by_kind<float>(d, x, q, scales, stream);
    else if (d.x_type == ACCB_F16) e = by_kind<__half>(d, x, q, scales, stream);
    else e = by_kind<__nv_bfloat16>(d, x, q, scales, stream);
    if (e != cudaSuccess) { *err = cudaGetErrorString(e); return ACCB_ERR_CUDA; }
    note_launches(1);
    return 1;
}

}  // namespace accb
