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

#include <type_traits>

#include "accb_internal.h"

namespace accb {
namespace {

struct Params {
    int64_t rows, cols;
    int64_t xs0, xs1;
    int64_t qs;
    int64_t ss0, ss1;
    int64_t col_blocks;
    int64_t row_step;
    int groups32;                // all group numbers fit 32 bits
    int h;                       // exponent of the largest 8-bit value: 8 or 15
};

constexpr int kGroup = ACCB_FP8_BLOCK;
constexpr int kRowUnits = 4;     // groups a thread takes part in

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

template <bool E5M2>
__device__ __forceinline__ uint32_t pack2(float lo, float hi)
{
    uint16_t r;
    if constexpr (E5M2) asm("cvt.rn.satfinite.e5m2x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    else asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(r) : "f"(hi), "f"(lo));
    return r;
}

// Maxima are taken of the values' bits without the sign, which are ordered like the magnitudes: two 16-bit values to a word.
// Bits from kInf on are infinities and NaN.
template <typename T> struct Bits {
    static constexpr int kPer = 4 / (int)sizeof(T);           // values in a word
    static constexpr uint32_t kInf = sizeof(T) == 4 ? 0x7f800000u : std::is_same<T, __half>::value ? 0x7c00u : 0x7f80u;
    static __device__ __forceinline__ uint32_t of(uint32_t w) { return w & (kPer == 2 ? 0x7fff7fffu : 0x7fffffffu); }
    static __device__ __forceinline__ uint32_t max(uint32_t a, uint32_t b)
    {
        uint32_t r;
        if constexpr (kPer == 2) asm("max.u16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
        else r = a > b ? a : b;
        return r;
    }
    static __device__ __forceinline__ uint32_t get(uint32_t w, int i) { return kPer == 2 ? (i ? w >> 16 : w & 0xffffu) : w; }
    static __device__ __forceinline__ bool finite(uint32_t w) { return get(w, 0) < kInf && (kPer == 1 || get(w, 1) < kInf); }
    // the word with its infinities and NaN replaced by zero: they do not count
    static __device__ __forceinline__ uint32_t only_finite(uint32_t w)
    {
        if constexpr (kPer == 1) return w < kInf ? w : 0u;
        else return (get(w, 0) < kInf ? w & 0xffffu : 0u) | (get(w, 1) < kInf ? w & 0xffff0000u : 0u);
    }
    static __device__ __forceinline__ float value(uint32_t bits)
    {
        if constexpr (kPer == 1) return __uint_as_float(bits);
        else if constexpr (std::is_same<T, __half>::value) return __half2float(__ushort_as_half((unsigned short)bits));
        else return __uint_as_float(bits << 16);
    }
};

// 16 bytes of x as they were loaded: kept packed until the scale is known, which halves the registers that wait for it
template <typename T> union alignas(16) Vec16 {
    uint32_t w[4];
    T v[16 / sizeof(T)];
    __device__ Vec16() { w[0] = w[1] = w[2] = w[3] = 0u; }
};

// value i of w times inv; where the vector has an infinity, that becomes NaN (the conversion would clamp it)
template <typename T> __device__ __forceinline__ float scaled(const Vec16<T>& w, int i, float inv, bool finite)
{
    const float y = (float)w.v[i] * inv;
    return finite ? y : fmaf(y, 0.0f, y);
}

// Groups along the rows of x.  TILE = false: a group is 128 neighbours of a row, taken by 128 * sizeof(T) / 16 threads
// with one 16-byte load each.  TILE = true: a block takes one square tile.  A group's last lane to know its maximum is one
// warp reduction away (redux.sync), so the loads in flight come from the many warps that fit an SM.  8192 x 8192 bf16 to e4m3:
// rows 42 us, tiles 35 us; the bytes alone take 31 us.  fp32 to e4m3: rows 69 us, tiles 150 us (51 us); the 16 vectors a thread
// of an fp32 tile do not fit its 64 registers (924 bytes are spilled), nor do all of the rows' in 32 (68 to 80 bytes).
// Rows that are not whole vectors go by single elements: 16383 x 8191 bf16 197 us where 16384 x 8192 takes 81.
constexpr int kRowThreads = 256;

template <typename T, bool E5M2, bool TILE, bool VEC>
__global__ void __launch_bounds__(kRowThreads, VEC ? (TILE ? 4 : 8) : 2)
quantize_rows_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scales, const Params p)
{
    pdl_enter();
    using B = Bits<T>;
    constexpr int E = 16 / (int)sizeof(T);                    // values a thread holds of one group
    constexpr int kPer = kGroup / E;                          // threads that share a group's row: 16 or 32
    constexpr int kSets = kRowThreads / kPer;                 // rows (TILE) or groups a block takes at once
    constexpr int kUnits = TILE ? kGroup / kSets : kRowUnits;
    __shared__ uint32_t warp_max[kRowThreads / 32];
    const int set = threadIdx.x / kPer, part = threadIdx.x % kPer;
    Vec16<T> v[kUnits];
    // A thread's units lie row_step rows apart at the same column: in a tile the rows that the block takes at once, else a
    // kUnits-th of all rows, so that one division finds the place of all of them.
    int64_t row0, col;
    const int64_t row_step = TILE ? kSets : p.row_step;
    if constexpr (TILE) {
        row0 = (int64_t)(blockIdx.x / p.col_blocks) * kGroup + set;
        col = (int64_t)(blockIdx.x % p.col_blocks) * kGroup + part * E;
    } else {
        const int64_t g = (int64_t)blockIdx.x * kSets + set;
        row0 = p.groups32 ? (int64_t)((uint32_t)g / (uint32_t)p.col_blocks) : g / p.col_blocks;
        col = (g - row0 * p.col_blocks) * kGroup + part * E;
    }
    const int64_t last_row = TILE ? p.rows : min(p.rows, p.row_step);        // of the first unit
    auto inside = [&](int u) { return (TILE || row0 < last_row) && row0 + u * row_step < p.rows && col < p.cols; };
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        const int64_t row = row0 + u * row_step;
        if (!inside(u)) continue;
        if constexpr (VEC) *reinterpret_cast<uint4*>(v[u].w) = *reinterpret_cast<const uint4*>(x + row * p.xs0 + col);
        else {
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (col + e < p.cols) v[u].v[e] = x[row * p.xs0 + (col + e) * p.xs1];
        }
    }
    uint32_t top[kUnits];
    bool finite[kUnits];
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        uint32_t m = B::max(B::max(B::of(v[u].w[0]), B::of(v[u].w[1])), B::max(B::of(v[u].w[2]), B::of(v[u].w[3])));
        finite[u] = B::finite(m);
        if (!finite[u]) {
            m = 0u;
#pragma unroll
            for (int i = 0; i < 4; ++i) m = B::max(m, B::only_finite(B::of(v[u].w[i])));
        }
        if constexpr (B::kPer == 2) m = m >> 16 > (m & 0xffffu) ? m >> 16 : m & 0xffffu;
        top[u] = m;
    }
    if constexpr (TILE) {
        uint32_t m = 0u;
#pragma unroll
        for (int u = 0; u < kUnits; ++u) m = max(m, top[u]);
        m = __reduce_max_sync(0xffffffffu, m);
        if (threadIdx.x % 32 == 0) warp_max[threadIdx.x / 32] = m;
        __syncthreads();
        m = warp_max[0];
#pragma unroll
        for (int w = 1; w < kRowThreads / 32; ++w) m = max(m, warp_max[w]);
#pragma unroll
        for (int u = 0; u < kUnits; ++u) top[u] = m;
    } else {
        const uint32_t lanes = kPer == 32 ? 0xffffffffu : 0xffffu << (threadIdx.x & 16);
#pragma unroll
        for (int u = 0; u < kUnits; ++u) top[u] = __reduce_max_sync(lanes, top[u]);
    }
#pragma unroll
    for (int u = 0; u < kUnits; ++u) {
        float s, inv;
        group_scale(B::value(top[u]), p.h, s, inv);
        const int64_t row = row0 + u * row_step;
        const bool in = inside(u);
        if (TILE ? (u == 0 && threadIdx.x == 0) : (part == 0 && in))
            scales[(TILE ? row / kGroup : row) * p.ss0 + (col / kGroup) * p.ss1] = s;
        if (!in) continue;
        uint32_t w[E / 4];
#pragma unroll
        for (int e = 0; e < E; e += 4)
            w[e / 4] = pack2<E5M2>(scaled(v[u], e, inv, finite[u]), scaled(v[u], e + 1, inv, finite[u])) |
                       pack2<E5M2>(scaled(v[u], e + 2, inv, finite[u]), scaled(v[u], e + 3, inv, finite[u])) << 16;
        uint8_t* dst = q + row * p.qs + col;
        if constexpr (VEC) {
            if constexpr (E == 8) *reinterpret_cast<uint2*>(dst) = make_uint2(w[0], w[1]);
            else *reinterpret_cast<uint32_t*>(dst) = w[0];
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) if (col + e < p.cols) dst[e] = (uint8_t)(w[e / 4] >> (8 * (e % 4)));
        }
    }
}

// x contiguous along its rows' index (a transposed view): a block takes 128 columns of the view (which lie a pitch apart in
// memory) times a strip of its rows (contiguous), 64 rows or, for square tiles, 128.  A thread loads 16 bytes (E
// rows) of four neighbouring columns, so that it can store four bytes of a result row at a time to shared
// memory, from where rows of 128 bytes leave.  16384 x 8192 bf16 to e5m2: 85 us (4.8 TB/s); the bytes alone take 62 us.  Unaligned, 16383 x 8191: 192 us by single elements.
template <typename T, bool E5M2, bool TILE, bool VEC>
__global__ void __launch_bounds__(256, TILE ? 4 : 6)
quantize_across_kernel(const T* __restrict__ x, uint8_t* __restrict__ q, float* __restrict__ scales, const Params p, int64_t row_blocks,
                       int q_vec)
{
    pdl_enter();
    using B = Bits<T>;
    constexpr int E = 16 / (int)sizeof(T);
    constexpr int kStrip = 256 / 32 * E;                      // rows of the view that one set of loads covers: 64 or 32
    constexpr int kSets = TILE ? kGroup / kStrip : 1;
    constexpr int kRows = kSets * kStrip;
    constexpr int kPitch = kGroup + 4;
    __shared__ uint32_t bytes[kRows * kPitch / 4];
    __shared__ uint32_t row_max[8][kRows / B::kPer];
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
                if (k < p.cols && r < p.rows) *reinterpret_cast<uint4*>(v[z][c].w) = *reinterpret_cast<const uint4*>(x + k * p.xs1 + r);
            } else {
#pragma unroll
                for (int e = 0; e < E; ++e) if (k < p.cols && r + e < p.rows) v[z][c].v[e] = x[k * p.xs1 + r + e];
            }
        }
    // maxima of each row over its four columns here, over the warp's sixteen, over the block's 128
    bool finite = true;
#pragma unroll
    for (int z = 0; z < kSets; ++z)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t m = B::max(B::max(B::of(v[z][0].w[i]), B::of(v[z][1].w[i])), B::max(B::of(v[z][2].w[i]), B::of(v[z][3].w[i])));
            if (!B::finite(m)) {
                finite = false;
                m = 0u;
#pragma unroll
                for (int c = 0; c < 4; ++c) m = B::max(m, B::only_finite(B::of(v[z][c].w[i])));
            }
            m = B::max(m, __shfl_xor_sync(0xffffffffu, m, 8));
            m = B::max(m, __shfl_xor_sync(0xffffffffu, m, 16));
            if (lane < 8) row_max[warp][(z * kStrip + octet * E) / B::kPer + i] = m;
        }
    __syncthreads();
    uint32_t tile_max = 0u;
    if constexpr (TILE) {
        uint32_t m = 0u;
        for (int i = lane; i < 8 * kRows / B::kPer; i += 32) m = B::max(m, row_max[i / (kRows / B::kPer)][i % (kRows / B::kPer)]);
        if constexpr (B::kPer == 2) m = max(m >> 16, m & 0xffffu);
        tile_max = __reduce_max_sync(0xffffffffu, m);
    }
#pragma unroll
    for (int z = 0; z < kSets; ++z)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            uint32_t m = 0u;
            if constexpr (!TILE) {
                m = row_max[0][(z * kStrip + octet * E) / B::kPer + i];
#pragma unroll
                for (int w = 1; w < 8; ++w) m = B::max(m, row_max[w][(z * kStrip + octet * E) / B::kPer + i]);
            }
#pragma unroll
            for (int h = 0; h < B::kPer; ++h) {
                const int e = i * B::kPer + h, r = z * kStrip + octet * E + e;
                float s, inv;
                group_scale(B::value(TILE ? tile_max : B::get(m, h)), p.h, s, inv);
                if (TILE ? threadIdx.x == 0 && z == 0 && e == 0 : quad == 0 && row0 + r < p.rows)
                    scales[(TILE ? (int64_t)(blockIdx.x % row_blocks) : row0 + r) * p.ss0 + col_block * p.ss1] = s;
                bytes[r * (kPitch / 4) + quad] = pack2<E5M2>(scaled(v[z][0], e, inv, finite), scaled(v[z][1], e, inv, finite)) |
                                                 pack2<E5M2>(scaled(v[z][2], e, inv, finite), scaled(v[z][3], e, inv, finite)) << 16;
            }
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
    p.row_step = (d.rows + kRowUnits - 1) / kRowUnits;
    p.groups32 = p.row_step * p.col_blocks < ((int64_t)1 << 32) - kRowThreads;
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
    const int64_t blocks = TILE ? row_blocks * p.col_blocks : (p.row_step * p.col_blocks + kSets - 1) / kSets;
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
