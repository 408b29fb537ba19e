// Tensor-core GEMM of 8-bit floating point operands with one fp32 scale per block of 128 along K, for sm_100a:
//
//   C <- epi(alpha * sum over blocks b of (sa[i, b] sb[b, j]) (A[i, b] @ B[b, j])  +  beta * C + bias[j])
//
// A block is 128 bytes of K: one swizzle atom, one pipeline stage, four tcgen05.mma (kind::f8f6f4, K = 32 each).  The
// scales differ from block to block, so the sum over blocks cannot stay in TMEM: every block's product goes to a TMEM
// buffer of its own, from where the epilogue warps take it with tcgen05.ld and add it, times the product of its two
// scales, to fp32 sums in registers.  While they do, the tensor core works on the next block in the other buffer.
//
// Two kernels:
//   pair   256 x 256 tiles by CTA pairs (cta_group::2), persistent: every SM multiplies 128 x 256 x 128 a block, in
//          512 cycles at the nominal 8-bit rate.  Eight epilogue warps hold the sums, 128 fp32 a thread; while a warp adds
//          32 columns the next 32 are on their way from TMEM.  8192^3, e4m3 to bf16: 630 us call after call on three sets of
//          inputs (1.75 PFLOP/s under the power limit), 550 to 590 in short runs; the same loads and MMAs without the
//          additions take 397 us in short runs, so the loop is bound by the round trip of a TMEM buffer (MMAs done -
//          read by both CTAs' warps - MMA issued again), of which only two fit TMEM at this width.  Narrower tiles with
//          three or four buffers (160, 128 columns) were measured slower, 650 and 700 us in short runs: their operands alone
//          take 500 and 540.  With a scale per column 4096 x 8192 x 16384 takes 840 to 860 us (each product costs the
//          epilogue warps two instructions instead of one).  The 168 registers a thread do not hold everything: 52 to 92 bytes a
//          thread are spilled, 296 to 424 with a scale per column.
//          Problems with few tiles cut K into slices, whose fp32 sums gemm_splitk.cu adds in slice order.
//   tile   128 x BN tiles by single CTAs, for few rows of C, or few tiles: columns of C (weights) on the 128 TMEM
//          lanes, 16 to 64 rows of C (tokens) on BN = 16, 32 or 64 accumulator columns, K cut into up to eight slices
//          that a cluster multiplies side by side and adds, slice by slice, through distributed shared memory.
// Scales reach shared memory by cp.async up to sixteen blocks ahead, four blocks of a row in 16 bytes where they lie side by
// side (4 bytes at a time the copies themselves bound the pair kernel with a scale per column).
//
// Every wait is bounded as in gemm_umma.cu: one that runs out is recorded, all roles leave, the host reports
// ACCB_ERR_TIMEOUT.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstring>
#include <type_traits>

#include "accb_internal.h"
#define ACCB_WAIT_INLINE __forceinline__
#include "umma_device.h"

namespace accb {
namespace {

constexpr int kRowsX = 128;                 // TMEM lanes of a CTA
constexpr int kRing = 8;                    // blocks of scales in shared memory

struct F8Params {
    int64_t m, n;
    int64_t cs0, cs1;
    int64_t sa_row, sa_kb, sb_col, sb_kb;   // strides of the scales
    const float* sa;
    const float* sb;
    const float* bias;
    float alpha, beta;
    int relu;
    int a_shift, b_shift;                   // 0, or 7 where 128 rows of A / columns of B share a scale
    int sa_vec, sb_vec;                     // the scales of four neighbouring blocks of a row / column lie in 16 aligned bytes
    int a_mn, b_mn;                         // operand contiguous along M / N instead of K
    int num_kb;
    uint32_t idesc;
    int tiles_m, tiles_n, group_m;
    int slices;                             // parts that K is cut into: CTAs of a cluster (tile kernel), work items (pair kernel)
    int64_t slice_stride;                   // pair kernel: elements of C from one slice's sums to the next's
    int plain;                              // pair kernel: C is the sums alone, in rows of 16-byte vectors
    int c_mode;                             // pair kernel: 2 rows of 16-byte vectors, 1 contiguous rows, 0 any strides
    int* status;
    int launch_id;
    unsigned long long wait_ns;
    int drop_commit;                        // self-test of the time-out path: the commit of the last block's MMAs is left out
    int drop_scales;                        // the same: the arrival of a tile's last scales is left out
};

__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& lo, float& hi)
{
    uint32_t a, b;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(a), "=r"(b) : "l"(v));
    lo = __uint_as_float(a);
    hi = __uint_as_float(b);
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr)
        : "memory");
}
// as tmem_wait_ld: the registers pass through the wait so that their uses stay behind it
__device__ __forceinline__ void tmem_wait_ld16(uint32_t (&r)[16])
{
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                   "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}

// 4 bytes global -> shared, zero where !inside (the source is not read then)
__device__ __forceinline__ void copy_scale(uint32_t dst, const float* src, bool inside)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(inside ? 4 : 0) : "memory");
}
__device__ __forceinline__ void copy_scales4(uint32_t dst, const float* src, bool inside)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(inside ? 16 : 0) : "memory");
}
// arrives on the barrier once this thread's copies so far have landed; the barrier counts one arrival a lane
__device__ __forceinline__ void copies_arrive(uint32_t bar)
{
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
// Arrival on a barrier of the pair's rank 0 that only says "these TMEM columns have been read" (tcgen05.wait::ld and
// tcgen05.fence::before_thread_sync come before it): no memory of this thread needs to be visible with it.
__device__ __forceinline__ void mbar_arrive_pair(uint32_t bar)
{
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_test(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
    return ok != 0;
}
__device__ __forceinline__ uint32_t map_to_rank(uint32_t addr, uint32_t rank)
{
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float4 load_cluster4(uint32_t addr)
{
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr));
    return v;
}

// Four tcgen05.mma that multiply one stage (128 bytes of K a row) into a fresh accumulator, issued by the elected lane of
// a warp that runs converged, so that descriptors stay in uniform registers.  *_step: what 32 bytes of K add to a descriptor.
template <bool PAIR>
__device__ __forceinline__ void mma_block(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t a_step, uint32_t b_step, uint32_t elected)
{
#define ACCB_F8_MMA(GROUP, A, B, ADD) "@e tcgen05.mma.cta_group::" GROUP ".kind::f8f6f4 [%0], " A ", " B ", %3, " ADD ";\n\t"
#define ACCB_F8_BLOCK(GROUP)                                                                                          \
    asm volatile("{\n\t.reg .pred e, fresh, add;\n\t.reg .b64 as, bs, a1, a2, a3, b1, b2, b3;\n\t"                   \
                 "setp.ne.b32 e, %6, 0;\n\tsetp.ne.b32 fresh, 0, 0;\n\tsetp.eq.b32 add, 0, 0;\n\t"                   \
                 "cvt.u64.u32 as, %4;\n\tcvt.u64.u32 bs, %5;\n\t"                                                    \
                 "add.u64 a1, %1, as;\n\tadd.u64 b1, %2, bs;\n\tadd.u64 a2, a1, as;\n\tadd.u64 b2, b1, bs;\n\t"      \
                 "add.u64 a3, a2, as;\n\tadd.u64 b3, b2, bs;\n\t"                                                    \
                 ACCB_F8_MMA(GROUP, "%1", "%2", "fresh") ACCB_F8_MMA(GROUP, "a1", "b1", "add")                        \
                 ACCB_F8_MMA(GROUP, "a2", "b2", "add") ACCB_F8_MMA(GROUP, "a3", "b3", "add") "}"                      \
                 ::"r"(tmem_d), "l"(a), "l"(b), "r"(idesc), "r"(a_step), "r"(b_step), "r"(elected) : "memory")
    if constexpr (PAIR) ACCB_F8_BLOCK("2");
    else ACCB_F8_BLOCK("1");
#undef ACCB_F8_BLOCK
#undef ACCB_F8_MMA
}
__device__ __forceinline__ uint32_t elect_lane()
{
    uint32_t e;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(e));
    return e;
}
// operand descriptor of the ring's first stage, and what 32 bytes of K add to it
__device__ __forceinline__ uint64_t operand_desc(uint32_t smem, int mn) { return mn ? make_smem_desc_mn(smem, kSlabBytes * kSlabBytes) : make_smem_desc(smem); }
__device__ __forceinline__ uint32_t operand_step(int mn) { return (uint32_t)((mn ? kMmaKBytes * kSlabBytes : kMmaKBytes) >> 4); }

// alpha, beta * old, bias and ReLU of one value; a NaN stays NaN
__device__ __forceinline__ float finish(float acc, float old, float bias, const F8Params& p)
{
    float v = acc * p.alpha;
    if (p.beta != 0.0f) v = fmaf(p.beta, old, v);
    if (p.bias) v += bias;
    if (p.relu) v = v < 0.0f ? 0.0f : v;
    return v;
}

// ---------------------------------------------------------------------------------
// pair kernel
// ---------------------------------------------------------------------------------

struct PairPlan {
    static constexpr int kThreads = 384;                                // TMA, MMA, scales, an idle warp; eight epilogue warps
    static constexpr int kEpilogueWarp = 4;                             // first of them
    // Registers a thread: the launch gets 65536 / 384, rounded down to 168; the epilogue warps, with 128 sums and 64 values on
    // their way from TMEM, take what the first four warps give up: 4 * 40 + 8 * 232 = 12 * 168
    static constexpr int kFewRegisters = 40, kManyRegisters = 232;
    static constexpr int kGroup = 4, kSlots = 4;                        // scales: blocks a ring slot, slots
    static constexpr int kBN = 256;
    static constexpr int kStageBytes = 2 * kRowsX * kSlabBytes;         // 16 KB of A, 16 KB of B (this CTA's half of the columns)
    static constexpr int kStages = 5;
    static constexpr int kBoxBytes = 32 * 128;
    static constexpr int kScaleBytes = (kRowsX + kBN) * 4;
    static constexpr int kBoxes = kStages * kStageBytes;
    static constexpr int kScales = kBoxes + 8 * kBoxBytes;
    static constexpr int kBars = kScales + kSlots * kGroup * kScaleBytes;
    static constexpr int kTotal = kBars + 512 + 1024;                   // + manual alignment
    static_assert(kTotal <= 227 * 1024, "shared memory of a CTA");
};

// A box between shared memory and C.  Along rows lane / 8 is one of four rows, lane % 8 a 16-byte slot; a row's slots are
// stored at slot ^ (row % 8), so neither accesses along rows nor those of whole columns of slots collide in banks.  Rows of C
// that are not whole vectors go row by row instead, neighbouring elements by neighbouring lanes: 2000 x 2001 bf16 with
// K = 1024 took 28.8 us with a vector's elements one after the other by a lane, 21.2 this way.
template <typename TC>
__device__ __forceinline__ int box_byte(int r, int c) { const int b = c * (int)sizeof(TC); return r * 128 + (((b >> 4) ^ (r & 7)) << 4) + (b & 15); }
template <typename TC>
__device__ __forceinline__ void box_in(uint8_t* box, const TC* C, int64_t row0, int64_t col0, int rows, int cols, int lane, const F8Params& p)
{
    constexpr int V = 16 / (int)sizeof(TC);
    const int r0 = lane >> 3, slot = lane & 7, in_slot = cols - slot * V;
    const TC* base = C + (row0 + r0) * p.cs0 + col0 + slot * V;
    const bool vec = in_slot >= V;
    if (p.c_mode != 2) {
#pragma unroll 4
        for (int r = 0; r < rows; ++r)
            for (int c = lane; c < cols; c += 32) *reinterpret_cast<TC*>(box + box_byte<TC>(r, c)) = C[(row0 + r) * p.cs0 + col0 + c];
        __syncwarp();
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + r0;
        uint8_t* at = box + r * 128 + ((slot ^ (r & 7)) << 4);
        const TC* src = base + (int64_t)(i * 4) * p.cs0;
        if (r >= rows) continue;
        if (vec) *reinterpret_cast<uint4*>(at) = *reinterpret_cast<const uint4*>(src);
        else
            for (int e = 0; e < V && e < in_slot; ++e) reinterpret_cast<TC*>(at)[e] = src[e];
    }
    __syncwarp();
}
template <typename TC>
__device__ __forceinline__ void box_out(const uint8_t* box, TC* C, int64_t row0, int64_t col0, int rows, int cols, int lane, const F8Params& p)
{
    constexpr int V = 16 / (int)sizeof(TC);
    const int r0 = lane >> 3, slot = lane & 7, in_slot = cols - slot * V;
    TC* base = C + (row0 + r0) * p.cs0 + col0 + slot * V;
    const bool vec = in_slot >= V;
    __syncwarp();
    if (p.c_mode != 2) {
#pragma unroll 4
        for (int r = 0; r < rows; ++r)
            for (int c = lane; c < cols; c += 32) C[(row0 + r) * p.cs0 + col0 + c] = *reinterpret_cast<const TC*>(box + box_byte<TC>(r, c));
        __syncwarp();
        return;
    }
    if (rows == 32 && cols == 8 * V) {
        // a box inside the matrix, as nearly all are: all reads, then all writes
        uint4 w[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = *reinterpret_cast<const uint4*>(box + (i * 4 + r0) * 128 + ((slot ^ ((i * 4 + r0) & 7)) << 4));
#pragma unroll
        for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(base + (int64_t)(i * 4) * p.cs0) = w[i];
        __syncwarp();
        return;
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const int r = i * 4 + r0;
        const uint8_t* at = box + r * 128 + ((slot ^ (r & 7)) << 4);
        TC* dst = base + (int64_t)(i * 4) * p.cs0;
        if (r >= rows) continue;
        if (vec) *reinterpret_cast<uint4*>(dst) = *reinterpret_cast<const uint4*>(at);
        else
            for (int e = 0; e < V && e < in_slot; ++e) dst[e] = reinterpret_cast<const TC*>(at)[e];
    }
    __syncwarp();
}

// One box (32 rows of 128 bytes, this thread's row in `v`) of the tile to C, through shared memory
template <typename TC>
__device__ __forceinline__ void store_box(float (&v)[128 / sizeof(TC)], uint8_t* box, TC* C, int64_t row0, int64_t col0, int lane, const F8Params& p)
{
    constexpr int W = 128 / (int)sizeof(TC), V = 16 / (int)sizeof(TC);
    const int cols = (int)(p.n - col0 < W ? p.n - col0 : W), rows = (int)(p.m - row0 < 32 ? p.m - row0 : 32);
    if (p.alpha != 1.0f) {
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] *= p.alpha;
    }
    if (p.c_mode == 0) {
        if (lane < rows) {
            TC* d = C + (row0 + lane) * p.cs0 + col0 * p.cs1;
#pragma unroll
            for (int j = 0; j < W; ++j) {
                if (j >= cols) break;
                float x = v[j];
                if (p.beta != 0.0f) x = fmaf(p.beta, (float)d[j * p.cs1], x);
                if (p.bias) x += __ldg(p.bias + col0 + j);
                if (p.relu) x = x < 0.0f ? 0.0f : x;
                d[j * p.cs1] = (TC)x;
            }
        }
        return;
    }
    uint8_t* own = box + lane * 128;                         // this thread's row; its slots are at s ^ (lane & 7)
    const int flip = (lane & 7) << 4;
    if (p.beta != 0.0f) {
        box_in<TC>(box, C, row0, col0, rows, cols, lane, p);
#pragma unroll
        for (int s = 0; s < 8; ++s) {
            const uint4 w = *reinterpret_cast<const uint4*>(own + ((s << 4) ^ flip));
            const TC* h = reinterpret_cast<const TC*>(&w);
#pragma unroll
            for (int e = 0; e < V; ++e) v[s * V + e] = fmaf(p.beta, (float)h[e], v[s * V + e]);
        }
    }
    if (p.bias) {
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] += j < cols ? __ldg(p.bias + col0 + j) : 0.0f;
    }
    if (p.relu) {
#pragma unroll
        for (int j = 0; j < W; ++j) v[j] = v[j] < 0.0f ? 0.0f : v[j];
    }
#pragma unroll
    for (int s = 0; s < 8; ++s) {
        uint4 w;
        TC* h = reinterpret_cast<TC*>(&w);
#pragma unroll
        for (int e = 0; e < V; ++e) h[e] = (TC)v[s * V + e];
        *reinterpret_cast<uint4*>(own + ((s << 4) ^ flip)) = w;
    }
    box_out<TC>(box, C, row0, col0, rows, cols, lane, p);
}

// The same for a thread that holds pairs of neighbouring columns of four rows, as tcgen05.ld.16x256b gives them: value(h, j, i) is
// row 16 h + 8 (i / 2) + lane / 4, column 8 j + 2 (lane % 4) + i % 2 of the box.
template <typename TC, typename F>
__device__ __forceinline__ void store_box_pairs(F value, uint8_t* box, TC* C, int64_t row0, int64_t col0, int lane, const F8Params& p)
{
    constexpr int W = 128 / (int)sizeof(TC);
    struct alignas(2 * sizeof(TC)) Pair { TC v[2]; };
    const int cols = (int)(p.n - col0 < W ? p.n - col0 : W), rows = (int)(p.m - row0 < 32 ? p.m - row0 : 32);
    const bool boxed = p.c_mode != 0;
    if (boxed && p.beta != 0.0f) box_in<TC>(box, C, row0, col0, rows, cols, lane, p);
#pragma unroll
    for (int j = 0; j < W / 8; ++j) {
        const int col = 8 * j + 2 * (lane & 3);
        float bias[2] = { 0.0f, 0.0f };
        if (p.bias) {
            if (col < cols) bias[0] = __ldg(p.bias + col0 + col);
            if (col + 1 < cols) bias[1] = __ldg(p.bias + col0 + col + 1);
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int row = 8 * h + (lane >> 2);
            const float lo = value(h >> 1, j, 2 * (h & 1)), hi = value(h >> 1, j, 2 * (h & 1) + 1);
            if (boxed) {
                const int byte = col * (int)sizeof(TC);
                Pair* at = reinterpret_cast<Pair*>(box + row * 128 + (((byte >> 4) ^ (row & 7)) << 4) + (byte & 15));
                Pair y = {};
                if (p.beta != 0.0f) y = *at;
                y.v[0] = (TC)finish(lo, (float)y.v[0], bias[0], p);
                y.v[1] = (TC)finish(hi, (float)y.v[1], bias[1], p);
                *at = y;
            } else if (row < rows) {
                TC* d = C + (row0 + row) * p.cs0 + (col0 + col) * p.cs1;
                if (col < cols) d[0] = (TC)finish(lo, p.beta != 0.0f ? (float)d[0] : 0.0f, bias[0], p);
                if (col + 1 < cols) d[p.cs1] = (TC)finish(hi, p.beta != 0.0f ? (float)d[p.cs1] : 0.0f, bias[1], p);
            }
        }
    }
    if (boxed) box_out<TC>(box, C, row0, col0, rows, cols, lane, p);
}

// work item -> tile and range of blocks of K
template <bool SPLIT>
__device__ __forceinline__ void pair_item(int t, const F8Params& p, int& tm, int& tn, int& slice, int& kb_begin, int& kb_end)
{
    slice = 0; kb_begin = 0; kb_end = p.num_kb;
    if (SPLIT) {
        slice = t % p.slices;
        t /= p.slices;
        kb_begin = (int)((int64_t)p.num_kb * slice / p.slices);
        kb_end = (int)((int64_t)p.num_kb * (slice + 1) / p.slices);
    }
    const int group_size = p.group_m * p.tiles_n;
    const int group = t / group_size;
    const int first_m = group * p.group_m;
    const int rows = min(p.tiles_m - first_m, p.group_m);
    const int in = t - group * group_size;
    tm = first_m + in % rows;
    tn = in / rows;
}

// 32 columns of a block's product, times one scale, to the sums
__device__ __forceinline__ void add_scaled(float* acc, const uint32_t (&x)[32], float f)
{
#pragma unroll
    for (int j = 0; j < 32; ++j) acc[j] = fmaf(__uint_as_float(x[j]), f, acc[j]);
}
// 32 columns of 32 lanes as two 16x256b loads: register 16 h + 4 j + i of lane l is row 16 h + 8 (i / 2) + l / 4, column
// 8 j + 2 (l % 4) + i % 2
__device__ __forceinline__ void tmem_ld_pairs(uint32_t taddr, uint32_t (&r)[32])
{
#pragma unroll
    for (int h = 0; h < 2; ++h)
        asm volatile(
            "tcgen05.ld.sync.aligned.16x256b.x4.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
            : "=r"(r[16 * h]), "=r"(r[16 * h + 1]), "=r"(r[16 * h + 2]), "=r"(r[16 * h + 3]), "=r"(r[16 * h + 4]), "=r"(r[16 * h + 5]),
              "=r"(r[16 * h + 6]), "=r"(r[16 * h + 7]), "=r"(r[16 * h + 8]), "=r"(r[16 * h + 9]), "=r"(r[16 * h + 10]), "=r"(r[16 * h + 11]),
              "=r"(r[16 * h + 12]), "=r"(r[16 * h + 13]), "=r"(r[16 * h + 14]), "=r"(r[16 * h + 15])
            : "r"(taddr + ((uint32_t)(16 * h) << 16))
            : "memory");
}
// the same columns, times a scale for each of this thread's four rows and each of its two columns in eight (at col_scale,
// four floats a column)
__device__ __forceinline__ void add_scaled_pairs(float* acc, const uint32_t (&x)[32], const float (&f)[4], const float* col_scale)
{
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float2 w = make_float2(col_scale[32 * j], col_scale[32 * j + 4]);
#pragma unroll
        for (int h = 0; h < 4; ++h) {
            const int i = 16 * (h >> 1) + 4 * j + 2 * (h & 1);
            acc[i] = fmaf(__uint_as_float(x[i]), f[h] * w.x, acc[i]);
            acc[i + 1] = fmaf(__uint_as_float(x[i + 1]), f[h] * w.y, acc[i + 1]);
        }
    }
}

// COLS: every column of B has a scale of its own (else 128 share one).  SPLIT: K is cut into slices, C holds their sums.
template <typename TC, bool COLS, bool SPLIT>
__global__ void __launch_bounds__(PairPlan::kThreads, 1)
gemm_fp8_pair_kernel(const __grid_constant__ CUtensorMap map_a, const __grid_constant__ CUtensorMap map_b, TC* __restrict__ C, const F8Params p)
{
    using Plan = PairPlan;
    constexpr int S = Plan::kStages;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t bars = smem_base + Plan::kBars;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    // A block's MMAs are complete: its stage may be loaded again and its accumulator read.  One commit a block for both,
    // because the issuing thread pays for each; neither side can be a whole turn of the ring behind.
    auto done_bar = [&](int s) { return bars + 8u * (S + s); };
    auto tmem_empty_bar = [&](int b) { return bars + 8u * (2 * S + b); };
    auto scale_full_bar = [&](int r) { return bars + 8u * (2 * S + 2 + r); };
    auto scale_empty_bar = [&](int r) { return bars + 8u * (2 * S + 2 + Plan::kSlots + r); };
    volatile uint32_t* tmem_holder = reinterpret_cast<volatile uint32_t*>(smem_gen + Plan::kBars + 8 * (2 * S + 2 + 2 * Plan::kSlots));
    volatile uint32_t* gave_up = tmem_holder + 2;        // one word a CTA of the pair, each CTA with a copy of both

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WaitCtx wctx{p.status, p.launch_id, p.wait_ns};
    const uint32_t rank = cluster_ctarank();
    const bool leader = rank == 0;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");

    auto record_give_up = [&]() {
        gave_up[rank] = 1u;
        asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(map_to_rank(smem_u32((const void*)(gave_up + rank)), rank ^ 1u)), "r"(1u) : "memory");
    };
    if (threadIdx.x == 0) {
        gave_up[0] = 0u;
        gave_up[1] = 0u;
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_a)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_b)) : "memory");
        for (int s = 0; s < S; ++s) { mbar_init(full_bar(s), 1); mbar_init(done_bar(s), 1); }
        for (int b = 0; b < 2; ++b) mbar_init(tmem_empty_bar(b), 16);                          // the epilogue warps of both CTAs
        for (int r = 0; r < Plan::kSlots; ++r) { mbar_init(scale_full_bar(r), 32); mbar_init(scale_empty_bar(r), 8); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_holder)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync_all();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *tmem_holder;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    const int num_tiles = p.tiles_m * p.tiles_n * (SPLIT ? p.slices : 1);
    const int num_units = (int)gridDim.x / 2, unit = (int)blockIdx.x / 2;

    if (warp < Plan::kEpilogueWarp) {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(Plan::kFewRegisters));
    if (warp == 0) {
        // ---------------- TMA producer ----------------
        if (lane == 0) {
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int t = unit; t < num_tiles && ok; t += num_units) {
                int tm, tn, slice, kb_begin, kb_end;
                pair_item<SPLIT>(t, p, tm, tn, slice, kb_begin, kb_end);
                const int row_a = (tm * 2 + (int)rank) * kRowsX, row_b = tn * Plan::kBN + (int)rank * 128;
                for (int kb = kb_begin; kb < kb_end; ++kb) {
                    if (!mbar_wait(done_bar(s), ph ^ 1u, wctx, SITE_PRODUCER_EMPTY, kb)) { ok = false; break; }
                    const uint32_t sa = smem_base + s * Plan::kStageBytes, sb = sa + kRowsX * kSlabBytes;
                    if (leader) mbar_arrive_expect_tx(full_bar(s), 2u * Plan::kStageBytes);
                    if (p.a_mn) tma_load_2d_pair(sa, &map_a, full_bar(s), row_a, kb * kSlabBytes, 0);
                    else tma_load_2d_pair(sa, &map_a, full_bar(s), kb * kSlabBytes, row_a, 0);
                    if (p.b_mn) tma_load_2d_pair(sb, &map_b, full_bar(s), row_b, kb * kSlabBytes, 0);
                    else tma_load_2d_pair(sb, &map_b, full_bar(s), kb * kSlabBytes, row_b, 0);
                    if (++s == S) { s = 0; ph ^= 1u; }
                }
            }
            if (!ok) record_give_up();
        }
    } else if (warp == 2) {
        // ---------------- scales ----------------
        int r = 0;
        uint32_t rph = 0;
        bool ok = true;
        for (int t = unit; t < num_tiles && ok; t += num_units) {
            int tm, tn, slice, kb_begin, kb_end;
            pair_item<SPLIT>(t, p, tm, tn, slice, kb_begin, kb_end);
            const int64_t row_a = (int64_t)(tm * 2 + (int)rank) * kRowsX + lane, col_b = (int64_t)tn * Plan::kBN + lane * (COLS ? 1 : 128);
            for (int kb0 = kb_begin; kb0 < kb_end; kb0 += Plan::kGroup) {
                ok = __all_sync(0xffffffffu, mbar_wait(scale_empty_bar(r), rph ^ 1u, wctx, SITE_PRODUCER_EMPTY, kb0));
                if (!ok) break;
                const int blocks = min(Plan::kGroup, kb_end - kb0);
                const uint32_t slot = smem_base + Plan::kScales + r * Plan::kGroup * Plan::kScaleBytes;
                auto copy = [&](const float* base, int64_t first, int64_t count, int64_t step, int shift, int64_t s_row, int64_t s_kb, int loads, int at, int vec) {
                    for (int i = 0; i < loads; ++i) {
                        const int64_t row = first + i * step;
                        const bool inside = row < count;
                        const float* src = base + (inside ? (row >> shift) * s_row : 0) + kb0 * s_kb;
                        const uint32_t dst = slot + (at + i * 32 + lane) * 16;
                        if (vec) copy_scales4(dst, src, inside);
                        else
                            for (int j = 0; j < blocks; ++j) copy_scale(dst + 4 * j, src + j * s_kb, inside);
                    }
                };
                const bool whole = blocks == Plan::kGroup && kb0 % Plan::kGroup == 0;
                copy(p.sa, row_a, p.m, 32, p.a_shift, p.sa_row, p.sa_kb, 4, 0, p.sa_vec && whole);
                if (COLS || lane < 2) copy(p.sb, col_b, p.n, 32, p.b_shift, p.sb_col, p.sb_kb, COLS ? 8 : 1, kRowsX, p.sb_vec && whole);
                if (!(p.drop_scales && kb0 + Plan::kGroup >= kb_end)) copies_arrive(scale_full_bar(r));
                if (++r == Plan::kSlots) { r = 0; rph ^= 1u; }
            }
        }
        if (!ok && lane == 0) record_give_up();
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == 1) {
        // ---------------- MMA issuer (rank 0 of the pair) ----------------
        if (leader) {
            const uint64_t a0 = operand_desc(smem_base, p.a_mn), b0 = operand_desc(smem_base + kRowsX * kSlabBytes, p.b_mn);
            const uint32_t a_step = operand_step(p.a_mn), b_step = operand_step(p.b_mn), elected = elect_lane();
            int blocks = 0;
            for (int t = unit; t < num_tiles; t += num_units) {
                int tm, tn, slice, kb_begin, kb_end;
                pair_item<SPLIT>(t, p, tm, tn, slice, kb_begin, kb_end);
                blocks += kb_end - kb_begin;
            }
            int s = 0;
            uint32_t ph = 0;
            bool ok = true;
            for (int g = 0; g < blocks; ++g) {
                ok = mbar_wait(full_bar(s), ph, wctx, SITE_MMA_FULL, g) &&
                     mbar_wait(tmem_empty_bar(g & 1), ((g >> 1) & 1u) ^ 1u, wctx, SITE_MMA_TMEM_EMPTY, g);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                const uint64_t stage = (uint64_t)(s * (Plan::kStageBytes >> 4));
                mma_block<true>(tmem_base + (uint32_t)((g & 1) * Plan::kBN), a0 + stage, b0 + stage, p.idesc, a_step, b_step, elected);
                if (elected && !(p.drop_commit && g == blocks - 1)) umma_commit<true>(done_bar(s));
                __syncwarp();
                if (++s == S) { s = 0; ph ^= 1u; }
            }
            if (!ok && lane == 0) record_give_up();
        }
    }
    } else {
        // ---------------- epilogue warps ----------------
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(Plan::kManyRegisters));
        const int q = warp & 3, ew = warp - Plan::kEpilogueWarp, half = ew >> 2;     // TMEM lane quarter, half of the tile's columns
        uint8_t* box = smem_gen + Plan::kBoxes + ew * Plan::kBoxBytes;
        const float* scales = reinterpret_cast<const float*>(smem_gen + Plan::kScales);
        const uint32_t taddr0 = tmem_base + ((uint32_t)(q * 32) << 16) + (uint32_t)(half * 128);
        int g = 0, r = 0, s = 0;
        uint32_t rph = 0, ph = 0;
        bool ok = true;
        for (int t = unit; t < num_tiles && ok; t += num_units) {
            int tm, tn, slice, kb_begin, kb_end;
            pair_item<SPLIT>(t, p, tm, tn, slice, kb_begin, kb_end);
            float acc[128];
#pragma unroll
            for (int i = 0; i < 128; ++i) acc[i] = 0.0f;
            // One load of 32 columns is always on its way while the 32 before it are added: the first of a block is issued
            // before the last of the block before it is added, if that block's MMAs are done by then.
            uint32_t x0[32], x1[32];
            bool loading = false;
            const int num_kb = SPLIT ? kb_end - kb_begin : p.num_kb;
            for (int kb = 0; kb < num_kb; ++kb, ++g) {
                const int buf = g & 1, in_group = kb % Plan::kGroup;
                const uint32_t taddr = taddr0 + (uint32_t)(buf * Plan::kBN);
                // The lanes leave a wait one by one; the vote after it brings them together for the warp-wide tcgen05.ld and wait::ld,
                // and all of them stay or leave.  With the block's load already on its way, only a new slot of scales is waited for.
                if (in_group == 0 || !loading) {
                    ok = in_group != 0 || mbar_wait(scale_full_bar(r), rph, wctx, SITE_EPI_SCALES, kb);
                    ok = ok && (loading || mbar_wait(done_bar(s), ph, wctx, SITE_EPI_TMEM_FULL, kb));
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) {
                        if (loading) tmem_wait_ld(x0);           // no load may be in flight when TMEM is given back
                        break;
                    }
                }
                if (!loading) {
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    if constexpr (COLS) tmem_ld_pairs(taddr, x0);
                    else tmem_ld32(taddr, x0);
                }
                if (++s == S) { s = 0; ph ^= 1u; }
                // a slot holds the scales of a row, or column, of four blocks side by side
                const float* sc = scales + r * Plan::kGroup * (Plan::kScaleBytes / 4) + in_group;
                const float* col_scale = sc + 4 * (kRowsX + (COLS ? half * 128 : half));
                // A column's scale for each thread that holds the column costs shared memory as much bandwidth as the sums cost
                // TMEM, 1024 cycles a block with a row a thread.  With pairs of columns of four rows a thread it is a quarter.
                float f[COLS ? 4 : 1];
                if constexpr (COLS) {
                    col_scale += 8 * (lane & 3);
#pragma unroll
                    for (int i = 0; i < 4; ++i) f[i] = sc[4 * (q * 32 + (lane >> 2) + 8 * i)];
                } else {
                    f[0] = sc[4 * (q * 32 + lane)] * col_scale[0];
                }
                auto load = [&](uint32_t at, uint32_t (&x)[32]) { if constexpr (COLS) tmem_ld_pairs(at, x); else tmem_ld32(at, x); };
                auto add = [&](int c, const uint32_t (&x)[32]) {
                    if constexpr (COLS) add_scaled_pairs(acc + 32 * c, x, f, col_scale + 128 * c);
                    else add_scaled(acc + 32 * c, x, f[0]);
                };
                tmem_wait_ld(x0);
                load(taddr + 32, x1);
                add(0, x0);
                tmem_wait_ld(x1);
                load(taddr + 64, x0);
                add(1, x1);
                tmem_wait_ld(x0);
                load(taddr + 96, x1);
                const bool next = kb + 1 < num_kb && mbar_test(done_bar(s), ph);
                add(2, x0);
                tmem_wait_ld(x1);
                // this warp has read the buffer: the MMA issuer of the pair may overwrite it
                asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
                loading = __all_sync(0xffffffffu, next);
                if (lane == 0) mbar_arrive_pair(tmem_empty_bar(buf) & kPeerMask);
                if (loading) {
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    load(taddr0 + (uint32_t)((buf ^ 1) * Plan::kBN), x0);
                }
                add(3, x1);
                if (in_group == Plan::kGroup - 1 || kb == num_kb - 1) {
                    __syncwarp();
                    if (lane == 0) mbar_arrive(scale_empty_bar(r));
                    if (++r == Plan::kSlots) { r = 0; rph ^= 1u; }
                }
            }
            if (!ok) break;
            const int64_t row0 = (int64_t)(tm * 2 + (int)rank) * kRowsX + q * 32, col0 = (int64_t)tn * Plan::kBN + half * 128;
            constexpr int W = 128 / (int)sizeof(TC);
            TC* dst = SPLIT ? C + slice * p.slice_stride : C;
            if (p.plain && row0 + 32 <= p.m && col0 + 128 <= p.n) {
                // Nothing but the sums, all inside the matrix.  This code runs once a tile and is not in the instruction cache then,
                // so the common case is kept short and without branches (7 % of the time of 8192^3 with a scale per column).
                constexpr int V = 16 / (int)sizeof(TC);
                const int r0 = lane >> 3, slot = lane & 7;
                uint8_t* out = reinterpret_cast<uint8_t*>(dst + (row0 + r0) * p.cs0 + col0 + slot * V);
                const int64_t step = 4 * p.cs0 * (int64_t)sizeof(TC);
                const uint8_t* from = box + r0 * 128 + ((slot ^ r0) << 4), *from4 = box + r0 * 128 + ((slot ^ r0 ^ 4) << 4);
#pragma unroll
                for (int b = 0; b < 128 / W; ++b) {
                    if constexpr (COLS) {
                        struct alignas(2 * sizeof(TC)) Pair { TC v[2]; };
#pragma unroll
                        for (int j = 0; j < W / 8; ++j)
#pragma unroll
                            for (int h = 0; h < 4; ++h) {
                                const int row = 8 * h + (lane >> 2), byte = (8 * j + 2 * (lane & 3)) * (int)sizeof(TC);
                                const int i = b * W + 32 * (j / 4) + 16 * (h >> 1) + 4 * (j % 4) + 2 * (h & 1);
                                *reinterpret_cast<Pair*>(box + row * 128 + (((byte >> 4) ^ (row & 7)) << 4) + (byte & 15)) = Pair{ { (TC)acc[i], (TC)acc[i + 1] } };
                            }
                    } else {
#pragma unroll
                        for (int k = 0; k < 8; ++k) {
                            uint4 w;
                            TC* e = reinterpret_cast<TC*>(&w);
#pragma unroll
                            for (int j = 0; j < V; ++j) e[j] = (TC)acc[b * W + k * V + j];
                            *reinterpret_cast<uint4*>(box + lane * 128 + ((k ^ (lane & 7)) << 4)) = w;
                        }
                    }
                    __syncwarp();
                    uint4 w[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) w[i] = *reinterpret_cast<const uint4*>((i & 1 ? from4 : from) + i * 512);
#pragma unroll
                    for (int i = 0; i < 8; ++i) *reinterpret_cast<uint4*>(out + b * 128 + i * step) = w[i];
                    __syncwarp();
                }
                continue;
            }
#pragma unroll
            for (int b = 0; b < 128 / W; ++b) {
                if (row0 >= p.m || col0 + b * W >= p.n) continue;
                if constexpr (COLS) {
                    store_box_pairs<TC>([&](int h, int j, int i) { return acc[b * W + 32 * (j / 4) + 16 * h + 4 * (j % 4) + i]; }, box, dst, row0, col0 + b * W, lane, p);
                } else {
                    float v[W];
#pragma unroll
                    for (int j = 0; j < W; ++j) v[j] = acc[b * W + j];
                    store_box<TC>(v, box, dst, row0, col0 + b * W, lane, p);
                }
            }
        }
        if (!ok && lane == 0) record_give_up();
    }

    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    cluster_sync_all();
    if ((gave_up[0] | gave_up[1]) != 0u) {
        // give loads that are still in flight time to land before shared memory is released
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
        cluster_sync_all();
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(512) : "memory");
    }
}

// ---------------------------------------------------------------------------------
// tile kernel
// ---------------------------------------------------------------------------------

template <int BN> struct TilePlan {
    static constexpr int kThreads = 192;                                 // TMA + scales, MMA, four epilogue warps
    static constexpr int kStageBytes = (kRowsX + BN) * kSlabBytes;       // 128 columns of C (weights), BN rows of C (tokens)
    static constexpr int kStages = BN == 64 ? 4 : 5;
    static constexpr int kBuffers = BN == 64 ? 4 : 8;    // TMEM accumulators of BN columns
    static constexpr int kTmemCols = kBuffers * BN;
    static constexpr int kScaleBytes = (kRowsX + BN) * 4;
    static constexpr int kScales = kStages * kStageBytes;
    static constexpr int kBars = kScales + kRing * kScaleBytes;
    static constexpr int kTotal = kBars + 512 + 1024;
    static_assert(kTotal <= 113 * 1024, "two CTAs share an SM");
    static_assert(BN * kRowsX * 4 <= kStages * kStageBytes, "the sums of a slice fit the operand ring");
};

template <typename TC, int BN>
__global__ void __launch_bounds__(TilePlan<BN>::kThreads, 2)
gemm_fp8_tile_kernel(const __grid_constant__ CUtensorMap map_w, const __grid_constant__ CUtensorMap map_t, TC* __restrict__ C, const F8Params p)
{
    using Plan = TilePlan<BN>;
    constexpr int S = Plan::kStages, NB = Plan::kBuffers;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t smem_base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* smem_gen = smem_raw + (smem_base - smem_u32(smem_raw));
    const uint32_t bars = smem_base + Plan::kBars;
    auto full_bar = [&](int s) { return bars + 8u * s; };
    auto empty_bar = [&](int s) { return bars + 8u * (S + s); };
    auto tmem_full_bar = [&](int b) { return bars + 8u * (2 * S + b); };
    auto tmem_empty_bar = [&](int b) { return bars + 8u * (2 * S + NB + b); };
    auto scale_full_bar = [&](int r) { return bars + 8u * (2 * S + 2 * NB + r); };
    auto scale_empty_bar = [&](int r) { return bars + 8u * (2 * S + 2 * NB + kRing + r); };
    static_assert(8 * (2 * S + 2 * NB + 2 * kRing) + 16 <= 512, "barriers");
    volatile uint32_t* tmem_holder = reinterpret_cast<volatile uint32_t*>(smem_gen + Plan::kBars + 8 * (2 * S + 2 * NB + 2 * kRing));
    volatile uint32_t* gave_up = tmem_holder + 2;

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const WaitCtx wctx{p.status, p.launch_id, p.wait_ns};
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    if (threadIdx.x == 0) {
        gave_up[0] = 0u;
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_w)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&map_t)) : "memory");
        for (int s = 0; s < S; ++s) { mbar_init(full_bar(s), 1); mbar_init(empty_bar(s), 1); }
        for (int b = 0; b < NB; ++b) { mbar_init(tmem_full_bar(b), 1); mbar_init(tmem_empty_bar(b), 4); }
        for (int r = 0; r < kRing; ++r) { mbar_init(scale_full_bar(r), 32); mbar_init(scale_empty_bar(r), 4); }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32((const void*)tmem_holder)), "r"(Plan::kTmemCols) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
    const uint32_t tmem_base = *tmem_holder;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    // neighbouring tiles share their weights, which are the larger operand
    const int tile = (int)blockIdx.x / p.slices, slice = (int)blockIdx.x % p.slices;
    const int row0 = (tile / p.tiles_m) * kRowsX;                        // first column of C (weight)
    const int col0 = (tile % p.tiles_m) * BN;                            // first row of C (token)
    const int kb_begin = (int)((int64_t)p.num_kb * slice / p.slices), kb_end = (int)((int64_t)p.num_kb * (slice + 1) / p.slices);

    uint64_t acc[BN / 2];
#pragma unroll
    for (int i = 0; i < BN / 2; ++i) acc[i] = 0ull;

    if (warp == 0) {
        int s = 0, r = 0;
        uint32_t ph = 0, rph = 0;
        bool ok = true;
        const float* src_w[4];
        bool in_w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int64_t row = (int64_t)row0 + i * 32 + lane;
            in_w[i] = row < p.n;
            src_w[i] = p.sb + (in_w[i] ? (row >> p.b_shift) * p.sb_col : 0);
        }
        constexpr int kColLoads = (BN + 31) / 32;
        const float* src_t[kColLoads];
        bool in_t[kColLoads];
#pragma unroll
        for (int i = 0; i < kColLoads; ++i) {
            const int64_t col = (int64_t)col0 + i * 32 + lane;
            in_t[i] = col < p.m && i * 32 + lane < BN;
            src_t[i] = p.sa + (in_t[i] ? (col >> p.a_shift) * p.sa_row : 0);
        }
        for (int kb = kb_begin; kb < kb_end; ++kb) {
            // the operands first: the scales are needed only once a block has been multiplied
            if (lane == 0) {
                ok = mbar_wait(empty_bar(s), ph ^ 1u, wctx, SITE_PRODUCER_EMPTY, kb);
                if (ok) {
                    const uint32_t sw = smem_base + s * Plan::kStageBytes, st = sw + kRowsX * kSlabBytes;
                    mbar_arrive_expect_tx(full_bar(s), (uint32_t)Plan::kStageBytes);
                    if (p.b_mn) tma_load_2d(sw, &map_w, full_bar(s), row0, kb * kSlabBytes, 0);
                    else tma_load_2d(sw, &map_w, full_bar(s), kb * kSlabBytes, row0, 0);
                    tma_load_2d(st, &map_t, full_bar(s), kb * kSlabBytes, col0, 0);
                }
            }
            if (++s == S) { s = 0; ph ^= 1u; }
            ok = __all_sync(0xffffffffu, ok && mbar_wait(scale_empty_bar(r), rph ^ 1u, wctx, SITE_PRODUCER_EMPTY, kb));
            if (!ok) break;
            const uint32_t sc = smem_base + Plan::kScales + r * Plan::kScaleBytes;
#pragma unroll
            for (int i = 0; i < 4; ++i) copy_scale(sc + (i * 32 + lane) * 4, src_w[i] + kb * p.sb_kb, in_w[i]);
#pragma unroll
            for (int i = 0; i < kColLoads; ++i)
                if (i * 32 + lane < BN) copy_scale(sc + (kRowsX + i * 32 + lane) * 4, src_t[i] + kb * p.sa_kb, in_t[i]);
            if (!(p.drop_scales && kb == kb_end - 1)) copies_arrive(scale_full_bar(r));
            if (++r == kRing) { r = 0; rph ^= 1u; }
        }
        if (!ok && lane == 0) gave_up[0] = 1u;
        asm volatile("cp.async.wait_all;" ::: "memory");
    } else if (warp == 1) {
        if (lane == 0) {
            auto issue = [&](auto w_mn_tag, auto t_mn_tag) {
                constexpr bool W_MN = decltype(w_mn_tag)::value, T_MN = decltype(t_mn_tag)::value;
                int s = 0, b = 0;
                uint32_t ph = 0, bph = 0;
                for (int kb = kb_begin; kb < kb_end; ++kb) {
                    if (!mbar_wait(tmem_empty_bar(b), bph ^ 1u, wctx, SITE_MMA_TMEM_EMPTY, kb) || !mbar_wait(full_bar(s), ph, wctx, SITE_MMA_FULL, kb)) {
                        gave_up[0] = 1u;
                        break;
                    }
                    asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
                    const uint32_t sw = smem_base + s * Plan::kStageBytes;
                    issue_stage<KIND_F8F6F4, false, W_MN, T_MN>(tmem_base + (uint32_t)(b * BN), sw, sw + kRowsX * kSlabBytes, p.idesc, true);
                    umma_commit<false>(empty_bar(s));
                    if (!(p.drop_commit && kb == kb_end - 1)) umma_commit<false>(tmem_full_bar(b));
                    if (++s == S) { s = 0; ph ^= 1u; }
                    if (++b == NB) { b = 0; bph ^= 1u; }
                }
            };
            if (!p.b_mn) issue(std::false_type{}, std::false_type{});
            else issue(std::true_type{}, std::false_type{});
        }
    } else {
        const int q = warp & 3;
        const float* scales = reinterpret_cast<const float*>(smem_gen + Plan::kScales);
        const uint32_t taddr0 = tmem_base + ((uint32_t)(q * 32) << 16);
        int b = 0, r = 0;
        uint32_t bph = 0, rph = 0;
        bool ok = true;
        for (int kb = kb_begin; kb < kb_end; ++kb) {
            ok = mbar_wait(scale_full_bar(r), rph, wctx, SITE_EPI_SCALES, kb) && mbar_wait(tmem_full_bar(b), bph, wctx, SITE_EPI_TMEM_FULL, kb);
            ok = __all_sync(0xffffffffu, ok);
            if (!ok) break;
            asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
            const float* sc = scales + r * (Plan::kScaleBytes / 4);
            const float f = sc[q * 32 + lane];
            const uint64_t f2 = pack2(__float_as_uint(f), __float_as_uint(f));
            const uint32_t taddr = taddr0 + (uint32_t)(b * BN);
#pragma unroll
            for (int c = 0; c < BN / 16; ++c) {
                uint32_t x[16];
                tmem_ld16(taddr + (uint32_t)(16 * c), x);
                tmem_wait_ld16(x);
#pragma unroll
                for (int j = 0; j < 8; j += 2) {
                    const ulonglong2 w = *reinterpret_cast<const ulonglong2*>(sc + kRowsX + 16 * c + 2 * j);
                    acc[8 * c + j] = fma2(pack2(x[2 * j], x[2 * j + 1]), mul2(f2, w.x), acc[8 * c + j]);
                    acc[8 * c + j + 1] = fma2(pack2(x[2 * j + 2], x[2 * j + 3]), mul2(f2, w.y), acc[8 * c + j + 1]);
                }
            }
            asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
            __syncwarp();
            if (lane == 0) { mbar_arrive(tmem_empty_bar(b)); mbar_arrive(scale_empty_bar(r)); }
            if (++b == NB) { b = 0; bph ^= 1u; }
            if (++r == kRing) { r = 0; rph ^= 1u; }
        }
        if (!ok && lane == 0) gave_up[0] = 1u;
    }
    __syncwarp();
    asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
    __syncthreads();
    if (gave_up[0] != 0u) {
        for (int i = 0; i < 64; ++i) __nanosleep(1000);
        __syncthreads();
    }
    if (warp == 1) {
        asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"(Plan::kTmemCols) : "memory");
    }

    // All loads and MMAs of this CTA are done: the operand ring holds the slice's sums, [BN][128] fp32, which leave with four
    // weights a lane, so that a token's 128 results are one or two instructions of a warp.
    const int cols = (int)(p.m - col0 < BN ? p.m - col0 : BN);
    float* sums = reinterpret_cast<float*>(smem_gen);
    if (warp >= 2) {
        const int at = (warp & 3) * 32 + lane;
#pragma unroll
        for (int c = 0; c < BN; c += 2) {
            float lo, hi;
            unpack2(acc[c / 2], lo, hi);
            sums[c * kRowsX + at] = lo;
            sums[(c + 1) * kRowsX + at] = hi;
        }
    }
    const int64_t n0 = (int64_t)row0 + lane * 4;
    float bias[4] = {};
    if (p.bias) {
#pragma unroll
        for (int e = 0; e < 4; ++e) if (n0 + e < p.n) bias[e] = __ldg(p.bias + n0 + e);
    }
    if (p.slices > 1) cluster_sync_all(); else __syncthreads();
    if (warp >= 2 && n0 < p.n) {
        // This CTA's share of the columns: every slices-th, one a warp at a time; the slices' sums are added in their order
        // along K.  Reads from other CTAs take long, so those of two columns are issued together.
        struct alignas(4 * sizeof(TC)) Four { TC v[4]; };
        const bool vec = p.cs1 == 1 && n0 + 4 <= p.n && p.cs0 % 4 == 0 && reinterpret_cast<uintptr_t>(C) % sizeof(Four) == 0;
        const int step = p.slices * 4;
        for (int c = slice + p.slices * (warp - 2); c < cols; c += 2 * step) {
            float v[2][4] = {};
            const bool two = c + step < cols;
            const uint32_t mine = smem_base + (uint32_t)(c * kRowsX + lane * 4) * 4, second = two ? (uint32_t)(step * kRowsX) * 4 : 0u;
#pragma unroll 4
            for (int z = 0; z < p.slices; ++z) {
                const uint32_t from = p.slices > 1 ? map_to_rank(mine, (uint32_t)z) : mine;
                const float4 a = load_cluster4(from), b = load_cluster4(from + second);
                v[0][0] += a.x; v[0][1] += a.y; v[0][2] += a.z; v[0][3] += a.w;
                v[1][0] += b.x; v[1][1] += b.y; v[1][2] += b.z; v[1][3] += b.w;
            }
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                if (h == 1 && !two) break;
                TC* d = C + (col0 + c + h * step) * p.cs0 + n0 * p.cs1;
                if (vec) {
                    Four y = {};
                    if (p.beta != 0.0f) y = *reinterpret_cast<const Four*>(d);
#pragma unroll
                    for (int e = 0; e < 4; ++e) y.v[e] = (TC)finish(v[h][e], (float)y.v[e], bias[e], p);
                    *reinterpret_cast<Four*>(d) = y;
                } else {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (n0 + e < p.n) d[e * p.cs1] = (TC)finish(v[h][e], p.beta != 0.0f ? (float)d[e * p.cs1] : 0.0f, bias[e], p);
                }
            }
        }
    }
    if (p.slices > 1) cluster_sync_all();                                // nobody leaves while its sums are being read
}

// ---------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------

uint32_t f8_idesc(const accb_gemm_desc& d, bool swapped, int m, int n, bool a_mn, bool b_mn)
{
    const int x = swapped ? d.b_type : d.a_type, y = swapped ? d.a_type : d.b_type;
    const bool x_mn = swapped ? b_mn : a_mn, y_mn = swapped ? a_mn : b_mn;
    uint32_t i = 1u << 4;                                                // fp32 accumulator
    i |= (x == ACCB_E5M2 ? 1u : 0u) << 7;
    i |= (y == ACCB_E5M2 ? 1u : 0u) << 10;
    i |= (x_mn ? 1u : 0u) << 15;
    i |= (y_mn ? 1u : 0u) << 16;
    i |= (uint32_t)(n >> 3) << 17;
    i |= (uint32_t)(m >> 4) << 24;
    return i;
}

constexpr int kMaxDevices = 64;

template <typename TC, bool COLS, bool SPLIT>
cudaError_t launch_pair(const GemmFp8Launch& g, const CUtensorMap& ma, const CUtensorMap& mb, const F8Params& p)
{
    auto kernel = gemm_fp8_pair_kernel<TC, COLS, SPLIT>;
    cudaLaunchConfig_t cfg = {};
    cfg.blockDim = dim3(PairPlan::kThreads);
    cfg.dynamicSmemBytes = PairPlan::kTotal;
    cfg.stream = g.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = options().gemm_pdl == 0 ? 0 : 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    static std::atomic<int> resident[kMaxDevices];
    int units = g.device < kMaxDevices ? resident[g.device].load(std::memory_order_acquire) : 0;
    if (units == 0) {
        cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, PairPlan::kTotal);
        if (e != cudaSuccess) return e;
        cfg.gridDim = dim3(2 * (unsigned)(g.num_sms / 2));
        e = cudaOccupancyMaxActiveClusters(&units, kernel, &cfg);
        if (e != cudaSuccess) return e;
        if (units < 1) return cudaErrorLaunchOutOfResources;
        if (units > g.num_sms / 2) units = g.num_sms / 2;
        if (g.device < kMaxDevices) resident[g.device].store(units, std::memory_order_release);
    }
    if (g.d.max_ctas > 0 && units > (g.d.max_ctas + 1) / 2) units = (g.d.max_ctas + 1) / 2;
    const int64_t tiles = (int64_t)p.tiles_m * p.tiles_n * p.slices;
    if (units > tiles) units = (int)tiles;
    cfg.gridDim = dim3((unsigned)(2 * units));
    return cudaLaunchKernelEx(&cfg, kernel, ma, mb, (TC*)g.c, p);
}

template <typename TC, int BN>
cudaError_t launch_tile(const GemmFp8Launch& g, const CUtensorMap& mw, const CUtensorMap& mt, const F8Params& p)
{
    auto kernel = gemm_fp8_tile_kernel<TC, BN>;
    static std::atomic<bool> opted[kMaxDevices];
    if (g.device >= kMaxDevices || !opted[g.device].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, TilePlan<BN>::kTotal);
        if (e != cudaSuccess) return e;
        if (g.device < kMaxDevices) opted[g.device].store(true, std::memory_order_release);
    }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(p.tiles_m * p.tiles_n * p.slices));
    cfg.blockDim = dim3(TilePlan<BN>::kThreads);
    cfg.dynamicSmemBytes = TilePlan<BN>::kTotal;
    cfg.stream = g.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.slices; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = options().gemm_pdl == 0 ? 0 : 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, kernel, mw, mt, (TC*)g.c, p);
}

template <typename TC>
cudaError_t launch_c(const GemmFp8Launch& g, const CUtensorMap& ma, const CUtensorMap& mb, const F8Params& p, int bn)
{
    if (bn == 256) {
        if constexpr (std::is_same<TC, float>::value)
            if (p.slices > 1) return p.b_shift ? launch_pair<TC, false, true>(g, ma, mb, p) : launch_pair<TC, true, true>(g, ma, mb, p);
        return p.b_shift ? launch_pair<TC, false, false>(g, ma, mb, p) : launch_pair<TC, true, false>(g, ma, mb, p);
    }
    if (bn == 64) return launch_tile<TC, 64>(g, mb, ma, p);
    if (bn == 32) return launch_tile<TC, 32>(g, mb, ma, p);
    return launch_tile<TC, 16>(g, mb, ma, p);
}

}  // namespace

// Contiguous direction of an operand [rows, k] with element strides `s_rows`, `s_k`: 0 along K, 1 along its rows, -1 neither.
// Where both would do (one row, or K = 1) K comes first.
static int contiguous_direction(int64_t rows, int64_t k, int64_t s_rows, int64_t s_k)
{
    if (s_k == 1 || k == 1) return 0;
    if (s_rows == 1 || rows == 1) return 1;
    return -1;
}

int launch_gemm_fp8(const GemmFp8Launch& g0, const char** err)
{
    GemmFp8Launch g = g0;
    const accb_gemm_desc& d = g.d;
    const int a_dir = contiguous_direction(d.m, d.k, d.a_stride[0], d.a_stride[1]);
    const int b_dir = contiguous_direction(d.n, d.k, d.b_stride[1], d.b_stride[0]);
    if (d.k < 1 || a_dir < 0 || b_dir < 0 || !encode_tiled_fn()) return 0;

    // Operands as `lines` runs of `width` bytes, `pitch` bytes apart.  TMA wants 16-byte aligned runs that do not overlap: others
    // are copied.
    struct Operand { const void* base; int64_t lines, width, pitch; } op[2] = {
        { g.a, a_dir ? d.k : d.m, a_dir ? d.m : d.k, a_dir ? d.a_stride[1] : d.a_stride[0] },
        { g.b, b_dir ? d.k : d.n, b_dir ? d.n : d.k, b_dir ? d.b_stride[0] : d.b_stride[1] } };
    void* tmp[2] = { nullptr, nullptr };
    auto release = [&]() { for (void* t : tmp) temp_free(t, g.stream); };
    int launches = 0;
    for (int i = 0; i < 2; ++i) {
        Operand& o = op[i];
        if (o.lines == 1) o.pitch = (o.width + 15) / 16 * 16;            // never followed
        if (o.pitch % 16 == 0 && o.pitch >= o.width && (reinterpret_cast<uintptr_t>(o.base) & 15) == 0) continue;
        const int64_t pitch = (o.width + 15) / 16 * 16;
        tmp[i] = temp_alloc(g.device, (size_t)(pitch * o.lines), g.stream);
        if (!tmp[i]) { release(); *err = "no device memory for an aligned copy of an operand"; return ACCB_ERR_CUDA; }
        const int rc = launch_repack_rows(o.base, o.pitch, o.lines, o.width, 1, tmp[i], pitch, o.lines, g.stream, err);
        if (rc < 0) { release(); return rc; }
        note_launches(rc);
        launches += rc;
        o.base = tmp[i];
        o.pitch = pitch;
    }

    F8Params p;
    memset(&p, 0, sizeof p);
    p.m = d.m; p.n = d.n;
    p.cs0 = d.c_stride[0]; p.cs1 = d.c_stride[1];
    p.sa = g.a_scales; p.sb = g.b_scales; p.bias = g.bias;
    p.sa_row = g.s.a_stride[0]; p.sa_kb = g.s.a_stride[1]; p.sb_kb = g.s.b_stride[0]; p.sb_col = g.s.b_stride[1];
    p.a_shift = g.s.a_block == 1 ? 0 : 7; p.b_shift = g.s.b_block == 1 ? 0 : 7;
    p.alpha = d.alpha; p.beta = d.beta; p.relu = d.epilogue == ACCB_EPI_RELU;
    p.a_mn = a_dir; p.b_mn = b_dir;
    p.sa_vec = p.sa_kb == 1 && p.sa_row % 4 == 0 && (reinterpret_cast<uintptr_t>(p.sa) & 15) == 0;
    p.sb_vec = p.sb_kb == 1 && p.sb_col % 4 == 0 && (reinterpret_cast<uintptr_t>(p.sb) & 15) == 0;
    p.num_kb = (int)((d.k + kSlabBytes - 1) / kSlabBytes);
    p.status = g.status; p.launch_id = g.launch_id;
    const Options& o = options();
    p.drop_commit = o.gemm_test_drop_commit;
    p.drop_scales = o.gemm_fp8_test_drop_scales;
    p.wait_ns = o.gemm_wait_limit_us > 0 ? (unsigned long long)o.gemm_wait_limit_us * 1000ull : 1000000000ull;

    // Which kernel, and how many slices of K, by estimated microseconds, fitted to measured launches (graph replays).
    //   pair   a round of tiles takes 0.55 a block of K and 6 at its ends; slices add a second pass: 6, and its bytes at 4 TB/s
    //          (fitted with one scale per 128 columns; a scale per column takes about 0.95 a block, which the choice does not know)
    //   tile   a wave of CTAs (two an SM) takes 0.6, 0.7, 0.9 a block for 16, 32, 64 rows, two thirds of it with one CTA an SM;
    //          4 at its ends and 1, 2, 3 more for the sum over a cluster, which only pays within one wave
    // For example 64 x 4096 x 4096: tile with 8 slices 10.4, pair at best 19; 256 x 4096 x 4096: 19 and 20.6; 128 x 32000 x 4096: 62 and 49.
    const int64_t pair_tiles = ((d.m + 255) / 256) * ((d.n + 255) / 256), pair_units = g.num_sms / 2;
    auto pair_cost = [&](int64_t sl) {
        return (double)((pair_tiles * sl + pair_units - 1) / pair_units) * ((double)((p.num_kb + sl - 1) / sl) * 0.55 + 6.0) +
               (sl > 1 ? 6.0 + (double)(sl + 1) * (double)d.m * (double)d.n * 4.0 / 4.0e6 : 0.0);
    };
    int pair_slices = 1;
    for (int sl = 2; sl <= 16 && pair_tiles * sl <= pair_units && sl * 2 <= p.num_kb; ++sl)
        if (pair_cost(sl) < 0.95 * pair_cost(pair_slices)) pair_slices = sl;
    const int tile_bn = d.m <= 16 ? 16 : d.m <= 32 ? 32 : 64;
    const int64_t tiles = ((d.m + tile_bn - 1) / tile_bn) * ((d.n + kRowsX - 1) / kRowsX);
    auto tile_cost = [&](int64_t sl) {
        const int64_t ctas = tiles * sl;
        const double block = (tile_bn == 16 ? 0.6 : tile_bn == 32 ? 0.7 : 0.9) * (ctas <= g.num_sms ? 0.65 : 1.0);
        return (double)((ctas + 2 * g.num_sms - 1) / (2 * g.num_sms)) * (double)((p.num_kb + sl - 1) / sl) * block + 4.0 + (sl > 1 ? (tile_bn == 16 ? 1.0 : tile_bn == 32 ? 2.0 : 3.0) : 0.0);
    };
    int tile_slices = 1;
    for (int sl = 2; sl <= 8 && sl <= p.num_kb && tiles * sl <= 2 * g.num_sms; sl *= 2)
        if (tile_cost(sl) < tile_cost(tile_slices)) tile_slices = sl;
    bool pair = pair_cost(pair_slices) <= tile_cost(tile_slices);
    if (o.gemm_fp8_kernel) pair = o.gemm_fp8_kernel == 1;
    if (d.max_ctas > 0 || a_dir == 1) pair = true;      // persistent; and the tile kernel takes no A that is contiguous along M
    int bn = 256;
    GemmFp8Launch part = g;                  // what the kernel computes: g, or the fp32 sums of the slices of K
    void* sums = nullptr;
    if (pair) {
        p.tiles_m = (int)((d.m + 255) / 256); p.tiles_n = (int)((d.n + 255) / 256);
        p.group_m = 8;
        p.idesc = f8_idesc(d, false, 256, 256, a_dir, b_dir);
        if (pair_tiles > 0x3ffffff) { release(); *err = "too many tiles"; return ACCB_ERR_ARG; }
        // with a bounded grid the units are fewer than the estimate's
        int slices = d.max_ctas > 0 ? 1 : pair_slices;
        if (o.gemm_fp8_slices > 0) slices = o.gemm_fp8_slices < p.num_kb ? o.gemm_fp8_slices : p.num_kb;
        if (slices > 1) sums = temp_alloc(g.device, (size_t)slices * (size_t)d.m * (size_t)d.n * 4, g.stream);
        p.slices = sums ? slices : 1;        // (no memory to spare: one slice)
        if (sums) {
            p.slice_stride = d.m * d.n;
            p.cs0 = d.n; p.cs1 = 1;
            p.alpha = 1.0f; p.beta = 0.0f; p.bias = nullptr; p.relu = 0;
            part.c = sums;
            part.d.c_type = ACCB_F32;
        }
        const int es = elem_size(part.d.c_type);
        p.c_mode = p.cs1 != 1 ? 0 : (p.cs0 * es % 16 == 0 && (reinterpret_cast<uintptr_t>(part.c) & 15) == 0 && p.slice_stride * es % 16 == 0) ? 2 : 1;
    } else {
        bn = tile_bn;
        p.tiles_m = (int)((d.m + bn - 1) / bn); p.tiles_n = (int)((d.n + kRowsX - 1) / kRowsX);
        p.idesc = f8_idesc(d, true, kRowsX, bn, a_dir, b_dir);
        int slices = tile_slices;
        if (o.gemm_fp8_slices > 0) { slices = o.gemm_fp8_slices; while (slices > p.num_kb) slices /= 2; }
        p.slices = slices;
        if (tiles * slices > 0x7fffffff) { release(); *err = "too many tiles"; return ACCB_ERR_ARG; }
    }
    p.plain = p.c_mode == 2 && p.alpha == 1.0f && p.beta == 0.0f && !p.bias && !p.relu;
    CUtensorMap ma, mb;
    if (!make_operand_map(&ma, op[0].base, d.a_type, d.m, d.k, op[0].pitch, pair ? kRowsX : bn, a_dir == 1) ||
        !make_operand_map(&mb, op[1].base, d.b_type, d.n, d.k, op[1].pitch, kRowsX, b_dir == 1)) {
        temp_free(sums, g.stream);
        release();
        *err = "cuTensorMapEncodeTiled failed";
        return ACCB_ERR_CUDA;
    }
    cudaError_t e;
    if (part.d.c_type == ACCB_F32) e = launch_c<float>(part, ma, mb, p, bn);
    else if (part.d.c_type == ACCB_F16) e = launch_c<__half>(part, ma, mb, p, bn);
    else e = launch_c<__nv_bfloat16>(part, ma, mb, p, bn);
    int n = 0;
    if (e == cudaSuccess) {
        note_launches(1);
        n = launches + 1;
        if (sums) {
            const int r = launch_splitk_reduce(sums, p.slices, d, g.c, g.bias, g.stream, err, true);
            n = r < 0 ? r : n + r;
        }
    }
    temp_free(sums, g.stream);
    release();
    if (e != cudaSuccess) { *err = cudaGetErrorString(e); (void)cudaGetLastError(); return ACCB_ERR_CUDA; }
    return n;
}

}  // namespace accb
