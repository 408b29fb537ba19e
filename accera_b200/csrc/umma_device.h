// What the tcgen05 kernels share: bounded mbarrier waits, TMA loads, shared-memory descriptors, tcgen05.mma / commit / ld,
// and the tensor maps of operands.  Included by the kernel files; everything is local to the file that includes it.
#pragma once

#include <cuda.h>

#include "accb_internal.h"

namespace accb {
namespace {

constexpr int kSlabBytes = 128;       // bytes of K per stage row: one 128B swizzle atom
constexpr int kMmaKBytes = 32;        // bytes of K one tcgen05.mma consumes
constexpr uint32_t kPeerMask = 0xFEFFFFFFu;  // clears the CTA-rank bit of a shared::cluster address (rank 0 of a pair)

enum { KIND_F16 = 0, KIND_TF32 = 1, KIND_I8 = 2, KIND_F8F6F4 = 3 };

// where a bounded wait gave up (status word 1, bits 31..24)
enum { SITE_PRODUCER_EMPTY = 1, SITE_MMA_FULL = 2, SITE_MMA_TMEM_EMPTY = 3, SITE_EPI_TMEM_FULL = 4, SITE_COPY_TILE = 5, SITE_EPI_SCALES = 6 };

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count)
{
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive_expect_tx(uint32_t bar, uint32_t bytes)
{
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
// arrive on a barrier addressed in the cluster window (own CTA or the pair's rank 0)
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ uint32_t mbar_try_wait(uint32_t bar, uint32_t parity)
{
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    return ok;
}

__device__ __forceinline__ unsigned long long global_timer_ns()
{
    unsigned long long t;
    asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
    return t;
}

// ACCB_WAIT_INLINE: how a file takes the waiting loop.  Out of line keeps the code small; a kernel that moves registers
// between its warps (setmaxnreg) must not contain calls.
#ifndef ACCB_WAIT_INLINE
#define ACCB_WAIT_INLINE __noinline__
#endif

// Bounded wait.  Returns false when it gave up: after `wait_ns` (a second unless the caller asked otherwise), or as
// soon as a CTA of THIS launch has recorded a failure.  The first failure of a launch is recorded with the launch's
// id; a record left by an earlier launch is not this launch's business and neither stops it nor is overwritten.
__device__ ACCB_WAIT_INLINE bool mbar_wait_slow(uint32_t bar, uint32_t parity, int* status, int launch_id, unsigned long long wait_ns,
                                            int site, int detail)
{
    const unsigned long long t0 = global_timer_ns();
    for (uint32_t spin = 0;; ++spin) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((spin & 0x3f) == 0x3f) {
            if (*(volatile int*)(status + ST_GEMM_ID) == launch_id) return false;   // another CTA of this launch already failed
            if (global_timer_ns() - t0 > wait_ns) {
                atomicAdd(status + ST_GEMM_COUNT, 1);
                if (atomicCAS(status + ST_GEMM_ID, 0, launch_id) == 0) {
                    status[ST_GEMM_SITE] = (site << 24) | (int)(blockIdx.x & 0xffffff);
                    status[ST_GEMM_STEP] = detail;
                }
                return false;
            }
        }
    }
}
struct WaitCtx { int* status; int launch_id; unsigned long long wait_ns; };
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, const WaitCtx& w, int site, int detail)
{
    if (__builtin_expect(mbar_try_wait(bar, parity), 1)) return true;
    return mbar_wait_slow(bar, parity, w.status, w.launch_id, w.wait_ns, site, detail);
}

// L2 eviction-priority policy for the operand loads; 0 = none (the plain load form is used)
__device__ __forceinline__ uint64_t make_l2_policy(int hint)
{
    uint64_t pol = 0;
    if (hint == 1) asm volatile("createpolicy.fractional.L2::evict_first.b64 %0, 1.0;" : "=l"(pol));
    else if (hint == 2) asm volatile("createpolicy.fractional.L2::evict_last.b64 %0, 1.0;" : "=l"(pol));
    return pol;
}

__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, uint64_t pol)
{
    if (pol == 0)
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
            ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
            ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "l"(pol)
            : "memory");
}
// CTA-pair form: the transaction bytes are signalled on the barrier of the pair's rank-0 CTA
__device__ __forceinline__ void tma_load_2d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, uint64_t pol)
{
    if (pol == 0)
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
            ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar & kPeerMask), "r"(c0), "r"(c1)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes.L2::cache_hint [%0], [%1, {%3, %4}], [%2], %5;"
            ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar & kPeerMask), "r"(c0), "r"(c1), "l"(pol)
            : "memory");
}

// Rank-3 forms for batched operands: the box is [1][rows][128 bytes], laid out in shared memory like the rank-2 box
__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}
__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap* map, uint32_t bar, int c0, int c1, int c2)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
        ::"r"(dst), "l"(reinterpret_cast<uint64_t>(map)), "r"(bar & kPeerMask), "r"(c0), "r"(c1), "r"(c2)
        : "memory");
}

// TMA store of one shared-memory box into a C replica (rows / columns outside the tensor are clipped)
__device__ __forceinline__ void tma_store_2d(const CUtensorMap* map, uint32_t src, int c0, int c1)
{
    asm volatile("cp.async.bulk.tensor.2d.global.shared::cta.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(reinterpret_cast<uint64_t>(map)), "r"(src), "r"(c0), "r"(c1) : "memory");
}

// Shared-memory matrix descriptor of a K-major tile stored as rows of 128 bytes
// with the 128-byte swizzle (what TMA writes): 8-row groups are 1024 bytes apart.
__device__ __forceinline__ uint64_t make_smem_desc(uint32_t smem_addr)
{
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3fff);        // start address, 16-byte units
    d |= (uint64_t)1 << 16;                            // leading byte offset (unused with swizzle): 1
    d |= (uint64_t)(1024 >> 4) << 32;                  // stride byte offset between 8-row groups
    d |= (uint64_t)1 << 46;                            // descriptor version of sm_100
    d |= (uint64_t)2 << 61;                            // layout: 128-byte swizzle
    return d;
}

// MN-major operand tile as TMA writes it from an MN-contiguous array: boxes of [k rows][128 bytes of MN] with
// the 128-byte swizzle; 8 k-rows form one 1024-byte swizzle atom (stride byte offset), consecutive 128-byte
// MN blocks are `mn_block_bytes` apart (leading byte offset).
__device__ __forceinline__ uint64_t make_smem_desc_mn(uint32_t smem_addr, uint32_t mn_block_bytes)
{
    uint64_t d = 0;
    d |= (uint64_t)((smem_addr >> 4) & 0x3fff);
    d |= (uint64_t)((mn_block_bytes >> 4) & 0x3fff) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}

template <int KIND, bool TWO_SM>
__device__ __forceinline__ void umma(uint32_t tmem_d, uint64_t adesc, uint64_t bdesc, uint32_t idesc, uint32_t accumulate)
{
    if constexpr (!TWO_SM) {
        if constexpr (KIND == KIND_F16)
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                         "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                         ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
        else if constexpr (KIND == KIND_TF32)
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                         "tcgen05.mma.cta_group::1.kind::tf32 [%0], %1, %2, %3, p;\n\t}"
                         ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
        else if constexpr (KIND == KIND_F8F6F4)
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                         "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                         ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
        else
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                         "tcgen05.mma.cta_group::1.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                         ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
    } else {
        if constexpr (KIND == KIND_F16)
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                         "tcgen05.mma.cta_group::2.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                         ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
        else if constexpr (KIND == KIND_TF32)
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                         "tcgen05.mma.cta_group::2.kind::tf32 [%0], %1, %2, %3, p;\n\t}"
                         ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
        else if constexpr (KIND == KIND_F8F6F4)
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                         "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
                         ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
        else
            asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                         "tcgen05.mma.cta_group::2.kind::i8 [%0], %1, %2, %3, p;\n\t}"
                         ::"r"(tmem_d), "l"(adesc), "l"(bdesc), "r"(idesc), "r"(accumulate) : "memory");
    }
}

// Make `bar` (same offset in every CTA of cta_mask) complete once all tcgen05.mma
// issued so far by this thread have finished reading shared memory / writing TMEM.
template <bool TWO_SM>
__device__ __forceinline__ void umma_commit(uint32_t bar)
{
    if constexpr (!TWO_SM) {
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
    } else {
        const uint16_t mask = 3;
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                     ::"r"(bar), "h"(mask) : "memory");
    }
}

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
        "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr)
        : "memory");
}

// Waits for this thread's outstanding tcgen05.ld.  The registers of the load are passed through the statement so
// that the compiler orders every use of them after the wait (a load may be issued well before its data is needed).
__device__ __forceinline__ void tmem_wait_ld(uint32_t (&r)[32])
{
    asm volatile(
        "tcgen05.wait::ld.sync.aligned;"
        : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
          "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
          "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]),
          "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
        :
        : "memory");
}

__device__ __forceinline__ void cluster_sync_all()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}

__device__ __forceinline__ uint32_t cluster_ctarank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

template <int KIND> struct ElemBytes { static constexpr int value = (KIND == KIND_F16) ? 2 : (KIND == KIND_TF32) ? 4 : 1; };

// Issues the tcgen05.mma instructions that consume one stage (128 bytes of K per row).
//   K-major operand:  advancing K inside the swizzle atom is +32 bytes on the descriptor's start address
//   MN-major operand: one MMA consumes (32 / element bytes) k-rows of 128 bytes each
template <int KIND, bool TWO_SM, bool A_MN, bool B_MN>
__device__ __forceinline__ void issue_stage(uint32_t tmem_d, uint32_t sa, uint32_t sb, uint32_t idesc, bool first_kb)
{
    constexpr int EB = ElemBytes<KIND>::value;
    constexpr uint32_t kBoxBytes = (uint32_t)(kSlabBytes * (kSlabBytes / EB));
    constexpr uint64_t kStepMn = (uint64_t)(((kMmaKBytes / EB) * kSlabBytes) >> 4);
    constexpr uint64_t kStepK = (uint64_t)(kMmaKBytes >> 4);
    const uint64_t adesc = A_MN ? make_smem_desc_mn(sa, kBoxBytes) : make_smem_desc(sa);
    const uint64_t bdesc = B_MN ? make_smem_desc_mn(sb, kBoxBytes) : make_smem_desc(sb);
#pragma unroll
    for (int j = 0; j < kSlabBytes / kMmaKBytes; ++j)
        umma<KIND, TWO_SM>(tmem_d, adesc + (uint64_t)j * (A_MN ? kStepMn : kStepK), bdesc + (uint64_t)j * (B_MN ? kStepMn : kStepK),
                           idesc, (!first_kb || j > 0) ? 1u : 0u);
}

// ---------------------------------------------------------------------------------
// host side
// ---------------------------------------------------------------------------------

typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                  const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                  CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_tiled_fn()
{
    // resolved through the runtime so that the library has no link-time dependency on the driver library
    static EncodeTiledFn fn = [] {
        void* f = nullptr;
        cudaDriverEntryPointQueryResult qres;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &qres) != cudaSuccess ||
            qres != cudaDriverEntryPointSuccess)
            f = nullptr;
        return (EncodeTiledFn)f;
    }();
    return fn;
}

int elem_size(int t)
{
    switch (t) {
    case ACCB_F32: case ACCB_S32: return 4;
    case ACCB_F16: case ACCB_BF16: case ACCB_S16: return 2;
    default: return 1;
    }
}

// K-major operand [rows, k] with `ld` elements between rows; box = 128 bytes of K by box_rows rows
bool make_operand_map(CUtensorMap* map, const void* base, int type, int64_t rows, int64_t k, int64_t ld, int box_rows,
                      bool mn_major = false, int64_t batch = 1, int64_t batch_stride = 0)
{
    EncodeTiledFn enc = encode_tiled_fn();
    if (!enc) return false;
    CUtensorMapDataType dt;
    switch (type) {
    case ACCB_F16: dt = CU_TENSOR_MAP_DATA_TYPE_FLOAT16; break;
    case ACCB_BF16: dt = CU_TENSOR_MAP_DATA_TYPE_BFLOAT16; break;
    case ACCB_F32: dt = CU_TENSOR_MAP_DATA_TYPE_FLOAT32; break;
    default: dt = CU_TENSOR_MAP_DATA_TYPE_UINT8; break;
    }
    const int es = elem_size(type);
    // K-major: [rows][k], k contiguous, box = 128 bytes of k by box_rows rows.
    // MN-major: the array is [k][rows] with `rows` (M or N) contiguous; box = 128 bytes of M/N by (128 / es) k-rows.
    // Batched (batch > 1 with a non-zero batch stride): a third, outermost dimension walks the problems; the box
    // is one problem thick, so it lands in shared memory exactly like the rank-2 box.
    const bool rank3 = batch > 1 && batch_stride > 0;
    cuuint64_t dims[3] = { (cuuint64_t)(mn_major ? rows : k), (cuuint64_t)(mn_major ? k : rows), (cuuint64_t)batch };
    cuuint64_t strides[2] = { (cuuint64_t)(ld * es), (cuuint64_t)(batch_stride * es) };
    cuuint32_t box[3] = { (cuuint32_t)(kSlabBytes / es), (cuuint32_t)(mn_major ? kSlabBytes / es : box_rows), 1 };
    cuuint32_t estr[3] = { 1, 1, 1 };
    CUresult r = enc(map, dt, rank3 ? 3 : 2, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS;
}

}  // namespace
}  // namespace accb
