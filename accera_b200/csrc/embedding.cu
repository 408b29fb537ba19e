// Token table for sm_100a: lookup with a scale, and its gradient by sorted tokens.
//
//   lookup     rows[t, :]  = scale * table[ids[t], :]
//   gradient   table[v, :] = beta * table[v, :] + scale * sum of rows[t, :] over the tokens t with ids[t] == v
//
// Both are HBM traffic: a lookup reads and writes every row once, a gradient reads every row once and writes the table
// once.  The gradient's additions have to happen in an order that does not depend on the run, so the tokens are sorted by id
// first (stably: a word's rows are added in token order) and sums are cut only at places that the sorted list fixes.
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

#include "accb_internal.h"

namespace accb {
namespace {

template <typename T, int E> struct alignas(E * sizeof(T) > 16 ? 16 : E * sizeof(T)) Vec { T v[E]; };

// a store that should not displace what is read again (the table) from L2
template <typename T, int E>
__device__ __forceinline__ void store_streaming(T* dst, const Vec<T, E>& x)
{
    constexpr int kBytes = E * (int)sizeof(T);
    if constexpr (kBytes % 16 == 0) {
        const uint4* w = reinterpret_cast<const uint4*>(&x);
#pragma unroll
        for (int i = 0; i < kBytes / 16; ++i) __stcs(reinterpret_cast<uint4*>(dst) + i, w[i]);
    } else if constexpr (kBytes == 8) __stcs(reinterpret_cast<uint2*>(dst), *reinterpret_cast<const uint2*>(&x));
    else *reinterpret_cast<Vec<T, E>*>(dst) = x;
}

// ---------------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------------

struct LookupParams {
    int64_t table_stride, rows_stride;
    int64_t tokens;
    uint32_t vocab;
    uint32_t vecs;              // vectors in a row
    int shift;                  // log2 of the threads that share a row
    uint32_t parts;             // blocks that share a row: each thread takes U vectors of it; 0: one vector of U rows
    float scale;
    int id_bytes;
    int launch_id;
};

constexpr int kLookupBlock = 256;

__device__ __forceinline__ int64_t load_id(const void* ids, int64_t t, int id_bytes)
{
    return id_bytes == 8 ? __ldg((const long long*)ids + t) : (int64_t)__ldg((const int*)ids + t);
}

// A thread moves U vectors, with all loads in flight: U of its row, or, where a row has no more vectors than threads, one
// each of U rows.  Threads find their row without a division.  U = 2 for vectors of 16 bytes, the loads in flight coming from
// eight resident blocks an SM: 16384 rows of 4096 bf16 take 40 us, 44 with a division a vector, 58 with four vectors a thread (and
// three blocks an SM).  U = 8 for rows that have to go by single elements: 9968 rows of 3283 fp16 take 93 us, with U = 2 142.
template <typename TT, typename TR, int E, int U>
__global__ void __launch_bounds__(kLookupBlock, U == 2 ? 8 : 4)
embedding_kernel(const TT* __restrict__ table, const void* __restrict__ ids, TR* __restrict__ rows, int* __restrict__ status,
                 const LookupParams p)
{
    pdl_enter();
    const uint32_t x = threadIdx.x & ((1u << p.shift) - 1u);
    const int groups = kLookupBlock >> p.shift, sub = threadIdx.x >> p.shift;
    int64_t row0;
    uint32_t vec0, vec_step;
    int row_step;
    if (p.parts) {
        row0 = (int64_t)(blockIdx.x / p.parts) * groups + sub;
        row_step = 0;
        vec0 = x + ((U * (blockIdx.x % p.parts)) << p.shift);
        vec_step = 1u << p.shift;
    } else {
        row0 = (int64_t)blockIdx.x * (U * groups) + sub;
        row_step = groups;
        vec0 = x;
        vec_step = 0;
    }
    Vec<TT, E> v[U];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t row = row0 + u * row_step;
        const uint32_t vec = vec0 + u * vec_step;
        ok[u] = false;
        if (row < p.tokens && vec < p.vecs) {
            const int64_t id = load_id(ids, row, p.id_bytes);
            ok[u] = (uint64_t)id < p.vocab;
            if (!ok[u] && vec == 0) { atomicAdd(status + ST_EMBED_COUNT, 1); status[ST_EMBED_ID] = p.launch_id; }
            if (ok[u]) v[u] = *reinterpret_cast<const Vec<TT, E>*>(table + id * p.table_stride + vec * (int64_t)E);
        }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const int64_t row = row0 + u * row_step;
        const uint32_t vec = vec0 + u * vec_step;
        if (row >= p.tokens || vec >= p.vecs) continue;
        Vec<TR, E> y;
#pragma unroll
        for (int e = 0; e < E; ++e) y.v[e] = ok[u] ? (TR)((float)v[u].v[e] * p.scale) : (TR)0.0f;
        store_streaming<TR, E>(rows + row * p.rows_stride + vec * (int64_t)E, y);
    }
}

template <typename TT, typename TR>
cudaError_t launch_lookup(const EmbeddingLaunch& l, const void* table, void* rows)
{
    const accb_embedding_desc& d = l.d;
    // elements per vector: 16 bytes on the wider side; single elements when rows do not all start on a vector boundary
    constexpr int E = 16 / (int)(sizeof(TT) > sizeof(TR) ? sizeof(TT) : sizeof(TR));
    auto aligned = [](const void* p, int64_t stride, int64_t es) { return (reinterpret_cast<uintptr_t>(p) % (E * es)) == 0 && stride % E == 0; };
    const bool vec = d.dim % E == 0 && aligned(table, d.table_stride, sizeof(TT)) && aligned(rows, d.rows_stride, sizeof(TR));
    LookupParams p;
    p.table_stride = d.table_stride; p.rows_stride = d.rows_stride;
    p.tokens = d.tokens;
    p.vocab = (uint32_t)d.vocab;
    p.vecs = (uint32_t)(vec ? d.dim / E : d.dim);
    p.scale = d.scale; p.id_bytes = d.id_bytes; p.launch_id = l.launch_id;
    const uint32_t each = vec ? 2 : 8;
    // threads to a row: the power of two that leaves the fewest of them idle, the larger one of equals; all of a block for
    // long rows of single elements, whose parts by fewer threads share too many lines (3283 fp16: 283 us by 64 threads)
    p.shift = 0;
    uint32_t best = 0;
    for (int shift = !vec && p.vecs > 1024 ? 8 : 0; shift <= 8; ++shift) {
        const uint32_t t = 1u << shift, turns = (p.vecs + t - 1) / t, used = (uint32_t)((uint64_t)p.vecs * 1024 / ((uint64_t)(turns == 1 ? 1 : (turns + each - 1) / each * each) * t));
        if (used >= best) { best = used; p.shift = shift; }
    }
    const uint32_t turns = (p.vecs + (1u << p.shift) - 1) >> p.shift;
    p.parts = turns == 1 ? 0 : (turns + each - 1) / each;
    const int64_t groups = kLookupBlock >> p.shift;
    const int64_t blocks = p.parts ? (d.tokens + groups - 1) / groups * p.parts : (d.tokens + each * groups - 1) / (each * groups);
    if (blocks > 0x7fffffff) return cudaErrorInvalidConfiguration;
    const dim3 grid((unsigned)blocks), block(kLookupBlock);
    return vec ? launch_pdl(embedding_kernel<TT, TR, E, 2>, grid, block, l.stream, (const TT*)table, l.ids, (TR*)rows, l.status, p)
               : launch_pdl(embedding_kernel<TT, TR, 1, 8>, grid, block, l.stream, (const TT*)table, l.ids, (TR*)rows, l.status, p);
}

// ---------------------------------------------------------------------------------
// gradient, step 1: tokens sorted by id
// ---------------------------------------------------------------------------------
// A stable radix sort of (id, token) pairs by one cluster of up to eight CTAs in one launch: CTA r owns the r-th part of
// the list, each of its warps a run of it.  A pass counts the run's digits per warp (shared memory), turns the counts
// into places (digit by digit over all CTAs through distributed shared memory, then over the CTA's warps) and moves the
// pairs, 32 at a time in list order, so that equal digits keep their order.  A padding or out-of-range id becomes the
// key `vocab`, which sorts behind every word and is left out by step 2.

constexpr int kSortThreads = 1024;
constexpr int kSortWarps = kSortThreads / 32;
constexpr int kMaxDigitBits = 9;
constexpr int kMaxBins = 1 << kMaxDigitBits;
constexpr int kSortCluster = 8;
constexpr size_t kSortSmem = ((size_t)kSortWarps * kMaxBins + 2 * kMaxBins + kSortWarps) * 4;

// An id outside the table is a mistake unless it is the padding id; a negative padding_id stands for none, so that no id equals it
__device__ __forceinline__ bool bad_id(int64_t id, int vocab, int64_t padding_id)
{
    return (uint64_t)id >= (uint64_t)vocab && (id < 0 || id != padding_id);
}

struct SortParams {
    int n;
    int vocab;
    int64_t padding_id;
    int id_bytes;
    int passes, digit_bits;
    int launch_id;
};

__device__ __forceinline__ void cluster_barrier()
{
    asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
__device__ __forceinline__ uint32_t cluster_rank() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ uint32_t cluster_size() { uint32_t r; asm volatile("mov.u32 %0, %%cluster_nctarank;" : "=r"(r)); return r; }
__device__ __forceinline__ int load_remote(const int* own_copy, uint32_t rank)
{
    uint32_t a;
    int v;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(a) : "r"((uint32_t)__cvta_generic_to_shared(own_copy)), "r"(rank));
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}

// One digit of 32 items of a warp: the lanes with the same digit, inactive lanes in a group of their own
__device__ __forceinline__ uint32_t same_digit(int digit, bool active) { return __match_any_sync(0xffffffffu, active ? digit : -1); }

// keys[0], tokens[0] and keys[1], tokens[1]: two buffers of n entries; the result is in buffer (passes - 1) & 1
__device__ void sort_tokens(const void* ids, int* keys0, int* tokens0, int* keys1, int* tokens1, int* status, const SortParams& p, int* smem)
{
    int (*hist)[kMaxBins] = reinterpret_cast<int (*)[kMaxBins]>(smem);      // per warp: counts, then next free place
    int* cta_count = smem + kSortWarps * kMaxBins;
    int* bin_base = cta_count + kMaxBins;
    int* warp_sum = bin_base + kMaxBins;
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    const int rank = (int)cluster_rank(), ctas = (int)cluster_size();
    const int runs = ctas * kSortWarps;
    const int run_len = ((p.n + runs - 1) / runs + 31) / 32 * 32;
    const int64_t run_begin = (int64_t)(rank * kSortWarps + warp) * run_len;
    const int begin = (int)(run_begin < p.n ? run_begin : p.n);
    const int end = p.n - begin < run_len ? p.n : begin + run_len;
    const int bins = 1 << p.digit_bits;
    int bad = 0;
    for (int pass = 0; pass < p.passes; ++pass) {
        const int* src_k = (pass & 1) ? keys0 : keys1;
        const int* src_t = (pass & 1) ? tokens0 : tokens1;
        int* dst_k = (pass & 1) ? keys1 : keys0;
        int* dst_t = (pass & 1) ? tokens1 : tokens0;
        const int shift = pass * p.digit_bits;
        auto key_at = [&](int i) -> int {
            if (pass > 0) return __ldcg(src_k + i);
            const int64_t id = load_id(ids, i, p.id_bytes);
            return ((uint64_t)id < (uint64_t)p.vocab && id != p.padding_id) ? (int)id : p.vocab;
        };
        for (int b = threadIdx.x; b < kSortWarps * kMaxBins; b += kSortThreads) smem[b] = 0;
        __syncthreads();
        for (int i = begin + lane; i < end; i += 32) {
            if (pass == 0) {
                const int64_t id = load_id(ids, i, p.id_bytes);
                bad += bad_id(id, p.vocab, p.padding_id);
            }
            atomicAdd(&hist[warp][(key_at(i) >> shift) & (bins - 1)], 1);
        }
        __syncthreads();
        // counts -> places among this CTA's items of the digit
        if (threadIdx.x < kMaxBins) {
            int sum = 0;
            for (int w = 0; w < kSortWarps; ++w) {
                const int c = hist[w][threadIdx.x];
                hist[w][threadIdx.x] = sum;
                sum += c;
            }
            cta_count[threadIdx.x] = sum;
        }
        cluster_barrier();
        int all = 0, before = 0;
        if (threadIdx.x < bins)
            for (int r = 0; r < ctas; ++r) {
                const int c = load_remote(cta_count + threadIdx.x, r);
                if (r < rank) before += c;
                all += c;
            }
        // exclusive scan of the digit totals over the first kMaxBins threads
        int scan = all;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, scan, o); if (lane >= o) scan += v; }
        if (lane == 31) warp_sum[warp] = scan;
        __syncthreads();
        if (threadIdx.x < bins) {
            int base = 0;
            for (int w = 0; w < warp; ++w) base += warp_sum[w];
            bin_base[threadIdx.x] = base + scan - all + before;
        }
        __syncthreads();
        for (int b = threadIdx.x; b < kSortWarps * kMaxBins; b += kSortThreads) smem[b] += bin_base[b % kMaxBins];
        __syncthreads();
        for (int i0 = begin; i0 < end; i0 += 32) {
            const int i = i0 + lane;
            const bool active = i < end;
            int key = 0, token = 0;
            if (active) { key = key_at(i); token = pass > 0 ? __ldcg(src_t + i) : i; }
            const int digit = (key >> shift) & (bins - 1);
            const uint32_t peers = same_digit(digit, active);
            if (active) {
                const int place = hist[warp][digit] + __popc(peers & ((1u << lane) - 1));
                dst_k[place] = key;
                dst_t[place] = token;
            }
            __syncwarp();
            if (active && (peers >> lane) == 1u) hist[warp][digit] += __popc(peers);      // the highest lane of each digit
            __syncwarp();
        }
        // the pairs are visible to the whole cluster before the next pass reads them; nobody still reads cta_count
        __threadfence();
        cluster_barrier();
    }
    for (int o = 16; o; o >>= 1) bad += __shfl_down_sync(0xffffffffu, bad, o);
    if (lane == 0 && bad) { atomicAdd(status + ST_EMBED_COUNT, bad); status[ST_EMBED_ID] = p.launch_id; }
}

__global__ void __launch_bounds__(kSortThreads, 1)
sort_tokens_kernel(const void* __restrict__ ids, int* keys0, int* tokens0, int* keys1, int* tokens1, int* long_words, int* status, const SortParams p)
{
    extern __shared__ int smem[];
    pdl_enter();
    if (blockIdx.x == 0 && threadIdx.x == 0) *long_words = 0;
    sort_tokens(ids, keys0, tokens0, keys1, tokens1, status, p, smem);
}

// ---------------------------------------------------------------------------------
// gradient: words without a token
// ---------------------------------------------------------------------------------
// They get their final value, zero or beta times the old one, from blocks behind those of the sums in the same grid.

struct ClearParams {
    int64_t stride;
    int dim;
    int vec;                     // rows are whole 16-byte vectors, 16-byte aligned
    float beta;
    int ctas;                    // CTA i owns rows i, i + ctas, ..., so that all CTAs together write one stretch of memory after the other
};

// One row's value by per_row threads, x of them this one
template <typename TT>
__device__ __forceinline__ void clear_row(TT* row, int x, int per_row, const ClearParams& c)
{
    constexpr int V = 16 / (int)sizeof(TT);
    if (c.beta != 0.0f) {
        for (int i = x; i < c.dim; i += per_row) row[i] = (TT)(c.beta * (float)row[i]);
    } else if (c.vec) {
        for (int v = x; v < c.dim / V; v += per_row) reinterpret_cast<uint4*>(row)[v] = make_uint4(0u, 0u, 0u, 0u);
    } else {
        // a row that starts or ends within a vector: its whole vectors, and the elements before and after them
        const int head = min(c.dim, (int)((16 - (reinterpret_cast<uintptr_t>(row) & 15)) & 15) / (int)sizeof(TT)), vecs = (c.dim - head) / V;
        for (int v = x; v < vecs; v += per_row) reinterpret_cast<uint4*>(row + head)[v] = make_uint4(0u, 0u, 0u, 0u);
        const int tail = head + vecs * V;
        if (x < head) row[x] = (TT)0.0f;
        if (tail + x < c.dim && x < V) row[tail + x] = (TT)0.0f;
    }
}
// as many threads side by side as a row has vectors, a power of two from 32 to `most`
template <typename TT>
__device__ __forceinline__ int clear_width(const ClearParams& c, int most)
{
    constexpr int V = 16 / (int)sizeof(TT);
    const int width = c.beta == 0.0f ? (c.dim + V - 1) / V : c.dim;
    int per_row = 32;
    while (per_row < most && per_row < width) per_row *= 2;
    return per_row;
}

// seen: one bit of shared memory for each of the CTA's rows
template <typename TT, int kThreads>
__device__ __forceinline__ void clear_rows(TT* table, const void* ids, int part, const SortParams& p, const ClearParams& c, uint32_t* seen)
{
    if (part >= p.vocab) return;
    const int rows = (int)(((int64_t)p.vocab - part + c.ctas - 1) / c.ctas);
    for (int i = threadIdx.x; i < (rows + 31) / 32; i += kThreads) seen[i] = 0u;
    __syncthreads();
#pragma unroll 8
    for (int i = threadIdx.x; i < p.n; i += kThreads) {
        const int64_t id = load_id(ids, i, p.id_bytes);
        if ((uint64_t)id >= (uint64_t)p.vocab || id == p.padding_id) continue;
        const uint32_t at = (uint32_t)id / (uint32_t)c.ctas;
        if ((uint32_t)id - at * (uint32_t)c.ctas == (uint32_t)part) atomicOr(seen + at / 32, 1u << (at % 32));
    }
    __syncthreads();
    // the CTA writes one stretch of memory after the other
    const int per_row = clear_width<TT>(c, 256);
    const int sub = threadIdx.x / per_row, x = threadIdx.x % per_row;
    const int groups = kThreads / per_row;                    // a power of two, at most 16: group g takes every groups-th row
    uint32_t every = 0u;
    for (int i = sub; i < 32; i += groups) every |= 1u << i;
    for (int w = 0; w * 32 < rows; ++w) {
        uint32_t todo = ~seen[w] & every & (rows - w * 32 < 32 ? (1u << (rows - w * 32)) - 1u : 0xffffffffu);
        while (todo) {
            const int r = w * 32 + __ffs(todo) - 1;
            todo &= todo - 1u;
            clear_row<TT>(table + (part + (int64_t)r * c.ctas) * c.stride, x, per_row, c);
        }
    }
}

// The first place from `lo` of the sorted list whose key is not below `word`, found by a whole warp with 32 probes a step
__device__ __forceinline__ int first_place(const int* keys, int lo, int n, int word)
{
    int hi = n;
    while (lo < hi) {
        const int step = (hi - lo + 31) / 32;
        const int64_t at = lo + (int64_t)(threadIdx.x % 32) * step;
        const int below = __popc(__ballot_sync(0xffffffffu, at < hi && keys[at] < word));
        // probe `below` is not below the word (or behind the range), the one before it is
        if (below < 32) hi = (int)min((int64_t)hi, lo + (int64_t)below * step);
        if (below > 0) lo += (below - 1) * step + 1;
    }
    return lo;
}

// The clearing of up to 32 rows from the sorted list.  Every warp finds the first place that is not before them and the words
// in the 32 places from there; where those places do not reach the rows' end, each lane looks for its own word.
template <typename TT, int kThreads>
__device__ __forceinline__ void clear_unlisted(TT* table, const int* keys, int n, int first, int rows, int vocab, const ClearParams& c)
{
    const int lane = threadIdx.x % 32;
    rows = min(rows, vocab - first);
    int lo = first_place(keys, 0, n, first);
    const int key = lo + lane < n ? keys[lo + lane] : vocab;
    uint32_t listed = __reduce_or_sync(0xffffffffu, key - first < rows ? 1u << (key - first) : 0u);
    if (__shfl_sync(0xffffffffu, key, 31) < first + rows) {
        const int word = first + lane;
        int hi = n;
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (keys[mid] < word) lo = mid + 1; else hi = mid;
        }
        listed = __ballot_sync(0xffffffffu, lo < n && keys[lo] == word);
    }
    uint32_t todo = ~listed & (rows < 32 ? (1u << rows) - 1u : 0xffffffffu);
    const int per_row = clear_width<TT>(c, kThreads), sub = threadIdx.x / per_row, x = threadIdx.x % per_row;
    for (int at = 0; todo; ++at, todo &= todo - 1u)
        if (at % (kThreads / per_row) == sub) clear_row<TT>(table + (int64_t)(first + __ffs(todo) - 1) * c.stride, x, per_row, c);
}

// ---------------------------------------------------------------------------------
// gradient, step 2: sums over the sorted list
// ---------------------------------------------------------------------------------
// A block owns kChunk places of the list times a slab of columns, a thread one vector of columns.  A word with up to
// kChunk tokens belongs to the chunk it starts in, however far it runs into the next one; a longer ("long") word is cut
// at chunk borders and its pieces' fp32 sums go to `partial`, two slots a chunk (slot 0: the piece of a word that began
// in an earlier chunk, slot 1: of one that begins here and runs on), which step 3 adds in chunk order.  So the order
// of additions is fixed by the sorted list, and only words that are long anyway pay for a second pass.

constexpr int kChunk = 32;
constexpr int kSumThreads = 128;
// A thread has two rows on their way with sixteen blocks an SM, eight with four blocks.  Up to kSumDeep blocks of sums an SM, the
// time of one block counts: 6271 tokens of 112 columns took 47 us with two rows, 38 with eight; beyond, the blocks do each
// other's waiting (16384 tokens of 4096 columns: 132 us with two rows, 141 with eight).
constexpr int kSumDeep = 6;
// The blocks behind those of the sums give words without a token their value, as many rows each as make kClearBytes, so
// that all of them together write one stretch of memory after the other and the sums' loads have stores beside them: 16384
// tokens into 32000 x 4096 fp32 take 137 us at 32 KB a block, 197 at 512 KB, 160 with the clearing beside the sort instead.
constexpr int64_t kClearBytes = 32768;

struct SumParams {
    int n, vocab, dim;
    int64_t table_stride, rows_stride;
    float scale, beta;
    int chunks;
    int slabs;
    int clear_rows;              // of words without a token that a block behind those of the sums looks after: up to 32
};

template <typename TT, int E>
__device__ __forceinline__ void write_sum(TT* table, int64_t word, int64_t stride, int col, const float (&acc)[E], float scale, float beta)
{
    Vec<TT, E>* dst = reinterpret_cast<Vec<TT, E>*>(table + word * stride + col);
    Vec<TT, E> y;
    if (beta != 0.0f) {
        const Vec<TT, E> old = *dst;
#pragma unroll
        for (int e = 0; e < E; ++e) y.v[e] = (TT)fmaf(beta, (float)old.v[e], scale * acc[e]);
    } else {
#pragma unroll
        for (int e = 0; e < E; ++e) y.v[e] = (TT)(scale * acc[e]);
    }
    *dst = y;
}

template <typename TT, typename TR, int E, int U>
__global__ void __launch_bounds__(kSumThreads, U == 2 ? 16 : 4)
sum_rows_kernel(const TR* __restrict__ rows, const int* __restrict__ keys, const int* __restrict__ tokens, TT* __restrict__ table,
                float* __restrict__ partial, int* __restrict__ long_words, const SumParams p, const ClearParams c)
{
    pdl_enter();
    if ((int)blockIdx.x >= p.chunks * p.slabs) {
        clear_unlisted<TT, kSumThreads>(table, keys, p.n, ((int)blockIdx.x - p.chunks * p.slabs) * p.clear_rows, p.clear_rows, p.vocab, c);
        return;
    }
    const int chunk = blockIdx.x / p.slabs, slab = blockIdx.x % p.slabs;
    const int i0 = chunk * kChunk, i1 = min(p.n, i0 + kChunk);
    __shared__ int key[3 * kChunk + 1];                      // places i0 - kChunk ..
    __shared__ int64_t row_at[2 * kChunk];                   // places i0 ..: where the token's row begins
    for (int j = threadIdx.x; j < 3 * kChunk; j += kSumThreads) {
        const int i = i0 - kChunk + j;
        key[j] = (i >= 0 && i < p.n) ? keys[i] : -1;
        if (j >= kChunk) row_at[j - kChunk] = i < p.n ? (int64_t)tokens[i] * p.rows_stride : 0;
    }
    if (threadIdx.x == 0) key[3 * kChunk] = -1;
    __syncthreads();
    const int* k = key + kChunk;                             // k[i] = key of place i0 + i
    const int len = i1 - i0;
    // Lane l of every warp looks at places l - kChunk, l and l + kChunk of the chunk; ballots give the runs of equal keys.
    static_assert(kChunk == 32, "one place a lane");
    const int lane = threadIdx.x % 32;
    const int k_first = k[0], k_last = k[len - 1];
    const uint32_t before = __ballot_sync(0xffffffffu, k[lane - kChunk] == k_first);
    const uint32_t same_first = __ballot_sync(0xffffffffu, k[lane] == k_first), beyond_first = __ballot_sync(0xffffffffu, k[lane + kChunk] == k_first);
    const uint32_t same_last = __ballot_sync(0xffffffffu, k[lane] == k_last), beyond_last = __ballot_sync(0xffffffffu, k[lane + kChunk] == k_last);
    auto ones = [](uint32_t m) { return m == 0xffffffffu ? 32 : __ffs(~m) - 1; };            // consecutive ones from bit 0
    const int back = before == 0xffffffffu ? 32 : __clz(~before);
    const int ahead_first = same_first == 0xffffffffu ? 32 + ones(beyond_first) : ones(same_first);
    // the piece of a word that began earlier: skipped when that word is short (its first chunk takes it all)
    int first = 0;
    bool first_long = false;
    if (back > 0) {
        first_long = back + ahead_first > kChunk;
        if (!first_long) first = ahead_first < len ? ahead_first : len;
    }
    // the word that runs past the chunk's end: taken to its end when short, to the border when long
    int last = len;
    bool last_long = false;
    if (first < len && len == kChunk && (beyond_last & 1u)) {
        const uint32_t other = ~same_last;                                                    // the list is sorted
        const int start = other ? 32 - __clz(other) : 0;
        const int end = kChunk + ones(beyond_last);
        if (start > 0 || back == 0) {
            last_long = end - start > kChunk;
            if (!last_long) last = end;
        }
    }
    last_long = last_long && k_last < p.vocab;
    if (threadIdx.x == 0 && slab == 0 && last_long) long_words[1 + atomicAdd(long_words, 1)] = chunk;
    // ids that stand for no word come last
    const int valid = __popc(__ballot_sync(0xffffffffu, (uint32_t)k[lane] < (uint32_t)p.vocab)) +
                      __popc(__ballot_sync(0xffffffffu, (uint32_t)k[lane + kChunk] < (uint32_t)p.vocab));
    last = min(last, valid);
    // places whose word ends there, the next one being another's
    const uint64_t ends = (uint64_t)__ballot_sync(0xffffffffu, k[lane] != k[lane + 1]) | (uint64_t)__ballot_sync(0xffffffffu, k[lane + kChunk] != k[lane + kChunk + 1]) << 32;
    const int col = (slab * kSumThreads + threadIdx.x) * E;
    if (col >= p.dim || first >= last) return;
    // U rows are always on their way: a place's register takes the row U places on as soon as it is added
    const TR* src = rows + col;
    Vec<TR, E> x[U];
#pragma unroll
    for (int u = 0; u < U; ++u) x[u] = *reinterpret_cast<const Vec<TR, E>*>(src + row_at[min(first + u, last - 1)]);
    float acc[E] = {};
    for (int j0 = first; j0 < last; j0 += U) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int j = j0 + u;
            if (j >= last) break;
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += (float)x[u].v[e];
            if (j + U < last) x[u] = *reinterpret_cast<const Vec<TR, E>*>(src + row_at[j + U]);
            if (j + 1 == last || (ends >> j & 1u)) {
                const bool head = first_long && k[j] == k_first, tail = last_long && j + 1 == last;
                if (head || tail) {
                    Vec<float, E> y;
#pragma unroll
                    for (int e = 0; e < E; ++e) y.v[e] = acc[e];
                    float* dst = partial + ((int64_t)chunk * 2 + (head ? 0 : 1)) * p.dim + col;
                    if constexpr (E == 1) *dst = acc[0];
                    else *reinterpret_cast<Vec<float, E>*>(dst) = y;
                } else {
                    write_sum<TT, E>(table, k[j], p.table_stride, col, acc, p.scale, p.beta);
                }
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = 0.0f;
            }
        }
    }
}

// step 3: the pieces of the long words.  long_words[0] of them begin in chunks long_words[1 ..] (in any order: each is a sum
// of its own).  A block takes kJoinCols columns of one word at a time: kJoinLanes threads a column add every kJoinLanes-th
// piece, and their sums are added in lane order.
constexpr int kJoinCols = 32, kJoinLanes = 8;

template <typename TT, int E>
__global__ void __launch_bounds__(kJoinCols * kJoinLanes)
join_rows_kernel(const float* __restrict__ partial, const int* __restrict__ keys, const int* __restrict__ long_words, TT* __restrict__ table,
                 const SumParams p)
{
    pdl_enter();
    __shared__ Vec<float, E> part[kJoinLanes][kJoinCols];
    const int x = threadIdx.x % kJoinCols, y = threadIdx.x / kJoinCols;
    const int col_blocks = (p.dim + kJoinCols * E - 1) / (kJoinCols * E);
    const int64_t total = (int64_t)long_words[0] * col_blocks;
    for (int64_t w = blockIdx.x; w < total; w += gridDim.x) {
        const int chunk = long_words[1 + w / col_blocks], col = ((int)(w % col_blocks) * kJoinCols + x) * E;
        const int word = keys[chunk * kChunk + kChunk - 1];
        const int last_chunk = (first_place(keys, chunk * kChunk + kChunk, p.n, word + 1) - 1) / kChunk;
        Vec<float, E> acc = {};
        if (col < p.dim) {
#pragma unroll 8
            for (int c = chunk + y; c <= last_chunk; c += kJoinLanes) {
                const Vec<float, E> v = *reinterpret_cast<const Vec<float, E>*>(partial + ((int64_t)c * 2 + (c == chunk ? 1 : 0)) * p.dim + col);
#pragma unroll
                for (int e = 0; e < E; ++e) acc.v[e] += v.v[e];
            }
        }
        part[y][x] = acc;
        __syncthreads();
        if (y == 0 && col < p.dim) {
            float sum[E] = {};
#pragma unroll
            for (int l = 0; l < kJoinLanes; ++l)
#pragma unroll
                for (int e = 0; e < E; ++e) sum[e] += part[l][x].v[e];
            write_sum<TT, E>(table, word, p.table_stride, col, sum, p.scale, p.beta);
        }
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------
// gradient of few tokens: one launch, no workspace
// ---------------------------------------------------------------------------------
// Up to kFewTokens tokens, every block can look at all of them.  The block of (token, slab of columns) does nothing unless
// it is its word's first token; else it collects the word's tokens in order and adds their rows: a thread one vector of
// columns, or, for more than kFewSplit tokens, kFewLanes threads a vector, each a kFewLanes-th of the list, whose
// sums are added in lane order.  Blocks behind those give words without a token their value.
// Above kFewTokens the list is sorted: 1598 tokens of 144 columns take 18 us here and 46 sorted, 3708 of 128 columns 45 and 31.
constexpr int kFewTokens = 2048, kFewThreads = 256, kFewLanes = 8, kFewSplit = 16, kFewUnroll = 8;

template <typename TT, typename TR, int E, int kRounds>
__global__ void __launch_bounds__(kFewThreads)
few_tokens_kernel(const TR* __restrict__ rows, const void* __restrict__ ids, TT* __restrict__ table, int* __restrict__ status, const SortParams sp,
                  const ClearParams c, const SumParams p)
{
    pdl_enter();
    constexpr int kWarps = kFewThreads / 32;
    __shared__ uint32_t list[kRounds * kFewThreads];
    __shared__ int count[(kRounds * kWarps + 31) / 32 * 32];        // of a round and warp, in list order
    __shared__ float part[kFewLanes][kFewThreads / kFewLanes][E + 1];
    const int sum_blocks = sp.n * p.slabs;
    if ((int)blockIdx.x >= sum_blocks) {
        clear_rows<TT, kFewThreads>(table, ids, (int)blockIdx.x - sum_blocks, sp, c, list);
        return;
    }
    const int token = blockIdx.x / p.slabs, slab = blockIdx.x % p.slabs;
    const int64_t word = load_id(ids, token, sp.id_bytes);
    if ((uint64_t)word >= (uint64_t)sp.vocab || word == sp.padding_id) {
        if (bad_id(word, sp.vocab, sp.padding_id) && slab == 0 && threadIdx.x == 0) { atomicAdd(status + ST_EMBED_COUNT, 1); status[ST_EMBED_ID] = sp.launch_id; }
        return;
    }
    const int warp = threadIdx.x / 32, lane = threadIdx.x % 32;
    uint32_t mine[kRounds];
    bool earlier = false;
#pragma unroll
    for (int r = 0; r < kRounds; ++r) {
        const int i = r * kFewThreads + threadIdx.x;
        const bool same = i < sp.n && load_id(ids, i, sp.id_bytes) == word;
        earlier |= same && i < token;
        mine[r] = __ballot_sync(0xffffffffu, same);
        if (lane == 0) count[r * kWarps + warp] = __popc(mine[r]);
    }
    if (__syncthreads_or(earlier)) return;
    // every warp adds the counts up for itself
    int n = 0;
#pragma unroll
    for (int r0 = 0; r0 < kRounds; r0 += 32 / kWarps) {
        const int own = r0 * kWarps + lane < kRounds * kWarps ? count[r0 * kWarps + lane] : 0;
        int sum = own;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) { const int v = __shfl_up_sync(0xffffffffu, sum, o); if (lane >= o) sum += v; }
#pragma unroll
        for (int r = r0; r < kRounds && r < r0 + 32 / kWarps; ++r) {
            const int before = n + __shfl_sync(0xffffffffu, sum - own, (r - r0) * kWarps + warp);
            if (mine[r] >> lane & 1u) list[before + __popc(mine[r] & ((1u << lane) - 1u))] = (uint32_t)(r * kFewThreads + threadIdx.x);
        }
        n += __shfl_sync(0xffffffffu, sum, 31);
    }
    __syncthreads();
    if (n <= kFewSplit) {
        const int col = (slab * kFewThreads + threadIdx.x) * E;
        if (col >= p.dim) return;
        float acc[E] = {};
        for (int j0 = 0; j0 < n; j0 += kFewUnroll) {
            Vec<TR, E> x[kFewUnroll];
#pragma unroll
            for (int u = 0; u < kFewUnroll; ++u)
                if (j0 + u < n) x[u] = *reinterpret_cast<const Vec<TR, E>*>(rows + (int64_t)list[j0 + u] * p.rows_stride + col);
#pragma unroll
            for (int u = 0; u < kFewUnroll; ++u)
                if (j0 + u < n) {
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[e] += (float)x[u].v[e];
                }
        }
        write_sum<TT, E>(table, word, p.table_stride, col, acc, p.scale, p.beta);
        return;
    }
    // kAtOnce of the slab's eighths together: their loads of a row do not wait for one another
    constexpr int kCols = kFewThreads / kFewLanes, kAtOnce = E == 1 ? 8 : 2;
    const int x = threadIdx.x % kCols, y = threadIdx.x / kCols;
    for (int v0 = 0; v0 < kFewThreads; v0 += kCols * kAtOnce) {
        float acc[kAtOnce][E] = {};
        const int col0 = (slab * kFewThreads + v0 + x) * E;
#pragma unroll 2
        for (int j = y; j < n; j += kFewLanes) {
            const TR* row = rows + (int64_t)list[j] * p.rows_stride;
            Vec<TR, E> v[kAtOnce];
#pragma unroll
            for (int a = 0; a < kAtOnce; ++a)
                if (col0 + a * kCols * E < p.dim) v[a] = *reinterpret_cast<const Vec<TR, E>*>(row + col0 + a * kCols * E);
#pragma unroll
            for (int a = 0; a < kAtOnce; ++a)
                if (col0 + a * kCols * E < p.dim) {
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[a][e] += (float)v[a].v[e];
                }
        }
#pragma unroll
        for (int a = 0; a < kAtOnce; ++a) {
            const int col = col0 + a * kCols * E;
#pragma unroll
            for (int e = 0; e < E; ++e) part[y][x][e] = acc[a][e];
            __syncthreads();
            if (y == 0 && col < p.dim) {
                float sum[E] = {};
#pragma unroll
                for (int e = 0; e < E; ++e)
#pragma unroll
                    for (int l = 0; l < kFewLanes; ++l) sum[e] += part[l][x][e];
                write_sum<TT, E>(table, word, p.table_stride, col, sum, p.scale, p.beta);
            }
            __syncthreads();
        }
    }
}

// Vectors of a row for the gradient kernels: 16 bytes of the rows that are read, however many that are of the table
template <typename TT, typename TR>
bool vector_rows(const accb_embedding_desc& d, const void* table, const void* rows)
{
    constexpr int E = 16 / (int)sizeof(TR);
    constexpr size_t kTableAlign = E * sizeof(TT) > 16 ? 16 : E * sizeof(TT);
    return d.dim % E == 0 && d.rows_stride % E == 0 && (d.table_stride * sizeof(TT)) % kTableAlign == 0 && (reinterpret_cast<uintptr_t>(rows) & 15) == 0 &&
           reinterpret_cast<uintptr_t>(table) % kTableAlign == 0;
}

template <typename TT>
ClearParams clear_params(const accb_embedding_desc& d, const void* table, int64_t ctas)
{
    ClearParams c;
    c.stride = d.table_stride; c.dim = (int)d.dim; c.beta = d.beta;
    c.vec = (d.dim * sizeof(TT)) % 16 == 0 && (d.table_stride * sizeof(TT)) % 16 == 0 && (reinterpret_cast<uintptr_t>(table) & 15) == 0;
    c.ctas = (int)ctas;
    return c;
}

cudaError_t launch_sort(const EmbeddingLaunch& l, const SortParams& s, int* keys0, int* tokens0, int* keys1, int* tokens1, int* long_words)
{
    static std::atomic<bool> opted[64];
    if (l.device >= 64 || !opted[l.device].load(std::memory_order_acquire)) {
        const cudaError_t e = cudaFuncSetAttribute(sort_tokens_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSortSmem);
        if (e != cudaSuccess) return e;
        if (l.device < 64) opted[l.device].store(true, std::memory_order_release);
    }
    const bool pdl = options().stream_pdl != 0;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(kSortCluster); cfg.blockDim = dim3(kSortThreads); cfg.dynamicSmemBytes = kSortSmem; cfg.stream = l.stream;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = kSortCluster; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = pdl ? 1 : 0;
    cfg.attrs = attr; cfg.numAttrs = 2;
    return cudaLaunchKernelEx(&cfg, sort_tokens_kernel, l.ids, keys0, tokens0, keys1, tokens1, long_words, l.status, s);
}

template <typename TT, typename TR>
int launch_grad(const EmbeddingLaunch& l, const void* rows, void* table, const char** err)
{
    const accb_embedding_desc& d = l.d;
    constexpr int E = 16 / (int)sizeof(TR);
    const int64_t n = d.tokens;
    const bool vec = vector_rows<TT, TR>(d, table, rows), clear = d.beta != 1.0f;
    SortParams s;
    s.n = (int)n; s.vocab = (int)d.vocab; s.padding_id = d.padding_id;
    s.id_bytes = d.id_bytes;
    int bits = 1;
    while (((int64_t)1 << bits) <= d.vocab) ++bits;          // keys 0 .. vocab
    s.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
    s.digit_bits = (bits + s.passes - 1) / s.passes;
    s.launch_id = l.launch_id;
    SumParams p;
    p.n = (int)n; p.vocab = (int)d.vocab; p.dim = (int)d.dim;
    p.table_stride = d.table_stride; p.rows_stride = d.rows_stride;
    p.scale = d.scale; p.beta = d.beta;
    p.chunks = (int)((n + kChunk - 1) / kChunk);
    const int64_t cols_per_slab = (int64_t)(n <= kFewTokens ? kFewThreads : kSumThreads) * (vec ? E : 1);
    p.slabs = (int)((d.dim + cols_per_slab - 1) / cols_per_slab);
    auto cuda_failed = [&](cudaError_t e) { *err = cudaGetErrorString(e); return (int)ACCB_ERR_CUDA; };

    if (n <= kFewTokens) {
        // a few rows a clearing block, four blocks an SM, and no more rows than a block's bit list holds
        const int rounds = n <= 2 * kFewThreads ? 2 : n <= 4 * kFewThreads ? 4 : 8;
        const int64_t most = (int64_t)rounds * kFewThreads * 32;
        int64_t ctas = clear ? (d.vocab + 7) / 8 : 0;
        if (ctas > 4 * l.num_sms) ctas = 4 * l.num_sms;
        if (clear && (d.vocab + most - 1) / most > ctas) ctas = (d.vocab + most - 1) / most;
        const ClearParams c = clear_params<TT>(d, table, ctas > 0 ? ctas : 1);
        const dim3 grid((unsigned)(n * p.slabs + ctas)), block(kFewThreads);
        auto kernel = rounds == 2 ? (vec ? few_tokens_kernel<TT, TR, E, 2> : few_tokens_kernel<TT, TR, 1, 2>)
                    : rounds == 4 ? (vec ? few_tokens_kernel<TT, TR, E, 4> : few_tokens_kernel<TT, TR, 1, 4>)
                                  : (vec ? few_tokens_kernel<TT, TR, E, 8> : few_tokens_kernel<TT, TR, 1, 8>);
        const cudaError_t e = launch_pdl(kernel, grid, block, l.stream, (const TR*)rows, l.ids, (TT*)table, l.status, s, c, p);
        if (e != cudaSuccess) return cuda_failed(e);
        note_launches(1);
        return 1;
    }

    const int64_t blocks = (int64_t)p.chunks * p.slabs;
    if (blocks > 0x7fffffff) return cuda_failed(cudaErrorInvalidConfiguration);
    const size_t list = ((size_t)n * 4 + 15) / 16 * 16, words = ((size_t)(p.chunks + 1) * 4 + 15) / 16 * 16;
    char* ws = (char*)temp_alloc(l.device, 4 * list + words + (size_t)p.chunks * 2 * (size_t)d.dim * 4, l.stream);
    if (!ws) { *err = "no device memory for the workspace"; return ACCB_ERR_CUDA; }
    int *keys0 = (int*)ws, *tokens0 = (int*)(ws + list), *keys1 = (int*)(ws + 2 * list), *tokens1 = (int*)(ws + 3 * list), *long_words = (int*)(ws + 4 * list);
    float* partial = (float*)(ws + 4 * list + words);
    const int* keys = (s.passes & 1) ? keys0 : keys1;
    const int* tokens = (s.passes & 1) ? tokens0 : tokens1;
    cudaError_t e = cudaSuccess;
    const ClearParams c = clear_params<TT>(d, table, 1);
    p.clear_rows = 32;
    while (p.clear_rows > 1 && p.clear_rows * d.dim * (int64_t)sizeof(TT) > kClearBytes) p.clear_rows /= 2;
    if (e == cudaSuccess) e = launch_sort(l, s, keys0, tokens0, keys1, tokens1, long_words);
    const int64_t rest = clear ? (d.vocab + p.clear_rows - 1) / p.clear_rows : 0;
    if (blocks + rest > 0x7fffffff) { temp_free(ws, l.stream); return cuda_failed(cudaErrorInvalidConfiguration); }
    const dim3 grid((unsigned)(blocks + rest)), block(kSumThreads);
    const bool deep = blocks <= kSumDeep * (int64_t)l.num_sms;
    auto sum = vec ? (deep ? sum_rows_kernel<TT, TR, E, 8> : sum_rows_kernel<TT, TR, E, 2>) : (deep ? sum_rows_kernel<TT, TR, 1, 8> : sum_rows_kernel<TT, TR, 1, 2>);
    if (e == cudaSuccess) e = launch_pdl(sum, grid, block, l.stream, (const TR*)rows, keys, tokens, (TT*)table, partial, long_words, p, c);
    if (e == cudaSuccess)
        e = launch_pdl(vec ? join_rows_kernel<TT, 4> : join_rows_kernel<TT, 1>, dim3((unsigned)(8 * l.num_sms)), dim3(kJoinCols * kJoinLanes), l.stream,
                       (const float*)partial, keys, (const int*)long_words, (TT*)table, p);
    temp_free(ws, l.stream);
    if (e != cudaSuccess) return cuda_failed(e);
    note_launches(3);
    return 3;
}

template <template <typename, typename> class F, typename... Args>
auto by_types(int table_type, int rows_type, Args... args)
{
    auto rows = [&](auto tt) {
        using TT = decltype(tt);
        if (rows_type == ACCB_F32) return F<TT, float>::run(args...);
        if (rows_type == ACCB_F16) return F<TT, __half>::run(args...);
        return F<TT, __nv_bfloat16>::run(args...);
    };
    if (table_type == ACCB_F32) return rows(float());
    if (table_type == ACCB_F16) return rows(__half());
    return rows(__nv_bfloat16());
}
template <typename TT, typename TR> struct Lookup {
    static cudaError_t run(const EmbeddingLaunch* l, const void* table, void* rows) { return launch_lookup<TT, TR>(*l, table, rows); }
};
template <typename TT, typename TR> struct Grad {
    static int run(const EmbeddingLaunch* l, const void* rows, void* table, const char** err) { return launch_grad<TT, TR>(*l, rows, table, err); }
};

}  // namespace

int launch_embedding(const EmbeddingLaunch& l, const void* table, void* rows, const char** err)
{
    const cudaError_t e = by_types<Lookup>(l.d.table_type, l.d.rows_type, &l, table, rows);
    if (e != cudaSuccess) { *err = cudaGetErrorString(e); return ACCB_ERR_CUDA; }
    note_launches(1);
    return 1;
}

int launch_embedding_grad(const EmbeddingLaunch& l, const void* rows, void* table, const char** err)
{
    if (l.d.tokens == 0 && l.d.beta == 1.0f) return 0;
    return by_types<Grad>(l.d.table_type, l.d.rows_type, &l, rows, table, err);
}

}  // namespace accb
