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

// ---------------------------------------------------------------------------------
// lookup
// ---------------------------------------------------------------------------------

struct LookupParams {
    int64_t table_stride, rows_stride;
    uint32_t vocab;
    uint32_t vecs_per_row;
    uint64_t total;             // vectors in all rows
    float scale;
    int id_bytes;
    int launch_id;
};

constexpr int kLookupBlock = 256;
constexpr int kLookupUnroll = 4;

__device__ __forceinline__ int64_t load_id(const void* ids, int64_t t, int id_bytes)
{
    return id_bytes == 8 ? __ldg((const long long*)ids + t) : (int64_t)__ldg((const int*)ids + t);
}

// A block moves kLookupBlock * kLookupUnroll neighbouring vectors of the flattened rows, so that short and odd rows
// fill it as well as long ones; a thread has its kLookupUnroll id -> row chains in flight together.
template <typename TT, typename TR, int E>
__global__ void __launch_bounds__(kLookupBlock)
embedding_kernel(const TT* __restrict__ table, const void* __restrict__ ids, TR* __restrict__ rows, int* __restrict__ status,
                 const LookupParams p)
{
    pdl_enter();
    const uint64_t base = (uint64_t)blockIdx.x * (kLookupBlock * kLookupUnroll) + threadIdx.x;
    Vec<TT, E> x[kLookupUnroll];
    uint64_t row[kLookupUnroll];
    uint32_t col[kLookupUnroll];
    bool ok[kLookupUnroll];
#pragma unroll
    for (int u = 0; u < kLookupUnroll; ++u) {
        const uint64_t v = base + (uint64_t)u * kLookupBlock;
        ok[u] = false;
        row[u] = p.total <= 0xffffffffu ? (uint32_t)v / p.vecs_per_row : v / p.vecs_per_row;
        col[u] = (uint32_t)(v - row[u] * p.vecs_per_row);
        if (v < p.total) {
            const int64_t id = load_id(ids, (int64_t)row[u], p.id_bytes);
            ok[u] = (uint64_t)id < p.vocab;
            if (!ok[u] && col[u] == 0) { atomicAdd(status + ST_EMBED_COUNT, 1); status[ST_EMBED_ID] = p.launch_id; }
            if (ok[u]) x[u] = *reinterpret_cast<const Vec<TT, E>*>(table + id * p.table_stride + (int64_t)col[u] * E);
        }
    }
#pragma unroll
    for (int u = 0; u < kLookupUnroll; ++u) {
        if (base + (uint64_t)u * kLookupBlock >= p.total) continue;
        Vec<TR, E> y;
#pragma unroll
        for (int e = 0; e < E; ++e) y.v[e] = ok[u] ? (TR)((float)x[u].v[e] * p.scale) : (TR)0.0f;
        *reinterpret_cast<Vec<TR, E>*>(rows + (int64_t)row[u] * p.rows_stride + (int64_t)col[u] * E) = y;
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
    p.vocab = (uint32_t)d.vocab;
    p.vecs_per_row = (uint32_t)(vec ? d.dim / E : d.dim);
    p.total = (uint64_t)d.tokens * p.vecs_per_row;
    p.scale = d.scale; p.id_bytes = d.id_bytes; p.launch_id = l.launch_id;
    const uint64_t blocks = (p.total + kLookupBlock * kLookupUnroll - 1) / (kLookupBlock * kLookupUnroll);
    if (blocks > 0x7fffffffu) return cudaErrorInvalidConfiguration;
    const dim3 grid((unsigned)blocks), block(kLookupBlock);
    return vec ? launch_pdl(embedding_kernel<TT, TR, E>, grid, block, l.stream, (const TT*)table, l.ids, (TR*)rows, l.status, p)
               : launch_pdl(embedding_kernel<TT, TR, 1>, grid, block, l.stream, (const TT*)table, l.ids, (TR*)rows, l.status, p);
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
                bad += !((uint64_t)id < (uint64_t)p.vocab) && id != p.padding_id;
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
sort_tokens_kernel(const void* __restrict__ ids, int* keys0, int* tokens0, int* keys1, int* tokens1, int* status, const SortParams p)
{
    extern __shared__ int smem[];
    pdl_enter();
    sort_tokens(ids, keys0, tokens0, keys1, tokens1, status, p, smem);
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
constexpr int kSumThreads = 256;
constexpr int kSumUnroll = 8;

struct SumParams {
    int n, vocab, dim;
    int64_t table_stride, rows_stride;
    float scale, beta;
    int chunks;
    int slabs;
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

template <typename TT, typename TR, int E>
__global__ void __launch_bounds__(kSumThreads)
sum_rows_kernel(const TR* __restrict__ rows, const int* __restrict__ keys, const int* __restrict__ tokens, TT* __restrict__ table,
                float* __restrict__ partial, int* __restrict__ runs_on, const SumParams p)
{
    pdl_enter();
    const int chunk = blockIdx.x / p.slabs, slab = blockIdx.x % p.slabs;
    const int i0 = chunk * kChunk, i1 = min(p.n, i0 + kChunk);
    __shared__ int key[3 * kChunk], token[2 * kChunk];      // places i0 - kChunk .. and i0 ..
    for (int j = threadIdx.x; j < 3 * kChunk; j += kSumThreads) {
        const int i = i0 - kChunk + j;
        key[j] = (i >= 0 && i < p.n) ? keys[i] : -1;
        if (j >= kChunk) token[j - kChunk] = i < p.n ? tokens[i] : 0;
    }
    __syncthreads();
    const int* k = key + kChunk;                             // k[i] = key of place i0 + i
    const int len = i1 - i0;
    // the piece of a word that began earlier: skipped when that word is short (its first chunk takes it all)
    int first = 0;
    bool first_long = false;
    if (k[-1] == k[0]) {
        int back = 1, ahead = 0;
        while (back < kChunk && k[-back - 1] == k[0]) ++back;
        while (ahead < 2 * kChunk && k[ahead] == k[0]) ++ahead;
        first_long = back + ahead > kChunk;
        if (!first_long) first = ahead < len ? ahead : len;
    }
    // the word that runs past the chunk's end: taken to its end when short, to the border when long
    int last = len;
    bool last_long = false;
    if (first < len && i1 < p.n && k[len] == k[len - 1]) {
        const int w = k[len - 1];
        int start = len - 1, ahead = len;
        while (start > 0 && k[start - 1] == w) --start;
        const bool from_before = start == 0 && k[-1] == w;
        while (ahead < 2 * kChunk && k[ahead] == w) ++ahead;
        if (!from_before) {
            last_long = ahead - start > kChunk;
            if (!last_long) last = ahead;
        }
    }
    if (threadIdx.x == 0 && slab == 0) runs_on[chunk] = last_long;
    const int col = (slab * kSumThreads + threadIdx.x) * E;
    if (col >= p.dim) return;
    float acc[E] = {};
    for (int j0 = first; j0 < last; j0 += kSumUnroll) {
        Vec<TR, E> x[kSumUnroll];
#pragma unroll
        for (int u = 0; u < kSumUnroll; ++u)
            if (j0 + u < last && k[j0 + u] < p.vocab)
                x[u] = *reinterpret_cast<const Vec<TR, E>*>(rows + (int64_t)token[j0 + u] * p.rows_stride + col);
#pragma unroll
        for (int u = 0; u < kSumUnroll; ++u) {
            const int j = j0 + u;
            if (j < last && k[j] < p.vocab) {
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] += (float)x[u].v[e];
                const bool ends = j + 1 == last || k[j + 1] != k[j];
                if (ends) {
                    const bool head = first_long && k[j] == k[0], tail = last_long && j + 1 == last;
                    if (head || tail) {
                        float* dst = partial + ((int64_t)chunk * 2 + (head ? 0 : 1)) * p.dim + col;
#pragma unroll
                        for (int e = 0; e < E; ++e) dst[e] = acc[e];
                    } else {
                        write_sum<TT, E>(table, k[j], p.table_stride, col, acc, p.scale, p.beta);
                    }
#pragma unroll
                    for (int e = 0; e < E; ++e) acc[e] = 0.0f;
                }
            }
        }
    }
}

// step 3: the pieces of the long words.  Lane l of a warp looks at chunk 32 * blockIdx.x + l; the block then takes the long
// words that begin there one by one: kJoinLanes threads a column add every kJoinLanes-th piece, and their sums are added
// in lane order.
constexpr int kJoinCols = 32, kJoinLanes = 8;

template <typename TT>
__global__ void __launch_bounds__(kJoinCols * kJoinLanes)
join_rows_kernel(const float* __restrict__ partial, const int* __restrict__ keys, const int* __restrict__ runs_on, TT* __restrict__ table,
                 const SumParams p)
{
    pdl_enter();
    __shared__ float part[kJoinLanes][kJoinCols];
    const int x = threadIdx.x % kJoinCols, y = threadIdx.x / kJoinCols;
    const int base = blockIdx.x * 32;
    uint32_t todo = __ballot_sync(0xffffffffu, base + x < p.chunks && runs_on[base + x]);
    const int col = blockIdx.y * kJoinCols + x;
    while (todo) {
        const int chunk = base + __ffs(todo) - 1;
        todo &= todo - 1;
        const int word = keys[chunk * kChunk + kChunk - 1];
        // the word's last place: the list is sorted
        int lo = chunk * kChunk + kChunk, hi = p.n;
        while (lo < hi) { const int mid = lo + (hi - lo) / 2; if (keys[mid] <= word) lo = mid + 1; else hi = mid; }
        const int last_chunk = (lo - 1) / kChunk;
        float acc = 0.0f;
        if (col < p.dim && word < p.vocab)
            for (int c = chunk + y; c <= last_chunk; c += kJoinLanes)
                acc += partial[((int64_t)c * 2 + (c == chunk ? 1 : 0)) * p.dim + col];
        part[y][x] = acc;
        __syncthreads();
        if (y == 0 && col < p.dim && word < p.vocab) {
            float sum[1] = { 0.0f };
#pragma unroll
            for (int l = 0; l < kJoinLanes; ++l) sum[0] += part[l][x];
            write_sum<TT, 1>(table, word, p.table_stride, col, sum, p.scale, p.beta);
        }
        __syncthreads();
    }
}

// Rows of the table before any sum is added: zero (beta = 0) or scaled by beta.  `touched` words are overwritten afterwards
// when beta = 0; with another beta the sums read the old value themselves, so only untouched words are scaled here.
template <typename TT>
__global__ void __launch_bounds__(256)
untouched_rows_kernel(const int* __restrict__ keys, int n, TT* __restrict__ table, int64_t vocab, int64_t dim, int64_t stride, float beta)
{
    pdl_enter();
    for (int64_t v = blockIdx.x; v < vocab; v += gridDim.x) {
        int lo = 0, hi = n;
        while (lo < hi) { const int mid = lo + (hi - lo) / 2; if (keys[mid] < v) lo = mid + 1; else hi = mid; }
        if (lo < n && keys[lo] == v) continue;
        TT* row = table + v * stride;
        if (beta == 0.0f) for (int64_t c = threadIdx.x; c < dim; c += 256) row[c] = (TT)0.0f;
        else for (int64_t c = threadIdx.x; c < dim; c += 256) row[c] = (TT)(beta * (float)row[c]);
    }
}

struct GradWork { int *keys0, *tokens0, *keys1, *tokens1, *runs_on; float* partial; };

template <typename TT, typename TR>
cudaError_t launch_sums(const EmbeddingLaunch& l, const void* rows, void* table, const GradWork& w, const int* keys, const int* tokens)
{
    const accb_embedding_desc& d = l.d;
    constexpr int E = 16 / (int)(sizeof(TT) > sizeof(TR) ? sizeof(TT) : sizeof(TR));
    auto aligned = [](const void* p, int64_t stride, int64_t es) { return (reinterpret_cast<uintptr_t>(p) % (E * es)) == 0 && stride % E == 0; };
    const bool vec = d.dim % E == 0 && aligned(table, d.table_stride, sizeof(TT)) && aligned(rows, d.rows_stride, sizeof(TR));
    cudaError_t e = cudaSuccess;
    if (d.beta != 1.0f) {
        const unsigned blocks = (unsigned)(d.vocab < 148 * 16 ? d.vocab : 148 * 16);
        e = launch_pdl(untouched_rows_kernel<TT>, dim3(blocks), dim3(256), l.stream, keys, (int)d.tokens, (TT*)table, d.vocab, d.dim, d.table_stride, d.beta);
        if (e != cudaSuccess) return e;
    }
    if (d.tokens == 0) return cudaSuccess;
    SumParams p;
    p.n = (int)d.tokens; p.vocab = (int)d.vocab; p.dim = (int)d.dim;
    p.table_stride = d.table_stride; p.rows_stride = d.rows_stride;
    p.scale = d.scale; p.beta = d.beta;
    p.chunks = (p.n + kChunk - 1) / kChunk;
    const int64_t cols_per_slab = (int64_t)kSumThreads * (vec ? E : 1);
    p.slabs = (int)((d.dim + cols_per_slab - 1) / cols_per_slab);
    if ((int64_t)p.chunks * p.slabs > 0x7fffffff || (d.dim + kJoinCols - 1) / kJoinCols > 65535) return cudaErrorInvalidConfiguration;
    const dim3 grid((unsigned)(p.chunks * p.slabs)), block(kSumThreads);
    e = vec ? launch_pdl(sum_rows_kernel<TT, TR, E>, grid, block, l.stream, (const TR*)rows, keys, tokens, (TT*)table, w.partial, w.runs_on, p)
            : launch_pdl(sum_rows_kernel<TT, TR, 1>, grid, block, l.stream, (const TR*)rows, keys, tokens, (TT*)table, w.partial, w.runs_on, p);
    if (e != cudaSuccess) return e;
    return launch_pdl(join_rows_kernel<TT>, dim3((unsigned)((p.chunks + 31) / 32), (unsigned)((d.dim + kJoinCols - 1) / kJoinCols)),
                      dim3(kJoinCols * kJoinLanes), l.stream, (const float*)w.partial, keys, (const int*)w.runs_on, (TT*)table, p);
}

template <template <typename, typename> class F, typename... Args>
cudaError_t by_types(int table_type, int rows_type, Args... args)
{
    auto rows = [&](auto tt) -> cudaError_t {
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
template <typename TT, typename TR> struct Sums {
    static cudaError_t run(const EmbeddingLaunch* l, const void* rows, void* table, const GradWork* w, const int* keys, const int* tokens)
    {
        return launch_sums<TT, TR>(*l, rows, table, *w, keys, tokens);
    }
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
    const accb_embedding_desc& d = l.d;
    const int64_t n = d.tokens;
    if (n == 0 && d.beta == 1.0f) return 0;
    const int64_t chunks = (n + kChunk - 1) / kChunk;
    const size_t list = ((size_t)n * 4 + 15) / 16 * 16;
    const size_t bytes = 4 * list + ((size_t)chunks * 4 + 15) / 16 * 16 + (size_t)chunks * 2 * (size_t)d.dim * 4 + 16;
    char* ws = (char*)temp_alloc(l.device, bytes, l.stream);
    if (!ws) { *err = "no device memory for the workspace"; return ACCB_ERR_CUDA; }
    GradWork w;
    w.keys0 = (int*)ws; w.tokens0 = (int*)(ws + list); w.keys1 = (int*)(ws + 2 * list); w.tokens1 = (int*)(ws + 3 * list);
    w.runs_on = (int*)(ws + 4 * list);
    w.partial = (float*)(ws + 4 * list + ((size_t)chunks * 4 + 15) / 16 * 16);

    SortParams s;
    s.n = (int)n; s.vocab = (int)d.vocab; s.padding_id = d.padding_id < 0 ? -1 : d.padding_id; s.id_bytes = d.id_bytes;
    int bits = 1;
    while (((int64_t)1 << bits) <= d.vocab) ++bits;          // keys 0 .. vocab
    s.passes = (bits + kMaxDigitBits - 1) / kMaxDigitBits;
    s.digit_bits = (bits + s.passes - 1) / s.passes;
    s.launch_id = l.launch_id;
    const int* keys = (s.passes & 1) ? w.keys0 : w.keys1;
    const int* tokens = (s.passes & 1) ? w.tokens0 : w.tokens1;
    cudaError_t e = cudaSuccess;
    if (n > 0) {
        static std::atomic<bool> opted[64];
        if (l.device < 0 || l.device >= 64 || !opted[l.device]) {
            e = cudaFuncSetAttribute(sort_tokens_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)kSortSmem);
            if (e == cudaSuccess && l.device >= 0 && l.device < 64) opted[l.device] = true;
        }
        const unsigned ctas = n <= 2048 ? 1 : n <= 4096 ? 2 : n <= 8192 ? 4 : kSortCluster;
        cudaLaunchConfig_t cfg = {};
        cfg.gridDim = dim3(ctas); cfg.blockDim = dim3(kSortThreads); cfg.dynamicSmemBytes = kSortSmem; cfg.stream = l.stream;
        cudaLaunchAttribute attr[2];
        attr[0].id = cudaLaunchAttributeClusterDimension;
        attr[0].val.clusterDim.x = ctas; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
        attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attr[1].val.programmaticStreamSerializationAllowed = options().stream_pdl == 0 ? 0 : 1;
        cfg.attrs = attr; cfg.numAttrs = 2;
        if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, sort_tokens_kernel, l.ids, w.keys0, w.tokens0, w.keys1, w.tokens1, l.status, s);
    }
    if (e == cudaSuccess) e = by_types<Sums>(d.table_type, d.rows_type, &l, rows, table, (const GradWork*)&w, keys, tokens);
    temp_free(ws, l.stream);
    if (e != cudaSuccess) { *err = cudaGetErrorString(e); return ACCB_ERR_CUDA; }
    note_launches((n > 0 ? 3 : 0) + (d.beta != 1.0f ? 1 : 0));
    return 1;
}

}  // namespace accb
