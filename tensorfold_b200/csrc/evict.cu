// Which cached keys are used, and the eviction of those that are not.
//
// attention_mass: after a commit, every cached key of every layer and KV head gets the attention weight that the kept rows
// gave it: mass[j] += sum over kept rows t and the KV head's query heads h of exp(scale q_th . k_j - lse_th), j <= L + t; a key that
// the commit brought starts at that sum and takes its row's position.
//
// evict: a sequence of more than `budget` slots is cut back to it, every (layer, KV head) by itself: the slots whose position is below
// `sinks` or among the `recent` latest stay, then those of the largest mass, ties to the lower slot. Kept slots above the budget
// move into the evicted ones below it, in order (keys carry their rotation, so their order does not matter): a slot that
// stays below the budget is not touched, and the fewest possible rows travel.

#include "common.cuh"

namespace tf {
namespace {

constexpr int kPage = 16;
constexpr float kLog2e = 1.4426950408889634f;

struct MassArgs {
    const __nv_bfloat16* q;        // [layers, R, H, D]
    const float* lse;              // [layers, R, H]
    const __nv_bfloat16* k_pages;  // [layers, pages, HK, 16, D]
    const int *page_table, *seq_lens, *seq_start, *keep, *row_pos;
    float* mass;                   // [layers, pages, HK, 16]
    int* pos;
    int* status;
    int num_pages, max_pages, H, HK, R, S, max_context;
    float scale_log2;
};

// First form: a block per (page, KV head, layer and sequence), a warp per four keys, rows one by one.
template <int D>
__global__ void __launch_bounds__(128) mass_kernel(const MassArgs a) {
    constexpr int PER = D / 32;
    pdl_launch_dependents();
    pdl_wait();
    const int kvh = blockIdx.y, layer = blockIdx.z / a.S, seq = blockIdx.z % a.S, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int r0 = a.seq_start[seq], n = a.seq_start[seq + 1] - r0, L = a.seq_lens[seq], kept = min(max(a.keep[seq], 0), n);
    if (L + kept > a.max_context && threadIdx.x == 0) report(a.status, TF_EINVAL);
    const int j0 = blockIdx.x * kPage, end = min(L + kept, min(a.max_context, a.max_pages * kPage));
    if (kept == 0 || j0 >= end) return;
    const int page = a.page_table[(size_t)seq * a.max_pages + blockIdx.x];
    if (page < 0 || page >= a.num_pages) { report(a.status, TF_EINVAL); return; }
    const int G = a.H / a.HK;
    const size_t cell0 = (((size_t)layer * a.num_pages + page) * a.HK + kvh) * kPage;
    for (int jj = warp; jj < kPage && j0 + jj < end; jj += 4) {
        const int j = j0 + jj;
        float k[PER], sum = 0.f;
#pragma unroll
        for (int i = 0; i < PER; ++i) k[i] = bf2f(a.k_pages[(cell0 + jj) * D + lane * PER + i]);
        for (int t = max(0, j - L); t < kept; ++t)
            for (int g = 0; g < G; ++g) {
                const size_t row = ((size_t)layer * a.R + r0 + t) * a.H + kvh * G + g;
                float s = 0.f;
#pragma unroll
                for (int i = 0; i < PER; ++i) s = fmaf(k[i], bf2f(a.q[row * D + lane * PER + i]), s);
                sum += exp2f(warp_sum(s) * a.scale_log2 - a.lse[row] * kLog2e);
            }
        if (lane == 0) {
            a.mass[cell0 + jj] = j < L ? a.mass[cell0 + jj] + sum : sum;
            if (j >= L) a.pos[cell0 + jj] = a.row_pos[r0 + j - L];
        }
    }
}

// ---- eviction ------------------------------------------------------------------------------------------
constexpr int kSelThreads = 1024;
constexpr int kBins = 2048;
constexpr int kSelKeys = 49152;      // slots whose keys fit the block's shared memory; longer sequences are ranked from global memory

struct EvictArgs {
    __nv_bfloat16 *k_pages, *v_pages;   // [layers, pages, HK, 16, D]
    const int *page_table, *seq_lens, *next_pos;
    float* mass;                        // [layers, pages, HK, 16]
    int* pos;
    int* moved;                         // [layers, S, HK]
    int* list;                          // [layers, S, HK][2][most]: evicted slots below the budget, kept slots above it
    int* status;
    int num_pages, max_pages, HK, S, budget, recent, sinks, max_context, most;
};

// Exclusive prefix sum over the block (kSelThreads threads) of two counts below 2^32 packed in one word; `total`: the sum.
__device__ __forceinline__ unsigned long long block_scan(unsigned long long v, unsigned long long* warp_s, unsigned long long& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned long long x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();                  // an earlier scan's sums have been read
    if (lane == 31) warp_s[warp] = x;
    __syncthreads();
    unsigned long long before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kSelThreads / 32; ++w) {
        const unsigned long long s = warp_s[w];
        before += w < warp ? s : 0;
        total += s;
    }
    return before + x - v;
}

template <bool STAGED>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
    extern __shared__ uint32_t keys_s[];
    __shared__ unsigned hist[kBins];
    __shared__ unsigned long long warp_s[kSelThreads / 32];
    __shared__ unsigned digit_s, above_s;
    pdl_launch_dependents();
    pdl_wait();
    const int kvh = blockIdx.x, seq = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x;
    const size_t item = ((size_t)layer * a.S + seq) * a.HK + kvh;
    const int L = a.seq_lens[seq], n = min(L, min(a.max_context, a.max_pages * kPage));
    if (L > n && tid == 0) report(a.status, TF_EINVAL);
    if (n <= a.budget) {
        if (tid == 0) a.moved[item] = 0;
        return;
    }
    const int* pt = a.page_table + (size_t)seq * a.max_pages;
    const int safe_from = a.next_pos[seq] - a.recent;
    // a slot's rank: protected first, then by mass; NaN counts as -inf
    auto rank_of = [&](int j) -> uint32_t {
        const int page = pt[j / kPage];
        if (page < 0 || page >= a.num_pages) { report(a.status, TF_EINVAL); return 0u; }
        const size_t cell = (((size_t)layer * a.num_pages + page) * a.HK + kvh) * kPage + j % kPage;
        const int p = a.pos[cell];
        if (p < a.sinks || p >= safe_from) return 0xFFFFFFFFu;
        const float m = a.mass[cell] + 0.f;            // -0 ranks as 0
        if (m != m) return 0x007FFFFFu;                // the rank of -inf
        const uint32_t u = __float_as_uint(m);
        return u & 0x80000000u ? ~u : u | 0x80000000u;
    };
    auto key = [&](int j) -> uint32_t { return STAGED ? keys_s[j] : rank_of(j); };
    if (STAGED)
        for (int j = tid; j < n; j += kSelThreads) keys_s[j] = rank_of(j);

    // the budget-th largest key, 11 + 11 + 10 bits at a time
    uint32_t prefix = 0, need = a.budget;
    for (int pass = 0; pass < 3; ++pass) {
        const int bits = pass == 2 ? 10 : 11, shift = pass == 0 ? 21 : pass == 1 ? 10 : 0;
        __syncthreads();
        for (int b = tid; b < kBins; b += kSelThreads) hist[b] = 0;
        __syncthreads();
        for (int j = tid; j < n; j += kSelThreads) {
            const uint32_t k = key(j);
            if (pass == 0 || (k >> (shift + bits)) == prefix) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1u);
        }
        __syncthreads();
        // thread i holds bins 2047 - 2i and 2046 - 2i: prefix sums from the largest digit down
        const unsigned c0 = hist[kBins - 1 - 2 * tid], c1 = hist[kBins - 2 - 2 * tid];
        unsigned long long total;
        const unsigned before = (unsigned)block_scan(c0 + c1, warp_s, total);
        if (before < need && before + c0 >= need) { digit_s = kBins - 1 - 2 * tid; above_s = before; }
        else if (before + c0 < need && before + c0 + c1 >= need) { digit_s = kBins - 2 - 2 * tid; above_s = before + c0; }
        __syncthreads();
        prefix = prefix << bits | digit_s;
        need -= above_s;
    }
    // kept: every key above `prefix` and the first `need` slots of that key. Each thread takes a run of slots (an odd number of
    // words: no bank conflicts)
    const int per = ((n + kSelThreads - 1) / kSelThreads) | 1, lo = min(n, tid * per), hi = min(n, lo + per);
    unsigned long long equal = 0, total;
    for (int j = lo; j < hi; ++j) equal += key(j) == prefix;
    const unsigned eq0 = (unsigned)block_scan(equal, warp_s, total);
    unsigned eq = eq0;
    unsigned long long counts = 0;               // holes below the budget | kept slots above it
    for (int j = lo; j < hi; ++j) {
        const uint32_t k = key(j);
        const bool kept = k > prefix || (k == prefix && eq++ < need);
        if (j < a.budget) counts += !kept;
        else counts += (unsigned long long)kept << 32;
    }
    const unsigned long long at = block_scan(counts, warp_s, total);
    int* holes = a.list + item * 2 * a.most;
    int* fills = holes + a.most;
    unsigned h = (unsigned)at, f = (unsigned)(at >> 32);
    eq = eq0;
    for (int j = lo; j < hi; ++j) {
        const uint32_t k = key(j);
        const bool kept = k > prefix || (k == prefix && eq++ < need);
        if (j < a.budget) { if (!kept) holes[h++] = j; }
        else if (kept) fills[f++] = j;
    }
    if (tid == 0) a.moved[item] = (int)(unsigned)total;
}

constexpr int kMoveWarps = 8;
template <int D>
__global__ void __launch_bounds__(kMoveWarps * 32) evict_move_kernel(const EvictArgs a) {
    pdl_launch_dependents();
    pdl_wait();
    const int kvh = blockIdx.y, seq = blockIdx.z % a.S, layer = blockIdx.z / a.S, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const size_t item = ((size_t)layer * a.S + seq) * a.HK + kvh;
    const int count = a.moved[item];
    const int* holes = a.list + item * 2 * a.most;
    const int* fills = holes + a.most;
    const int* pt = a.page_table + (size_t)seq * a.max_pages;
    auto cell = [&](int j, bool& ok) -> size_t {
        const int page = pt[j / kPage];
        ok = ok && page >= 0 && page < a.num_pages;
        return (((size_t)layer * a.num_pages + page) * a.HK + kvh) * kPage + j % kPage;
    };
    for (int i = blockIdx.x * kMoveWarps + warp; i < count; i += gridDim.x * kMoveWarps) {
        bool ok = true;
        const size_t to = cell(holes[i], ok), from = cell(fills[i], ok);
        if (!ok) continue;
        if (D == 256) {
            const uint4 k = reinterpret_cast<const uint4*>(a.k_pages + from * D)[lane], v = reinterpret_cast<const uint4*>(a.v_pages + from * D)[lane];
            reinterpret_cast<uint4*>(a.k_pages + to * D)[lane] = k;
            reinterpret_cast<uint4*>(a.v_pages + to * D)[lane] = v;
        } else {
            __nv_bfloat16* base = lane < 16 ? a.k_pages : a.v_pages;
            const uint4 x = reinterpret_cast<const uint4*>(base + from * D)[lane & 15];
            reinterpret_cast<uint4*>(base + to * D)[lane & 15] = x;
        }
        if (lane == 0) { a.mass[to] = a.mass[from]; a.pos[to] = a.pos[from]; }
    }
}

}  // namespace
}  // namespace tf

extern "C" {

int tf_attention_mass(const void* q, const float* lse, const void* k_pages, int num_pages, const int* page_table, int max_pages,
                      const int* seq_lens, const int* seq_start, const int* keep, const int* row_pos, float* mass, int* pos, int layers,
                      int rows, int n_seqs, int max_window, int max_context, int heads, int kv_heads, int head_dim, float scale, int* status,
                      void* stream) {
    if (layers < 1 || rows < 1 || n_seqs < 1 || max_window < 1 || max_context < max_window || heads < 1 || kv_heads < 1 || heads % kv_heads) return TF_EINVAL;
    if ((head_dim != 128 && head_dim != 256) || heads / kv_heads > 16 || !(scale > 0.f) || !(scale < INFINITY) || num_pages < 1 || max_pages < 1)
        return TF_EINVAL;
    if (!q || !lse || !k_pages || !page_table || !seq_lens || !seq_start || !keep || !row_pos || !mass || !pos) return TF_EINVAL;
    if (((uintptr_t)q | (uintptr_t)k_pages) & 15 || ((uintptr_t)mass | (uintptr_t)pos | (uintptr_t)lse) & 3) return TF_EALIGN;
    if ((long long)layers * n_seqs > 65535 || kv_heads > 65535) return TF_EINVAL;
    tf::MassArgs a{static_cast<const __nv_bfloat16*>(q), lse, static_cast<const __nv_bfloat16*>(k_pages), page_table, seq_lens, seq_start, keep,
                   row_pos, mass, pos, status, num_pages, max_pages, heads, kv_heads, rows, n_seqs, max_context, scale * tf::kLog2e};
    void* args[] = {&a};
    const void* kern = head_dim == 256 ? (const void*)tf::mass_kernel<256> : (const void*)tf::mass_kernel<128>;
    if (tf::launch_pdl(kern, dim3((max_context + tf::kPage - 1) / tf::kPage, kv_heads, layers * n_seqs), dim3(128), 0, static_cast<cudaStream_t>(stream),
                       args) != cudaSuccess) { cudaGetLastError(); return TF_ECUDA; }
    return TF_OK;
}

size_t tf_evict_scratch_bytes(int layers, int n_seqs, int kv_heads, int budget, int max_context) {
    if (layers < 1 || n_seqs < 1 || kv_heads < 1 || budget < 1 || max_context < 1) return 0;
    const size_t most = max_context <= budget ? 1 : (size_t)(max_context - budget < budget ? max_context - budget : budget);
    return (size_t)layers * n_seqs * kv_heads * 2 * most * sizeof(int);
}

int tf_kv_evict(void* k_pages, void* v_pages, int num_pages, const int* page_table, int max_pages, const int* seq_lens, const int* next_pos,
                float* mass, int* pos, int* moved, void* scratch, size_t scratch_bytes, int layers, int n_seqs, int budget, int recent, int sinks,
                int max_context, int kv_heads, int head_dim, int* status, void* stream) {
    if (layers < 1 || n_seqs < 1 || kv_heads < 1 || budget < 1 || recent < 0 || sinks < 0 || (long long)recent + sinks > budget || max_context < 1)
        return TF_EINVAL;
    if ((head_dim != 128 && head_dim != 256) || num_pages < 1 || max_pages < 1) return TF_EINVAL;
    if (!k_pages || !v_pages || !page_table || !seq_lens || !next_pos || !mass || !pos || !moved) return TF_EINVAL;
    if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15 || ((uintptr_t)mass | (uintptr_t)pos | (uintptr_t)moved | (uintptr_t)scratch) & 3) return TF_EALIGN;
    if ((long long)layers * n_seqs > 65535 || kv_heads > 65535) return TF_EINVAL;
    if (!scratch || scratch_bytes < tf_evict_scratch_bytes(layers, n_seqs, kv_heads, budget, max_context)) return TF_ESCRATCH;
    const int most = max_context <= budget ? 1 : (max_context - budget < budget ? max_context - budget : budget);
    tf::EvictArgs a{static_cast<__nv_bfloat16*>(k_pages), static_cast<__nv_bfloat16*>(v_pages), page_table, seq_lens, next_pos, mass, pos, moved,
                    static_cast<int*>(scratch), status, num_pages, max_pages, kv_heads, n_seqs, budget, recent, sinks, max_context, most};
    void* args[] = {&a};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool staged = max_context <= tf::kSelKeys;
    static bool configured[64] = {};       // the opt-in is per device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return TF_ECUDA; }
    if (!configured[dev]) {
        if (cudaFuncSetAttribute(tf::evict_select_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize, tf::kSelKeys * 4) != cudaSuccess) {
            cudaGetLastError();
            return TF_ECUDA;
        }
        configured[dev] = true;
    }
    const void* select = staged ? (const void*)tf::evict_select_kernel<true> : (const void*)tf::evict_select_kernel<false>;
    if (tf::launch_pdl(select, dim3(kv_heads, n_seqs, layers), dim3(tf::kSelThreads), staged ? (size_t)max_context * 4 : 0, st, args) != cudaSuccess) {
        cudaGetLastError();
        return TF_ECUDA;
    }
    const int blocks = min((most + tf::kMoveWarps - 1) / tf::kMoveWarps, 32);
    const void* move = head_dim == 256 ? (const void*)tf::evict_move_kernel<256> : (const void*)tf::evict_move_kernel<128>;
    if (tf::launch_pdl(move, dim3(blocks, kv_heads, layers * n_seqs), dim3(tf::kMoveWarps * 32), 0, st, args) != cudaSuccess) {
        cudaGetLastError();
        return TF_ECUDA;
    }
    return TF_OK;
}

}  // extern "C"
