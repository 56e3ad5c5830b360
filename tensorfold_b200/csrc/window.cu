// Lane attention with a sliding window and sinks over the paged KV cache.
//
// Row t of a sequence's window stands at slot p = L + t (L committed keys) and sees key j when j <= p and
// (p - j < window or j < sinks): softmax of its scores over those keys, the weighted sum of their values, and the
// log-sum-exp of the scores.
//
// First form: one block per (row, head), a warp per key in turn, online softmax in fp32.

#include "common.cuh"

namespace tf {
namespace {

constexpr int kPage = 16, kWarps = 4;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

struct WindowArgs {
    const __nv_bfloat16 *q, *k_new, *v_new, *k_pages, *v_pages;
    const int *page_table, *seq_lens, *seq_start;
    __nv_bfloat16* out;            // [R, H, D] or null
    float* lse;                    // [R, H] or null
    const __nv_bfloat16* qg;       // output gate or null
    size_t qg_stride;
    uint8_t* out_packed;           // or null
    int* status;
    int num_pages, max_pages, H, HK, R, S, window, sinks, max_context, group;
    float scale_log2;
};

// The sequence that holds packed row `row`: the last one that starts at or before it (a sequence without rows starts where the
// next one does, and is passed over); -1 for a row behind the last sequence. Whole warps.
__device__ __forceinline__ int seq_of(const int* seq_start, int S, int row) {
    const int lane = threadIdx.x & 31;
    if (row >= seq_start[S]) return -1;
    int found = -1;
    for (int s0 = 0; s0 < S; s0 += 32) {
        const bool before = s0 + lane < S && seq_start[s0 + lane] <= row;
        const unsigned m = __ballot_sync(0xffffffffu, before);
        if (m) found = s0 + 31 - __clz(m);
        if (m != 0xffffffffu) break;
    }
    return found;
}

template <int D>
__global__ void __launch_bounds__(kWarps * 32) window_kernel(const WindowArgs a) {
    constexpr int PER = D / 32;
    __shared__ float sm_m[kWarps], sm_l[kWarps];
    __shared__ float sm_o[kWarps][D];
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.y, head = blockIdx.x, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int Mp = tf_padded_rows(a.R);
    const int seq = row < a.R ? seq_of(a.seq_start, a.S, row) : -1;
    if (seq < 0) {
        if (row >= a.R && a.out_packed != nullptr && warp == 0 && lane < D / 8) {
            if (a.group == 64) packed_store<64>(a.out_packed, Mp, row, head * (D / 8) + lane, make_uint4(0, 0, 0, 0), 0.f);
            else packed_store<32>(a.out_packed, Mp, row, head * (D / 8) + lane, make_uint4(0, 0, 0, 0), 0.f);
        }
        return;
    }
    const int r0 = a.seq_start[seq], L = a.seq_lens[seq], p = L + row - r0;
    if (p >= a.max_context) { if (threadIdx.x == 0) report(a.status, TF_EINVAL); return; }
    const int kvh = head / (a.H / a.HK);
    const int first = max(0, p + 1 - a.window), nsink = min(a.sinks, first), n = nsink + p + 1 - first;
    float q[PER], acc[PER];
#pragma unroll
    for (int i = 0; i < PER; ++i) { q[i] = bf2f(a.q[((size_t)row * a.H + head) * D + lane * PER + i]); acc[i] = 0.f; }
    float m = -INFINITY, l = 0.f;
    for (int i = warp; i < n; i += kWarps) {
        const int j = i < nsink ? i : first + i - nsink;
        const __nv_bfloat16 *k, *v;
        if (j < L) {
            const int page = a.page_table[(size_t)seq * a.max_pages + j / kPage];
            if (page < 0 || page >= a.num_pages) { report(a.status, TF_EINVAL); continue; }
            const size_t off = (((size_t)page * a.HK + kvh) * kPage + j % kPage) * D;
            k = a.k_pages + off; v = a.v_pages + off;
        } else {
            const size_t off = ((size_t)(r0 + j - L) * a.HK + kvh) * D;
            k = a.k_new + off; v = a.v_new + off;
        }
        float s = 0.f;
#pragma unroll
        for (int e = 0; e < PER; ++e) s = fmaf(q[e], bf2f(k[lane * PER + e]), s);
        s = warp_sum(s) * a.scale_log2;
        const float mn = fmaxf(m, s), ms = mn == -INFINITY ? 0.f : mn;
        const float al = exp2f(m - ms), w = exp2f(s - ms);
        l = fmaf(l, al, w);
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] = fmaf(acc[e], al, w * bf2f(v[lane * PER + e]));
        m = mn;
    }
    if (lane == 0) { sm_m[warp] = m; sm_l[warp] = l; }
#pragma unroll
    for (int e = 0; e < PER; ++e) sm_o[warp][lane * PER + e] = acc[e];
    __syncthreads();
    if (warp != 0) return;
    for (int w = 1; w < kWarps; ++w) {
        const float mn = fmaxf(m, sm_m[w]), ms = mn == -INFINITY ? 0.f : mn, sa = exp2f(m - ms), sb = exp2f(sm_m[w] - ms);
        l = l * sa + sm_l[w] * sb;
#pragma unroll
        for (int e = 0; e < PER; ++e) acc[e] = acc[e] * sa + sm_o[w][lane * PER + e] * sb;
        m = mn;
    }
    if (a.lse != nullptr && lane == 0) a.lse[(size_t)row * a.H + head] = (m + log2f(l)) * kLn2;
    float o[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) o[e] = round_bf16(acc[e] / l);
    if (a.qg != nullptr) {
        const __nv_bfloat16* g = a.qg + (size_t)row * a.qg_stride + (size_t)head * 2 * D + D + lane * PER;
#pragma unroll
        for (int e = 0; e < PER; ++e) o[e] = round_bf16(o[e] * sigmoidf_(bf2f(g[e])));
    }
    if (a.out != nullptr) {
#pragma unroll
        for (int e = 0; e < PER; ++e) a.out[((size_t)row * a.H + head) * D + lane * PER + e] = f2bf(o[e]);
    }
    if (a.out_packed != nullptr) {
        // a lane takes 8 values: at D = 128 the first 16 lanes, from the lanes 2c and 2c + 1 that hold chunk c
        float o8[8];
#pragma unroll
        for (int e = 0; e < 8; ++e)
            o8[e] = PER == 8 ? o[e % PER] : __shfl_sync(0xffffffffu, o[e % PER], (2 * lane + e / PER) & 31);
        const uint4 v = pack8(o8);
        const float sum = a.group == 64 ? group_sum8<64>(v) : group_sum8<32>(v);
        if (lane < D / 8) {
            const int c = head * (D / 8) + lane;
            if (a.group == 64) packed_store<64>(a.out_packed, Mp, row, c, v, sum);
            else packed_store<32>(a.out_packed, Mp, row, c, v, sum);
        }
    }
}

}  // namespace
}  // namespace tf

extern "C" {

int tf_window_slots(int window, int sinks, int max_window, int max_context, int chunk_keys) {
    if (window < 0 || sinks < 0 || max_window < 1 || max_context < max_window || chunk_keys < 64 || chunk_keys % 64) return 0;
    return 1;
}

size_t tf_window_scratch_bytes(int rows, int heads, int head_dim, int slots) {
    if (rows < 1 || heads < 1 || head_dim < 1 || slots < 1) return 0;
    return (size_t)slots * rows * heads * (head_dim + 2) * sizeof(float);
}

int tf_window_attention(const void* q, const void* k_new, const void* v_new, const void* k_pages, const void* v_pages, int num_pages,
                        const int* page_table, int max_pages, const int* seq_lens, const int* seq_start, void* out, float* lse,
                        const void* qg, size_t qg_stride, void* out_packed, int group, void* scratch, size_t scratch_bytes, int rows,
                        int n_seqs, int max_window, int max_context, int window, int sinks, int chunk_keys, int heads, int kv_heads,
                        int head_dim, float scale, int* status, void* stream) {
    if (!out && !out_packed) return TF_EINVAL;
    if ((group != 64 && group != 32) || (qg && (qg_stride % 8 || qg_stride < (size_t)heads * 2 * head_dim)) || (out_packed && rows > TF_QMM_MAX_ROWS)) return TF_EINVAL;
    if (rows < 1 || n_seqs < 1 || max_window < 1 || heads < 1 || kv_heads < 1 || heads % kv_heads || num_pages < 1 || max_pages < 1) return TF_EINVAL;
    if ((head_dim != 128 && head_dim != 256) || heads / kv_heads > 16 || !(scale > 0.f) || !(scale < INFINITY)) return TF_EINVAL;
    const int slots = tf_window_slots(window, sinks, max_window, max_context, chunk_keys);
    if (slots < 1) return TF_EINVAL;
    if (!q || !k_new || !v_new || !k_pages || !v_pages || !page_table || !seq_lens || !seq_start) return TF_EINVAL;
    if (((uintptr_t)q | (uintptr_t)k_new | (uintptr_t)v_new | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)qg | (uintptr_t)out_packed |
         (uintptr_t)out) & 15) return TF_EALIGN;
    if (!scratch || ((uintptr_t)scratch & 15) || scratch_bytes < tf_window_scratch_bytes(rows, heads, head_dim, slots)) return TF_ESCRATCH;
    if (rows > 65535) return TF_EINVAL;
    tf::WindowArgs a{};
    a.q = static_cast<const __nv_bfloat16*>(q);
    a.k_new = static_cast<const __nv_bfloat16*>(k_new); a.v_new = static_cast<const __nv_bfloat16*>(v_new);
    a.k_pages = static_cast<const __nv_bfloat16*>(k_pages); a.v_pages = static_cast<const __nv_bfloat16*>(v_pages);
    a.page_table = page_table; a.seq_lens = seq_lens; a.seq_start = seq_start;
    a.out = static_cast<__nv_bfloat16*>(out); a.lse = lse;
    a.qg = static_cast<const __nv_bfloat16*>(qg); a.qg_stride = qg_stride;
    a.out_packed = static_cast<uint8_t*>(out_packed); a.status = status;
    a.num_pages = num_pages; a.max_pages = max_pages; a.H = heads; a.HK = kv_heads; a.R = rows; a.S = n_seqs;
    a.window = window > 0 ? window : 1 << 30; a.sinks = window > 0 ? sinks : 0; a.max_context = max_context; a.group = group;
    a.scale_log2 = scale * tf::kLog2e;
    void* args[] = {&a};
    const int grid_rows = out_packed ? tf::tf_padded_rows(rows) : rows;
    const void* kern = head_dim == 256 ? (const void*)tf::window_kernel<256> : (const void*)tf::window_kernel<128>;
    if (tf::launch_pdl(kern, dim3(heads, grid_rows), dim3(tf::kWarps * 32), 0, static_cast<cudaStream_t>(stream), args) != cudaSuccess) {
        cudaGetLastError();
        return TF_ECUDA;
    }
    return TF_OK;
}

}  // extern "C"
