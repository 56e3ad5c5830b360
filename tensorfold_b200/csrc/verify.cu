// Verification of drafted tokens against the target's probabilities, from given random numbers.
//
// A sequence's window is its last token and n - 1 drafts; row t's logits are the target's for the place after row t, and the draft
// for that place is the input token x of row t + 1. With p = softmax(logits_t / T) and q the drafter's distribution for the same
// place (softmax of the draft logits of row t + 1 over their own temperature, or all of it on x where there are none):
//
//   row t + 1 is kept while u1_t q(x) < p(x); the first one that is not is replaced by a draw from max(p - q, 0), and
//   after a window that is kept whole the next token is drawn from p of its last row.
//
// The draw is the first token in vocabulary order whose cumulative weight is above u2 times the total.
//
// Two launches. Row statistics: a slice of 8192 logits a block, its maximum and the sum of 2^((x - max) log2e / T) - bound by the
// bytes of the logits. Choice: a cluster of blocks per sequence; every block forms the acceptances from the slices' sums (64 bits), then the cluster
// goes over the one row that is drawn from. An acceptance is one comparison, so 32-bit exponentials (relative error of
// p and q near 3e-7) decide all but one in some million draws as exact arithmetic would; a draw compares one
// number with up to a million borders, so its weights and sums are in 64 bits throughout. A NaN logit counts as -inf and +inf as the
// largest bf16 value.

#include <cooperative_groups.h>

#include "common.cuh"

namespace tf {
namespace {
namespace cg = cooperative_groups;

constexpr int kStatThreads = 256, kStatChunks = 4;                  // chunks of 8 logits a thread
constexpr int kSlice = kStatThreads * kStatChunks * 8;              // logits a slice
constexpr int kChoiceThreads = 512, kCluster = 8, kChoiceWarps = kChoiceThreads / 32;
constexpr int kSegment = 256;                                       // logits a warp takes at a time
constexpr int kMaxVocab = 1 << 20;
constexpr int kMaxSegments = kMaxVocab / kCluster / kSegment + 2;

struct VerifyArgs {
    const __nv_bfloat16 *logits, *draft;      // rows of V; draft may be null
    size_t stride, draft_stride;
    const int *tokens, *seq_start;
    const void* uniforms;                     // [R, 2]
    int *keep, *next;
    float2* stats;                            // [2 (target, draft)][R][slices]: maximum, sum
    int V, R, S, slices, u64;
    float c, draft_c;                         // log2e / temperature
    double inv, draft_inv;                    // 1 / temperature
};

__device__ __forceinline__ float tame(float x) {       // NaN -> -inf, +inf -> the largest bf16
    return x != x ? -INFINITY : fminf(x, 3.3895313892515355e38f);
}

// A row seen as chunks of eight logits on 16-byte boundaries: chunk c holds logits 8c - skew .. 8c - skew + 7, those that exist.
struct Row {
    const __nv_bfloat16* p;
    int skew, V;
    __device__ Row(const __nv_bfloat16* row, int V_) : p(row), skew((int)((reinterpret_cast<uintptr_t>(row) & 15) >> 1)), V(V_) {}
    __device__ int chunks() const { return (V + skew + 7) >> 3; }
    __device__ int first(int c) const { return 8 * c - skew; }
    __device__ void load(int c, float (&x)[8]) const {
        const int i = first(c);
        if (i >= 0 && i + 8 <= V) {
            unpack8(*reinterpret_cast<const uint4*>(p + i), x);
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = tame(x[e]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = i + e >= 0 && i + e < V ? tame(bf2f(p[i + e])) : -INFINITY;
        }
    }
};

__global__ void __launch_bounds__(kStatThreads) verify_stats_kernel(const VerifyArgs a) {
    __shared__ float red[kStatThreads / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool drafter = blockIdx.y >= (unsigned)a.R;
    const int row = blockIdx.y - (drafter ? a.R : 0);
    // rows behind the last sequence are nobody's, a first row was not drafted
    bool skip = row >= a.seq_start[a.S];
    if (drafter)
        for (int s = tid; s < a.S; s += kStatThreads) skip |= a.seq_start[s] == row;
    if (__syncthreads_or(skip)) return;
    const Row r(drafter ? a.draft + (size_t)row * a.draft_stride : a.logits + (size_t)row * a.stride, a.V);
    const float c = drafter ? a.draft_c : a.c;
    const int chunks = r.chunks(), c0 = blockIdx.x * (kSlice / 8) + tid;
    float x[kStatChunks][8], m = -INFINITY;
#pragma unroll
    for (int k = 0; k < kStatChunks; ++k) {
        if (c0 + k * kStatThreads < chunks) {
            r.load(c0 + k * kStatThreads, x[k]);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[k][e] = -INFINITY;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) m = fmaxf(m, x[k][e]);
    }
    m = warp_max(m);
    if (lane == 0) red[warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kStatThreads / 32; ++w) m = fmaxf(m, red[w]);
    __syncthreads();
    float s = 0.f;
    if (m > -INFINITY) {
#pragma unroll
        for (int k = 0; k < kStatChunks; ++k)
#pragma unroll
            for (int e = 0; e < 8; ++e) s += exp2f((x[k][e] - m) * c);
    }
    s = warp_sum(s);
    if (lane == 0) red[warp] = s;
    __syncthreads();
    if (tid == 0) {
        for (int w = 1; w < kStatThreads / 32; ++w) s += red[w];
        a.stats[(size_t)blockIdx.y * a.slices + blockIdx.x] = make_float2(m, s);
    }
}

// A row's maximum and sum from its slices, in 64 bits. Whole warps.
__device__ __forceinline__ void row_stats(const float2* st, int slices, double inv, float& m, double& z) {
    const int lane = threadIdx.x & 31;
    m = -INFINITY;
    for (int i = lane; i < slices; i += 32) m = fmaxf(m, st[i].x);
    m = warp_max(m);
    z = 0.0;
    if (m > -INFINITY)
        for (int i = lane; i < slices; i += 32)
            if (st[i].x > -INFINITY) z += st[i].y * exp(((double)st[i].x - m) * inv);
#pragma unroll
    for (int o = 16; o; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
}

__device__ __forceinline__ double block_sum(double v, double* warp_s) {     // every thread gets it
#pragma unroll
    for (int o = 16; o; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    __syncthreads();
    if ((threadIdx.x & 31) == 0) warp_s[threadIdx.x >> 5] = v;
    __syncthreads();
    double s = 0.0;
    for (int w = 0; w < kChoiceWarps; ++w) s += warp_s[w];
    return s;
}

enum Weights { kAll, kWithout, kResidual };     // p; p without the draft; max(p - q, 0)

__global__ void __launch_bounds__(kChoiceThreads) verify_choice_kernel(const VerifyArgs a) {
    __shared__ double warp_s[kChoiceWarps], seg[kMaxSegments], cum[kMaxSegments], share[4];
    __shared__ int first_out;
    pdl_launch_dependents();
    pdl_wait();
    cg::cluster_group cluster = cg::this_cluster();
    const int seq = blockIdx.x / kCluster, rank = blockIdx.x % kCluster;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int r0 = a.seq_start[seq], n = a.seq_start[seq + 1] - r0;
    if (n < 1) {                                 // a sequence without rows: the whole cluster leaves
        if (rank == 0 && tid == 0) { a.keep[seq] = 0; a.next[seq] = -1; }
        return;
    }
    auto uniform = [&](int row, int i) -> double {
        return a.u64 ? static_cast<const double*>(a.uniforms)[2 * (size_t)row + i] : (double)static_cast<const float*>(a.uniforms)[2 * (size_t)row + i];
    };
    // ---- which drafts are kept ----
    if (tid == 0) first_out = n - 1;
    __syncthreads();
    for (int t = warp; t < n - 1; t += kChoiceWarps) {
        const int row = r0 + t, x = a.tokens[row + 1];
        bool taken = false;
        if (x >= 0 && x < a.V) {
            float mp, mq = 0.f;
            double zp, zq = 1.0, q = 1.0;
            row_stats(a.stats + (size_t)row * a.slices, a.slices, a.inv, mp, zp);
            if (a.draft != nullptr) {
                row_stats(a.stats + ((size_t)a.R + row + 1) * a.slices, a.slices, a.draft_inv, mq, zq);
                q = exp(((double)tame(bf2f(a.draft[(size_t)(row + 1) * a.draft_stride + x])) - mq) * a.draft_inv) / zq;
            }
            const double p = exp(((double)tame(bf2f(a.logits[(size_t)row * a.stride + x])) - mp) * a.inv) / zp;
            taken = uniform(row, 0) * q < p;     // no probabilities (NaN): not taken
        }
        if (!taken && lane == 0) atomicMin(&first_out, t);
    }
    __syncthreads();
    const int last = first_out, row = r0 + last;
    if (rank == 0 && tid == 0) a.keep[seq] = last + 1;
    // ---- the weights that the next token is drawn from ----
    const bool full = last == n - 1;
    int mode = full ? kAll : a.draft == nullptr ? kWithout : kResidual;
    const int x = full ? -1 : a.tokens[row + 1];
    if (mode == kWithout && (x < 0 || x >= a.V)) mode = kAll;
    const Row p(a.logits + (size_t)row * a.stride, a.V), q(mode == kResidual ? a.draft + (size_t)(row + 1) * a.draft_stride : a.logits, a.V);
    float mp, mq = 0.f;
    double unused;
    row_stats(a.stats + (size_t)row * a.slices, a.slices, a.inv, mp, unused);
    if (mode == kResidual) row_stats(a.stats + ((size_t)a.R + row + 1) * a.slices, a.slices, a.draft_inv, mq, unused);
    const int chunks = p.chunks(), per = ((chunks + kCluster - 1) / kCluster + 31) / 32 * 32;
    const int lo = min(chunks, rank * per), hi = min(chunks, lo + per), segs = (hi - lo + 31) / 32;
    double zp = 1.0, zq = 1.0;
    auto target = [&](float v) -> double { return v > -INFINITY ? exp(((double)v - mp) * a.inv) : 0.0; };
    auto drafted = [&](int i) -> double {
        const float v = tame(bf2f(q.p[i]));
        return v > -INFINITY ? exp(((double)v - mq) * a.draft_inv) : 0.0;
    };
    if (mode == kResidual) {
        double sp = 0.0, sq = 0.0;
        for (int c = lo + tid; c < hi; c += kChoiceThreads) {
            float v[8];
            p.load(c, v);
            const int i = p.first(c);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                sp += target(v[e]);
                if (i + e >= 0 && i + e < a.V) sq += drafted(i + e);
            }
        }
        sp = block_sum(sp, warp_s);
        sq = block_sum(sq, warp_s);
        if (tid == 0) { share[0] = sp; share[1] = sq; }
        cluster.sync();
        zp = zq = 0.0;
        for (int k = 0; k < kCluster; ++k) {
            const double* o = cluster.map_shared_rank(share, k);
            zp += o[0];
            zq += o[1];
        }
        if (!(zq > 0.0)) zq = INFINITY;          // a drafter without any probability: nothing is taken off
    }
    auto weight = [&](float v, int i) -> double {
        if (i < 0 || i >= a.V || (mode == kWithout && i == x)) return 0.0;
        const double w = target(v);
        return mode == kResidual ? fmax(w / zp - drafted(i) / zq, 0.0) : w;
    };
    double before = 0.0, total = 0.0;
    int attempt = 0;
    for (;; ++attempt) {
        for (int s = warp; s < segs; s += kChoiceWarps) {
            double w = 0.0;
            const int c = lo + s * 32 + lane;
            if (c < hi) {
                float v[8];
                p.load(c, v);
                const int i = p.first(c);
#pragma unroll
                for (int e = 0; e < 8; ++e) w += weight(v[e], i + e);
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
            if (lane == 0) seg[s] = w;
        }
        __syncthreads();
        if (warp == 0) {                         // cumulative weights of the block's segments
            double base = 0.0;
            for (int s0 = 0; s0 < segs; s0 += 32) {
                double w = s0 + lane < segs ? seg[s0 + lane] : 0.0;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double y = __shfl_up_sync(0xffffffffu, w, o);
                    if (lane >= o) w += y;
                }
                if (s0 + lane < segs) cum[s0 + lane] = base + w;
                base += __shfl_sync(0xffffffffu, w, 31);
            }
            if (lane == 0) share[2 + attempt] = base;
        }
        cluster.sync();
        before = total = 0.0;
        for (int k = 0; k < kCluster; ++k) {
            const double w = *cluster.map_shared_rank(share + 2 + attempt, k);
            if (k < rank) before += w;
            total += w;
        }
        // nothing is left where p is nowhere above q but for rounding, or all of it is on the rejected draft: p itself
        if (total > 0.0 || mode == kAll) break;
        mode = kAll;                             // at most once: the second pass ends above
    }
    // ---- the first token whose cumulative weight is above the target ----
    if (warp == 0) {
        const double goal = uniform(row, 1) * total;
        // the block that holds it: the first whose end is above, the last one that has any weight if rounding leaves none
        int owner = -1;
        double sum = 0.0;
        for (int k = 0; k < kCluster; ++k) {
            const double w = *cluster.map_shared_rank(share + 2 + attempt, k);
            const bool reached = owner >= 0 && goal < sum;
            sum += w;
            if (w > 0.0 && !reached) owner = k;
        }
        if (owner < 0) {
            if (rank == 0 && lane == 0) a.next[seq] = -1;        // a row without any probability
        } else if (owner == rank) {
            const double at = goal - before;
            int found = -1;
            for (int s0 = 0; s0 < segs && found < 0; s0 += 32) {
                const unsigned m = __ballot_sync(0xffffffffu, s0 + lane < segs && seg[s0 + lane] > 0.0 && cum[s0 + lane] > at);
                if (m) found = s0 + __ffs(m) - 1;
            }
            if (found < 0)                       // rounding: the last segment with any weight
                for (int s = 0; s < segs; ++s)
                    if (seg[s] > 0.0) found = s;
            double w[8], own = 0.0;
            const int c = lo + found * 32 + lane, i = p.first(c);
            float v[8];
            if (c < hi) p.load(c, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) { w[e] = c < hi ? weight(v[e], i + e) : 0.0; own += w[e]; }
            double run = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += y;
            }
            run += (found > 0 ? cum[found - 1] : 0.0) - own;
            int hit = -1, positive = -1;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                run += w[e];
                if (w[e] > 0.0) {
                    positive = i + e;
                    if (hit < 0 && run > at) hit = i + e;
                }
            }
            const unsigned m = __ballot_sync(0xffffffffu, hit >= 0), any = __ballot_sync(0xffffffffu, positive >= 0);
            const int token = m ? __shfl_sync(0xffffffffu, hit, __ffs(m) - 1) : __shfl_sync(0xffffffffu, positive, 31 - __clz(any));
            if (lane == 0) a.next[seq] = token;
        }
    }
    cluster.sync();                              // nobody leaves while another block may read its sums
}

}  // namespace
}  // namespace tf

extern "C" {

size_t tf_verify_scratch_bytes(int rows, int vocab) {
    if (rows < 1 || vocab < 1 || vocab > tf::kMaxVocab) return 0;
    return (size_t)2 * rows * ((vocab + 7 + tf::kSlice - 1) / tf::kSlice) * sizeof(float2);
}

int tf_verify_rows(const void* logits, size_t row_stride, const void* draft_logits, size_t draft_stride, const int* tokens, const int* seq_start,
                   const void* uniforms, int uniforms_f64, int* keep, int* next, void* scratch, size_t scratch_bytes, int rows, int vocab,
                   int n_seqs, double temperature, double draft_temperature, void* stream) {
    if (rows < 1 || rows > 32767 || vocab < 1 || vocab > tf::kMaxVocab || n_seqs < 1 || n_seqs > (1 << 24)) return TF_EINVAL;
    if (!(temperature > 0.0) || !(draft_temperature > 0.0) || !(temperature < INFINITY) || !(draft_temperature < INFINITY)) return TF_EINVAL;
    if (!logits || !tokens || !seq_start || !uniforms || !keep || !next || row_stride < (size_t)vocab || (draft_logits && draft_stride < (size_t)vocab))
        return TF_EINVAL;
    if (((uintptr_t)logits | (uintptr_t)draft_logits) & 1 || (uintptr_t)uniforms & (uniforms_f64 ? 7 : 3) || (uintptr_t)scratch & 7) return TF_EALIGN;
    if (!scratch || scratch_bytes < tf_verify_scratch_bytes(rows, vocab)) return TF_ESCRATCH;
    tf::VerifyArgs a{static_cast<const __nv_bfloat16*>(logits), static_cast<const __nv_bfloat16*>(draft_logits), row_stride, draft_stride, tokens, seq_start,
                     uniforms, keep, next, static_cast<float2*>(scratch), vocab, rows, n_seqs, (vocab + 7 + tf::kSlice - 1) / tf::kSlice, uniforms_f64,
                     (float)(1.4426950408889634 / temperature), (float)(1.4426950408889634 / draft_temperature), 1.0 / temperature, 1.0 / draft_temperature};
    void* args[] = {&a};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (tf::launch_pdl((const void*)tf::verify_stats_kernel, dim3(a.slices, draft_logits ? 2 * rows : rows), dim3(tf::kStatThreads), 0, st, args) !=
        cudaSuccess) { cudaGetLastError(); return TF_ECUDA; }
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n_seqs * tf::kCluster);
    cfg.blockDim = dim3(tf::kChoiceThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = tf::kCluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = tf::pdl_enabled(0) ? 2 : 1;
    if (cudaLaunchKernelExC(&cfg, (const void*)tf::verify_choice_kernel, args) != cudaSuccess) { cudaGetLastError(); return TF_ECUDA; }
    return TF_OK;
}

}  // extern "C"
