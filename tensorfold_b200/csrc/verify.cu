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
// Two launches. Row statistics: a slice of 8192 logits a block, an offset o, the largest y = logit * log2e / T, and the sum of 2^(y - o) -
// bound by the bytes of the logits (128 + 112 rows of 248320: 24 us, 5 TB/s). Choice: a cluster of blocks per sequence; every
// block forms the acceptances from the slices' sums (64 bits), then the cluster goes over the one row that is drawn from, twice where a
// drafter's distribution has to be normalised too. 16 rows of 248320 with a drafter: 39 us, on the 96 SMs that 16 clusters of 6 take and
// with their 64-bit pipe busy 38 % of the time: the acceptances in front, loads that each warp waits for, the search and the cluster's
// barriers are the rest. One row without a drafter: 11 us, mostly its dependent steps. An acceptance is one comparison, so 32-bit exponentials (relative
// error of p and q near 1e-6) decide all but one in a million draws as exact arithmetic would; a draw compares one number with
// up to a million borders, so its weights and sums are in 64 bits throughout (relative error 1e-13). A NaN logit counts as -inf, +inf as a very
// large one (tame).

#include <cooperative_groups.h>

#include <utility>

#include "tc.cuh"

namespace tf {
namespace {
namespace cg = cooperative_groups;

constexpr int kStatThreads = 256, kStatChunks = 4;                  // chunks of 8 logits a thread
constexpr int kSlice = kStatThreads * kStatChunks * 8;              // logits a slice
constexpr int kChoiceThreads = 1024, kChoiceWarps = kChoiceThreads / 32;
constexpr int kKept = 128;                                          // window rows whose offsets are kept between the two steps
constexpr int kSegment = 256;                                       // logits a warp takes at a time
constexpr int kMaxVocab = 1 << 20;
constexpr uint32_t kNone = 0xFF80FF80u;                              // two bf16 -inf
constexpr int kSpan = 8;                                            // segments a span: the unit that sums are formed in and blocks are given
constexpr int kMaxSpans = kMaxVocab / (kSegment * kSpan) + 2, kLeastBlocks = 4, kMost = kMaxSpans / kLeastBlocks + 1;   // most: spans a block

struct VerifyArgs {
    const __nv_bfloat16 *logits, *draft;      // rows of V; draft may be null
    size_t stride, draft_stride;
    const int *tokens, *seq_start;
    const void* uniforms;                     // [R, 2]
    int *keep, *next;
    float2* stats;                            // [2 (target, draft)][R][slices]: maximum, sum
    int V, R, S, slices, u64;
    float c, draft_c, most, draft_most;       // log2e / temperature; the largest logit (see tame)
    double c64, draft_c64;
};

// NaN -> -inf; more than `most` -> `most`: logit / temperature up to 7e8, where an offset in 32 bits still leaves 2^(y - offset) in range
__device__ __forceinline__ float tame(float x, float most) { return x != x ? -INFINITY : fminf(x, most); }

// A row seen as chunks of eight logits on 16-byte boundaries: chunk c holds logits 8c - skew .. 8c - skew + 7, those that exist.
struct Row {
    const __nv_bfloat16* p;
    int skew, V;
    float most;
    __device__ Row(const __nv_bfloat16* row, int V_, float most_) : p(row), skew((int)((reinterpret_cast<uintptr_t>(row) & 15) >> 1)), V(V_), most(most_) {}
    __device__ int chunks() const { return (V + skew + 7) >> 3; }
    __device__ int first(int c) const { return 8 * c - skew; }
    __device__ uint4 raw(int c) const {          // -inf where there is none
        const int i = first(c);
        return i >= 0 && i + 8 <= V ? *reinterpret_cast<const uint4*>(p + i) : edge(i);
    }
    __device__ __noinline__ uint4 edge(int i) const {
        uint32_t u[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t lo = i + 2 * e >= 0 && i + 2 * e < V ? __bfloat16_as_ushort(p[i + 2 * e]) : kNone & 0xFFFFu;
            const uint32_t hi = i + 2 * e + 1 >= 0 && i + 2 * e + 1 < V ? __bfloat16_as_ushort(p[i + 2 * e + 1]) : kNone & 0xFFFFu;
            u[e] = lo | hi << 16;
        }
        return make_uint4(u[0], u[1], u[2], u[3]);
    }
};

// the larger of two bf16 pairs, a NaN losing to any number
__device__ __forceinline__ uint32_t max_pair(uint32_t x, uint32_t y) {
    const __nv_bfloat162 m = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&x), *reinterpret_cast<const __nv_bfloat162*>(&y));
    return *reinterpret_cast<const uint32_t*>(&m);
}

__global__ void __launch_bounds__(kStatThreads) verify_stats_kernel(const VerifyArgs a) {
    __shared__ float red[2][kStatThreads / 32];
    pdl_launch_dependents();
    pdl_wait();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const bool drafter = blockIdx.y >= (unsigned)a.R;
    const int row = blockIdx.y - (drafter ? a.R : 0);
    // rows behind the last sequence are nobody's, a first row was not drafted
    bool skip = row >= a.seq_start[a.S];
    if (drafter) {
        for (int s = tid; s < a.S; s += kStatThreads) skip |= a.seq_start[s] == row;
        if (__syncthreads_or(skip)) return;
    }
    const Row r(drafter ? a.draft + (size_t)row * a.draft_stride : a.logits + (size_t)row * a.stride, a.V,
                drafter ? a.draft_most : a.most);
    const float c = drafter ? a.draft_c : a.c;
    const int chunks = r.chunks(), c0 = blockIdx.x * (kSlice / 8) + tid;
    uint4 v[kStatChunks];
#pragma unroll
    for (int k = 0; k < kStatChunks; ++k) v[k] = c0 + k * kStatThreads < chunks ? r.raw(c0 + k * kStatThreads) : make_uint4(kNone, kNone, kNone, kNone);
    if (skip) return;                            // the whole block, where it is not a drafter's
    uint32_t m2 = kNone;
#pragma unroll
    for (int k = 0; k < kStatChunks; ++k) m2 = max_pair(max_pair(m2, max_pair(v[k].x, v[k].y)), max_pair(v[k].z, v[k].w));
    float m = warp_max(fmaxf(bf16_lo(m2), bf16_hi(m2)));
    if (lane == 0) red[0][warp] = m;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < kStatThreads / 32; ++w) m = fmaxf(m, red[0][w]);
    const float o = fminf(m, r.most) * c;
    float s = 0.f;
    if (o > -INFINITY) {
        const unsigned long long c2 = pair_of(c, c), o2 = pair_of(-o, -o);
        unsigned long long sum[2] = {0, 0};              // two zeros each
#pragma unroll
        for (int k = 0; k < kStatChunks; ++k) {
            const uint32_t u[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                float x, y;
                split_pair(fma_pair(pair_of(bf16_lo(u[e]), bf16_hi(u[e])), c2, o2), x, y);
                sum[e & 1] = add_pair(sum[e & 1], pair_of(fast_exp2(x), fast_exp2(y)));
            }
        }
        float x, y;
        split_pair(add_pair(sum[0], sum[1]), x, y);
        s = x + y;
    }
    s = warp_sum(s);
    if (lane == 0) red[1][warp] = s;
    __syncthreads();
    s = red[1][0];
#pragma unroll
    for (int w = 1; w < kStatThreads / 32; ++w) s += red[1][w];
    if (!(s < INFINITY)) {                       // a NaN or +inf among the logits: again, one by one
        s = 0.f;
#pragma unroll 1
        for (int k = 0; k < kStatChunks; ++k) {
            float x[8];
            unpack8(c0 + k * kStatThreads < chunks ? r.raw(c0 + k * kStatThreads) : make_uint4(kNone, kNone, kNone, kNone), x);
            for (int e = 0; e < 8; ++e) s += fast_exp2(fmaf(tame(x[e], r.most), c, -o));
        }
        s = warp_sum(s);
        __syncthreads();
        if (lane == 0) red[1][warp] = s;
        __syncthreads();
        s = red[1][0];
        for (int w = 1; w < kStatThreads / 32; ++w) s += red[1][w];
    }
    if (tid == 0) a.stats[(size_t)blockIdx.y * a.slices + blockIdx.x] = make_float2(o, s);
}

// A weight 2^(logit c - offset) in 64 bits, in the two factors of which the second is a table's: t = 16 (logit c - offset) = n + r, a table of
// 2^(j/16) times a factor of the row's own (128 bytes: no two entries share a bank; the high words less j << 16, so that adding n << 16 sets the
// exponent), and the series of 2^(r/16) to the fifth power (the next term is 1.5e-13 at |r| = 1/2). Ten operations of the 64-bit pipe
// with the product and eight others (a pass over a row is its weights' instructions and its loads). Weights end at 2^-900, which stands for 0 (NaN and
// -inf too): sums and weights up to kZero are none.
constexpr int kTable = 16;
constexpr double kZero = 1e-240;
__device__ __forceinline__ double table_entry(double value, int j) { return __hiloint2double(__double2hiint(value) - (j << 16), __double2loint(value)); }
struct Weight {
    double slope, shift;                         // 16 c, 16 offset
    float least, most;                           // logit of 2^-900, of the largest that counts
    const double* table;                         // shared memory
    // (a row of nothing has no offset: any will do)
    __device__ Weight(double c, float offset, float most_, const double* table_)
        : slope(kTable * c), shift(offset > -INFINITY ? kTable * (double)offset : 0.0), least((float)((shift / kTable - 900.0) / c)), most(most_), table(table_) {}
    __device__ void operator()(float v, double& series, double& factor) const {
        constexpr double l = 0.69314718055994530942 / kTable, shifter = 6755399441055744.0;   // 1.5 * 2^52: adding it leaves the nearest integer in the low word
        const double t = fma((double)fminf(fmaxf(v, least), most), slope, -shift), big = t + shifter, r = t - (big - shifter);
        const int n = __double2loint(big);
        double y = fma(r, l * l * l * l * l / 120, l * l * l * l / 24);
        y = fma(r, y, l * l * l / 6);
        y = fma(r, y, l * l / 2);
        y = fma(r, y, l);
        series = fma(r, y, 1.0);
        const double p = table[n & (kTable - 1)];
        factor = __hiloint2double(__double2hiint(p) + (n << 16), __double2loint(p));
    }
    __device__ double operator()(float v) const {
        double y, f;
        (*this)(v, y, f);
        return y * f;
    }
};

// A row's offset and sum from its slices. Whole warps.
__device__ __forceinline__ float row_offset(const float2* st, int slices) {
    float o = -INFINITY;
    for (int i = threadIdx.x & 31; i < slices; i += 32) o = fmaxf(o, st[i].x);
    return warp_max(o);
}
__device__ __forceinline__ double row_sum(const float2* st, int slices, float o, const double* table) {
    const Weight w(1.0, o, 3e9f, table);
    double z = 0.0;
    for (int i = threadIdx.x & 31; i < slices; i += 32) z += st[i].y * w(st[i].x);           // a slice of nothing has the sum 0
#pragma unroll
    for (int k = 16; k; k >>= 1) z += __shfl_xor_sync(0xffffffffu, z, k);
    return z;
}

enum Weights { kAll, kWithout, kResidual };     // p; p without the draft; max(p - q, 0)

__global__ void __launch_bounds__(kChoiceThreads, 1) verify_choice_kernel(const VerifyArgs a) {
    // sums of the block's spans: [0] p, [1] q, then the weights of the first and the second attempt; of its segments; of every block's spans
    __shared__ double table[kTable], table_p[kTable], table_q[kTable], span_s[4][kMost], seg[2 * kMost * kSpan], all_s[2][kMaxSpans];
    __shared__ float offset_s[2][kKept];         // target's and drafter's, of the window's first rows
    __shared__ int first_out;
    cg::cluster_group cluster = cg::this_cluster();
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    if (tid < kTable) table[tid] = table_p[tid] = table_q[tid] = table_entry(exp2(tid / (double)kTable), tid);
    pdl_launch_dependents();
    pdl_wait();
    const int blocks = cluster.num_blocks(), rank = cluster.block_rank(), seq = blockIdx.x / blocks;
    const int r0 = a.seq_start[seq], n = a.seq_start[seq + 1] - r0;
    if (r0 < 0 || n < 1 || r0 > a.R - n) {       // a sequence without rows, or not among the call's: the whole cluster leaves
        if (rank == 0 && tid == 0) { a.keep[seq] = 0; a.next[seq] = -1; }
        return;
    }
    auto uniform = [&](int row, int i) -> double {
        return a.u64 ? static_cast<const double*>(a.uniforms)[2 * (size_t)row + i] : (double)static_cast<const float*>(a.uniforms)[2 * (size_t)row + i];
    };
    // ---- which drafts are kept ----
    if (tid == 0) first_out = n - 1;
    __syncthreads();
    for (int t = warp; t < n; t += kChoiceWarps) {
        const int row = r0 + t;
        const float2 *st = a.stats + (size_t)row * a.slices, *sq = a.stats + ((size_t)a.R + min(row + 1, a.R - 1)) * a.slices;
        const float op = row_offset(st, a.slices);
        if (t == n - 1) {
            if (lane == 0 && t < kKept) offset_s[0][t] = op;
            break;
        }
        const int x = a.tokens[row + 1];
        const float oq = a.draft != nullptr ? row_offset(sq, a.slices) : 0.f;
        if (lane == 0 && t < kKept) { offset_s[0][t] = op; offset_s[1][t] = oq; }
        bool taken = false;
        if (x >= 0 && x < a.V) {
            const float vp = tame(bf2f(a.logits[(size_t)row * a.stride + x]), a.most);
            const float vq = a.draft != nullptr ? tame(bf2f(a.draft[(size_t)(row + 1) * a.draft_stride + x]), a.draft_most) : 0.f;
            const double u = uniform(row, 0);
            const double q = a.draft == nullptr ? 1.0 : Weight(a.draft_c, oq, a.draft_most, table)(vq) / row_sum(sq, a.slices, oq, table);
            const double p = vp > -INFINITY ? Weight(a.c, op, a.most, table)(vp) / row_sum(st, a.slices, op, table) : 0.0;
            taken = u * q < p;                   // no probabilities (NaN): not taken
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
    const Row p(a.logits + (size_t)row * a.stride, a.V, a.most), q(mode == kResidual ? a.draft + (size_t)(row + 1) * a.draft_stride : a.logits, a.V, a.draft_most);
    const bool abreast = p.skew == q.skew;       // the two rows' chunks hold the same tokens
    // any offset that keeps the largest weight near 1 will do: the statistics' one
    const float op = last < kKept ? offset_s[0][last] : row_offset(a.stats + (size_t)row * a.slices, a.slices);
    const float oq = mode != kResidual ? 0.f : last < kKept ? offset_s[1][last] : row_offset(a.stats + ((size_t)a.R + row + 1) * a.slices, a.slices);
    const double goal_u = uniform(row, 1);
    // the row in spans of 512 chunks, dealt out in runs; sums are formed by span and then over the spans in order, so that they do not depend
    // on how many blocks the cluster has
    const int chunks = p.chunks(), spans = (chunks + kSpan * 32 - 1) / (kSpan * 32), least = spans / blocks, more = spans - least * blocks;
    const int first = rank * least + min(rank, more), mine = least + (rank < more), lo = first * kSpan * 32, segs = mine * kSpan;
    // the block that holds span `tid`, and where
    const int in_more = more * (least + 1), holder = tid < in_more ? tid / (least + 1) : more + (tid - in_more) / max(least, 1);
    const int held_at = tid - holder * least - min(holder, more);
    const Weight target(a.c64, op, a.most, table_p), drafted(a.draft_c64, oq, a.draft_most, table_q);
    auto load_q = [&](int c, float (&v)[8]) { unpack8(abreast ? q.raw(c) : q.edge(p.first(c)), v); };
    // the sums over all spans of the cluster, in order, of `which` of the span sums and (two) of the next; all_s keeps them. The whole
    // block; the clusters' span sums are complete (a cluster barrier lies before).
    auto gather = [&](int which, bool two, double& second) -> double {
        static_assert(kMaxSpans <= kChoiceThreads, "a thread a span");
        __syncthreads();                         // all_s is no longer read
        if (tid < spans) {
            const double* from = cluster.map_shared_rank(&span_s[which][held_at], holder);
            const double x = from[0], y = two ? from[kMost] : 0.0;
            all_s[0][tid] = x;
            if (two) all_s[1][tid] = y;
        }
        __syncthreads();
        double sum = 0.0;
        second = 0.0;
        for (int i = lane; i < spans; i += 32) {
            sum += all_s[0][i];
            if (two) second += all_s[1][i];
        }
#pragma unroll
        for (int k = 16; k; k >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, k);
            if (two) second += __shfl_xor_sync(0xffffffffu, second, k);
        }
        return sum;
    };
    if (mode == kResidual) {
        // a warp a segment of 256 tokens; p and q of the span's segments are added by its sixteen warps' lanes below
        for (int s = warp; s < segs; s += kChoiceWarps) {
            double sp = 0.0, sq = 0.0;
            const int c = lo + s * 32 + lane;
            if (c < chunks) {
                float v[8], w[8];
                unpack8(p.raw(c), v);
                load_q(c, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) { sp += target(v[e]); sq += drafted(w[e]); }
            }
#pragma unroll
            for (int k = 16; k; k >>= 1) { sp += __shfl_xor_sync(0xffffffffu, sp, k); sq += __shfl_xor_sync(0xffffffffu, sq, k); }
            if (lane == 0) { seg[s] = sp; seg[segs + s] = sq; }
        }
        __syncthreads();
        for (int i = tid; i < 2 * mine; i += kChoiceThreads) {
            const double* from = seg + (i < mine ? 0 : segs) + (i < mine ? i : i - mine) * kSpan;
            double sum = 0.0;
#pragma unroll
            for (int k = 0; k < kSpan; ++k) sum += from[k];
            span_s[i < mine ? 0 : 1][i < mine ? i : i - mine] = sum;
        }
        cluster.sync();
        double zq;
        const double zp = gather(0, true, zq);
        // the normalisers go into the tables; a drafter without any probability takes nothing off (2^-900 a token)
        if (tid < kTable) {
            const double whole = exp2(tid / (double)kTable);
            table_p[tid] = table_entry(zp > kZero ? whole / zp : whole, tid);
            table_q[tid] = table_entry(zq > kZero ? whole / zq : whole, tid);
        }
        __syncthreads();
    }
    auto weights = [&](int c, double (&w)[8]) {  // of chunk c
        float v[8];
        unpack8(p.raw(c), v);
        const int i = p.first(c);
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = target(v[e]);
        if (mode == kResidual) {
            load_q(c, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                double y, f;
                drafted(v[e], y, f);
                const double rest = fma(-y, f, w[e]);
                w[e] = __double2hiint(rest) < 0 ? 0.0 : rest;
            }
        } else if (mode == kWithout) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (i + e == x) w[e] = 0.0;
        }
    };
    double total, unused;
    for (int attempt = 0;; ++attempt) {
        for (int s = warp; s < segs; s += kChoiceWarps) {
            double sum = 0.0;
            const int c = lo + s * 32 + lane;
            if (c < chunks) {
                double w[8];
                weights(c, w);
#pragma unroll
                for (int e = 0; e < 8; ++e) sum += w[e];
            }
#pragma unroll
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            if (lane == 0) seg[s] = sum;
        }
        __syncthreads();
        for (int i = tid; i < mine; i += kChoiceThreads) {
            double sum = 0.0;
#pragma unroll
            for (int k = 0; k < kSpan; ++k) sum += seg[i * kSpan + k];
            span_s[2 + attempt][i] = sum;
        }
        cluster.sync();
        total = gather(2 + attempt, false, unused);
        // nothing is left where p is nowhere above q but for rounding, or all of it is on the refused draft: p itself
        if (total > kZero || mode == kAll) break;
        mode = kAll;                             // at most once: the second pass ends above
    }
    auto others = cluster.barrier_arrive();      // this block has read what it needs of the others
    // ---- the first token whose cumulative weight is above the goal ----
    if (warp == 0) {
        const double goal = goal_u * total;
        // a warp's search in `count` weights: the first whose cumulative weight is above `at`, or the last with any if rounding leaves none; `at`
        // becomes what is left of it there. -1: no weight at all
        auto search = [&](const double* w, int count, double& at) -> int {
            double base = 0.0, start_of_last = 0.0;
            int last_with = -1;
            for (int i0 = 0; i0 < count; i0 += 32) {
                const double v = i0 + lane < count ? w[i0 + lane] : 0.0;
                double run = v;
#pragma unroll
                for (int o = 1; o < 32; o <<= 1) {
                    const double y = __shfl_up_sync(0xffffffffu, run, o);
                    if (lane >= o) run += y;
                }
                run += base;
                const unsigned above = __ballot_sync(0xffffffffu, v > kZero && run > at), any = __ballot_sync(0xffffffffu, v > kZero);
                const int who = above ? __ffs(above) - 1 : 31 - __clz(any);
                if (any) {
                    last_with = i0 + who;
                    start_of_last = __shfl_sync(0xffffffffu, run - v, who);
                }
                if (above) break;
                base = __shfl_sync(0xffffffffu, run, 31);
            }
            at -= start_of_last;
            return last_with;
        };
        double at = goal;
        const int span = search(all_s[0], spans, at);
        if (span < 0) {
            if (rank == 0 && lane == 0) a.next[seq] = -1;        // a row without any probability
        } else if (span >= first && span < first + mine) {
            const int found = (span - first) * kSpan + search(seg + (span - first) * kSpan, kSpan, at);
            double w[8] = {0, 0, 0, 0, 0, 0, 0, 0}, own = 0.0;
            const int c = lo + found * 32 + lane, i = p.first(c);
            if (c < chunks) weights(c, w);
#pragma unroll
            for (int e = 0; e < 8; ++e) own += w[e];
            double run = own;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double y = __shfl_up_sync(0xffffffffu, run, o);
                if (lane >= o) run += y;
            }
            run -= own;
            int hit = -1, positive = -1;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                run += w[e];
                if (w[e] > kZero) {
                    positive = i + e;
                    if (hit < 0 && run > at) hit = i + e;
                }
            }
            const unsigned m = __ballot_sync(0xffffffffu, hit >= 0), any = __ballot_sync(0xffffffffu, positive >= 0);
            const int token = m ? __shfl_sync(0xffffffffu, hit, __ffs(m) - 1) : __shfl_sync(0xffffffffu, positive, 31 - __clz(any));
            if (lane == 0) a.next[seq] = token;
        }
    }
    cluster.barrier_wait(std::move(others));     // nobody leaves while another block may read its sums
}

// Blocks a sequence: as many as still let all sequences' clusters run at the same time, which the GPU is asked once. Of 148 SMs 7 clusters of 16,
// 11 of 10, 15 of 9 (and of 8 or 7), 22 of 6, 26 of 5, 33 of 4 fit: 16 sequences as clusters of 8 took two rounds, 53 us against 50 of 6 at the
// time; 24 of 5 take 78.6 us, of 4 84.8. All 26 of 5 do not always run at once (46 us without a drafter, 40 of 4): one less. Four where even those
// do not fit.
int cluster_for(int n_seqs) {
    constexpr int kSizes[] = {16, 10, 9, 6, 5, kLeastBlocks}, kCount = 6;
    static std::atomic<int> fits[64][kCount];    // per device; the last one 0: not asked yet (threads that ask at the same time find the same)
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return 0; }
    if (fits[dev][kCount - 1] == 0) {
        if (cudaFuncSetAttribute(verify_choice_kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess) { cudaGetLastError(); return 0; }
        for (int i = 0; i < kCount; ++i) {
            cudaLaunchConfig_t cfg = {};
            cfg.gridDim = dim3(kSizes[i]);
            cfg.blockDim = dim3(kChoiceThreads);
            cudaLaunchAttribute attr[1];
            attr[0].id = cudaLaunchAttributeClusterDimension;
            attr[0].val.clusterDim.x = kSizes[i];
            attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
            cfg.attrs = attr;
            cfg.numAttrs = 1;
            int n = 0;
            if (cudaOccupancyMaxActiveClusters(&n, verify_choice_kernel, &cfg) != cudaSuccess) { cudaGetLastError(); n = 0; }
            fits[dev][i] = n < 1 ? -1 : n;
        }
    }
    for (int i = 0; i + 1 < kCount; ++i)
        if (fits[dev][i] - (kSizes[i] == 5) >= n_seqs) return kSizes[i];
    return fits[dev][kCount - 1] > 0 ? kLeastBlocks : 0;
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
    if (!(temperature >= 1e-6) || !(draft_temperature >= 1e-6) || !(temperature <= 1e6) || !(draft_temperature <= 1e6)) return TF_EINVAL;
    if (!logits || !tokens || !seq_start || !uniforms || !keep || !next || row_stride < (size_t)vocab || (draft_logits && draft_stride < (size_t)vocab))
        return TF_EINVAL;
    if (((uintptr_t)logits | (uintptr_t)draft_logits) & 1 || (uintptr_t)uniforms & (uniforms_f64 ? 7 : 3) || (uintptr_t)scratch & 7) return TF_EALIGN;
    if (!scratch || scratch_bytes < tf_verify_scratch_bytes(rows, vocab)) return TF_ESCRATCH;
    const double c = 1.4426950408889634 / temperature, draft_c = 1.4426950408889634 / draft_temperature, top = 1 << 30;
    tf::VerifyArgs a{static_cast<const __nv_bfloat16*>(logits), static_cast<const __nv_bfloat16*>(draft_logits), row_stride, draft_stride, tokens, seq_start,
                     uniforms, keep, next, static_cast<float2*>(scratch), vocab, rows, n_seqs, (vocab + 7 + tf::kSlice - 1) / tf::kSlice, uniforms_f64,
                     (float)c, (float)draft_c, (float)(top / c), (float)(top / draft_c), c, draft_c};
    void* args[] = {&a};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    if (tf::launch_pdl((const void*)tf::verify_stats_kernel, dim3(a.slices, draft_logits ? 2 * rows : rows), dim3(tf::kStatThreads), 0, st, args) !=
        cudaSuccess) { cudaGetLastError(); return TF_ECUDA; }
    const int blocks = tf::cluster_for(n_seqs);
    if (blocks < 1) return TF_ECUDA;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(n_seqs * blocks);
    cfg.blockDim = dim3(tf::kChoiceThreads);
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = blocks;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = tf::pdl_enabled(0) ? 2 : 1;
    if (cudaLaunchKernelExC(&cfg, (const void*)tf::verify_choice_kernel, args) != cudaSuccess) { cudaGetLastError(); return TF_ECUDA; }
    return TF_OK;
}

}  // extern "C"
