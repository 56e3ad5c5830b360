// Lane attention with a sliding window and sinks over the paged KV cache, on the 5th-generation tensor cores.
//
// Row t of a sequence's window stands at slot p = L + t (L committed keys) and sees key j when j <= p and
// (p - j < window or j < sinks): softmax of its scores over those keys, the weighted sum of their values, and the
// log-sum-exp of the scores.
//
// The key axis is cut by ABSOLUTE position into chunks; a block handles one chunk of one (sequence, KV head) for up to 128 query
// rows (window rows x the KV head's query heads, row = t * G + head). A row's chunks are joined in order by a second kernel or, where rows and chunks are
// few, by the cluster of blocks that holds them; a row of one chunk is finished by its block. In a block the keys go by in tiles of 64:
//
//   S = Q K^T        tcgen05, both operands in shared memory, 128 x 64 sums in tensor memory (two buffers)
//   P = 2^(S - m)    four warps, a thread a row: no shuffles; P goes where S was, as bf16. m is a maximum that is only moved when a score exceeds it by 2^8, so the
//                    sums so far are rescaled seldom (exactly the rows that need it change: multiplying by 1 keeps bits)
//   O += P V         tcgen05, P in tensor memory, V in shared memory as it lies in the cache (rows are the contraction's index)
//
// P is rounded to bf16 because the tensor core takes both operands in one type and V is bf16: at most 2^-8 of a term, without bias, beside the
// results' own 2^-8 (relative error of the results in the 2-norm against 64 bits 0.0021 to 0.0024, 0.0017 where only the results are rounded;
// the older lane attention rounds P the same way). Scores, maxima, the sums of the unrounded P and the log-sum-exps are fp32. A remainder of P as a second operand would
// take its place in shared memory or double the products, and was not tried.
//
// What bounds it. Many users: memory (16 users, 2 to 8 rows, a window of 4096: 262 MB in 53 us, 4.9 TB/s, with 4 us before for the plan and 5
// behind for the join). A prompt's rows with heads of 128: the chain scores - maximum - weights - product of a tile, of which two blocks an SM hide
// a part (2900 rows, a window of 1024: 45 us for 19 GFLOP, 63 with one block and a join). One row: latency (10 us for a window of 1024 keys, 14 of 4096).
//
// K and V arrive by tiled copies (TMA), a page of 16 keys at a time, into rings of their own. A page that not all rows see whole
// (around the committed length, the window's far edge, the sinks' end) is written by its producer warp instead, keys that no
// row sees as zeros without being read. There a value that is not finite is written as zero and noted: the results of rows that see its key
// become NaN (their log-sum-exps, which do not depend on values, stay), rows that do not keep their bits. Keys on a page that is none
// (reported) are NaN, and so are the rows that see them. Every step of a row's arithmetic is fixed by its own position and keys and by the
// chunk size, so a row alone, in a window and as a serial step has the same bits.

#include <cooperative_groups.h>

#include <utility>

#include "tc.cuh"

namespace tf {
namespace {
namespace cg = cooperative_groups;

constexpr int kPage = 16, kTile = 64, kRows = 128;     // keys a page, keys a tile, query rows a block (the tensor core's M)
constexpr int kSoftWarps = 4, kMmaWarp = 4, kQWarp = 5, kKWarp = 6, kVWarp = 8, kProducers = 2, kThreads = 10 * 32, kSms = 148;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr uint32_t kNan2 = 0x7FC07FC0u;                // two bf16 NaN
constexpr float kSlack = 8.f;                          // how far (log2) a score may exceed the running maximum

// n / d for 0 <= n < 2^31 without a division: d's reciprocal as a 32-bit fraction, rounded up (exact for n below 2^31 with the
// shift that makes the fraction's error less than 1 / n).
struct FastDiv {
    unsigned d, mul, shift;
    __device__ int operator()(int n) const { return d == 1 ? n : (int)(__umulhi((unsigned)n, mul) >> shift); }
};
inline FastDiv fast_div(int d) {
    unsigned bits = 0;
    while ((1ull << bits) < (unsigned long long)d) ++bits;                     // ceil(log2 d)
    if (d == 1) return {1u, 0u, 0u};
    return {(unsigned)d, (unsigned)(((1ull << (31 + bits)) + d - 1) / d), bits - 1};
}

struct WindowArgs {
    const __nv_bfloat16 *q, *k_new, *v_new, *k_pages, *v_pages;
    const int *page_table, *seq_lens, *seq_start;
    float *part_o, *part_m, *part_l;   // [slots, R, H, D], [slots, R, H] (m in the log2 domain)
    __nv_bfloat16* out;                // [R, H, D] or null
    float* lse;                        // [R, H] or null
    const __nv_bfloat16* qg;           // output gate or null
    size_t qg_stride;
    uint8_t* out_packed;               // or null
    int* status;
    int num_pages, max_pages, H, HK, R, S, window, sinks, max_context, max_window, group;
    int chunk, first_slots, near_slots, slots;         // keys a chunk; slots of the sinks' chunks, of the window's, of both
    int qgroups, group_rows, items;                    // groups of window rows, rows a group; (group, slot, KV head, sequence) in all
    FastDiv by_group, by_slot, by_head, by_G, by_chunk;
    int* plan;                         // [rounds, blocks] items by block, -1: none; null: block b takes items b, b + blocks, ...
    int rounds, blocks;                // blocks: of a full GPU
    bool direct;                       // one chunk a row and nothing to be done to the results: no join
    float scale_log2;
};

// The slots of a call's partials: the chunks that hold sinks keep their own, the window's go round the others. A sequence's
// rows see at most window + max_window - 1 keys apart from the sinks, which lie in at most near_slots consecutive chunks.
struct Slots {
    int first, near;
};
__host__ __device__ inline Slots slots_for(int window, int sinks, int max_window, int max_context, int chunk) {
    const int total = (max_context + chunk - 1) / chunk;
    if (window == 0) return {0, total};
    const long long keys = (long long)window + max_window - 1;
    const int first = sinks >= max_context ? total : (sinks + chunk - 1) / chunk;
    const long long touched = (keys + chunk - 2) / chunk + 1;
    return {first, (int)(touched < total - first ? touched : total - first)};
}
__device__ __forceinline__ int slot_of(int chunk, int first, int near) { return chunk < first ? chunk : first + (chunk - first) % near; }

// The sequence that holds packed row `row`: the last one that starts at or before it (a sequence without rows starts where the
// next one does, and is passed over), and where it starts; -1 for a row behind the last sequence. Whole warps; one load for up to 31
// sequences.
__device__ __forceinline__ int seq_of(const int* seq_start, int S, int row, int& start) {
    const int lane = threadIdx.x & 31;
    int found = -1;
    for (int s0 = 0; s0 <= S; s0 += 32) {
        const int v = s0 + lane <= S ? seq_start[s0 + lane] : 0x7FFFFFFF;
        const unsigned m = __ballot_sync(0xffffffffu, v <= row);
        if (m) {
            found = s0 + 31 - __clz(m);
            start = __shfl_sync(0xffffffffu, v, 31 - __clz(m));
        }
        if (m != 0xffffffffu) break;
    }
    return found >= S ? -1 : found;              // at or behind seq_start[S]
}

// One chunk of one (sequence, KV head) for one group of window rows; every role of a block forms it by itself.
struct Work {
    int seq, kvh, slot, t0, r0, n, L, p_first, p_last, lo_first, lo_last, nq, key0, head_tiles, far_tile, tiles, sinks;
    // tile i of the block: those of the sinks, then those of the window
    __device__ int base(int i) const { return key0 + (i < head_tiles ? i : far_tile + i - head_tiles) * kTile; }
    // 0: a committed page that every row sees whole, 1: 16 window rows that every row sees, 2: anything else
    __device__ int kind(int j) const {
        if (j + kPage > p_first + 1 || !(j >= lo_last || j + kPage <= sinks)) return 2;
        return j + kPage <= L ? 0 : j >= L ? 1 : 2;
    }
    // every row sees the tile whole, and no page of it is part committed, part new: nothing to mask, nothing noted
    __device__ bool plain(int j) const {
        return j + kTile <= p_first + 1 && (j >= lo_last || j + kTile <= sinks) && !((L & (kPage - 1)) != 0 && j < L && L < j + kTile);
    }
    __device__ bool any_sees(int j) const { return j <= p_last && (j >= lo_first || j < sinks); }
};
struct Raw {           // what an item needs from memory
    int r0, r1, L;
};
__device__ __forceinline__ Raw fetch(const WindowArgs& a, int item) {
    if (item < 0) return {0, 0, 0};
    const int seq = a.by_head(a.by_slot(a.by_group(item)));
    return {a.seq_start[seq], a.seq_start[seq + 1], a.seq_lens[seq]};
}
__device__ __forceinline__ Work work_of(const WindowArgs& a, int item, Raw raw, bool speaks) {
    Work w;
    const int G = (int)a.by_G.d, in_group = a.by_group(item), in_slot = a.by_slot(in_group);
    w.seq = a.by_head(in_slot);
    w.kvh = in_slot - w.seq * a.HK;
    w.slot = in_group - in_slot * a.slots;
    w.t0 = (item - in_group * a.qgroups) * a.group_rows;
    w.r0 = raw.r0;
    w.n = raw.r1 - raw.r0;
    w.L = raw.L;
    w.sinks = a.sinks;
    w.tiles = 0;
    const int rows = min(a.group_rows, w.n - w.t0);
    w.nq = 0;
    if (w.n < 1) return w;
    if (w.n > a.max_window || w.L < 0 || w.L > a.max_context - w.n || w.r0 < 0 || w.r0 > a.R - w.n) {     // not what the call was made for
        if (speaks) report(a.status, TF_EINVAL);
        return w;
    }
    if (rows < 1) return w;
    w.p_first = w.L + w.t0;
    w.p_last = w.p_first + rows - 1;
    w.nq = rows * G;
    w.lo_first = max(0, w.p_first + 1 - a.window);
    w.lo_last = max(0, w.p_last + 1 - a.window);
    int chunk = w.slot;
    if (chunk >= a.first_slots) {
        const int lowest = max(a.first_slots, a.by_chunk(max(0, w.L + 1 - a.window)));        // of the sequence: its rows share the slots
        chunk = lowest + ((w.slot - lowest) % a.near_slots + a.near_slots) % a.near_slots;
    }
    w.key0 = chunk * a.chunk;
    if (w.key0 > w.p_last) return w;
    const int in_chunk = (min(w.key0 + a.chunk, w.p_last + 1) - w.key0 + kTile - 1) / kTile;
    w.head_tiles = w.sinks > w.key0 ? min(in_chunk, (w.sinks - w.key0 + kTile - 1) / kTile) : 0;
    w.far_tile = max(w.head_tiles, w.lo_first > w.key0 ? (w.lo_first - w.key0) / kTile : 0);
    w.tiles = w.head_tiles + max(0, in_chunk - w.far_tile);
    return w;
}

// A role's walk over its block's items. What the next one needs is fetched while the one before it is worked on.
struct Walk {
    int item, next, k = 0;
    Raw raw;
    __device__ explicit Walk(const WindowArgs& a) : item(at(a, 0)), next(at(a, 1)), raw(fetch(a, item)) {}
    __device__ static int at(const WindowArgs& a, int k) {
        if (a.plan != nullptr) return k < a.rounds ? a.plan[k * a.blocks + blockIdx.x] : -1;
        const int i = blockIdx.x + k * gridDim.x;
        return i < a.items ? i : -1;
    }
    __device__ Work work(const WindowArgs& a, bool speaks) {
        const Work w = work_of(a, item, raw, speaks);
        raw = fetch(a, next);
        return w;
    }
    __device__ void step(const WindowArgs& a) {
        item = next;
        next = at(a, ++k + 1);
    }
};

// Which block takes which items, where a block takes several: the items that have work, by falling weight, dealt out back and forth, so that
// the blocks end together (16 users: 40 tiles of 64 keys on the busiest block without it, 28 on average). One block; the
// order among equals does not matter, no item's result depends on where it runs.
constexpr int kPlanThreads = 1024, kPlanItems = 8192, kPlanBins = 128;
constexpr size_t kPlanBytes = ((kPlanItems + 2 * kSms) * sizeof(int) + 255) / 256 * 256;
__global__ void __launch_bounds__(kPlanThreads) window_plan_kernel(const WindowArgs a) {
    __shared__ int count[kPlanBins], start[kPlanBins];
    pdl_launch_dependents();
    const int tid = threadIdx.x;
    if (tid < kPlanBins) count[tid] = 0;
    pdl_wait();                                  // the plan may still be the one of a call before this
    for (int i = tid; i < a.rounds * a.blocks; i += kPlanThreads) a.plan[i] = -1;
    __syncthreads();
    constexpr int PER = kPlanItems / kPlanThreads;
    int place[PER];                              // bin << 16 | rank in it
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        const int item = tid + k * kPlanThreads;
        place[k] = -1;
        if (item >= a.items) continue;
        const int tiles = work_of(a, item, fetch(a, item), true).tiles;
        if (tiles == 0) continue;
        const int bin = kPlanBins - 1 - min(tiles, kPlanBins - 1);
        place[k] = bin << 16 | atomicAdd(&count[bin], 1);
    }
    __syncthreads();
    if (tid < 32) {
        int before = 0;
        for (int b0 = 0; b0 < kPlanBins; b0 += 32) {
            const int c = count[b0 + tid];
            int x = c;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (tid >= o) x += y;
            }
            start[b0 + tid] = before + x - c;
            before += __shfl_sync(0xffffffffu, x, 31);
        }
    }
    __syncthreads();
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        if (place[k] < 0) continue;
        const int at = start[place[k] >> 16] + (place[k] & 0xFFFF), round = at / a.blocks, in_round = at - round * a.blocks;
        a.plan[round * a.blocks + (round & 1 ? a.blocks - 1 - in_round : in_round)] = tid + k * kPlanThreads;
    }
}

// Blocks an SM: with heads of 128 a second one fits, and one's softmax runs beside the other's products; heads of 256 fill the
// shared memory.
__host__ __device__ constexpr int blocks_of(int head_dim) { return head_dim == 128 ? 2 : 1; }

template <int D, int QR>
struct Cfg {
    static constexpr int SLABS = D / 64;                 // 64 values of a row: one 128-byte swizzle row
    static constexpr int Q_SLAB = QR * 128, Q_BYTES = SLABS * Q_SLAB;
    static constexpr int TILE_BYTES = kTile * D * 2, K_SLAB = kTile * 128, PAGE_BYTES = kPage * D * 2;
    static constexpr int BLOCKS = blocks_of(D), MEMORY = (BLOCKS == 2 ? 113 : 227) * 1024;
    // results on their way out: 16 or 32 partial values a row, or 32 finished ones
    static constexpr int STAGE = BLOCKS == 2 ? 16 : 32, STAGE_ROW = STAGE * 4 + 16, STAGE_BYTES = kSoftWarps * 32 * STAGE_ROW;
    static constexpr int FIT = (MEMORY - 2560 - STAGE_BYTES - Q_BYTES) / TILE_BYTES;
    static constexpr int KS = FIT / 2 > 4 ? 4 : FIT / 2, VS = FIT - FIT / 2 > 4 ? 4 : FIT - FIT / 2;
    static constexpr int NBARS = 2 * KS + 2 * VS + 6 + 2;
    static constexpr int SMEM = Q_BYTES + (KS + VS) * TILE_BYTES + STAGE_BYTES + NBARS * 8 + VS * 8 + 1024;
    // tensor memory: O and two buffers of S; P (bf16 pairs) takes the place of the scores it is made from
    static constexpr int O_COL = 0, S_COL = D, COLS = D == 128 ? 256 : 512;
    static_assert(KS >= 2 && SMEM + 64 <= MEMORY, "the rings do not fit");
    static_assert(S_COL + 2 * kTile <= COLS, "tensor memory");
    // a block of fewer than 128 rows leaves the last rows of the tensor core's Q operand to whatever follows in shared memory
    static_assert((kRows - QR) * 128 <= (KS + VS) * TILE_BYTES, "the operand's rows lie inside the block's memory");
};

// The chunks of a row at slot p, joined in order, eight columns a lane: `read` fetches a slot's maximum, sum and columns, B at a time. Chunks in
// which the row sees nothing are passed over, so the join does not depend on which chunks the rows beside it needed.
template <int B, class Read>
__device__ __forceinline__ void join_chunks(const WindowArgs& a, int p, Read read, float (&acc)[8], float& m, float& l) {
    const int lo = max(0, p + 1 - a.window);
    // chunks with sinks below the window, then the window's
    const int head_chunks = min(a.sinks, lo) > 0 ? a.by_chunk(min(a.sinks, lo) - 1) + 1 : 0;
    const int far = max(head_chunks, a.by_chunk(lo)), count = head_chunks + a.by_chunk(p) + 1 - far;
    m = -INFINITY;
    l = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    for (int i0 = 0; i0 < count; i0 += B) {
        float cm[B], cl[B];
        float4 po[B][2];
#pragma unroll
        for (int k = 0; k < B; ++k) {
            cl[k] = 0.f;
            if (i0 + k >= count) continue;
            const int i = i0 + k, chunk = i < head_chunks ? i : far + i - head_chunks;
            read(slot_of(chunk, a.first_slots, a.near_slots), cm[k], cl[k], po[k]);
        }
#pragma unroll
        for (int k = 0; k < B; ++k) {
            if (cl[k] == 0.f) continue;                                // NaN goes on
            const float mn = fmaxf(m, cm[k]), sa = fast_exp2(m - mn), sb = fast_exp2(cm[k] - mn);      // m = -inf: sa = 0
            const float x[8] = {po[k][0].x, po[k][0].y, po[k][0].z, po[k][0].w, po[k][1].x, po[k][1].y, po[k][1].z, po[k][1].w};
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = fmaf(x[e], sb, acc[e] * sa);
            l = fmaf(cl[k], sb, l * sa);
            m = mn;
        }
    }
}

// A joined row on its way out. Whole warps (the packed form's group sums), `there`: this lane has a row.
template <int D>
__device__ __forceinline__ void finish_row(const WindowArgs& a, int row, int head, int li, bool there, const float (&acc)[8], float m, float l) {
    if (a.lse != nullptr && li == 0 && there) a.lse[(size_t)row * a.H + head] = (m + log2f(l)) * kLn2;
    const float inv = 1.f / l;               // (one chunk: the same operations as where the chunk kernel writes the results)
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = round_bf16(acc[e] * inv);
    if (a.qg != nullptr && there) {
        float g[8];
        unpack8(*reinterpret_cast<const uint4*>(a.qg + (size_t)row * a.qg_stride + (size_t)head * 2 * D + D + li * 8), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = round_bf16(o[e] * sigmoidf_(g[e]));
    }
    const uint4 v = pack8(o);
    if (a.out != nullptr && there) *reinterpret_cast<uint4*>(a.out + ((size_t)row * a.H + head) * D + li * 8) = v;
    if (a.out_packed != nullptr) {
        const int Mp = tf_padded_rows(a.R), c8 = head * (D / 8) + li;
        const float sum = a.group == 64 ? group_sum8<64>(v) : group_sum8<32>(v);
        if (there) {
            if (a.group == 64) packed_store<64>(a.out_packed, Mp, row, c8, v, sum);
            else packed_store<32>(a.out_packed, Mp, row, c8, v, sum);
        }
    }
}
// Padding rows of the packed buffer are zero.
__device__ __forceinline__ void zero_packed(const WindowArgs& a, int row, int c8) {
    const int Mp = tf_padded_rows(a.R);
    if (a.group == 64) packed_store<64>(a.out_packed, Mp, row, c8, make_uint4(0, 0, 0, 0), 0.f);
    else packed_store<32>(a.out_packed, Mp, row, c8, make_uint4(0, 0, 0, 0), 0.f);
}

__device__ __forceinline__ float max3(float x, float y, float z) {
    float v;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(v) : "f"(x), "f"(y), "f"(z));
    return v;
}

// CLUSTER: the blocks of a cluster hold all chunks of a (sequence, KV head), one each, and join them through each other's shared memory.
template <int D, int QR, bool CLUSTER>
__global__ void __launch_bounds__(kThreads, blocks_of(D)) window_chunk_kernel(const __grid_constant__ WindowArgs a, const __grid_constant__ CUtensorMap q_map,
                                                                   const __grid_constant__ CUtensorMap k_map, const __grid_constant__ CUtensorMap v_map,
                                                                   const __grid_constant__ CUtensorMap kn_map, const __grid_constant__ CUtensorMap vn_map) {
    using C = Cfg<D, QR>;
    constexpr int KS = C::KS, VS = C::VS, CPR = D / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t tmem_s;
    __shared__ float2 sums_s[CLUSTER ? QR : 1];    // CLUSTER: maximum and sum of the block's rows; their values lie where K and V were
    constexpr int JOIN_ROW = D * 4 + 16;
    static_assert(!CLUSTER || QR * JOIN_ROW <= (KS + VS) * C::TILE_BYTES, "the rows' values fit");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t* q_s = smem + ((1024u - (smem_u32(smem) & 1023u)) & 1023u);
    uint8_t* k_s = q_s + C::Q_BYTES;
    uint8_t* v_s = k_s + KS * C::TILE_BYTES;
    uint8_t* stage_s = v_s + VS * C::TILE_BYTES;
    const uint32_t bars = smem_u32(stage_s + C::STAGE_BYTES);
    uint32_t* bad_s = reinterpret_cast<uint32_t*>(stage_s + C::STAGE_BYTES + C::NBARS * 8);      // [VS][2]
    auto k_full = [&](int s) { return bars + 8u * s; };
    auto k_empty = [&](int s) { return bars + 8u * (KS + s); };
    auto v_full = [&](int s) { return bars + 8u * (2 * KS + s); };
    auto v_empty = [&](int s) { return bars + 8u * (2 * KS + VS + s); };
    auto s_full = [&](int s) { return bars + 8u * (2 * KS + 2 * VS + s); };
    auto p_full = [&](int s) { return bars + 8u * (2 * KS + 2 * VS + 2 + s); };
    auto o_done = [&](int s) { return bars + 8u * (2 * KS + 2 * VS + 4 + s); };      // P V of a tile is complete
    const uint32_t q_full = bars + 8u * (2 * KS + 2 * VS + 6), q_empty = q_full + 8;

    if (tid == 0) {
        for (int s = 0; s < KS; ++s) { mbar_init(k_full(s), kProducers); mbar_init(k_empty(s), 1); }
        for (int s = 0; s < VS; ++s) { mbar_init(v_full(s), kProducers); mbar_init(v_empty(s), 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(s_full(s), 1); mbar_init(p_full(s), kSoftWarps); mbar_init(o_done(s), 1); }
        mbar_init(q_full, 1);
        mbar_init(q_empty, 1);
        mbar_fence_init();
    }
    if (warp == kMmaWarp) tc_alloc(smem_u32(&tmem_s), C::COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_s;
    Waits wait(a.status);
    pdl_launch_dependents();
    pdl_wait();

    // All roles go through the block's items and their tiles in the same order and keep step by barriers: nobody is more than a ring ahead.
    Walk walk(a);
    if (warp >= kKWarp) {
        // ------------------------------- producers: two warps for K, two for V, half a tile each -----------------------
        const bool is_v = warp >= kVWarp;
        const int half = (warp - kKWarp) & 1;
        const CUtensorMap *pages = is_v ? &v_map : &k_map, *rows = is_v ? &vn_map : &kn_map;
        const __nv_bfloat16 *src_pages = is_v ? a.v_pages : a.k_pages, *src_new = is_v ? a.v_new : a.k_new;
        uint8_t* const ring_s = is_v ? v_s : k_s;
        const uint32_t full0 = is_v ? v_full(0) : k_full(0), empty0 = is_v ? v_empty(0) : k_empty(0);
        if (lane == 0) { tma_prefetch_map(pages); tma_prefetch_map(rows); }
        Ring ring(is_v ? VS : KS, 1);
        for (; walk.item >= 0; walk.step(a)) {
            const Work w = walk.work(a, false);
            const int* pt = a.page_table + (size_t)w.seq * a.max_pages;
            // page numbers of eight tiles at a time, a lane each, a batch ahead
            auto numbers = [&](int i) -> int {
                const int t = i + (lane >> 2);
                if (t >= w.tiles) return -1;
                const int j = w.base(t) + (lane & 3) * kPage;
                if (j >= w.L || !(w.any_sees(min(j + kPage - 1, w.p_last)) || w.any_sees(j))) return -1;      // nobody sees it: not followed
                const int num = j / kPage < a.max_pages ? pt[j / kPage] : -1;
                if (num < 0 || num >= a.num_pages) { report(a.status, TF_EINVAL); return -1; }
                return num;
            };
            int now = 0, next = numbers(0);
            for (int i = 0; i < w.tiles; ++i) {
                if ((i & 7) == 0) { now = next; next = numbers(i + 8); }
                const int j0 = w.base(i) + half * 2 * kPage, at = (i & 7) * 4 + half * 2;
                const int num[2] = {__shfl_sync(0xffffffffu, now, at), __shfl_sync(0xffffffffu, now, at + 1)};
                const int kinds[2] = {w.kind(j0), w.kind(j0 + kPage)};
                const bool copy[2] = {kinds[0] == 1 || (kinds[0] == 0 && num[0] >= 0), kinds[1] == 1 || (kinds[1] == 0 && num[1] >= 0)};
                const uint32_t full = full0 + 8u * ring.i;
                uint8_t* const tile = ring_s + ring.i * C::TILE_BYTES;
                wait(empty0 + 8u * ring.i, ring.phase);
                const bool both = copy[0] && copy[1];
                if (lane == 0 && (copy[0] || copy[1])) {
                    if (both) {
                        if (is_v) bad_s[ring.i * 2 + half] = 0;
                        mbar_arrive_expect_tx(full, 2 * C::PAGE_BYTES);
                    } else {
                        mbar_expect_tx(full, C::PAGE_BYTES);
                    }
#pragma unroll
                    for (int k = 0; k < 2; ++k) {
                        if (!copy[k]) continue;
                        const int pg = half * 2 + k;
                        const CUtensorMap* map = kinds[k] == 0 ? pages : rows;
                        const int y = kinds[k] == 0 ? (num[k] * a.HK + w.kvh) * kPage : w.r0 + j0 + k * kPage - w.L, head = kinds[k] == 0 ? 0 : w.kvh;
                        if (is_v) {
                            tma_4d(smem_u32(tile + pg * C::PAGE_BYTES), map, 0, y, 0, head, full);
                        } else {
#pragma unroll
                            for (int c = 0; c < C::SLABS; ++c) tma_4d(smem_u32(tile + c * C::K_SLAB + pg * (kPage * 128)), map, 0, y, c, head, full);
                        }
                    }
                }
                if (!both) {
                    // by the warp: lane takes 16-byte column `c` of one or two rows at a time, all on the way together. Bit r of `read`: the key
                    // j0 + r is to be read (others become zeros); of `part`: some rows see it and some do not
                    constexpr int RPI = 32 / CPR;
                    const int c = lane % CPR, key = j0 + lane, first_new = w.L - j0;
                    const bool wanted = !(lane < kPage ? copy[0] : copy[1]) && w.any_sees(key) && (lane >= first_new || (lane < kPage ? num[0] : num[1]) >= 0);
                    const unsigned read = __ballot_sync(0xffffffffu, wanted);
                    const unsigned part = __ballot_sync(0xffffffffu, wanted && !(key <= w.p_first && (key >= w.lo_last || key < w.sinks)));
                    const __nv_bfloat16* from_new = src_new + ((ptrdiff_t)(w.r0 - first_new) * a.HK + w.kvh) * D + c * 8;
                    uint8_t* const to = tile + (is_v ? half * 2 * C::PAGE_BYTES + (c >> 3) * (kPage * 128) : (c >> 3) * C::K_SLAB + half * 2 * (kPage * 128));
#pragma unroll 1
                    for (int k = 0; k < 2; ++k) {
                        if (k ? copy[1] : copy[0]) continue;
                        const __nv_bfloat16* from_page = src_pages + ((size_t)max(k ? num[1] : num[0], 0) * a.HK + w.kvh) * (kPage * D) + c * 8;
                        const uint32_t dst = smem_u32(to + k * (is_v ? C::PAGE_BYTES : kPage * 128));
#pragma unroll 8
                        for (int x = 0; x < kPage; x += RPI) {
                            const int r = x + lane / CPR, at = k * kPage + r;
                            cp_async16_or_zero(dst + r * 128 + (((c ^ r) & 7) << 4), at >= first_new ? from_new + (ptrdiff_t)at * a.HK * D : from_page + r * D, read >> at & 1);
                        }
                    }
                    cp_async_commit();
                    cp_async_wait<0>();
                    uint32_t bad = 0;
                    if (is_v) {
                        for (unsigned left = part; left != 0; left &= left - 1) {
                            const int at = __ffs(left) - 1, r = at & (kPage - 1);
                            bool odd = false;
                            uint4* cell = reinterpret_cast<uint4*>(to + (at >> 4) * C::PAGE_BYTES + r * 128 + (((c ^ r) & 7) << 4));
                            if (lane / CPR == at % RPI) {            // the lanes that wrote it; a value that is not finite: exponent all ones in either half
                                const uint4 u = *cell;
                                const uint32_t e[4] = {u.x, u.y, u.z, u.w};
#pragma unroll
                                for (int y = 0; y < 4; ++y) odd |= (e[y] & 0x7F80u) == 0x7F80u || (e[y] & 0x7F800000u) == 0x7F800000u;
                                if (odd) *cell = make_uint4(0, 0, 0, 0);
                            }
                            if (__any_sync(0xffffffffu, odd)) bad |= 1u << at;
                        }
                    } else {
                        // a page that is none (reported): keys of NaN, and with them the scores of the rows that see it
                        unsigned left = __ballot_sync(0xffffffffu, !(lane < kPage ? copy[0] : copy[1]) && w.any_sees(key) && lane < first_new && (lane < kPage ? num[0] : num[1]) < 0);
                        for (; left != 0; left &= left - 1) {
                            const int at = __ffs(left) - 1, r = at & (kPage - 1);
                            if (lane / CPR == at % RPI)
                                *reinterpret_cast<uint4*>(to + (at >> 4) * (kPage * 128) + r * 128 + (((c ^ r) & 7) << 4)) = make_uint4(kNan2, kNan2, kNan2, kNan2);
                        }
                    }
                    if (is_v && lane == 0) bad_s[ring.i * 2 + half] = bad;
                    fence_proxy_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(full);
                }
                ring.next();
            }
        }
    } else if (warp == kQWarp) {
        // ------------------------------- Q: row = t * G + head, once an item -------------------------------------------
        Ring ring(1, 1);
        for (; walk.item >= 0; walk.step(a)) {
            const Work w = walk.work(a, false);
            if (w.tiles == 0) continue;
            wait(q_empty, ring.phase);
            ring.next();
            if (lane == 0) {
                const int G = (int)a.by_G.d;
                mbar_arrive_expect_tx(q_full, C::SLABS * a.group_rows * G * 128);
#pragma unroll
                for (int c = 0; c < C::SLABS; ++c) tma_4d(smem_u32(q_s + c * C::Q_SLAB), &q_map, 0, w.kvh * G, w.r0 + w.t0, c, q_full);
            }
            __syncwarp();
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------- tensor-core issuer: Q K^T a tile ahead of P V ------------------------------------
        // The tensor core works in order: scores go where those of the tile before last were once P V, issued before, has read their P; and
        // that P was there means that they had been read.
        constexpr uint32_t qk_desc = tc_idesc(kTile, false), pv_desc = tc_idesc(D, true);
        const bool leader = elect_one();
        // descriptors as low words that advance by constants; everything the loop depends on is uniform in the compiler's eyes, too: a
        // product of 64 keys takes about as long as the moves into uniform registers that its operands would need otherwise
        const uint32_t q_lo = desc_lo(smem_u32(q_s), 1);
        Ring kr(KS, 0), vr(VS, 0), qr(1, 0);
        int it = 0;                                      // tiles so far, over all items
        for (;; walk.step(a)) {
            const int tiles = __reduce_max_sync(0xffffffffu, walk.item >= 0 ? walk.work(a, false).tiles : -1);
            if (tiles < 0) break;
            if (tiles == 0) continue;
            wait(q_full, qr.phase);
            qr.next();
            for (int i = 0; i <= tiles; ++i) {
                if (i < tiles) {
                    const int t = it + i, b = t & 1;
                    wait(k_full(kr.i), kr.phase);
                    tc_fence_after();
                    const uint32_t k_lo = desc_lo(smem_u32(k_s) + kr.i * C::TILE_BYTES, 1), d = tmem + C::S_COL + b * kTile;
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks)
                        tc_mma_ss(leader, d, q_lo + (((ks >> 2) * C::Q_SLAB + (ks & 3) * 32) >> 4), k_lo + (((ks >> 2) * C::K_SLAB + (ks & 3) * 32) >> 4), qk_desc, ks > 0);
                    if (leader) {
                        tc_commit(s_full(b));
                        tc_commit(k_empty(kr.i));
                        if (i + 1 == tiles) tc_commit(q_empty);
                    }
                    kr.next();
                    __syncwarp();
                }
                if (i > 0) {
                    const int t = it + i - 1, b = t & 1;
                    wait(v_full(vr.i), vr.phase);
                    wait(p_full(b), (uint32_t)((t >> 1) & 1));
                    tc_fence_after();
                    const uint32_t v_lo = desc_lo(smem_u32(v_s) + vr.i * C::TILE_BYTES, kPage * 128 / 16);
#pragma unroll
                    for (int pg = 0; pg < kTile / kPage; ++pg)
                        tc_mma_ts(leader, tmem + C::O_COL, tmem + C::S_COL + b * kTile + pg * 8, v_lo + pg * (C::PAGE_BYTES >> 4), pv_desc, i > 1 || pg > 0);
                    if (leader) { tc_commit(o_done(b)); tc_commit(v_empty(vr.i)); }
                    vr.next();
                    __syncwarp();
                }
            }
            it += tiles;
        }
    } else {
        // ------------------------------- softmax: thread = query row ---------------------------------------------
        const uint32_t row = tmem + ((uint32_t)(warp * 32) << 16);
        uint8_t* const mine_s = stage_s + warp * 32 * C::STAGE_ROW;
        const unsigned long long scale2 = pair_of(a.scale_log2, a.scale_log2);
        Ring vr(VS, 0);
        int it = 0;
        for (; walk.item >= 0; walk.step(a)) {
            const Work w = walk.work(a, tid == 0);
            if (w.tiles == 0) continue;
            if (warp * 32 >= w.nq) {                     // no rows: keeps step with the others, tile by tile
                for (int i = 0; i < w.tiles; ++i, ++it, vr.next()) {
                    wait(s_full(it & 1), (uint32_t)((it >> 1) & 1));
                    if (lane == 0) mbar_arrive(p_full(it & 1));
                }
                continue;
            }
            const bool mine = tid < w.nq;
            const int G = (int)a.by_G.d, dt = a.by_G(mine ? tid : 0), p = w.p_first + dt, lo = max(0, p + 1 - a.window);
            const int q_row = (w.r0 + w.t0 + dt) * a.H + w.kvh * G + (mine ? tid : 0) - dt * G;
            float m = -INFINITY, l = 0.f;
#pragma unroll 1
            for (int i = 0; i < w.tiles; ++i, ++it) {
                const int b = it & 1, j0 = w.base(i);
                const uint32_t round = (uint32_t)((it >> 1) & 1);
                const bool plain = w.plain(j0);
                wait(s_full(b), round);
                tc_fence_after();
                // a part of the scores at a time, read twice where there are two (two blocks an SM have 96 registers a thread)
                constexpr int PART = C::BLOCKS == 2 ? kTile / 2 : kTile;
                uint32_t see[2] = {~0u, ~0u};            // bit e: the row sees key j0 + e; up to p, and from lo on or below the sinks' end
                bool spoilt = false;                     // it sees a value that is not finite
                if (!plain) {                            // the V tile's notes are there once it is (and stay until P V)
                    uint32_t bad[2] = {0, 0};
                    if (w.p_first != w.p_last) {         // (a row alone sees all that is read)
                        wait(v_full(vr.i), vr.phase);
                        bad[0] = bad_s[vr.i * 2];
                        bad[1] = bad_s[vr.i * 2 + 1];
                    }
                    auto below = [](int x) -> unsigned long long { return x <= 0 ? 0ull : x >= kTile ? ~0ull : (1ull << x) - 1; };
                    const unsigned long long sees = below(p + 1 - j0) & (~below(lo - j0) | below(w.sinks - j0));
                    see[0] = (uint32_t)sees;
                    see[1] = (uint32_t)(sees >> 32);
                    spoilt = ((see[0] & bad[0]) | (see[1] & bad[1])) != 0;
                }
                vr.next();
                float s[PART];
                auto scores = [&](int e0) {
#pragma unroll
                    for (int c = 0; c < PART; c += 32) tc_ld32(row + C::S_COL + b * kTile + e0 + c, *reinterpret_cast<float(*)[32]>(s + c));
                    tc_wait_ld();
                    if (!plain) {
#pragma unroll
                        for (int e = 0; e < PART; ++e) s[e] = see[PART == kTile ? e >> 5 : e0 >> 5] >> (e & 31) & 1 ? s[e] : -INFINITY;
                    }
                };
                float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int e0 = 0; e0 < kTile; e0 += PART) {
                    scores(e0);
#pragma unroll
                    for (int e = 0; e < PART; e += 8) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) tops[k] = max3(tops[k], s[e + 2 * k], s[e + 2 * k + 1]);
                    }
                }
                const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])) * a.scale_log2;
                // move the maximum only where it must: a row's choice looks at its own scores alone
                float alpha = 1.f;
                if (top > m + kSlack || (m == -INFINITY && top > m)) {
                    alpha = m == -INFINITY ? 1.f : fast_exp2(m - top);       // nothing summed yet: all is zero
                    m = top;
                    l *= alpha;
                }
                if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                    wait(o_done((it - 1) & 1), (uint32_t)(((it - 1) >> 1) & 1));
                    tc_fence_after();
#pragma unroll 1
                    for (int c = 0; c < D; c += 32) {
                        float o[32];
                        uint32_t u[32];
                        tc_ld32(row + C::O_COL + c, o);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 32; ++e) u[e] = __float_as_uint(o[e] * alpha);
                        tc_st32(row + C::O_COL + c, u);
                    }
                }
                const float off = m == -INFINITY ? 0.f : -m;
                const unsigned long long off2 = pair_of(off, off);
                unsigned long long sum[4] = {0, 0, 0, 0};            // two zeros each
#pragma unroll
                for (int e0 = 0; e0 < kTile; e0 += PART) {
                    if (PART < kTile) scores(e0);
                    uint32_t pk[PART / 2];
#pragma unroll
                    for (int e = 0; e < PART; e += 2) {
                        float x, y;
                        split_pair(fma_pair(pair_of(s[e], s[e + 1]), scale2, off2), x, y);
                        x = fast_exp2(x);
                        y = fast_exp2(y);
                        sum[(e >> 1) & 3] = add_pair(sum[(e >> 1) & 3], pair_of(x, y));
                        const __nv_bfloat162 xy = __floats2bfloat162_rn(x, y);
                        pk[e >> 1] = *reinterpret_cast<const uint32_t*>(&xy);
                    }
                    if (e0 == 0 && spoilt) pk[0] = kNan2;     // NaN weights, of this row's results only
                    if constexpr (PART == kTile) tc_st32(row + C::S_COL + b * kTile, pk);
                    else tc_st16(row + C::S_COL + b * kTile + e0 / 2, pk);
                }
                float s0, s1;
                split_pair(add_pair(add_pair(sum[0], sum[1]), add_pair(sum[2], sum[3])), s0, s1);
                l += s0 + s1;
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(b));
            }
            // ---- the chunk's partials, or the results where a row has one chunk: 32 columns at a time through shared memory, so that a
            // store covers whole sectors ----
            if constexpr (CLUSTER) {
                if (mine) sums_s[tid] = make_float2(m, l);
                wait(o_done((it - 1) & 1), (uint32_t)(((it - 1) >> 1) & 1));
                tc_fence_after();
#pragma unroll 1
                for (int c = 0; c < D; c += 32) {
                    float o[32];
                    tc_ld32(row + C::O_COL + c, o);
                    tc_wait_ld();
                    // fours in two halves, the even ones first: a reader's lanes, eight columns each, lie beside one another
                    float4* to = reinterpret_cast<float4*>(k_s + tid * JOIN_ROW) + c / 8;
                    if (tid < QR) {
#pragma unroll
                        for (int e = 0; e < 8; ++e) to[(e & 1) * (D / 8) + (e >> 1)] = make_float4(o[4 * e], o[4 * e + 1], o[4 * e + 2], o[4 * e + 3]);
                    }
                }
                continue;
            }
            const int rows_here = min(32, w.nq - warp * 32);
            constexpr int LANES = C::STAGE / 4, ROWS = 32 / LANES;       // lanes a row of partials, rows a store
            const size_t first = (size_t)w.slot * a.R * a.H;
            float* to[LANES];
            float inv = 0.f;
            if (a.direct) {
                inv = 1.f / l;
                if (mine && a.lse != nullptr) a.lse[q_row] = (m + log2f(l)) * kLn2;
            } else {
                if (mine) { a.part_m[first + q_row] = m; a.part_l[first + q_row] = l; }
#pragma unroll
                for (int x = 0; x < LANES; ++x) to[x] = a.part_o + (first + __shfl_sync(0xffffffffu, q_row, x * ROWS + lane / LANES)) * D + lane % LANES * 4;
            }
            wait(o_done((it - 1) & 1), (uint32_t)(((it - 1) >> 1) & 1));
            tc_fence_after();
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                float o[32];
                tc_ld32(row + C::O_COL + c, o);
                tc_wait_ld();
                uint8_t* const cell = mine_s + lane * C::STAGE_ROW;
                if (a.direct) {
#pragma unroll
                    for (int e = 0; e < 32; e += 8) {
                        float x[8];
#pragma unroll
                        for (int y = 0; y < 8; ++y) x[y] = o[e + y] * inv;
                        *reinterpret_cast<uint4*>(cell + e * 2) = pack8(x);
                    }
                    __syncwarp();
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int r = x * 8 + (lane >> 2), at = __shfl_sync(0xffffffffu, q_row, r);
                        const uint4 v = *reinterpret_cast<const uint4*>(mine_s + r * C::STAGE_ROW + (lane & 3) * 16);
                        if (r < rows_here) *reinterpret_cast<uint4*>(a.out + (size_t)at * D + c + (lane & 3) * 8) = v;
                    }
                    __syncwarp();
                    continue;
                }
#pragma unroll
                for (int h = 0; h < 32; h += C::STAGE) {
#pragma unroll
                    for (int e = 0; e < C::STAGE; e += 4) *reinterpret_cast<float4*>(cell + e * 4) = make_float4(o[h + e], o[h + e + 1], o[h + e + 2], o[h + e + 3]);
                    __syncwarp();
                    float4 v[LANES];
#pragma unroll
                    for (int x = 0; x < LANES; ++x) v[x] = *reinterpret_cast<const float4*>(mine_s + (x * ROWS + lane / LANES) * C::STAGE_ROW + lane % LANES * 16);
#pragma unroll
                    for (int x = 0; x < LANES; ++x)
                        if (x * ROWS + lane / LANES < rows_here) *reinterpret_cast<float4*>(to[x] + c + h) = v[x];
                    __syncwarp();
                }
            }
            tc_fence_before();                           // the sums have been read: the next item's may overwrite them
        }
    }
    tc_fence_before();
    if constexpr (CLUSTER) {
        cg::cluster_group cluster = cg::this_cluster();
        __syncwarp();
        cluster.sync();
        const Work w = work_of(a, blockIdx.x, fetch(a, blockIdx.x), false);
        constexpr int LANES = D / 8;
        const int G = (int)a.by_G.d, rank = (int)cluster.block_rank(), step = (int)cluster.num_blocks() * kThreads;
        for (int i0 = rank * kThreads + warp * 32; i0 < w.nq * LANES; i0 += step) {
            const int r = (i0 + lane) / LANES, li = lane % LANES;
            const bool there = r < w.nq;
            const int at = there ? r : 0, dt = a.by_G(at);
            float acc[8], m, l;
            join_chunks<4>(a, w.p_first + dt, [&](int slot, float& cm, float& cl, float4 (&x)[2]) {
                const float2 sums = *cluster.map_shared_rank(&sums_s[at], slot);
                const float4* src = reinterpret_cast<const float4*>(cluster.map_shared_rank(k_s, slot) + at * JOIN_ROW) + li;
                cm = sums.x;
                cl = sums.y;
                x[0] = src[0];
                x[1] = src[LANES];
            }, acc, m, l);
            finish_row<D>(a, w.r0 + w.t0 + dt, w.kvh * G + at - dt * G, li, there, acc, m, l);
        }
        auto others = cluster.barrier_arrive();
        if (a.out_packed != nullptr && w.seq == 0 && rank == 0) {
            const int pads = tf_padded_rows(a.R) - a.R, columns = G * LANES;
            for (int i = tid; i < pads * columns; i += kThreads) zero_packed(a, a.R + i / columns, w.kvh * columns + i % columns);
        }
        cluster.barrier_wait(std::move(others));         // nobody leaves while another block may read its rows
    } else {
        __syncthreads();
    }
    if (warp == kMmaWarp) {
        tc_fence_after();
        tc_dealloc(tmem, C::COLS);
    }
}

// Joins the chunks of the rows: D / 8 lanes a (row, head), B chunks in flight.
template <int D, int B>
__global__ void __launch_bounds__(128) window_join_kernel(const WindowArgs a) {
    constexpr int LANES = D / 8, PER_WARP = 32 / LANES;
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = (blockIdx.x * 4 + warp) * PER_WARP + lane / LANES, li = lane % LANES;
    int start = 0;
    const int seq = row < a.R ? seq_of(a.seq_start, a.S, row, start) : -1;
    const bool there = head < a.H;
    if (seq < 0) {
        if (row >= a.R && a.out_packed != nullptr && there) zero_packed(a, row, head * LANES + li);
        return;
    }
    const int p = a.seq_lens[seq] + row - start;
    if (p < 0 || p >= a.max_context) return;                           // reported by the chunk kernel
    float acc[8], m, l;
    join_chunks<B>(a, p, [&](int slot, float& cm, float& cl, float4 (&x)[2]) {
        const size_t cell = ((size_t)slot * a.R + row) * a.H + (there ? head : 0);
        cm = a.part_m[cell];
        cl = a.part_l[cell];
        const float4* src = reinterpret_cast<const float4*>(a.part_o + cell * D + li * 8);
        x[0] = src[0];
        x[1] = src[1];
    }, acc, m, l);
    finish_row<D>(a, row, head, li, there, acc, m, l);
}

// ---- host side -----------------------------------------------------------------------------------------
// A cluster of a column's chunks joins them itself where rows and chunks are few and the clusters fit the GPU at once (of 148 SMs at least 7 of
// 16 and 15 of 8). One row of 6 heads a KV head, 15 chunks of a window of 4096 keys: 13.9 us, with partials in memory and a second launch 15.0;
// 4 chunks of 500 keys: 8.7 and 9.9. 24 query rows: 11.8 and 11.7; 48: 15.5 and 15.2, 11.0 and 10.1.
bool clustered(const WindowArgs& a) {
    const int columns = a.HK * a.S;
    return a.qgroups == 1 && a.group_rows * (a.H / a.HK) <= 24 && a.slots >= 2 && a.slots <= 16 && columns <= (a.slots > 8 ? 7 : 15);
}

template <int D, int QR, bool CLUSTER>
int launch_chunks(const WindowArgs& a, cudaStream_t st) {
    using C = Cfg<D, QR>;
    static std::atomic<bool> configured[64] = {};       // the opt-in is per device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return TF_ECUDA; }
    if (!configured[dev]) {
        if (cudaFuncSetAttribute(window_chunk_kernel<D, QR, CLUSTER>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess ||
            (CLUSTER && cudaFuncSetAttribute(window_chunk_kernel<D, QR, CLUSTER>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1) != cudaSuccess)) {
            cudaGetLastError();
            return TF_ECUDA;
        }
        configured[dev] = true;
    }
    CUtensorMap maps[5];
    const int G = a.H / a.HK;
    const unsigned long long H = a.H, HK = a.HK, R = a.R, rows = (unsigned long long)a.num_pages * HK * kPage;
    const size_t row = (size_t)D * 2;
    if (!describe_rows(&maps[0], a.q, D, H, row, R, row * H, true, G, a.group_rows, 1) ||
        !describe_rows(&maps[1], a.k_pages, D, rows, row, 1, row, false, kPage, 1, 1) || !describe_rows(&maps[2], a.v_pages, D, rows, row, 1, row, false, kPage, 1, D / 64) ||
        !describe_rows(&maps[3], a.k_new, D, R < 16 ? 16 : R, row * HK, HK, row, false, kPage, 1, 1) ||
        !describe_rows(&maps[4], a.v_new, D, R < 16 ? 16 : R, row * HK, HK, row, false, kPage, 1, D / 64))
        return TF_ECUDA;
    void* args[] = {const_cast<WindowArgs*>(&a), &maps[0], &maps[1], &maps[2], &maps[3], &maps[4]};
    if (launch_pdl((const void*)window_chunk_kernel<D, QR, CLUSTER>, dim3(a.items < a.blocks ? a.items : a.blocks), dim3(kThreads), C::SMEM, st, args, 0,
                   CLUSTER ? a.slots : 1) != cudaSuccess) {
        cudaGetLastError();
        return TF_ECUDA;
    }
    return TF_OK;
}

// Rows a group, groups of rows and items of a call; false where the items are more than the launch can count.
bool cut_rows(WindowArgs& a) {
    const int most = kRows / (a.H / a.HK);
    a.group_rows = a.max_window < most ? a.max_window : most;
    if (a.group_rows > a.R) a.group_rows = a.R;
    a.qgroups = (a.max_window + a.group_rows - 1) / a.group_rows;
    const long long items = (long long)a.qgroups * a.slots * a.HK * a.S;
    a.items = (int)items;
    return items <= (1 << 30);
}
// A plan only where a block takes several items, and not so many that they even out.
bool planned(const WindowArgs& a) { return a.items > a.blocks && a.items <= kPlanItems; }

template <int D>
int run(WindowArgs& a, cudaStream_t st) {
    const int G = a.H / a.HK;
    if (!cut_rows(a)) return TF_EINVAL;
    a.by_group = fast_div(a.qgroups); a.by_slot = fast_div(a.slots); a.by_head = fast_div(a.HK); a.by_G = fast_div(G); a.by_chunk = fast_div(a.chunk);
    a.blocks = kSms * blocks_of(D);
    a.rounds = (a.items + a.blocks - 1) / a.blocks;
    if (!planned(a)) a.plan = nullptr;
    if (a.plan != nullptr) {
        void* args[] = {&a};
        if (launch_pdl((const void*)window_plan_kernel, dim3(1), dim3(kPlanThreads), 0, st, args) != cudaSuccess) { cudaGetLastError(); return TF_ECUDA; }
    }
    if (clustered(a)) return launch_chunks<D, 64, true>(a, st);
    const int rc = a.group_rows * G <= 64 ? launch_chunks<D, 64, false>(a, st) : launch_chunks<D, 128, false>(a, st);
    if (rc != TF_OK || a.direct) return rc;
    void* join[] = {&a};
    const int heads = 4 * (32 / (D / 8)), out_rows = a.out_packed ? tf_padded_rows(a.R) : a.R;
    // (one row of 7 chunks: 11.3 us with eight in flight, 12 with four; 2900 rows of one or two: 14 and 24 us for this kernel)
    const void* kern = a.slots > 4 ? (const void*)window_join_kernel<D, 8> : (const void*)window_join_kernel<D, 4>;
    if (launch_pdl(kern, dim3((a.H + heads - 1) / heads, out_rows), dim3(128), 0, st, join) != cudaSuccess) {
        cudaGetLastError();
        return TF_ECUDA;
    }
    return TF_OK;
}

}  // namespace
}  // namespace tf

extern "C" {

// Few columns (sequence, KV head, group of up to 128 query rows): as many chunks as leave the SMs one each, but not below the size at
// which a chunk's tiles (0.95 us for 64 keys) and the join (0.36 us a chunk) cost the same, and one chunk where that saves the join for few
// tiles more (300 rows of up to 400 keys: 15.2 us in one, 19.7 in two). More columns: a quarter of what a group sees, so that the chunks
// can be dealt out evenly (16 x 4 columns of 4100 keys: 59.1 us in chunks of 1024, 59.6 of 2048, 64.8 of 512, 77 of 4096; with heads of
// 128 38.7, 48.7, 43.3 and 71.6). Very many, as for a prompt's rows: one chunk, without partials and join, where a group sees few
// keys (362 columns of 1040 keys: 45.5 us, 57 in chunks of 2048; 576 of 4000: 222 and 284), else 2048 (376 columns of 17500 keys:
// 511 us, 643 in one chunk, whose columns do not divide evenly).
int tf_window_chunk_keys(int n_seqs, int heads, int kv_heads, int max_window, int max_context, int window, int sinks) {
    if (n_seqs < 1 || kv_heads < 1 || heads < kv_heads || heads / kv_heads > tf::kRows || max_window < 1 || max_context < max_window ||
        max_context > (1 << 30) || window < 0 || sinks < 0) return 0;
    const auto over = [](long long x, long long y) { return (x + y - 1) / y; };
    const auto tiles_of = [&](long long keys) { return over(keys, tf::kTile) * tf::kTile; };
    const int most = tf::kRows / (heads / kv_heads), rows = max_window < most ? max_window : most;
    const long long columns = (long long)n_seqs * kv_heads * over(max_window, rows);
    const long long seen = (long long)window + rows - 1, keys = window == 0 || seen > max_context ? max_context : seen;
    const long long whole = tiles_of(max_context < 128 ? 128 : max_context);
    const long long spare = tf::kSms / columns - (window == 0 ? 0 : sinks > 0 ? 2 : 1);     // a window lies across one chunk more, sinks have their own
    long long chunk = 128;
    if (spare >= 1) {
        const long long even = (long long)sqrt(24.0 * keys), share = over(keys, spare);
        chunk = tiles_of(even > share ? even > 128 ? even : 128 : share > 128 ? share : 128);
        if (whole - chunk <= 256) chunk = whole;
    } else if (columns < 222) {
        chunk = tiles_of(over(keys, 4));
        chunk = chunk < 512 ? 512 : chunk > 2048 ? 2048 : chunk;
    } else {
        chunk = keys <= 4096 ? whole : 2048;
    }
    return (int)(chunk > 1 << 30 ? 1 << 30 : chunk);
}

int tf_window_slots(int window, int sinks, int max_window, int max_context, int chunk_keys) {
    if (window < 0 || sinks < 0 || max_window < 1 || max_context < max_window || max_context > (1 << 30) || chunk_keys < tf::kTile || chunk_keys > (1 << 30) ||
        chunk_keys % tf::kTile)
        return 0;
    const tf::Slots s = tf::slots_for(window, sinks, max_window, max_context, chunk_keys);
    return s.first + s.near;
}

size_t tf_window_scratch_bytes(int rows, int heads, int head_dim, int slots) {
    if (rows < 1 || heads < 1 || head_dim < 1 || slots < 1) return 0;
    return tf::kPlanBytes + (size_t)slots * rows * heads * (head_dim + 2) * sizeof(float);
}

int tf_window_launches(int rows, int n_seqs, int max_window, int slots, int heads, int kv_heads, int head_dim, int plain) {
    if (rows < 1 || n_seqs < 1 || max_window < 1 || slots < 1 || kv_heads < 1 || heads < kv_heads || heads / kv_heads > 16) return 0;
    tf::WindowArgs a{};
    a.R = rows; a.S = n_seqs; a.max_window = max_window; a.slots = slots; a.H = heads; a.HK = kv_heads;
    a.blocks = tf::kSms * tf::blocks_of(head_dim);
    return !tf::cut_rows(a) ? 0 : 1 + (tf::planned(a) ? 1 : 0) + ((slots == 1 && plain) || tf::clustered(a) ? 0 : 1);
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
    if (rows > 65535 || kv_heads > 65535 || (long long)rows * heads > 0x7FFFFFFFll || (long long)num_pages * kv_heads * 16 > 0x7FFFFFFFll) return TF_EINVAL;
    const int slots = tf_window_slots(window, sinks, max_window, max_context, chunk_keys);
    if (slots < 1) return TF_EINVAL;
    if (!q || !k_new || !v_new || !k_pages || !v_pages || !page_table || !seq_lens || !seq_start) return TF_EINVAL;
    if (((uintptr_t)q | (uintptr_t)k_new | (uintptr_t)v_new | (uintptr_t)k_pages | (uintptr_t)v_pages | (uintptr_t)qg | (uintptr_t)out_packed |
         (uintptr_t)out) & 15) return TF_EALIGN;
    if (!scratch || ((uintptr_t)scratch & 15) || scratch_bytes < tf_window_scratch_bytes(rows, heads, head_dim, slots)) return TF_ESCRATCH;
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
    a.max_window = max_window;
    a.chunk = chunk_keys; a.slots = slots;
    a.direct = slots == 1 && !qg && !out_packed;
    const tf::Slots cut = tf::slots_for(window, sinks, max_window, max_context, chunk_keys);
    a.first_slots = cut.first; a.near_slots = cut.near > 0 ? cut.near : 1;
    const size_t cells = (size_t)slots * rows * heads;
    a.plan = static_cast<int*>(scratch);
    a.part_o = reinterpret_cast<float*>(static_cast<char*>(scratch) + tf::kPlanBytes);
    a.part_m = a.part_o + cells * head_dim;
    a.part_l = a.part_m + cells;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return head_dim == 256 ? tf::run<256>(a, st) : tf::run<128>(a, st);
}

}  // extern "C"
