// Lane attention with a sliding window and sinks over the paged KV cache, on the 5th-generation tensor cores.
//
// Row t of a sequence's window stands at slot p = L + t (L committed keys) and sees key j when j <= p and
// (p - j < window or j < sinks): softmax of its scores over those keys, the weighted sum of their values, and the
// log-sum-exp of the scores.
//
// The key axis is cut by ABSOLUTE position into chunks; a block handles one chunk of one (sequence, KV head) for up to 128 query
// rows (window rows x the KV head's query heads, row = t * G + head), and a second kernel joins a row's chunks in order. In a block the
// keys go by in tiles of 64:
//
//   S = Q K^T        tcgen05, both operands in shared memory, 128 x 64 sums in tensor memory (two buffers)
//   P = 2^(S - m)    four warps, a thread a row: no shuffles. m is a maximum that is only moved when a score exceeds it by 2^8, so the
//                    sums so far are rescaled seldom (exactly the rows that need it change: multiplying by 1 keeps bits)
//   O += P V         tcgen05, P in tensor memory as bf16, V in shared memory as it lies in the cache (rows are the contraction's index)
//
// K and V arrive by tiled copies (TMA), a page of 16 keys at a time, into rings of their own. A page that not all rows see whole
// (around the committed length, the window's far edge, the sinks' end) is written by its producer warp instead, keys that no
// row sees as zeros without being read. There a value that is not finite is written as zero and noted: rows that see its key become
// NaN, rows that do not keep their bits. Every step of a row's arithmetic is fixed by its own position and keys and by the chunk
// size, so a row alone, in a window and as a serial step has the same bits.

#include <cudaTypedefs.h>

#include "tc.cuh"

namespace tf {
namespace {

constexpr int kPage = 16, kTile = 64, kRows = 128;     // keys a page, keys a tile, query rows a block (the tensor core's M)
constexpr int kSoftWarps = 4, kMmaWarp = 4, kKWarp = 5, kVWarp = 6, kThreads = 7 * 32;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr float kSlack = 8.f;                          // how far (log2) a score may exceed the running maximum

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
    int chunk, first_slots, near_slots, qgroups;       // keys a chunk; slots of the sinks' chunks and of the window's
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

// What a block works on: every thread forms it.
struct Work {
    int r0, L, p_first, p_last, lo_first, lo_last, nq, key0, head_tiles, far_tile, tiles, sinks;
    // tile i of the block: those of the sinks, then those of the window
    __device__ int base(int i) const { return key0 + (i < head_tiles ? i : far_tile + i - head_tiles) * kTile; }
    // 0: a committed page that every row sees whole, 1: 16 window rows that every row sees, 2: anything else
    __device__ int kind(int j) const {
        if (j + kPage > p_first + 1 || !(j >= lo_last || j + kPage <= sinks)) return 2;
        return j + kPage <= L ? 0 : j >= L ? 1 : 2;
    }
    __device__ bool mixed(int j) const { return kind(j) == 2 || kind(j + kPage) == 2 || kind(j + 2 * kPage) == 2 || kind(j + 3 * kPage) == 2; }
    __device__ bool any_sees(int j) const { return j <= p_last && (j >= lo_first || j < sinks); }
};

template <int D, int QR>
struct Cfg {
    static constexpr int SLABS = D / 64;                 // 64 values of a row: one 128-byte swizzle row
    static constexpr int Q_SLAB = QR * 128, Q_BYTES = SLABS * Q_SLAB;
    static constexpr int TILE_BYTES = kTile * D * 2, K_SLAB = kTile * 128, V_PAGE = kPage * D * 2;
    static constexpr int FIT = (227 * 1024 - 2048 - Q_BYTES) / TILE_BYTES;
    static constexpr int KS = FIT / 2 > 4 ? 4 : FIT / 2, VS = FIT - FIT / 2 > 4 ? 4 : FIT - FIT / 2;
    static constexpr int NBARS = 2 * KS + 2 * VS + 8 + 1;
    static constexpr int SMEM = Q_BYTES + (KS + VS) * TILE_BYTES + NBARS * 8 + VS * 8 + 1024;
    static constexpr int O_COL = 0, S_COL = D, P_COL = D + 2 * kTile, COLS = 512;
    static_assert(KS >= 2 && VS >= 2 && SMEM <= 227 * 1024, "the rings do not fit");
    static_assert(P_COL + 2 * (kTile / 2) <= COLS, "tensor memory");
    // a block of fewer than 128 rows leaves the last rows of the tensor core's Q operand to whatever follows in shared memory
    static_assert(Q_BYTES - Q_SLAB + kRows * 128 <= Q_BYTES + (KS + VS) * TILE_BYTES, "the operand's rows lie inside the block's memory");
};

template <int D, int QR>
__global__ void __launch_bounds__(kThreads, 1) window_chunk_kernel(const __grid_constant__ WindowArgs a, const __grid_constant__ CUtensorMap k_map,
                                                                   const __grid_constant__ CUtensorMap v_map, const __grid_constant__ CUtensorMap kn_map,
                                                                   const __grid_constant__ CUtensorMap vn_map) {
    using C = Cfg<D, QR>;
    constexpr int KS = C::KS, VS = C::VS, CPR = D / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t tmem_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t* q_s = smem + ((1024u - (smem_u32(smem) & 1023u)) & 1023u);
    uint8_t* k_s = q_s + C::Q_BYTES;
    uint8_t* v_s = k_s + KS * C::TILE_BYTES;
    const uint32_t bars = smem_u32(v_s + VS * C::TILE_BYTES);
    unsigned long long* bad_s = reinterpret_cast<unsigned long long*>(v_s + VS * C::TILE_BYTES + C::NBARS * 8);
    auto k_full = [&](int s) { return bars + 8u * s; };
    auto k_empty = [&](int s) { return bars + 8u * (KS + s); };
    auto v_full = [&](int s) { return bars + 8u * (2 * KS + s); };
    auto v_empty = [&](int s) { return bars + 8u * (2 * KS + VS + s); };
    auto s_full = [&](int s) { return bars + 8u * (2 * KS + 2 * VS + s); };
    auto s_empty = [&](int s) { return bars + 8u * (2 * KS + 2 * VS + 2 + s); };
    auto p_full = [&](int s) { return bars + 8u * (2 * KS + 2 * VS + 4 + s); };
    auto o_done = [&](int s) { return bars + 8u * (2 * KS + 2 * VS + 6 + s); };      // P V of a tile is complete
    const uint32_t q_full = bars + 8u * (2 * KS + 2 * VS + 8);

    pdl_launch_dependents();
    pdl_wait();
    // ---- which chunk, which rows, which tiles ----
    const int kvh = blockIdx.y, seq = blockIdx.z / a.qgroups, qg = blockIdx.z % a.qgroups, G = a.H / a.HK;
    Work w;
    w.r0 = a.seq_start[seq];
    w.L = a.seq_lens[seq];
    w.sinks = a.sinks;
    const int n = a.seq_start[seq + 1] - w.r0;
    if (n < 1) return;
    if (n > a.max_window || w.L < 0 || w.L + n > a.max_context || w.r0 < 0 || w.r0 + n > a.R) {     // not what the call was made for
        if (tid == 0) report(a.status, TF_EINVAL);
        return;
    }
    const int q0 = qg * QR, t_first = q0 / G;
    if (q0 >= n * G) return;
    w.nq = min(QR, n * G - q0);
    w.p_first = w.L + t_first;
    w.p_last = w.L + (q0 + w.nq - 1) / G;
    w.lo_first = max(0, w.p_first + 1 - a.window);
    w.lo_last = max(0, w.p_last + 1 - a.window);
    const int slot = blockIdx.x;
    int chunk = slot;
    if (slot >= a.first_slots) {
        const int lowest = max(a.first_slots, max(0, w.L + 1 - a.window) / a.chunk);        // of the sequence: its rows share the slots
        chunk = lowest + ((slot - lowest) % a.near_slots + a.near_slots) % a.near_slots;
    }
    w.key0 = chunk * a.chunk;
    const int end = min(w.key0 + a.chunk, w.p_last + 1), in_chunk = end > w.key0 ? (end - w.key0 + kTile - 1) / kTile : 0;
    w.head_tiles = w.sinks > w.key0 ? min(in_chunk, (w.sinks - w.key0 + kTile - 1) / kTile) : 0;
    w.far_tile = max(w.head_tiles, w.lo_first > w.key0 ? (w.lo_first - w.key0) / kTile : 0);
    w.tiles = w.head_tiles + max(0, in_chunk - w.far_tile);
    if (w.tiles == 0) return;
    const int live = (w.nq + 31) / 32;                   // softmax warps with rows

    if (tid == 0) {
        for (int s = 0; s < KS; ++s) { mbar_init(k_full(s), 1); mbar_init(k_empty(s), 1); }
        for (int s = 0; s < VS; ++s) { mbar_init(v_full(s), 1); mbar_init(v_empty(s), 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(s_full(s), 1); mbar_init(s_empty(s), live); mbar_init(p_full(s), live); mbar_init(o_done(s), 1); }
        mbar_init(q_full, kSoftWarps);
        mbar_fence_init();
    }
    if (warp == kMmaWarp) tc_alloc(smem_u32(&tmem_s), C::COLS);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = tmem_s;
    Waits wait(a.status);

    if (warp == kKWarp || warp == kVWarp) {
        // ------------------------------- producers: a warp for K, a warp for V --------------------------------
        const bool is_v = warp == kVWarp;
        const CUtensorMap *pages = is_v ? &v_map : &k_map, *rows = is_v ? &vn_map : &kn_map;
        const __nv_bfloat16 *src_pages = is_v ? a.v_pages : a.k_pages, *src_new = is_v ? a.v_new : a.k_new;
        const int* pt = a.page_table + (size_t)seq * a.max_pages;
        Ring ring(is_v ? VS : KS, 1);
        for (int i = 0; i < w.tiles; ++i) {
            const int j0 = w.base(i);
            const uint32_t full = is_v ? v_full(ring.i) : k_full(ring.i), empty = is_v ? v_empty(ring.i) : k_empty(ring.i);
            uint8_t* const tile = is_v ? v_s + ring.i * C::TILE_BYTES : k_s + ring.i * C::TILE_BYTES;
            wait(empty, ring.phase);
            // the four pages' numbers, looked up together
            int page = -1;
            if (lane < 4 && j0 + lane * kPage < w.L && w.any_sees(min(j0 + lane * kPage + kPage - 1, w.p_last)) | w.any_sees(j0 + lane * kPage)) {
                const int at = (j0 + lane * kPage) / kPage;
                page = at < a.max_pages ? pt[at] : -1;
                if (page < 0 || page >= a.num_pages) { report(a.status, TF_EINVAL); page = -1; }
            }
            unsigned copied = 0;
#pragma unroll
            for (int pg = 0; pg < 4; ++pg) {
                const int kind = w.kind(j0 + pg * kPage), num = __shfl_sync(0xffffffffu, page, pg);
                if (kind == 1 || (kind == 0 && num >= 0)) copied |= 1u << pg;
            }
            if (lane == 0 && copied) mbar_expect_tx(full, __popc(copied) * C::V_PAGE);
            __syncwarp();
            unsigned long long bad = 0;
#pragma unroll 1
            for (int pg = 0; pg < 4; ++pg) {
                const int j = j0 + pg * kPage, num = __shfl_sync(0xffffffffu, page, pg);
                if (copied >> pg & 1) {
                    if (lane == 0) {
                        const bool committed = w.kind(j) == 0;
                        const CUtensorMap* map = committed ? pages : rows;
                        const int y = committed ? (num * a.HK + kvh) * kPage : w.r0 + j - w.L, head = committed ? 0 : kvh;
                        if (is_v) {
                            tma_4d(smem_u32(tile + pg * C::V_PAGE), map, 0, y, 0, head, full);
                        } else {
#pragma unroll
                            for (int c = 0; c < C::SLABS; ++c) tma_4d(smem_u32(tile + c * C::K_SLAB + pg * (kPage * 128)), map, 0, y, c, head, full);
                        }
                    }
                    continue;
                }
                // by the warp: lane takes 16-byte column `c` of one or two rows at a time
                constexpr int RPI = 32 / CPR;
                const int c = lane % CPR;
#pragma unroll 4
                for (int rr = 0; rr < kPage; rr += RPI) {
                    const int r = rr + lane / CPR, key = j + r;
                    uint4 v = make_uint4(0, 0, 0, 0);
                    if (w.any_sees(key)) {
                        if (key >= w.L) v = *reinterpret_cast<const uint4*>(src_new + ((size_t)(w.r0 + key - w.L) * a.HK + kvh) * D + c * 8);
                        else if (num >= 0) v = *reinterpret_cast<const uint4*>(src_pages + (((size_t)num * a.HK + kvh) * kPage + r) * D + c * 8);
                    }
                    if (is_v) {                          // a value that is not finite: exponent all ones in either half
                        const uint32_t u[4] = {v.x, v.y, v.z, v.w};
                        bool odd = false;
#pragma unroll
                        for (int e = 0; e < 4; ++e) odd |= (u[e] & 0x7F80u) == 0x7F80u || (u[e] & 0x7F800000u) == 0x7F800000u;
                        const unsigned m = __ballot_sync(0xffffffffu, odd);
                        if (odd) v = make_uint4(0, 0, 0, 0);
#pragma unroll
                        for (int h = 0; h < RPI; ++h)
                            if (RPI == 1 ? m != 0 : (m >> (h * CPR) & ((1u << (CPR & 31)) - 1u)) != 0) bad |= 1ull << (pg * kPage + rr + h);
                        *reinterpret_cast<uint4*>(tile + pg * C::V_PAGE + (c >> 3) * (kPage * 128) + r * 128 + (((c ^ r) & 7) << 4)) = v;
                    } else {
                        *reinterpret_cast<uint4*>(tile + (c >> 3) * C::K_SLAB + (pg * kPage + r) * 128 + (((c ^ r) & 7) << 4)) = v;
                    }
                }
            }
            if (is_v && lane == 0) bad_s[ring.i] = bad;
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(full);
            ring.next();
        }
    } else if (warp == kMmaWarp) {
        // ------------------------------- tensor-core issuer: Q K^T one tile ahead of P V --------------------------
        constexpr uint32_t qk_desc = tc_idesc(kTile, false), pv_desc = tc_idesc(D, true);
        const bool leader = elect_one();
        const uint32_t qb = smem_u32(q_s);
        Ring kr(KS, 0), vr(VS, 0);
        wait(q_full, 0);
        for (int i = 0; i <= w.tiles; ++i) {
            if (i < w.tiles) {
                const int b = i & 1;
                wait(s_empty(b), (uint32_t)((i >> 1) & 1) ^ 1u);
                wait(k_full(kr.i), kr.phase);
                tc_fence_after();
                const uint32_t kb = smem_u32(k_s + kr.i * C::TILE_BYTES), d = tmem + C::S_COL + b * kTile;
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    const uint64_t ad = smem_desc(qb + (ks >> 2) * C::Q_SLAB + (ks & 3) * 32), bd = smem_desc(kb + (ks >> 2) * C::K_SLAB + (ks & 3) * 32);
                    if (leader) tc_mma_ss(d, ad, bd, qk_desc, ks > 0);
                }
                if (leader) { tc_commit(k_empty(kr.i)); tc_commit(s_full(b)); }
                kr.next();
                __syncwarp();
            }
            if (i > 0) {
                const int b = (i - 1) & 1;
                wait(v_full(vr.i), vr.phase);
                wait(p_full(b), (uint32_t)(((i - 1) >> 1) & 1));
                tc_fence_after();
                const uint32_t vb = smem_u32(v_s + vr.i * C::TILE_BYTES);
#pragma unroll
                for (int pg = 0; pg < kTile / kPage; ++pg) {
                    const uint64_t bd = smem_desc_mn(vb + pg * C::V_PAGE, kPage * 128);
                    if (leader) tc_mma_ts(tmem + C::O_COL, tmem + C::P_COL + b * (kTile / 2) + pg * 8, bd, pv_desc, i > 1 || pg > 0);
                }
                if (leader) { tc_commit(v_empty(vr.i)); tc_commit(o_done(b)); }
                vr.next();
                __syncwarp();
            }
        }
    } else {
        // ------------------------------- softmax: thread = query row ---------------------------------------------
        for (int e = tid; e < w.nq * CPR; e += kSoftWarps * 32) {
            const int r = e / CPR, c = e % CPR, qr = q0 + r, t = qr / G;
            const uint4 v = *reinterpret_cast<const uint4*>(a.q + ((size_t)(w.r0 + t) * a.H + kvh * G + qr - t * G) * D + c * 8);
            *reinterpret_cast<uint4*>(q_s + (c >> 3) * C::Q_SLAB + r * 128 + (((c ^ r) & 7) << 4)) = v;
        }
        fence_proxy_async();
        __syncwarp();
        if (lane == 0) mbar_arrive(q_full);
        if (warp < live) {
            const int qr = q0 + tid, t = min(qr / G, n - 1), p = w.L + t, lo = max(0, p + 1 - a.window);
            const uint32_t row = tmem + ((uint32_t)(warp * 32) << 16);
            float m = -INFINITY, l = 0.f;
            Ring vr(VS, 0);
            for (int i = 0; i < w.tiles; ++i) {
                const int b = i & 1, j0 = w.base(i);
                const uint32_t round = (uint32_t)((i >> 1) & 1);
                wait(s_full(b), round);
                tc_fence_after();
                float s[kTile];
                tc_ld32(row + C::S_COL + b * kTile, *reinterpret_cast<float(*)[32]>(s));
                tc_ld32(row + C::S_COL + b * kTile + 32, *reinterpret_cast<float(*)[32]>(s + 32));
                tc_wait_ld();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(s_empty(b));
                unsigned long long bad = 0;
                if (w.mixed(j0)) {                       // the V tile's notes are there once it is (and stay until P V)
                    wait(v_full(vr.i), vr.phase);
                    bad = bad_s[vr.i];
                }
                vr.next();
                const bool whole = j0 + kTile <= p + 1 && (j0 >= lo || j0 + kTile <= w.sinks);
                float top = -INFINITY;
                if (__all_sync(0xffffffffu, whole) && bad == 0) {
#pragma unroll
                    for (int e = 0; e < kTile; ++e) top = fmaxf(top, s[e]);
                } else {
#pragma unroll
                    for (int e = 0; e < kTile; ++e) {
                        const int j = j0 + e;
                        const bool sees = j <= p && (j >= lo || j < w.sinks);
                        s[e] = sees ? s[e] : -INFINITY;
                        if (sees && (bad >> e & 1)) l = __int_as_float(0x7FC00000);
                        top = fmaxf(top, s[e]);
                    }
                }
                top *= a.scale_log2;
                // move the maximum only where it must: a row's choice looks at its own scores alone
                float alpha = 1.f;
                if (top > m + kSlack || (m == -INFINITY && top > m)) {
                    alpha = m == -INFINITY ? 1.f : fast_exp2(m - top);       // nothing summed yet: all is zero
                    m = top;
                    l *= alpha;
                }
                const float off = m == -INFINITY ? 0.f : m;
                if (i > 0 && __any_sync(0xffffffffu, alpha != 1.f)) {
                    wait(o_done((i - 1) & 1), (uint32_t)(((i - 1) >> 1) & 1));
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
                    tc_wait_st();
                }
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
                uint32_t pk[kTile / 2];
#pragma unroll
                for (int e = 0; e < kTile; e += 2) {
                    const float x = fast_exp2(fmaf(s[e], a.scale_log2, -off)), y = fast_exp2(fmaf(s[e + 1], a.scale_log2, -off));
                    sum[(e >> 1) & 3] += x;
                    sum[(e >> 1) & 3] += y;
                    pk[e >> 1] = pack_bf16(x, y);
                }
                l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
                if (i > 1) wait(o_done(b), round ^ 1u);       // P V of tile i - 2 has read this buffer
                tc_fence_after();
                tc_st32(row + C::P_COL + b * (kTile / 2), pk);
                tc_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_full(b));
            }
            // ---- the chunk's partials ----
            wait(o_done((w.tiles - 1) & 1), (uint32_t)(((w.tiles - 1) >> 1) & 1));
            tc_fence_after();
            const size_t cell = ((size_t)slot * a.R + w.r0 + t) * a.H + kvh * G + qr - t * G;
            const bool mine = tid < w.nq;
            if (mine) { a.part_m[cell] = m; a.part_l[cell] = l; }
#pragma unroll 1
            for (int c = 0; c < D; c += 32) {
                float o[32];
                tc_ld32(row + C::O_COL + c, o);
                tc_wait_ld();
                if (mine) {
#pragma unroll
                    for (int e = 0; e < 32; e += 4) *reinterpret_cast<float4*>(a.part_o + cell * D + c + e) = make_float4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tc_dealloc(tmem, C::COLS);
    }
}

// Joins the chunks of a row, in order: D / 8 lanes a (row, head), eight values a lane. Chunks in which the row sees nothing are
// passed over, so the join does not depend on which chunks the rows beside it needed.
template <int D>
__global__ void __launch_bounds__(128) window_join_kernel(const WindowArgs a) {
    constexpr int LANES = D / 8, PER_WARP = 32 / LANES;
    pdl_launch_dependents();
    pdl_wait();
    const int row = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int head = (blockIdx.x * 4 + warp) * PER_WARP + lane / LANES, li = lane % LANES;
    const int Mp = tf_padded_rows(a.R);
    const int seq = row < a.R ? seq_of(a.seq_start, a.S, row) : -1;
    const bool there = head < a.H;
    const int c8 = head * LANES + li;
    if (seq < 0) {
        if (row >= a.R && a.out_packed != nullptr && there) {          // padding rows of the packed buffer are zero
            if (a.group == 64) packed_store<64>(a.out_packed, Mp, row, c8, make_uint4(0, 0, 0, 0), 0.f);
            else packed_store<32>(a.out_packed, Mp, row, c8, make_uint4(0, 0, 0, 0), 0.f);
        }
        return;
    }
    const int p = a.seq_lens[seq] + row - a.seq_start[seq];
    if (p < 0 || p >= a.max_context) return;                           // reported by the chunk kernel
    const int lo = max(0, p + 1 - a.window);
    // chunks with sinks below the window, then the window's
    const int head_chunks = min(a.sinks, lo) > 0 ? (min(a.sinks, lo) - 1) / a.chunk + 1 : 0;
    const int far = max(head_chunks, lo / a.chunk), count = head_chunks + p / a.chunk + 1 - far;
    float acc[8], m = -INFINITY, l = 0.f;
#pragma unroll
    for (int e = 0; e < 8; ++e) acc[e] = 0.f;
    constexpr int B = 4;                                               // chunks whose loads are in flight together
    for (int i0 = 0; i0 < count; i0 += B) {
        float cm[B], cl[B];
        float4 po[B][2];
#pragma unroll
        for (int k = 0; k < B; ++k) {
            const int i = min(i0 + k, count - 1), chunk = i < head_chunks ? i : far + i - head_chunks;
            const size_t cell = ((size_t)slot_of(chunk, a.first_slots, a.near_slots) * a.R + row) * a.H + (there ? head : 0);
            cm[k] = a.part_m[cell];
            cl[k] = i0 + k < count ? a.part_l[cell] : 0.f;
            const float4* src = reinterpret_cast<const float4*>(a.part_o + cell * D + li * 8);
            po[k][0] = src[0];
            po[k][1] = src[1];
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
    if (a.lse != nullptr && li == 0 && there) a.lse[(size_t)row * a.H + head] = (m + log2f(l)) * kLn2;
    float o[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) o[e] = round_bf16(acc[e] / l);
    if (a.qg != nullptr && there) {
        float g[8];
        unpack8(*reinterpret_cast<const uint4*>(a.qg + (size_t)row * a.qg_stride + (size_t)head * 2 * D + D + li * 8), g);
#pragma unroll
        for (int e = 0; e < 8; ++e) o[e] = round_bf16(o[e] * sigmoidf_(g[e]));
    }
    const uint4 v = pack8(o);
    if (a.out != nullptr && there) *reinterpret_cast<uint4*>(a.out + ((size_t)row * a.H + head) * D + li * 8) = v;
    if (a.out_packed != nullptr) {
        const float sum = a.group == 64 ? group_sum8<64>(v) : group_sum8<32>(v);
        if (there) {
            if (a.group == 64) packed_store<64>(a.out_packed, Mp, row, c8, v, sum);
            else packed_store<32>(a.out_packed, Mp, row, c8, v, sum);
        }
    }
}

// ---- host side -----------------------------------------------------------------------------------------
// Descriptors of the tiled copies: rows of D values seen as [row][64 values][D / 64 slabs], a box of 16 rows and one slab (K, whose
// slabs lie apart in a tile) or all of them (V).
bool describe(CUtensorMap* map, const void* base, unsigned long long rows, size_t row_bytes, int heads, size_t head_bytes, int D, bool all_slabs) {
    static const PFN_cuTensorMapEncodeTiled_v12000 encode = [] {
        void* fn = nullptr;
        cudaDriverEntryPointQueryResult got;
        if (cudaGetDriverEntryPointByVersion("cuTensorMapEncodeTiled", &fn, 12000, cudaEnableDefault, &got) != cudaSuccess || got != cudaDriverEntryPointSuccess)
            fn = nullptr;
        return reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
    }();
    if (encode == nullptr) return false;
    const cuuint64_t dims[4] = {64, rows < 16 ? 16 : rows, (cuuint64_t)(D / 64), (cuuint64_t)heads};
    const cuuint64_t strides[3] = {row_bytes, 128, head_bytes};
    const cuuint32_t box[4] = {64, kPage, all_slabs ? (cuuint32_t)(D / 64) : 1u, 1}, steps[4] = {1, 1, 1, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, steps, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <int D, int QR>
int launch_chunks(WindowArgs& a, int slots, cudaStream_t st) {
    using C = Cfg<D, QR>;
    static bool configured[64] = {};       // the opt-in is per device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return TF_ECUDA; }
    if (!configured[dev]) {
        if (cudaFuncSetAttribute(window_chunk_kernel<D, QR>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) {
            cudaGetLastError();
            return TF_ECUDA;
        }
        configured[dev] = true;
    }
    CUtensorMap maps[4];
    const unsigned long long rows = (unsigned long long)a.num_pages * a.HK * kPage;
    const size_t row = (size_t)D * 2;
    if (!describe(&maps[0], a.k_pages, rows, row, 1, row, D, false) || !describe(&maps[1], a.v_pages, rows, row, 1, row, D, true) ||
        !describe(&maps[2], a.k_new, a.R, row * a.HK, a.HK, row, D, false) || !describe(&maps[3], a.v_new, a.R, row * a.HK, a.HK, row, D, true))
        return TF_ECUDA;
    a.qgroups = (int)(((long long)a.max_window * (a.H / a.HK) + QR - 1) / QR);
    if ((long long)a.S * a.qgroups > 65535) return TF_EINVAL;
    void* args[] = {&a, &maps[0], &maps[1], &maps[2], &maps[3]};
    if (launch_pdl((const void*)window_chunk_kernel<D, QR>, dim3(slots, a.HK, a.S * a.qgroups), dim3(kThreads), C::SMEM, st, args) != cudaSuccess) {
        cudaGetLastError();
        return TF_ECUDA;
    }
    return TF_OK;
}

template <int D>
int run(WindowArgs& a, int slots, cudaStream_t st) {
    const bool small = a.max_window * (long long)(a.H / a.HK) <= 64;
    const int rc = small ? launch_chunks<D, 64>(a, slots, st) : launch_chunks<D, 128>(a, slots, st);
    if (rc != TF_OK) return rc;
    void* args[] = {&a};
    const int heads = 4 * (32 / (D / 8)), rows = a.out_packed ? tf_padded_rows(a.R) : a.R;
    if (launch_pdl((const void*)window_join_kernel<D>, dim3((a.H + heads - 1) / heads, rows), dim3(128), 0, st, args) != cudaSuccess) {
        cudaGetLastError();
        return TF_ECUDA;
    }
    return TF_OK;
}

}  // namespace
}  // namespace tf

extern "C" {

int tf_window_slots(int window, int sinks, int max_window, int max_context, int chunk_keys) {
    if (window < 0 || sinks < 0 || max_window < 1 || max_context < max_window || max_context > (1 << 30) || chunk_keys < tf::kTile || chunk_keys % tf::kTile)
        return 0;
    const tf::Slots s = tf::slots_for(window, sinks, max_window, max_context, chunk_keys);
    return s.first + s.near;
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
    if (rows > 65535 || kv_heads > 65535 || (long long)num_pages * kv_heads * 16 > 0x7FFFFFFFll) return TF_EINVAL;
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
    a.chunk = chunk_keys;
    const tf::Slots cut = tf::slots_for(window, sinks, max_window, max_context, chunk_keys);
    a.first_slots = cut.first; a.near_slots = cut.near > 0 ? cut.near : 1;
    const size_t cells = (size_t)slots * rows * heads;
    a.part_o = static_cast<float*>(scratch);
    a.part_m = a.part_o + cells * head_dim;
    a.part_l = a.part_m + cells;
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    return head_dim == 256 ? tf::run<256>(a, slots, st) : tf::run<128>(a, slots, st);
}

}  // extern "C"
