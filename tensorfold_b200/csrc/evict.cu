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

#include "tc.cuh"

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
    int num_pages, max_pages, H, HK, R, S, layers, max_window, max_context;
    float scale_log2;
};

// S^T = K Q^T on the tensor core: a tile of 128 keys is the A operand (its rows the tensor memory's lanes), the kept query rows, up to 128 at a
// time, the B operand, so that a key's scores lie in one thread's lane and its sum needs no shuffle and no atomic: thread = key, columns
// in row order, fp32. K arrives a page at a time by tiled copies; slots behind the last key are never added.
//
// The tiles of all (layer, KV head, sequence) columns form one sequence that is cut into equal runs, one a block: a block starts in the middle of a
// column and goes on into the next ones, its copies running ahead over the border. With up to 128 rows (the usual case) Q is staged once a
// column. What bounds it: the bytes of K (4 layers x 4 heads x 16 users of 2048 to 8192 keys: 767 MB in 135 us, 5.7 TB/s; with blocks that each took
// a share of one column, three rounds of them, 151 us); 2^x on the special-function units takes a quarter of a tile's 1.5 us. One user of 4096
// keys in 16 layers: 134 MB in 28 us, of which a block's start is 4.
constexpr int kMassKeys = 128, kMassRows = 128, kMassSum = 4, kMassMma = 4, kMassLoad = 5, kMassThreads = 6 * 32;

template <int D>
struct MassCfg {
    static constexpr int SLABS = D / 64, K_SLAB = kMassKeys * 128, TILE_BYTES = SLABS * K_SLAB, Q_SLAB = kMassRows * 128, Q_BYTES = SLABS * Q_SLAB;
    static constexpr int KS = D == 256 ? 2 : 4;
    static constexpr int NBARS = 2 * KS + 4 + 2;
    static constexpr int SMEM = Q_BYTES + KS * TILE_BYTES + kMassRows * 4 + NBARS * 8 + 1024;
    static_assert(SMEM <= 227 * 1024, "shared memory");
};

template <int D>
__global__ void __launch_bounds__(kMassThreads, 1) mass_kernel(const __grid_constant__ MassArgs a, const __grid_constant__ CUtensorMap k_map) {
    using C = MassCfg<D>;
    constexpr int KS = C::KS, CPR = D / 8;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint32_t tmem_s;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t* q_s = smem + ((1024u - (smem_u32(smem) & 1023u)) & 1023u);
    uint8_t* k_s = q_s + C::Q_BYTES;
    float* lse_s = reinterpret_cast<float*>(k_s + KS * C::TILE_BYTES);               // of the staged rows, log2 domain
    const uint32_t bars = smem_u32(lse_s + kMassRows);
    auto k_full = [&](int s) { return bars + 8u * s; };
    auto k_empty = [&](int s) { return bars + 8u * (KS + s); };
    auto s_full = [&](int s) { return bars + 8u * (2 * KS + s); };
    auto s_empty = [&](int s) { return bars + 8u * (2 * KS + 2 + s); };
    const uint32_t q_full = bars + 8u * (2 * KS + 4), q_empty = q_full + 8;
    if (tid == 0) {
        for (int s = 0; s < KS; ++s) { mbar_init(k_full(s), 1); mbar_init(k_empty(s), 1); }
        for (int s = 0; s < 2; ++s) { mbar_init(s_full(s), 1); mbar_init(s_empty(s), kMassSum); }
        mbar_init(q_full, kMassSum);
        mbar_init(q_empty, 1);
        mbar_fence_init();
    }
    if (warp == kMassMma) tc_alloc(smem_u32(&tmem_s), 2 * kMassRows);
    tc_fence_before();
    __syncthreads();
    pdl_launch_dependents();        // not before the tensor memory is this block's: a dependent that held it would wait for this kernel
    tc_fence_after();
    const uint32_t tmem = tmem_s;
    Waits wait(a.status);
    pdl_wait();
    // ---- the block's share of the tiles (it may have none) ----
    const int G = a.H / a.HK;
    // sequence s: first row, rows kept, length before the commit, tiles (0: not what the call was made for, reported, or nothing kept)
    auto column = [&](int s) -> int4 {
        if (s >= a.S) return make_int4(0, 0, 0, 0);
        const int r0 = a.seq_start[s], n = a.seq_start[s + 1] - r0, L = a.seq_lens[s], kept = min(max(a.keep[s], 0), n);
        if (kept < 1) return make_int4(0, 0, 0, 0);
        if (n > a.max_window || r0 < 0 || r0 > a.R - n || L < 0 || L > a.max_context - kept || L > a.max_pages * kPage - kept) {
            report(a.status, TF_EINVAL);
            return make_int4(0, 0, 0, 0);
        }
        return make_int4(r0, kept, L, (L + kept + kMassKeys - 1) / kMassKeys);
    };
    long long a_head = 0;                        // tiles of one (layer, KV head)
    for (int s0 = 0; s0 < a.S; s0 += 32) a_head += __reduce_add_sync(0xffffffffu, (unsigned)column(s0 + lane).w);
    const long long all = a_head * a.HK * a.layers;
    const long long begin = all * blockIdx.x / gridDim.x, end = all * (blockIdx.x + 1) / gridDim.x;
    struct Run {                                 // tiles first .. last - 1 of a column
        int layer, kvh, seq, r0, kept, L, keys, first, last;
    };
    // the block's run that starts at tile `x` of all. Whole warps; the columns are read again, from the cache
    auto run_at = [&](long long x) -> Run {
        const int head = (int)(x / a_head);
        long long left = x - head * a_head;
        Run r{head / a.HK, head % a.HK, 0, 0, 0, 0, 0, 0, 0};
        for (int s0 = 0; s0 < a.S; s0 += 32) {
            const int4 c = column(s0 + lane);
            int upto = c.w;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += y;
            }
            const unsigned m = __ballot_sync(0xffffffffu, upto > left);
            if (m == 0) {
                left -= __shfl_sync(0xffffffffu, upto, 31);
                continue;
            }
            const int who = __ffs(m) - 1, tiles = __shfl_sync(0xffffffffu, c.w, who);
            r.seq = s0 + who;
            r.r0 = __shfl_sync(0xffffffffu, c.x, who);
            r.kept = __shfl_sync(0xffffffffu, c.y, who);
            r.L = __shfl_sync(0xffffffffu, c.z, who);
            r.keys = r.L + r.kept;
            r.first = (int)(left - (__shfl_sync(0xffffffffu, upto, who) - tiles));
            r.last = end - x < tiles - r.first ? r.first + (int)(end - x) : tiles;
            break;
        }
        return r;
    };

    if (warp == kMassLoad) {
        Ring ring(KS, 1);
        // a lane copies 64 values of a page's 16 rows, the lanes of a page beside one another; page numbers are looked up a tile ahead; one
        // behind the last key or that is none (reported) is copied from page 0 and not used
        const int slab = lane % C::SLABS, at = lane / C::SLABS;
        for (long long x = begin; x < end;) {
            const Run w = run_at(x);
            x += w.last - w.first;
            const int* pt = a.page_table + (size_t)w.seq * a.max_pages;
            auto number = [&](int t) -> int {
                const int j = t * kMassKeys + at * kPage;
                if (at >= 8 || t >= w.last || j >= w.keys) return 0;
                const int page = pt[j / kPage];
                if (page >= 0 && page < a.num_pages) return page;
                report(a.status, TF_EINVAL);
                return 0;
            };
            int next = number(w.first);
            for (int t = w.first; t < w.last; ++t) {
                const int page = next;
                next = number(t + 1);
                wait(k_empty(ring.i), ring.phase);
                if (lane == 0) mbar_arrive_expect_tx(k_full(ring.i), C::TILE_BYTES);
                __syncwarp();
                if (at < 8) {
                    const int y = ((w.layer * a.num_pages + page) * a.HK + w.kvh) * kPage;
                    tma_4d(smem_u32(k_s) + ring.i * C::TILE_BYTES + slab * C::K_SLAB + at * (kPage * 128), &k_map, 0, y, slab, 0, k_full(ring.i));
                }
                __syncwarp();
                ring.next();
            }
        }
    } else if (warp == kMassMma) {
        const bool leader = elect_one();
        const uint32_t q_lo = desc_lo(smem_u32(q_s), 1);
        Ring kr(KS, 0), qr(1, 0), sr(2, 1);
        for (long long x = begin; x < end;) {
            const Run w = run_at(x);
            x += w.last - w.first;
            const int mine = __reduce_max_sync(0xffffffffu, w.last - w.first), least = __reduce_max_sync(0xffffffffu, w.kept * G);
            const int parts = (least + kMassRows - 1) / kMassRows;
            for (int t = 0; t < mine; ++t) {
                wait(k_full(kr.i), kr.phase);
                const uint32_t k_lo = desc_lo(smem_u32(k_s) + kr.i * C::TILE_BYTES, 1);
                for (int c = 0; c < parts; ++c) {
                    if (parts > 1 || t == 0) {
                        wait(q_full, qr.phase);
                        qr.next();
                    }
                    wait(s_empty(sr.i), sr.phase);
                    tc_fence_after();
                    // columns in sixteens (N of the tensor core with M = 128)
                    const uint32_t idesc = tc_idesc((min(kMassRows, least - c * kMassRows) + 15) & ~15, false);
#pragma unroll
                    for (int ks = 0; ks < D / 16; ++ks)
                        tc_mma_ss(leader, tmem + sr.i * kMassRows, k_lo + (((ks >> 2) * C::K_SLAB + (ks & 3) * 32) >> 4), q_lo + (((ks >> 2) * C::Q_SLAB + (ks & 3) * 32) >> 4),
                                  idesc, ks > 0);
                    if (leader) {
                        tc_commit(s_full(sr.i));
                        if (parts > 1 || t + 1 == mine) tc_commit(q_empty);
                        if (c + 1 == parts) tc_commit(k_empty(kr.i));
                    }
                    __syncwarp();
                    sr.next();
                }
                kr.next();
            }
        }
    } else {
        const uint32_t lanes = tmem + ((uint32_t)(warp * 32) << 16);
        Ring sr(2, 0), qr(1, 1);
        for (long long x = begin; x < end;) {
            const Run w = run_at(x);
            x += w.last - w.first;
            const int rows = w.kept * G, chunks = (rows + kMassRows - 1) / kMassRows;
            const size_t plane = (size_t)w.layer * a.num_pages * a.HK * kPage;
            const int* pt = a.page_table + (size_t)w.seq * a.max_pages;
            auto stage = [&](int c) {            // rows c * 128 ..: into shared memory, with their log-sum-exps
                wait(q_empty, qr.phase);         // the products of the rows before have read them ...
                qr.next();
                named_bar_sync(1, kMassSum * 32);        // ... and so have the sums
                const int q0 = c * kMassRows, count = min(kMassRows, rows - q0);
                const size_t row0 = (size_t)w.layer * a.R + w.r0;
                constexpr int B = 8, STEP = kMassSum * 32;       // loads in flight a thread
                for (int e0 = tid; e0 < count * CPR; e0 += B * STEP) {
                    uint4 v[B];
#pragma unroll
                    for (int k = 0; k < B; ++k) {
                        const int e = min(e0 + k * STEP, count * CPR - 1), r = e / CPR, y = e % CPR, t = (q0 + r) / G;
                        v[k] = *reinterpret_cast<const uint4*>(a.q + ((row0 + t) * a.H + w.kvh * G + q0 + r - t * G) * D + y * 8);
                    }
#pragma unroll
                    for (int k = 0; k < B; ++k) {
                        const int e = e0 + k * STEP, r = e / CPR, y = e % CPR;
                        if (e < count * CPR) *reinterpret_cast<uint4*>(q_s + (y >> 3) * C::Q_SLAB + r * 128 + (((y ^ r) & 7) << 4)) = v[k];
                    }
                }
                if (tid < count) {
                    const int t = (q0 + tid) / G;
                    lse_s[tid] = a.lse[(row0 + t) * a.H + w.kvh * G + q0 + tid - t * G] * kLog2e;
                }
                named_bar_sync(1, kMassSum * 32);            // the log-sum-exps are everybody's
                fence_proxy_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(q_full);
            };
            if (chunks == 1) stage(0);
            for (int t = w.first; t < w.last; ++t) {
                const int j = t * kMassKeys + tid;
                float sum = 0.f;
                // the key's old weight, under way while the scores are formed
                size_t cell = 0;
                float old = 0.f;
                bool real = j < w.keys;
                if (real) {
                    const int page = pt[j / kPage];
                    real = page >= 0 && page < a.num_pages;
                    cell = plane + ((size_t)(real ? page : 0) * a.HK + w.kvh) * kPage + j % kPage;
                    if (real && j < w.L) old = a.mass[cell];
                }
                const int from = max(0, j - w.L) * G;        // rows that come before the key itself
                for (int c = 0; c < chunks; ++c) {
                    if (chunks > 1) stage(c);
                    wait(s_full(sr.i), sr.phase);
                    tc_fence_after();
                    const int q0 = c * kMassRows, count = min(kMassRows, rows - q0);
                    for (int y = 0; y < count; y += 16) {
                        float s[16];
                        tc_ld16(lanes + sr.i * kMassRows + y, s);
                        tc_wait_ld();
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            const float p = fast_exp2(fmaf(s[e], a.scale_log2, -lse_s[y + e]));
                            sum += y + e < count && q0 + y + e >= from ? p : 0.f;
                        }
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s_empty(sr.i));
                    sr.next();
                }
                if (real) {
                    a.mass[cell] = old + sum;
                    if (j >= w.L) a.pos[cell] = a.row_pos[w.r0 + j - w.L];
                }
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kMassMma) {
        tc_fence_after();
        tc_dealloc(tmem, 2 * kMassRows);
    }
}

// ---- eviction ------------------------------------------------------------------------------------------
constexpr int kSelThreads = 1024;
constexpr int kBins = 8192;          // of the first histogram: 13 bits of a key; then 10 and 9 bits where many share those
constexpr int kRanked = kSelThreads / 4;
constexpr int kSelKeys = 45056;      // slots whose keys fit the block's shared memory; longer sequences are ranked from global memory

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

// Exclusive prefix sum over the block (kSelThreads threads) of counts (two below 2^32 in a 64-bit word); `total`: the sum. The warps' sums are scanned by
// every warp for itself.
template <class T>
__device__ __forceinline__ T block_scan(T v, unsigned long long* warp_s, T& total) {
    static_assert(kSelThreads == 32 * 32, "a lane a warp");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    auto inclusive = [&](T x) {
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const T y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        return x;
    };
    const T x = inclusive(v);
    __syncthreads();                  // an earlier scan's sums have been read
    if (lane == 31) warp_s[warp] = x;
    __syncthreads();
    const T sums = inclusive((T)warp_s[lane]);
    total = __shfl_sync(0xffffffffu, sums, 31);
    const T before = __shfl_sync(0xffffffffu, sums, (warp + 31) & 31);
    return (warp > 0 ? before : 0) + x - v;
}

// Bound by its chain of dependent steps (64 blocks of 4224 slots: 8.2 us): the page numbers, then weights and positions, a quarter page a
// thread; a histogram of the keys' first 13 bits, in which the slots that stay anyway take no part; the slots that share those bits with the
// threshold, few as a rule, ranked by comparison (two more histograms in their place: 10 us); a pass that counts, one that writes.
template <bool STAGED>
__global__ void __launch_bounds__(kSelThreads) evict_select_kernel(const EvictArgs a) {
    extern __shared__ uint32_t keys_s[];
    __shared__ __align__(16) unsigned hist[kBins];
    __shared__ unsigned long long ranked_s[kRanked];
    __shared__ unsigned long long warp_s[kSelThreads / 32];
    __shared__ unsigned digit_s, above_s, safe_s, count_s;
    pdl_launch_dependents();
    const int kvh = blockIdx.x, seq = blockIdx.y, layer = blockIdx.z, tid = threadIdx.x;
    const size_t item = ((size_t)layer * a.S + seq) * a.HK + kvh;
    for (int b = tid; b < kBins; b += kSelThreads) hist[b] = 0;
    if (tid == 0) safe_s = count_s = 0;
    pdl_wait();
    const int L = a.seq_lens[seq], n = min(L, min(a.max_context, a.max_pages * kPage)), safe_from = a.next_pos[seq] - a.recent;
    if (L > n && tid == 0) report(a.status, TF_EINVAL);
    if (n <= a.budget) {
        if (tid == 0) a.moved[item] = 0;
        return;
    }
    const int* pt = a.page_table + (size_t)seq * a.max_pages;
    constexpr uint32_t kSafe = 0xFFFFFFFFu;
    // a slot's rank: protected first, then by mass; NaN counts as -inf
    auto rank_of = [&](float m, int p) -> uint32_t {
        if (p < a.sinks || p >= safe_from) return kSafe;
        m += 0.f;                                      // -0 ranks as 0
        const uint32_t u = __float_as_uint(m);
        return m != m ? 0x007FFFFFu : u & 0x80000000u ? ~u : u | 0x80000000u;
    };
    auto cell_of = [&](int j, int page) -> size_t { return (((size_t)layer * a.num_pages + page) * a.HK + kvh) * kPage + j % kPage; };
    auto page_of = [&](int j) -> int {
        const int page = pt[j / kPage];
        if (page < 0 || page >= a.num_pages) { report(a.status, TF_EINVAL); return -1; }
        return page;
    };
    auto key = [&](int j) -> uint32_t {
        if (STAGED) return keys_s[j];
        const int page = page_of(j);
        return page < 0 ? 0u : rank_of(a.mass[cell_of(j, page)], a.pos[cell_of(j, page)]);
    };
    __syncthreads();
    unsigned safe = 0;
    if (STAGED) {
        // four slots a thread, two such quads in flight; the first histogram on the way
        for (int q0 = tid; q0 * 4 < n; q0 += 2 * kSelThreads) {
            int page[2];
            float4 m[2];
            int4 p[2];
#pragma unroll
            for (int k = 0; k < 2; ++k) page[k] = (q0 + k * kSelThreads) * 4 < n ? page_of((q0 + k * kSelThreads) * 4) : -1;
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const size_t cell = cell_of((q0 + k * kSelThreads) * 4, max(page[k], 0));
                m[k] = page[k] < 0 ? make_float4(0.f, 0.f, 0.f, 0.f) : *reinterpret_cast<const float4*>(a.mass + cell);
                p[k] = page[k] < 0 ? make_int4(0, 0, 0, 0) : *reinterpret_cast<const int4*>(a.pos + cell);
            }
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                const int j = (q0 + k * kSelThreads) * 4;
                const float mk[4] = {m[k].x, m[k].y, m[k].z, m[k].w};
                const int pk[4] = {p[k].x, p[k].y, p[k].z, p[k].w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (j + e >= n) continue;
                    const uint32_t r = page[k] < 0 ? 0u : rank_of(mk[e], pk[e]);
                    keys_s[j + e] = r;
                    if (r == kSafe) ++safe;
                    else atomicAdd(&hist[r >> 19], 1u);
                }
            }
        }
    } else {
        for (int j = tid; j < n; j += kSelThreads) {
            const uint32_t r = key(j);
            if (r == kSafe) ++safe;
            else atomicAdd(&hist[r >> 19], 1u);
        }
    }
    safe = __reduce_add_sync(0xffffffffu, safe);
    if ((tid & 31) == 0 && safe) atomicAdd(&safe_s, safe);
    __syncthreads();
    // the smallest key that stays: the need-th largest of those that are not protected. More protected slots than the budget holds (positions that
    // are none): the first of them stay
    uint32_t prefix = kSafe, need = a.budget;
    bool ties = true;
    if (safe_s < need) {
        need -= safe_s;
        // thread i holds bins 8191 - 8 i .. 8184 - 8 i: prefix sums from the largest digit down
        const uint4 *eight = reinterpret_cast<const uint4*>(hist + kBins - 8 - 8 * tid), hi4 = eight[1], lo4 = eight[0];
        const unsigned bins[8] = {hi4.w, hi4.z, hi4.y, hi4.x, lo4.w, lo4.z, lo4.y, lo4.x};
        unsigned mine = 0, all;
#pragma unroll
        for (int x = 0; x < 8; ++x) mine += bins[x];
        unsigned before = block_scan(mine, warp_s, all);
#pragma unroll
        for (int x = 0; x < 8; ++x) {
            if (before < need && before + bins[x] >= need) { digit_s = kBins - 1 - 8 * tid - x; above_s = before; }
            before += bins[x];
        }
        __syncthreads();
        prefix = digit_s;
        need -= above_s;
        const unsigned many = hist[prefix];
        if (STAGED && many <= kRanked) {
            // few enough to be ranked by comparing all with all, four threads a slot; the key becomes the decision
            for (int j = tid; j < n; j += kSelThreads) {
                const uint32_t k = keys_s[j];
                if (k >> 19 == prefix && k != kSafe) ranked_s[atomicAdd(&count_s, 1u)] = (unsigned long long)k << 32 | ~(uint32_t)j;
            }
            __syncthreads();
            const unsigned long long own = (tid >> 2) < many ? ranked_s[tid >> 2] : 0;
            unsigned above = 0;
            for (unsigned i = tid & 3; i < many; i += 4) above += ranked_s[i] > own;
            above += __shfl_xor_sync(0xffffffffu, above, 1);
            above += __shfl_xor_sync(0xffffffffu, above, 2);
            if ((tid >> 2) < many && (tid & 3) == 0) keys_s[~(uint32_t)own] = above < need ? kSafe : 0u;
            __syncthreads();
            prefix = prefix << 19 | 0x7FFFFu;
            need = 0;
            ties = false;
        } else {
            for (int pass = 0; pass < 2; ++pass) {
                const int bits = pass == 0 ? 10 : 9, shift = pass == 0 ? 9 : 0;
                __syncthreads();                 // the bins have been read
                hist[tid] = 0;
                __syncthreads();
                for (int j = tid; j < n; j += kSelThreads) {
                    const uint32_t k = key(j);
                    if ((k >> (shift + bits)) == prefix && k != kSafe) atomicAdd(&hist[(k >> shift) & ((1u << bits) - 1)], 1u);
                }
                __syncthreads();
                const unsigned c = hist[kSelThreads - 1 - tid];
                const unsigned higher = block_scan(c, warp_s, all);
                if (higher < need && higher + c >= need) { digit_s = kSelThreads - 1 - tid; above_s = higher; }
                __syncthreads();
                prefix = prefix << bits | digit_s;
                need -= above_s;
            }
        }
    }
    // kept: every key above `prefix` and the first `need` slots of that key. Each thread takes a run of slots (an odd number of
    // words: no bank conflicts)
    const int per = ((n + kSelThreads - 1) / kSelThreads) | 1, lo = min(n, tid * per), hi = min(n, lo + per);
    unsigned eq0 = 0;
    if (ties) {
        unsigned all;
        for (int j = lo; j < hi; ++j) eq0 += key(j) == prefix;
        eq0 = block_scan(eq0, warp_s, all);
    }
    unsigned eq = eq0;
    unsigned long long counts = 0, total;        // holes below the budget | kept slots above it
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
    // four slots a warp at a time: their places are looked up by four lanes, then eight rows (four of K, four of V) are on the way together
    constexpr int B = 4;
    for (int i0 = (blockIdx.x * kMoveWarps + warp) * B; i0 < count; i0 += gridDim.x * kMoveWarps * B) {
        bool ok = lane < B && i0 + lane < count;
        long long to = 0, from = 0;
        if (ok) {
            to = cell(holes[i0 + lane], ok);
            from = cell(fills[i0 + lane], ok);
        }
        const float m = ok ? a.mass[from] : 0.f;
        const int p = ok ? a.pos[from] : 0;
        const unsigned move = __ballot_sync(0xffffffffu, ok);
        constexpr int PARTS = D == 256 ? 2 : 1;          // 16-byte columns of K and V a lane has: D = 128 takes both in one go
        uint4 v[B][PARTS];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const long long f = __shfl_sync(0xffffffffu, from, b);
#pragma unroll
            for (int x = 0; x < PARTS; ++x) {
                const __nv_bfloat16* base = PARTS == 2 ? (x ? a.v_pages : a.k_pages) : lane < 16 ? a.k_pages : a.v_pages;
                if (move >> b & 1) v[b][x] = reinterpret_cast<const uint4*>(base + f * D)[PARTS == 2 ? lane : lane & 15];
            }
        }
#pragma unroll
        for (int b = 0; b < B; ++b) {
            const long long t = __shfl_sync(0xffffffffu, to, b);
#pragma unroll
            for (int x = 0; x < PARTS; ++x) {
                __nv_bfloat16* base = PARTS == 2 ? (x ? a.v_pages : a.k_pages) : lane < 16 ? a.k_pages : a.v_pages;
                if (move >> b & 1) reinterpret_cast<uint4*>(base + t * D)[PARTS == 2 ? lane : lane & 15] = v[b][x];
            }
        }
        if (ok) { a.mass[to] = m; a.pos[to] = p; }
    }
}

constexpr int kSms = 148;

template <int D>
int launch_mass(const MassArgs& a, int layers, cudaStream_t st) {
    using C = MassCfg<D>;
    static std::atomic<bool> configured[64] = {};       // the opt-in is per device
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) { cudaGetLastError(); return TF_ECUDA; }
    if (!configured[dev]) {
        if (cudaFuncSetAttribute(mass_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::SMEM) != cudaSuccess) {
            cudaGetLastError();
            return TF_ECUDA;
        }
        configured[dev] = true;
    }
    CUtensorMap map;
    if (!describe_rows(&map, a.k_pages, D, (unsigned long long)layers * a.num_pages * a.HK * kPage, (size_t)D * 2, 1, (size_t)D * 2, false, kPage, 1, 1)) return TF_ECUDA;
    const long long tiles = (long long)layers * a.S * a.HK * ((a.max_context + kMassKeys - 1) / kMassKeys);
    void* args[] = {const_cast<MassArgs*>(&a), &map};
    if (launch_pdl((const void*)mass_kernel<D>, dim3(tiles < kSms ? (unsigned)tiles : kSms), dim3(kMassThreads), C::SMEM, st, args) != cudaSuccess) {
        cudaGetLastError();
        return TF_ECUDA;
    }
    return TF_OK;
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
    if ((long long)layers * n_seqs > 65535 || kv_heads > 65535 || (long long)layers * num_pages * kv_heads * 16 > 0x7FFFFFFFll) return TF_EINVAL;
    tf::MassArgs a{static_cast<const __nv_bfloat16*>(q), lse, static_cast<const __nv_bfloat16*>(k_pages), page_table, seq_lens, seq_start, keep,
                   row_pos, mass, pos, status, num_pages, max_pages, heads, kv_heads, rows, n_seqs, layers, max_window, max_context, scale * tf::kLog2e};
    return head_dim == 256 ? tf::launch_mass<256>(a, layers, static_cast<cudaStream_t>(stream)) : tf::launch_mass<128>(a, layers, static_cast<cudaStream_t>(stream));
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
    if (((uintptr_t)k_pages | (uintptr_t)v_pages) & 15 || ((uintptr_t)mass | (uintptr_t)pos) & 15 || ((uintptr_t)moved | (uintptr_t)scratch) & 3) return TF_EALIGN;
    if ((long long)layers * n_seqs > 65535 || kv_heads > 65535) return TF_EINVAL;
    if (!scratch || scratch_bytes < tf_evict_scratch_bytes(layers, n_seqs, kv_heads, budget, max_context)) return TF_ESCRATCH;
    const int most = max_context <= budget ? 1 : (max_context - budget < budget ? max_context - budget : budget);
    tf::EvictArgs a{static_cast<__nv_bfloat16*>(k_pages), static_cast<__nv_bfloat16*>(v_pages), page_table, seq_lens, next_pos, mass, pos, moved,
                    static_cast<int*>(scratch), status, num_pages, max_pages, kv_heads, n_seqs, budget, recent, sinks, max_context, most};
    void* args[] = {&a};
    cudaStream_t st = static_cast<cudaStream_t>(stream);
    const bool staged = max_context <= tf::kSelKeys;
    static std::atomic<bool> configured[64] = {};       // the opt-in is per device
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
    const int blocks = min((most + 4 * tf::kMoveWarps - 1) / (4 * tf::kMoveWarps), 32);
    const void* move = head_dim == 256 ? (const void*)tf::evict_move_kernel<256> : (const void*)tf::evict_move_kernel<128>;
    if (tf::launch_pdl(move, dim3(blocks, kv_heads, layers * n_seqs), dim3(tf::kMoveWarps * 32), 0, st, args) != cudaSuccess) {
        cudaGetLastError();
        return TF_ECUDA;
    }
    return TF_OK;
}

}  // extern "C"
