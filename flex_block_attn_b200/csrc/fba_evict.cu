// Eviction from a paged cache by accumulated attention weight.
//
// Per (sequence, kv head) of n slots the n - budget tokens that come first in the order (protected, weight, slot) leave.
// One CTA per (sequence, kv head), or a cluster where the keys of its slots do not fit into one CTA's shared memory:
//   1. weights become 32-bit keys in their order, protected tokens the largest key;
//   2. the key T of the last token that leaves is found from its digits, 11 + 11 + 10 bits from the top: a histogram of a
//      digit per CTA, all of them added up by every CTA through distributed shared memory (reads of all the CTAs in
//      flight at once, as are those of pages and weights in step 1: one after the other they cost 9 us of 55);
//   3. counts per warp (tokens with the key T; slots that come free; tokens to be moved), exchanged the same way, give
//      every warp the place of its entries in the lists of slots to move from and to, which are in slot order
//      therefore, whatever the timing;
//   4. the rows on the lists are copied, by a second kernel where there can be many.
// In place, the i-th staying token behind slot `budget` goes to the i-th slot that came free before it: only as many rows
// move as tokens leave from there, and no row is both read and written.  Where one token is too many, as at every step of
// serving within a budget, the smallest key is all there is to find: 128 heads of 2049 slots take 5.3 us behind other work, 9
// by themselves and 10 with a cold L2; with two too many, which takes the lists, 8.7, 13 and 14.
// What bounds it: the rows copied, and with few rows the latency of the steps before.
#include <math.h>
#include <stdio.h>

#include <cooperative_groups.h>

#include "fba_paged.cuh"

namespace fba {

namespace cg = cooperative_groups;

constexpr int kEvThreads = 1024;
constexpr int kEvWarps = kEvThreads / 32;
constexpr int kEvBins = 2048;

struct EvictParams {
    const int32_t *seq_lens, *next_positions, *out_table;
    int32_t* out_lens;
    int32_t *from, *to;      // [B * Hkv, list]: slots; `to` is not used with an out_table
    uint32_t* status;
    int32_t* moves;          // [B * Hkv]: entries of the lists, for the second kernel; null: the first one copies
    int budget, sinks, recent, out_pages, list;
    int key_room;            // keys a CTA holds in shared memory; 0: read again on every use
};

struct EvictShared {
    uint32_t hist[2][kEvBins];     // in turns, so that one may be filled while other CTAs still read the other
    uint32_t scan[kEvWarps];
    uint2 least[kEvWarps], least_cta;   // smallest key and its slot
    uint2 count[2][kEvWarps];      // per warp: ties, then holes and moves
    uint2 total[2];                // of the CTA
    uint32_t digit, below, inside; // of the bin that holds the wanted rank: its number, how many keys lie before it and in it
};

__device__ __forceinline__ uint32_t evict_key(const EvictParams& p, int pos, float weight, long long recent_from) {
    if (pos < p.sinks || pos >= recent_from) return 0xffffffffu;
    const float w = weight + 0.f;          // -0 counts as 0
    if (isnan(w)) return 0xfffffffeu;      // above infinity
    const uint32_t u = __float_as_uint(w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

// Copies the entries i0, i0 + 1, ... < total of a head's lists, 32 at a time: a lane looks up one entry's rows, then the
// warp copies them one after the other, half a warp each for K and V in bf16 (16 bytes a lane), a quarter each in e4m3,
// then two tokens at a time.  `stride`: from one batch of the warp to its next.
template <bool e4m3>
__device__ __forceinline__ void copy_rows(const PagedDev& c, const EvictParams& p, int b, int h, const int32_t* from,
                                          const int32_t* to, int i0, int total, int stride) {
    const int lane = threadIdx.x & 31;
    constexpr int lanes = e4m3 ? 8 : 16, tokens = e4m3 ? 2 : 1;
    const int sub = lane / (2 * lanes), kv = lane / lanes & 1, l = lane % lanes;
    PagedDev dst_c = c;
    if (p.out_table) {
        dst_c.table = p.out_table;
        dst_c.max_pages = p.out_pages;
    }
    uint4* pool = reinterpret_cast<uint4*>(kv ? c.v : c.k);
    for (int base = i0; base < total; base += stride) {
        int src = -1, dst = -1;   // 32 bits do: 2^31 rows of keys and values are 512 GB
        if (base + lane < total) {
            const int f = from[base + lane], t = p.out_table ? base + lane : to[base + lane];
            const int f_page = paged_page(c, b, f), t_page = paged_page(dst_c, b, t);
            src = static_cast<int>(paged_row_in(c, f_page, h, f));
            dst = static_cast<int>(paged_row_in(dst_c, t_page, h, t));
            if (src < 0 || dst < 0) {   // a page that is not there
                report_paged(p.status, kBadPage, b, src < 0 ? f_page : t_page);
                dst = -1;
            } else {   // what there is one of per row
                float ks, vs;
                if (e4m3) {
                    ks = c.k_scale[src];
                    vs = c.v_scale[src];
                }
                const float w = c.weight[src];
                const int pos = c.position[src];
                c.weight[dst] = w;
                c.position[dst] = pos;
                if (e4m3) {
                    c.k_scale[dst] = ks;
                    c.v_scale[dst] = vs;
                }
            }
        }
        const int n = min(32, total - base);
        constexpr int kFlight = 8;   // rows a lane has under way
        for (int j0 = 0; j0 < n; j0 += kFlight * tokens) {
            uint4 x[kFlight];
            int d[kFlight];
#pragma unroll
            for (int u = 0; u < kFlight; ++u) {
                const int j = j0 + u * tokens + sub;   // below 32 + 16; lanes repeat modulo 32
                const int s = __shfl_sync(0xffffffffu, src, j & 31);
                d[u] = __shfl_sync(0xffffffffu, dst, j & 31);
                if (j >= n) d[u] = -1;
                if (d[u] >= 0) x[u] = pool[static_cast<long long>(s) * lanes + l];
            }
#pragma unroll
            for (int u = 0; u < kFlight; ++u)
                if (d[u] >= 0) pool[static_cast<long long>(d[u]) * lanes + l] = x[u];
        }
    }
}

// kCtas: CTAs a head, one cluster.  1024 threads leave 64 registers each, and 68 to 76 bytes are spilled; with 512 threads
// many heads took longer (126 -> 130, 99 -> 110 us).
template <int kCtas>
__global__ void __launch_bounds__(kEvThreads) paged_evict_kernel(const PagedDev c, const EvictParams p) {
    extern __shared__ __align__(16) uint32_t keys[];
    __shared__ EvictShared sh;
    pdl_launch_dependents();
    pdl_wait();
    cg::cluster_group cluster = cg::this_cluster();
    constexpr int ctas = kCtas;
    const int rank = ctas > 1 ? static_cast<int>(cluster.block_rank()) : 0;
    auto sync_all = [&]() {
        if (ctas > 1) cluster.sync();
        else __syncthreads();
    };
    const int head = blockIdx.x / ctas, b = head / c.Hkv, h = head - b * c.Hkv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = paged_length(c, p.seq_lens, b, p.status);
    const int left = min(n, p.budget), leave = n - left;
    if (h == 0 && rank == 0 && tid == 0) p.out_lens[b] = left;
    if (leave == 0 && !p.out_table) {   // the whole cluster, nothing to do
        if (p.moves && rank == 0 && tid == 0) p.moves[head] = 0;
        return;
    }
    const long long recent_from = static_cast<long long>(p.next_positions ? p.next_positions[b] : n) - p.recent;

    // This CTA's slots, and of them this warp's; but for the last, multiples of 32 and 128 long.
    const int per_cta = ((n + ctas - 1) / ctas + 31) / 32 * 32;
    const int begin = min(n, rank * per_cta), end = min(n, begin + per_cta);
    const int per_warp = ((end - begin + kEvWarps - 1) / kEvWarps + 127) / 128 * 128;
    const int w_begin = min(end, begin + warp * per_warp), w_end = min(end, w_begin + per_warp);
    const bool cached = per_cta <= p.key_room;
    if (cached) {
        constexpr int kFlight = 8;
        int bad_page = 0;
        bool bad = false;
        for (int i0 = begin + tid; i0 < end; i0 += kFlight * kEvThreads) {
            int page[kFlight];
            int row[kFlight];
            float w[kFlight];
            int pos[kFlight];
#pragma unroll
            for (int u = 0; u < kFlight; ++u) page[u] = paged_page(c, b, min(i0 + u * kEvThreads, end - 1));
#pragma unroll
            for (int u = 0; u < kFlight; ++u) {
                row[u] = static_cast<int>(paged_row_in(c, page[u], h, min(i0 + u * kEvThreads, end - 1)));
                if (row[u] < 0) bad_page = page[u], bad = true;
            }
#pragma unroll
            for (int u = 0; u < kFlight; ++u) {
                const bool is = row[u] >= 0 && i0 + u * kEvThreads < end;
                w[u] = is ? c.weight[row[u]] : 0.f;
                pos[u] = is ? c.position[row[u]] : 0;
            }
#pragma unroll
            for (int u = 0; u < kFlight; ++u) {
                const int i = i0 + u * kEvThreads;   // a page that is not there: the first to leave
                if (i < end) keys[i - begin] = row[u] >= 0 ? evict_key(p, pos[u], w[u], recent_from) : 0u;
            }
        }
        if (bad) report_paged(p.status, kBadPage, b, bad_page);
    }
    for (int i = tid; i < 2 * kEvBins; i += kEvThreads) sh.hist[0][i] = 0;
    __syncthreads();
    auto key_of = [&](int i) {
        if (cached) return keys[i - begin];
        const long long row = paged_row(c, b, h, i, p.status);
        return row >= 0 ? evict_key(p, c.position[row], c.weight[row], recent_from) : 0u;
    };

    // T, and how many tokens with a smaller key there are.
    int32_t* from = p.from + static_cast<long long>(head) * p.list;
    int32_t* to = p.to + static_cast<long long>(head) * p.list;
    uint32_t prefix = 0, below = 0;
    bool no_ties = leave == 0;   // all tokens with the key T leave
    int total = -1;              // entries of the lists
    if (leave == 1) {   // one token too many, as at every step of serving within a budget: the smallest key, in one round
        uint2 least = make_uint2(0xffffffffu, 0xffffffffu);
        auto smaller = [](uint2 x, uint2 y) { return y.x < x.x || (y.x == x.x && y.y < x.y) ? y : x; };
        auto least_of_warp = [](uint2 x) {
            const uint32_t key = __reduce_min_sync(0xffffffffu, x.x);
            return make_uint2(key, __reduce_min_sync(0xffffffffu, x.x == key ? x.y : 0xffffffffu));
        };
        for (int i = begin + tid; i < end; i += kEvThreads) least = smaller(least, make_uint2(key_of(i), i));
        least = least_of_warp(least);
        if (lane == 0) sh.least[warp] = least;
        __syncthreads();
        least = least_of_warp(sh.least[lane]);
        if (ctas > 1) {
            if (tid == 0) sh.least_cta = least;
            cluster.sync();
#pragma unroll
            for (int r = 0; r < ctas; ++r) least = smaller(least, *cluster.map_shared_rank(&sh.least_cta, r));
            cluster.sync();
        }
        if (!p.out_table) {   // the last token takes the slot of the one that leaves, unless it is that one
            total = static_cast<int>(least.y) < left;
            if (rank == 0 && tid == 0) {   // whose warp copies it
                from[0] = left;
                to[0] = static_cast<int>(least.y);
            }
            __syncwarp();
        }
        prefix = least.x;
    } else if (leave > 1) {
        uint32_t rank_left = leave - 1;   // of the last token that leaves, among those that share the digits so far
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            constexpr int kShift[3] = {21, 10, 0}, kBits[3] = {11, 11, 10};
            const int shift = kShift[pass], bins = 1 << kBits[pass];
            uint32_t* hist = sh.hist[pass & 1];
            for (int i = begin + tid; i < end; i += kEvThreads) {
                const uint32_t k = key_of(i);
                if (pass == 0 || (k >> kShift[pass ? pass - 1 : 0]) == prefix) atomicAdd(&hist[(k >> shift) & (bins - 1)], 1u);
            }
            sync_all();
            if (pass == 1)   // for the third pass: all have read what it held
                for (int i = tid; i < kEvBins; i += kEvThreads) sh.hist[0][i] = 0;
            // Thread t: bins 2 t and 2 t + 1 (t alone in the last pass) of all CTAs.
            constexpr int kPer = kEvBins / kEvThreads;
            static_assert(kPer == 2, "a thread reads two bins at once");
            uint32_t mine[kPer] = {}, sum = 0;
            const int per = bins / kEvThreads;
#pragma unroll
            for (int r = 0; r < ctas; ++r) {
                const uint32_t* other = ctas > 1 ? cluster.map_shared_rank(hist, r) : hist;
                if (per == 2) {
                    const uint2 y = reinterpret_cast<const uint2*>(other)[tid];
                    mine[0] += y.x;
                    mine[1] += y.y;
                } else {
                    mine[0] += other[tid];
                }
            }
#pragma unroll
            for (int x = 0; x < kPer; ++x) sum += mine[x];
            uint32_t upto = sum;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, upto, s);
                if (lane >= s) upto += y;
            }
            if (lane == 31) sh.scan[warp] = upto;
            __syncthreads();
            uint32_t before = upto - sum + __reduce_add_sync(0xffffffffu, lane < warp ? sh.scan[lane] : 0u);
            if (rank_left >= before && rank_left < before + sum) {
#pragma unroll
                for (int x = 0; x < kPer; ++x) {
                    if (rank_left >= before && rank_left < before + mine[x]) {
                        sh.digit = tid * per + x;
                        sh.below = before;
                        sh.inside = mine[x];
                    }
                    before += mine[x];
                }
            }
            __syncthreads();
            prefix = (prefix << kBits[pass]) | sh.digit;
            below += sh.below;
            rank_left -= sh.below;
            if (sh.inside == rank_left + 1) {   // the whole bin leaves: its upper end will do for T
                prefix = (prefix << shift) | ((1u << shift) - 1u);
                no_ties = true;
                break;
            }
        }
    }
    if (total < 0) {
        // Of the tokens with the key T the first so many leave.
        const uint32_t T = prefix, ties_leave = no_ties ? 0xffffffffu : leave - below;

        // Sums of a pair of counts over the warps ahead of this one, in this CTA and in those before it, and over the cluster.
        static_assert(kEvWarps == 32, "a lane reads a warp's counts");
        auto place = [&](int what, uint2 count, uint2& all) {
            if (lane == 0) sh.count[what][warp] = count;
            __syncthreads();
            const uint2 x = sh.count[what][lane];
            uint2 before = make_uint2(__reduce_add_sync(0xffffffffu, lane < warp ? x.x : 0u),
                                      __reduce_add_sync(0xffffffffu, lane < warp ? x.y : 0u));
            all = make_uint2(__reduce_add_sync(0xffffffffu, x.x), __reduce_add_sync(0xffffffffu, x.y));
            if (ctas > 1) {
                if (tid == 0) sh.total[what] = all;
                cluster.sync();
                all = make_uint2(0, 0);
#pragma unroll
                for (int r = 0; r < ctas; ++r) {
                    const uint2 y = *cluster.map_shared_rank(&sh.total[what], r);
                    all.x += y.x;
                    all.y += y.y;
                    if (r < rank) {
                        before.x += y.x;
                        before.y += y.y;
                    }
                }
            }
            return before;
        };
        uint32_t ties_before = 0;
        if (!no_ties) {
            uint32_t ties = 0;
            for (int i = w_begin + lane; i < w_end; i += 32) ties += key_of(i) == T;
            ties = __reduce_add_sync(0xffffffffu, ties);
            uint2 unused;
            ties_before = place(0, make_uint2(ties, 0), unused).x;
        }
        // Calls f(i, slots to be moved, slots that come free), as bits, for a lane's four slots from i on, the warp's slots 128
        // at a time.  With an out_table every token that stays is "moved", to its place among them.
        const bool out = p.out_table != nullptr;
        auto lanes_below = [&](uint32_t x, uint32_t& all) {   // sum of x over the lanes ahead, and over all
            uint32_t upto = x;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, upto, s);
                if (lane >= s) upto += y;
            }
            all = __shfl_sync(0xffffffffu, upto, 31);
            return upto - x;
        };
        auto for_slots = [&](auto f) {
            uint32_t tie = ties_before;
            for (int base = w_begin; base < w_end; base += 128) {
                const int i = base + 4 * lane;
                uint32_t k[4] = {}, less = 0, equal = 0;
                if (cached) {
                    if (i < w_end) {   // the room for keys is a multiple of 4
                        const uint4 x = *reinterpret_cast<const uint4*>(keys + (i - begin));
                        k[0] = x.x, k[1] = x.y, k[2] = x.z, k[3] = x.w;
                    }
                } else {
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (i + j < w_end) k[j] = key_of(i + j);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    less |= (k[j] < T ? 1u : 0u) << j;
                    equal |= (k[j] == T ? 1u : 0u) << j;
                }
                const uint32_t there = (1u << max(0, min(4, w_end - i))) - 1u;
                uint32_t goes = no_ties ? less | equal : less;
                equal &= there;
                if (!no_ties && __any_sync(0xffffffffu, equal != 0)) {
                    uint32_t sum;
                    const uint32_t ahead = tie + lanes_below(__popc(equal), sum);
                    tie += sum;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        if (ahead + __popc(equal & ((1u << j) - 1u)) < ties_leave) goes |= equal & (1u << j);
                }
                goes = leave > 0 ? goes & there : 0u;
                const uint32_t before = (1u << max(0, min(4, left - i))) - 1u;   // the budget
                f(i, there & ~goes & (out ? 15u : ~before), goes & before);
            }
        };
        uint32_t n_holes = 0, n_moves = 0;
        for_slots([&](int, uint32_t moves, uint32_t holes) {
            n_moves += __popc(moves);
            n_holes += __popc(holes);
        });
        uint2 all;
        const uint2 at = place(1, make_uint2(__reduce_add_sync(0xffffffffu, n_holes), __reduce_add_sync(0xffffffffu, n_moves)), all);
        uint32_t hole = at.x, move = at.y;
        for_slots([&](int i, uint32_t moves, uint32_t holes) {
            uint32_t sum;
            const uint32_t ahead = lanes_below(__popc(moves) | __popc(holes) << 16, sum);
            int32_t* f = from + move + (ahead & 0xffffu);
            int32_t* t = to + hole + (ahead >> 16);
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                if ((moves >> j) & 1u) *f++ = i + j;
                if (!out && ((holes >> j) & 1u)) *t++ = i + j;
            }
            move += sum & 0xffffu;
            hole += sum >> 16;
        });
        sync_all();   // the lists are written, and no CTA's shared memory is read any more

        total = static_cast<int>(all.y);
    }
    if (p.moves) {
        if (rank == 0 && tid == 0) p.moves[head] = total;
        return;
    }
    if (c.k_scale) copy_rows<true>(c, p, b, h, from, to, (rank * kEvWarps + warp) * 32, total, ctas * kEvWarps * 32);
    else copy_rows<false>(c, p, b, h, from, to, (rank * kEvWarps + warp) * 32, total, ctas * kEvWarps * 32);
}

// The copies, a warp per 32 entries of a head's lists.
// Seven CTAs an SM have 72 registers a thread (20 bytes spilled); eight, of 64, spill more: 32 heads of 4096 rows 48 us instead
// of 46, 512 of 2048 247 instead of 228.
constexpr int kMoveWarps = 4;
template <bool e4m3>
__global__ void __launch_bounds__(kMoveWarps * 32, 7) paged_move_kernel(const PagedDev c, const EvictParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int head = blockIdx.y, b = head / c.Hkv, h = head - b * c.Hkv;
    const int total = p.moves[head];
    copy_rows<e4m3>(c, p, b, h, p.from + static_cast<long long>(head) * p.list, p.to + static_cast<long long>(head) * p.list,
              (blockIdx.x * kMoveWarps + (threadIdx.x >> 5)) * 32, total, gridDim.x * kMoveWarps * 32);
}

}  // namespace fba

using namespace fba;

namespace {
// Up to so many rows a head are copied by the CTA that chose them; more by a kernel of their own, whose launch costs
// less than leaving most SMs idle.
constexpr int kMoveHere = 256;
int evict_list(int page_size, int max_pages, int budget) {
    const long long cap = static_cast<long long>(max_pages) * page_size;
    return static_cast<int>(cap < budget ? cap : budget);
}
}  // namespace

extern "C" int fba_paged_evict_workspace_bytes(int B, int Hkv, int page_size, int max_pages, int budget, uint64_t* bytes) {
    if (B <= 0 || Hkv <= 0 || page_size <= 0 || max_pages <= 0 || budget <= 0 || !bytes)
        return set_error(FBA_ERR_BAD_ARG, "fba_paged_evict_workspace_bytes: bad argument");
    if (static_cast<long long>(max_pages) * page_size >= 1 << 30)
        return set_error(FBA_ERR_TOO_LARGE, "fba_paged_evict_workspace_bytes: max_pages * page_size reaches 2^30");
    *bytes = static_cast<uint64_t>(B) * Hkv * (evict_list(page_size, max_pages, budget) * 2ull + 1) * sizeof(int32_t);
    return FBA_OK;
}

extern "C" int fba_paged_evict(const fba_paged_t* cache, int B, const int32_t* seq_lens, int budget, int sinks, int recent,
                               const int32_t* next_positions, const int32_t* out_table, int out_pages, int32_t* out_lens,
                               void* workspace, uint64_t workspace_bytes, uint32_t* status, void* stream) {
    ProfRange range("fba_paged_evict");
    PagedDev c;
    int rc = paged_args("fba_paged_evict", cache, B, &c);
    if (rc != FBA_OK) return rc;
    if (!seq_lens || !out_lens || !status) return set_error(FBA_ERR_BAD_ARG, "fba_paged_evict: null pointer argument");
    if (lens_overlap(out_lens, seq_lens, B) || lens_overlap(out_lens, next_positions, B))
        return set_error(FBA_ERR_BAD_ARG, "fba_paged_evict: out_lens must not overlap seq_lens or next_positions");
    if (!c.weight) return set_error(FBA_ERR_BAD_ARG, "fba_paged_evict: the cache has no weights");
    if (budget <= 0 || sinks < 0 || recent < 0 || static_cast<long long>(sinks) + recent > budget)
        return set_error(FBA_ERR_BAD_ARG, "fba_paged_evict: budget must be positive, and sinks + recent at most budget");
    if (out_table == c.table) return set_error(FBA_ERR_BAD_ARG, "fba_paged_evict: out_table must not be the cache's table");
    const int list = evict_list(c.page_size, c.max_pages, budget);
    if (out_table && (out_pages <= 0 || static_cast<long long>(out_pages) * c.page_size < list ||
                      static_cast<long long>(out_pages) * c.page_size >= 1 << 30))
        return set_error(FBA_ERR_BAD_ARG, "fba_paged_evict: out_table has no room for the budget");
    uint64_t need = 0;
    if ((rc = fba_paged_evict_workspace_bytes(B, c.Hkv, c.page_size, c.max_pages, budget, &need)) != FBA_OK) return rc;
    if (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 4 != 0)
        return set_error(FBA_ERR_BAD_ARG,
                         "fba_paged_evict: workspace must be 4-byte aligned, of fba_paged_evict_workspace_bytes() bytes");
    const long long heads = static_cast<long long>(B) * c.Hkv;
    if (heads > 65535) return set_error(FBA_ERR_TOO_LARGE, "fba_paged_evict: B * Hkv exceeds 65535");
    EvictParams p = {};
    p.seq_lens = seq_lens;
    p.next_positions = next_positions;
    p.out_table = out_table;
    p.out_lens = out_lens;
    p.from = static_cast<int32_t*>(workspace);
    p.to = p.from + heads * list;
    p.status = status;
    p.budget = budget;
    p.sinks = sinks;
    p.recent = recent;
    p.out_pages = out_pages;
    p.list = list;
    // The keys of a CTA's slots stay in shared memory beside the histogram, with a cluster of up to 8 CTAs if need be; a
    // cluster also where there are idle SMs and long stretches to go through (32 heads of up to 32768 slots, selection and
    // copies: 80 us with one CTA a head, 64 with two, 55 with four; with the loads of step 2 in parallel 46).  All of it for
    // what the table has room for, as the host does not know the lengths: 128 heads of 2049 slots, one too many, take 5.5 us
    // in tables for 2112, 8 for 16384, 21 for 131072.
    constexpr long long kMostKeys = 200 * 1024 / 4;
    const long long cap = static_cast<long long>(c.max_pages) * c.page_size;
    int ctas = 1;
    while (ctas < 8 && cap > kMostKeys * ctas) ctas *= 2;
    while (ctas < 8 && heads * ctas * 2 <= 148 && cap / (ctas * 2) >= 2048) ctas *= 2;
    const long long room = ((cap + ctas - 1) / ctas + 31) / 32 * 32;
    p.key_room = room <= kMostKeys ? static_cast<int>(room) : 0;
    // The most rows that a head can have to copy.
    const long long most = out_table ? list : (cap - budget < list ? cap - budget : list);
    if (most > kMoveHere) p.moves = p.to + heads * list;

    DeviceGuard guard;
    if ((rc = guard.bind(cache->k)) != FBA_OK) return rc;
    auto kernel = ctas == 1   ? paged_evict_kernel<1>
                  : ctas == 2 ? paged_evict_kernel<2>
                  : ctas == 4 ? paged_evict_kernel<4>
                              : paged_evict_kernel<8>;
    if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess) {
        cudaGetLastError();
        return set_error(FBA_ERR_LAUNCH, "fba_paged_evict: cannot raise the dynamic shared memory limit");
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(heads * ctas));
    config.blockDim = dim3(kEvThreads);
    config.dynamicSmemBytes = static_cast<size_t>(p.key_room) * 4;
    config.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attr;
    config.numAttrs = 2;
    cudaLaunchKernelEx(&config, kernel, c, p);
    if ((rc = check_launch("paged_evict_kernel")) != FBA_OK || !p.moves) return rc;
    // Blocks for all of a head's entries while the grid stays within 10 waves; a warp takes further batches beyond.  With 2.3
    // waves as the limit 320 heads of 2000 rows took 106 us instead of 97, 512 of 2048 228 instead of 216.
    long long blocks = (most + kMoveWarps * 32 - 1) / (kMoveWarps * 32);
    const long long enough = (148 * 64 + heads - 1) / heads;
    const dim3 grid(static_cast<unsigned>(blocks < enough ? blocks : enough), static_cast<unsigned>(heads));
    return launch_chained(cache->e4m3 ? paged_move_kernel<true> : paged_move_kernel<false>, grid, kMoveWarps * 32, 0,
                          static_cast<cudaStream_t>(stream), c, p);
}
