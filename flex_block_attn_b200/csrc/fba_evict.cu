// Eviction from a paged cache by accumulated attention weight.
//
// Per (sequence, kv head) of n slots the n - budget tokens that come first in the order (protected, weight, slot) leave.
// One cluster of CTAs per (sequence, kv head), each CTA with a contiguous stretch of the slots:
//   1. weights become 32-bit keys in their order (in shared memory where they fit), protected tokens the largest key;
//   2. the key T of the last token that leaves is found from its digits, 11 + 11 + 10 bits from the top: a histogram of a
//      digit per CTA, all of them added up by every CTA through distributed shared memory;
//   3. counts per warp (tokens with the key T; slots that come free; tokens to be moved), exchanged the same way, give
//      every warp the place of its entries in the lists of slots to move from and to, which are in slot order
//      therefore, whatever the timing;
//   4. all CTAs of the cluster divide the list and copy the rows.
// In place, the i-th staying token behind slot `budget` goes to the i-th slot that came free before it: only as many rows move as
// tokens leave from there, and no row is both read and written.
// What bounds it: the rows copied (and, with few rows, the latency of the steps before).
#include <math.h>
#include <stdio.h>

#include <cooperative_groups.h>

#include "fba_paged.cuh"

namespace fba {

namespace cg = cooperative_groups;

constexpr int kEvThreads = 512;
constexpr int kEvWarps = kEvThreads / 32;
constexpr int kEvBins = 2048;

struct EvictParams {
    const int32_t *seq_lens, *next_positions, *out_table;
    int32_t* out_lens;
    int32_t *from, *to;      // [B * Hkv, list]: slots; `to` is not used with an out_table
    uint32_t* status;
    int budget, sinks, recent, out_pages, list;
    int key_room;            // keys a CTA holds in shared memory; 0: read again on every use
};

struct EvictShared {
    uint32_t hist[kEvBins];
    uint32_t scan[kEvWarps];
    uint32_t count[3][kEvWarps];   // per warp: ties, holes, movers
    uint32_t total[3];             // of the CTA
    uint32_t digit, below;         // of the bin that holds the wanted rank: its number, and how many keys lie before it
};

__device__ __forceinline__ uint32_t evict_key(const PagedDev& c, const EvictParams& p, int b, int h, int slot, long long recent_from) {
    const long long row = paged_row(c, b, h, slot, p.status);
    if (row < 0) return 0u;   // a page that is not there: the first to leave
    const int pos = c.position[row];
    if (pos < p.sinks || pos >= recent_from) return 0xffffffffu;
    const float w = c.weight[row] + 0.f;   // -0 counts as 0
    if (isnan(w)) return 0xfffffffeu;      // above infinity
    const uint32_t u = __float_as_uint(w);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}

__global__ void __launch_bounds__(kEvThreads) paged_evict_kernel(const PagedDev c, const EvictParams p) {
    extern __shared__ uint32_t keys[];
    __shared__ EvictShared sh;
    cg::cluster_group cluster = cg::this_cluster();
    const int ctas = static_cast<int>(cluster.num_blocks()), rank = static_cast<int>(cluster.block_rank());
    const int head = blockIdx.x / ctas, b = head / c.Hkv, h = head - b * c.Hkv;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int n = paged_length(c, p.seq_lens, b, p.status);
    const int left = min(n, p.budget), leave = n - left;
    if (h == 0 && rank == 0 && tid == 0) p.out_lens[b] = left;
    if (leave == 0 && !p.out_table) return;   // the whole cluster, nothing to do
    const long long recent_from = static_cast<long long>(p.next_positions ? p.next_positions[b] : n) - p.recent;

    // This CTA's slots, and of them this warp's; both multiples of 32 long.
    const int per_cta = ((n + ctas - 1) / ctas + 31) / 32 * 32;
    const int begin = min(n, rank * per_cta), end = min(n, begin + per_cta);
    const int per_warp = ((end - begin + kEvWarps - 1) / kEvWarps + 31) / 32 * 32;
    const int w_begin = min(end, begin + warp * per_warp), w_end = min(end, w_begin + per_warp);
    const bool cached = per_cta <= p.key_room;
    if (cached)
        for (int i = begin + tid; i < end; i += kEvThreads) keys[i - begin] = evict_key(c, p, b, h, i, recent_from);
    __syncthreads();
    auto key_of = [&](int i) { return cached ? keys[i - begin] : evict_key(c, p, b, h, i, recent_from); };

    // T, and how many tokens with a smaller key there are.
    uint32_t prefix = 0, below = 0;
    if (leave > 0) {
        uint32_t rank_left = leave - 1;   // of the last token that leaves, among those that share the digits so far
#pragma unroll
        for (int pass = 0; pass < 3; ++pass) {
            constexpr int kShift[3] = {21, 10, 0}, kBits[3] = {11, 11, 10};
            const int shift = kShift[pass], bins = 1 << kBits[pass];
            for (int i = tid; i < bins; i += kEvThreads) sh.hist[i] = 0;
            __syncthreads();
            for (int i = begin + tid; i < end; i += kEvThreads) {
                const uint32_t k = key_of(i);
                if (pass == 0 || (k >> kShift[pass ? pass - 1 : 0]) == prefix) atomicAdd(&sh.hist[(k >> shift) & (bins - 1)], 1u);
            }
            cluster.sync();
            // Thread t: bins 4 t .. 4 t + 3 (2 t and 2 t + 1 in the last pass) of all CTAs.
            uint32_t mine[4] = {0, 0, 0, 0}, sum = 0;
            const int per = bins / kEvThreads;
            for (int r = 0; r < ctas; ++r) {
                const uint32_t* other = cluster.map_shared_rank(sh.hist, r);
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    if (x < per) mine[x] += other[tid * per + x];
            }
#pragma unroll
            for (int x = 0; x < 4; ++x) sum += mine[x];
            uint32_t upto = sum;
#pragma unroll
            for (int s = 1; s < 32; s <<= 1) {
                const uint32_t y = __shfl_up_sync(0xffffffffu, upto, s);
                if (lane >= s) upto += y;
            }
            if (lane == 31) sh.scan[warp] = upto;
            __syncthreads();
            uint32_t before = upto - sum;
            for (int w = 0; w < warp; ++w) before += sh.scan[w];
            if (rank_left >= before && rank_left < before + sum) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    if (rank_left >= before && rank_left < before + mine[x]) {
                        sh.digit = tid * per + x;
                        sh.below = before;
                    }
                    before += mine[x];
                }
            }
            cluster.sync();   // all have read the histograms, and `digit` is there
            prefix = (prefix << kBits[pass]) | sh.digit;
            below += sh.below;
            rank_left -= sh.below;
        }
    }
    const uint32_t T = prefix, ties_leave = leave - below;   // of the tokens with key T the first so many leave

    // Sums over the warps ahead of this one, in this CTA and in those before it, and over the cluster.
    auto place = [&](int what, uint32_t count, uint32_t& all) {
        if (lane == 0) sh.count[what][warp] = count;
        __syncthreads();
        if (tid == 0) {
            uint32_t t = 0;
            for (int w = 0; w < kEvWarps; ++w) t += sh.count[what][w];
            sh.total[what] = t;
        }
        cluster.sync();
        uint32_t before = 0;
        all = 0;
        for (int r = 0; r < ctas; ++r) {
            const uint32_t t = *cluster.map_shared_rank(&sh.total[what], r);
            all += t;
            if (r < rank) before += t;
        }
        for (int w = 0; w < warp; ++w) before += sh.count[what][w];
        return before;
    };
    uint32_t ties = 0, unused;
    for (int i = w_begin + lane; i < w_end; i += 32) ties += key_of(i) == T;
    ties = __reduce_add_sync(0xffffffffu, ties);
    const uint32_t ties_before = place(0, ties, unused);
    // Calls f(slot, stays) for the warp's slots, a full warp at a time.
    auto for_slots = [&](auto f) {
        uint32_t tie = ties_before;
        for (int base = w_begin; base < w_end; base += 32) {
            const int i = base + lane;
            const uint32_t k = i < w_end ? key_of(i) : 0u;
            const uint32_t eq = __ballot_sync(0xffffffffu, i < w_end && k == T);
            const bool goes = leave > 0 && (k < T || (k == T && tie + __popc(eq & ((1u << lane) - 1u)) < ties_leave));
            tie += __popc(eq);
            f(i, i < w_end && !goes, i < w_end && goes);
        }
    };
    // With an out_table every token that stays is "moved", to its place among them.
    const bool out = p.out_table != nullptr;
    uint32_t n_holes = 0, n_moves = 0;
    for_slots([&](int i, bool stays, bool goes) {
        n_moves += __popc(__ballot_sync(0xffffffffu, stays && (out || i >= left)));
        n_holes += __popc(__ballot_sync(0xffffffffu, goes && i < left));
    });
    uint32_t all_moves, all_holes;
    uint32_t move = place(2, n_moves, all_moves), hole = place(1, n_holes, all_holes);
    int32_t* from = p.from + static_cast<long long>(head) * p.list;
    int32_t* to = p.to + static_cast<long long>(head) * p.list;
    for_slots([&](int i, bool stays, bool goes) {
        const uint32_t mv = __ballot_sync(0xffffffffu, stays && (out || i >= left));
        const uint32_t hl = __ballot_sync(0xffffffffu, goes && i < left);
        const uint32_t ahead = (1u << lane) - 1u;
        if ((mv >> lane) & 1u) from[move + __popc(mv & ahead)] = i;
        if (!out && ((hl >> lane) & 1u)) to[hole + __popc(hl & ahead)] = i;
        move += __popc(mv);
        hole += __popc(hl);
    });
    cluster.sync();   // the lists are written, and no CTA's shared memory is read any more

    // Rows: half a warp each for K and V in bf16 (16 bytes a lane), a quarter each in e4m3, then two tokens at a time.
    const bool e4m3 = c.k_scale != nullptr;
    const int lanes = e4m3 ? 8 : 16, tokens = 16 / lanes;     // a warp's tokens at a time
    const int sub = lane / (2 * lanes), kv = lane / lanes & 1, l = lane % lanes;
    PagedDev dst_c = c;
    if (out) {
        dst_c.table = p.out_table;
        dst_c.max_pages = p.out_pages;
    }
    uint8_t* pool = kv ? c.v : c.k;
    const int total = static_cast<int>(all_moves);
    const int step = ctas * kEvWarps * tokens;
    constexpr int kFlight = 4;   // rows a lane has under way
    for (int i0 = (rank * kEvWarps + warp) * tokens + sub; i0 < total; i0 += step * kFlight) {
        long long dst[kFlight];
        uint4 x[kFlight];
        float f[kFlight];
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
            const int i = i0 + u * step;
            dst[u] = -1;
            if (i >= total) continue;
            const long long src = paged_row(c, b, h, from[i], p.status);
            dst[u] = paged_row(dst_c, b, h, out ? i : to[i], p.status);
            if (src < 0) dst[u] = -1;
            if (dst[u] < 0) continue;
            x[u] = reinterpret_cast<const uint4*>(pool)[src * lanes + l];
            // lane 0: the row's scale, lane 1: weight (by K's lanes) or position (by V's)
            if (l == 0 && e4m3) f[u] = (kv ? c.v_scale : c.k_scale)[src];
            if (l == 1) f[u] = kv ? __int_as_float(c.position[src]) : c.weight[src];
        }
#pragma unroll
        for (int u = 0; u < kFlight; ++u) {
            if (dst[u] < 0) continue;
            reinterpret_cast<uint4*>(pool)[dst[u] * lanes + l] = x[u];
            if (l == 0 && e4m3) (kv ? c.v_scale : c.k_scale)[dst[u]] = f[u];
            if (l == 1) {
                if (kv) c.position[dst[u]] = __float_as_int(f[u]);
                else c.weight[dst[u]] = f[u];
            }
        }
    }
}

}  // namespace fba

using namespace fba;

namespace {
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
    *bytes = static_cast<uint64_t>(B) * Hkv * evict_list(page_size, max_pages, budget) * 2 * sizeof(int32_t);
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
    if (out_lens == seq_lens) return set_error(FBA_ERR_BAD_ARG, "fba_paged_evict: out_lens must not be seq_lens");
    if (!c.weight) return set_error(FBA_ERR_BAD_ARG, "fba_paged_evict: the cache has no weights");
    if (budget <= 0 || sinks < 0 || recent < 0 || static_cast<long long>(sinks) + recent > budget)
        return set_error(FBA_ERR_BAD_ARG, "fba_paged_evict: budget must be positive, and sinks + recent at most budget");
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
    if (heads > 1 << 24) return set_error(FBA_ERR_TOO_LARGE, "fba_paged_evict: more than 2^24 heads of sequences");
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
    // A cluster grows while there are idle SMs and a CTA would have more than 2048 slots.
    const long long cap = static_cast<long long>(c.max_pages) * c.page_size;
    int ctas = 1;
    while (ctas < 8 && heads * ctas < 148 && cap / ctas > 2048) ctas *= 2;
    // The keys of a CTA's slots in shared memory where they fit beside the histogram.
    const long long room = ((cap + ctas - 1) / ctas + 31) / 32 * 32;
    p.key_room = room * 4 <= 200 * 1024 ? static_cast<int>(room) : 0;

    DeviceGuard guard;
    if ((rc = guard.bind(cache->k)) != FBA_OK) return rc;
    if (cudaFuncSetAttribute(paged_evict_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 200 * 1024) != cudaSuccess) {
        cudaGetLastError();
        return set_error(FBA_ERR_LAUNCH, "fba_paged_evict: cannot raise the dynamic shared memory limit");
    }
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(static_cast<unsigned>(heads * ctas));
    config.blockDim = dim3(kEvThreads);
    config.dynamicSmemBytes = static_cast<size_t>(p.key_room) * 4;
    config.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = ctas;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    if (cudaLaunchKernelEx(&config, paged_evict_kernel, c, p) != cudaSuccess) return check_launch("paged_evict_kernel");
    return check_launch("paged_evict_kernel");
}
