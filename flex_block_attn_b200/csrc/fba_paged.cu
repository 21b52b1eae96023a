// Paged key / value cache: the writer of new tokens and the attention of one new token per sequence.
#include <math.h>
#include <stdio.h>

#include "fba_paged.cuh"

namespace fba {

// ------------------------------------------------------------------------------------------ writer
struct AppendParams {
    const __nv_bfloat16 *k, *v;
    long long ks[3], vs[3];   // strides of batch, head and token, in elements
    const int32_t *seq_lens, *new_lens, *positions;
    int32_t* out_lens;
    uint32_t* status;
    int T;
};

__device__ __forceinline__ uint32_t max_nan_bf16x2(uint32_t a, uint32_t b) {   // per half; NaN if either is
    uint32_t d;
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(d) : "r"(a), "r"(b));
    return d;
}
// 16 values of a row of 128 in e4m3, where 8 neighbouring lanes hold the row; the scale by the way.
__device__ __forceinline__ uint4 quantise16(const uint4 (&x)[2], uint32_t lanes, float& scale) {
    const uint32_t* w = reinterpret_cast<const uint32_t*>(x);
    uint32_t m2 = w[0] & 0x7fff7fffu;
#pragma unroll
    for (int j = 1; j < 8; ++j) m2 = max_nan_bf16x2(m2, w[j] & 0x7fff7fffu);
#pragma unroll
    for (int s = 4; s > 0; s >>= 1) m2 = max_nan_bf16x2(m2, __shfl_xor_sync(lanes, m2, s));
    m2 = max_nan_bf16x2(m2, __byte_perm(m2, m2, 0x1032));
    const float m = __uint_as_float(m2 << 16);   // exact: one of the values
    // The floor keeps 1 / scale finite; a row with a NaN or an infinity gets a NaN.
    scale = m > 0.f ? fmaxf(m * (1.f / 448.f), 1.17549435e-38f) : 1.f;
    if (!(m < INFINITY)) scale = NAN;
    const float inv = 1.f / scale;
    uint32_t y[4];
#pragma unroll
    for (int j = 0; j < 4; ++j)
        y[j] = pack_e4m3x4(__uint_as_float(w[2 * j] << 16) * inv, __uint_as_float(w[2 * j] & 0xffff0000u) * inv,
                           __uint_as_float(w[2 * j + 1] << 16) * inv, __uint_as_float(w[2 * j + 1] & 0xffff0000u) * inv);
    return make_uint4(y[0], y[1], y[2], y[3]);
}

// Eight lanes per (token, kv head), 32 bytes each of the row of K and of the row of V; four tokens a warp at a time.  Bound by
// the rows read and written: what e4m3 computes (a row's maximum on packed bf16, 3 exchanges between lanes) is kept small
// enough for that.  4 x 8192 tokens of 8 heads to e4m3, 203 MB: 41 us; with 16 lanes a row 49; with two rows a lane in flight
// no faster, with four 63 (fewer warps).
template <bool kE4m3>
__global__ void __launch_bounds__(256) paged_append_kernel(const PagedDev c, const AppendParams p) {
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.y;
    const int lane = threadIdx.x & 31, l8 = lane & 7;
    const int start = paged_length(c, p.seq_lens, b, p.status);
    const int room = c.max_pages * c.page_size - start;
    int n = p.new_lens ? p.new_lens[b] : p.T;
    if (n < 0 || n > p.T || n > room) {
        if (threadIdx.x == 0 && blockIdx.x == 0) report_paged(p.status, kBadLength, b, n);
        n = max(0, min(min(n, p.T), room));
    }
    if (start != p.seq_lens[b]) n = 0;   // a length that is none: nothing is written anywhere
    if (p.out_lens && blockIdx.x == 0 && threadIdx.x == 0) p.out_lens[b] = start + n;
    const int pos0 = p.positions ? p.positions[b] : start;
    const int rows = n * c.Hkv;
    for (int r = (blockIdx.x * 256 + threadIdx.x) >> 3; r < rows; r += gridDim.x * 32) {
        const int tok = r / c.Hkv, h = r - tok * c.Hkv;
        const long long dst = paged_row(c, b, h, start + tok, p.status);
        const uint4* src[2] = {reinterpret_cast<const uint4*>(p.k + b * p.ks[0] + h * p.ks[1] + tok * p.ks[2]),
                               reinterpret_cast<const uint4*>(p.v + b * p.vs[0] + h * p.vs[1] + tok * p.vs[2])};
        uint4 x[2][2];
#pragma unroll
        for (int kv = 0; kv < 2; ++kv)
#pragma unroll
            for (int z = 0; z < 2; ++z)   // e4m3: a lane's 16 values are neighbours, so that it stores 16 bytes
                x[kv][z] = src[kv][kE4m3 ? 2 * l8 + z : l8 + 8 * z];
        if (dst < 0) continue;
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            uint4* pool = reinterpret_cast<uint4*>(kv ? c.v : c.k);
            if (kE4m3) {
                float scale;   // the lanes of other rows need not be here
                const uint4 y = quantise16(x[kv], 0xffu << (lane & 24), scale);
                pool[dst * 8 + l8] = y;
                if (l8 == 0) (kv ? c.v_scale : c.k_scale)[dst] = scale;
            } else {
                pool[dst * 16 + l8] = x[kv][0];
                pool[dst * 16 + l8 + 8] = x[kv][1];
            }
        }
        if (c.weight && l8 == 0) {
            c.weight[dst] = 0.f;
            c.position[dst] = pos0 + tok;
        }
    }
}

// ------------------------------------------------------------------------------------------ decode
//
// The rows of a (sequence, kv head) are taken 16 at a time ("tiles", which never straddle a page).  They are cut up in one of
// two ways (decode_plan has the rule), for every "row": sequence, kv head, group of at most 8 * NT of its query heads.
//   Many rows: each is cut into the same number of equal parts, one or more, with a CTA for each.
//   Few rows: all tiles of all rows form one list, which is cut into equal pieces, one per CTA; a piece may cover parts of
//   several rows, and a row may be cut over several pieces.
// The partial results of a row (running maximum, sum, unnormalised output) are joined by a second kernel.
//
// In a CTA the four warps take the tiles in turn, each with a ring of its own in shared memory that cp.async fills several
// tiles ahead, across the seams between rows; rows that the query does not see are filled with zeros instead of being
// read.  With so few queries the time goes into reading K and V (per tile 8 KB in bf16, for 2 x 16 x 128 x 8
// multiply-adds per 8 query heads), so the products run on the warp-level tensor instructions, keys as the 16 rows of
// a tile and query heads as its 8 columns:
//     S^T[16 keys x 8 heads] = K q^T,   O^T[128 x 8 heads] += V^T P^T,
// with K and V^T through ldmatrix from a swizzled ring and P^T turned in registers (movmatrix).  The running maximum is
// raised, and O^T rescaled, only when a score exceeds it by 2^8.  P is rounded to bf16 for its product like the prompt
// kernels' P; sums and statistics are fp32.
// e4m3: bytes become fp16 exactly, one conversion a pair, and the products run in fp16.  q goes to fp16 with a power of two per
// head that brings its largest element to 2^14 .. 2^15: bf16's 8 bits stay exact down to 2^-31 of that element.  A row's K
// scale multiplies its scores.  Its V scale multiplies its probabilities, relative to a power of two that is at least the
// largest V scale the warp has met (O^T is rescaled when a larger one comes) and times 2^7, so that they use fp16's range:
// below 2^15, 11 bits down to 2^-21 of the largest weight, absolute error 2^-32 of it beyond, where bf16 would keep 8
// bits.  (Bytes to bf16 by shifts and a multiplication by 2^120 took 288 of some 420 instructions a tile.)
constexpr int kDecThreads = 128;
constexpr int kTileKeys = 16;
constexpr int kDecMinTiles = 16;      // tiles a CTA gets at least: 256 keys, four tiles a warp
constexpr int kOStride = 132;         // floats between the heads of the exchange buffer (bank offset 4 a head)

template <bool kE4m3>
struct DecShape {
    static constexpr int kRow = kE4m3 ? 128 : 256;                                     // bytes
    static constexpr int kStage = 2 * kTileKeys * kRow + (kE4m3 ? 2 * kTileKeys * 4 : 0);   // K, V, scales
    static constexpr int kStages = 3;
    static constexpr int kCtas = kE4m3 ? 3 : 2;                                        // resident on an SM
    static constexpr int kRing = 4 * kStages * kStage;
    static constexpr int kSmem = kRing + 4 * 8 * kOStride * 4 + 4 * 8 * 2 * 4 + 4 * 8 * 4;
};
static_assert(DecShape<false>::kCtas * (DecShape<false>::kSmem + 1024) <= 233472 &&
              DecShape<true>::kCtas * (DecShape<true>::kSmem + 1024) <= 233472, "the CTAs must fit into an SM's shared memory");

struct DecodeParams {
    const __nv_bfloat16* q;
    long long qs[2];
    __nv_bfloat16* o;
    float* lse;
    const int32_t* seq_lens;
    uint32_t* status;
    float* part_o;       // [slot][8 NT][128]
    float* part_ml;      // [slot][8 NT][2]
    float* scores;       // accumulate: [B, Hq, score_stride] in units of log2, else null
    int score_stride;
    int B, Hq, group, q_tiles;      // query heads a kv head; groups of 8 NT of them
    int window, sinks;              // window 0: none; sinks: at most a row's slots (host-clamped: they are rounded up to tiles)
    int splits;                     // CTAs per row, each with an equal part of the row's own tiles; 0: the list of all tiles
    int n_ctas;                     //   is cut into this many pieces
    float scale_log2;
};

// A sequence's tiles: the first `sink_tiles`, then those from `first` on; nt in all.
struct SeqTiles {
    int n, sink_tiles, first, nt, lo;   // slots j < n with j < sinks or j >= lo are visible
};
__device__ __forceinline__ SeqTiles seq_tiles(int n, int window, int sinks) {
    SeqTiles s;
    s.n = n;
    s.lo = window > 0 && window < n ? n - window : 0;
    s.first = s.lo / kTileKeys;
    s.sink_tiles = min(s.first, (sinks + kTileKeys - 1) / kTileKeys);
    s.nt = s.sink_tiles + (n + kTileKeys - 1) / kTileKeys - s.first;
    return s;
}

// Tiles a CTA takes.
__device__ __forceinline__ long long list_piece(long long total, int n_ctas) {
    const long long per = (total + n_ctas - 1) / n_ctas;
    return per < kDecMinTiles ? kDecMinTiles : per;
}

// Where a CTA's piece of the list [sequence][head row][tile] begins.  Every lane of the warp takes part and gets the
// answers.
struct ListPlace {
    int b, length;       // the sequence, and its length in slots
    long long in;        // tiles of the sequence's head rows ahead of the piece
    long long count;     // tiles of the piece; 0: there is none
};
__device__ __forceinline__ ListPlace list_place(const PagedDev& c, const DecodeParams& p, int cta, int rows) {
    const int lane = threadIdx.x & 31;
    auto load = [&](int base, int& n) {   // tiles of one head row of the lane's sequence
        n = base + lane < p.B ? paged_length(c, p.seq_lens, base + lane, p.status) : 0;
        return base + lane < p.B ? seq_tiles(n, p.window, p.sinks).nt : 0;
    };
    int n0, all = 0;
    const int nt0 = load(0, n0);   // kept: with up to 32 sequences nothing is loaded twice
    for (int base = 32; base < p.B; base += 32) {
        int n;
        all += load(base, n);
    }
    all = __reduce_add_sync(0xffffffffu, all + nt0);
    const long long total = static_cast<long long>(all) * rows, per = list_piece(total, p.n_ctas), at = per * cta;
    ListPlace r = {0, 0, 0, 0};
    if (at >= total) return r;
    r.count = min(per, total - at);
    int before = 0;
    for (int base = 0; base < p.B; base += 32) {
        int n = n0, nt = nt0;
        if (base > 0) nt = load(base, n);
        int upto = nt;
#pragma unroll
        for (int s = 1; s < 32; s <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, upto, s);
            if (lane >= s) upto += x;
        }
        // the first sequence with tiles whose end lies behind `at`
        const uint32_t hit = __ballot_sync(0xffffffffu, nt > 0 && static_cast<long long>(before + upto) * rows > at);
        if (hit) {
            const int first = __ffs(hit) - 1;
            r.b = base + first;
            r.length = __shfl_sync(0xffffffffu, n, first);
            r.in = at - static_cast<long long>(before + __shfl_sync(0xffffffffu, upto - nt, first)) * rows;
            return r;
        }
        before += __shfl_sync(0xffffffffu, upto, 31);
    }
    r.count = 0;   // not reached: the last tile lies behind `at`
    return r;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
__device__ __forceinline__ void ldmatrix_x4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr) : "memory");
}
// 8 x 8 matrix of 16-bit elements, turned.
__device__ __forceinline__ uint32_t movmatrix(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// D[16 x 8] += A[16 x 16] B[16 x 8], bf16.
__device__ __forceinline__ void mma_16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The same in fp16.
__device__ __forceinline__ void mma_16816_f16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Four e4m3 bytes -> two fp16 pairs, exactly: (bytes 0, 1) and (bytes 2, 3).
__device__ __forceinline__ void e4m3_to_f16(uint32_t r, uint32_t& lo, uint32_t& hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\t"
        "cvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}" : "=r"(lo), "=r"(hi) : "r"(r));
}
__device__ __forceinline__ uint32_t pack_f16x2(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}
// 2^e for e in -126 .. 127.
__device__ __forceinline__ float pow2(int e) { return __int_as_float((e + 127) << 23); }
// Exponent of a positive finite number, rounded down (-127 for subnormals and 0).
__device__ __forceinline__ int exponent(float x) { return (__float_as_int(x) >> 23) - 127; }

// Weight of a part with maximum m; where no part has a finite score, the sums (0, or NaN) stand as they are.
__device__ __forceinline__ float part_scale(float m, float top) { return top == -INFINITY ? 1.f : ex2_approx(m - top); }

template <bool kE4m3, int NT>
__global__ void __launch_bounds__(kDecThreads, NT == 1 ? DecShape<kE4m3>::kCtas : 2) paged_decode_kernel(const PagedDev c, const DecodeParams p) {
    using Sh = DecShape<kE4m3>;
    extern __shared__ __align__(128) uint8_t smem[];
    pdl_wait();
    pdl_launch_dependents();   // in this order: the kernel behind reads lengths and tables ahead of its own wait
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int g = lane >> 2, t4 = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * Sh::kStages * Sh::kStage;
    float* ex_o = reinterpret_cast<float*>(smem + Sh::kRing);            // [warp][8][kOStride]
    float* ex_ml = ex_o + 4 * 8 * kOStride;                              // [warp][8][2]
    uint32_t* ring_vis = reinterpret_cast<uint32_t*>(ex_ml + 4 * 8 * 2) + warp * 8;   // [stage]: visible rows
    const int rows_per_seq = c.Hkv * p.q_tiles;

    // This CTA's piece: `left` tiles from tile `at` of row (b, hr) on.
    struct Cursor {
        int b, hr;           // sequence, head row (kv head * q_tiles + group)
        int i, end;          // next tile of this warp in the row, and where the CTA's part of the row ends
        long long left;      // tiles of the piece behind this row's part
        SeqTiles s;
    };
    Cursor first;
    if (p.splits > 0) {
        const int row = blockIdx.x / p.splits, part = blockIdx.x - row * p.splits;
        first.b = row / rows_per_seq;
        first.hr = row - first.b * rows_per_seq;
        first.s = seq_tiles(paged_length(c, p.seq_lens, first.b, p.status), p.window, p.sinks);
        const int per = static_cast<int>(list_piece(first.s.nt, p.splits));
        first.i = part * per;
        if (part > 0 && first.i >= first.s.nt) return;   // (part 0 of a row without a tile writes its zeros)
        first.end = min(first.s.nt, first.i + per);
        first.left = 0;
    } else {
        const ListPlace place = list_place(c, p, blockIdx.x, rows_per_seq);
        if (place.count == 0) return;
        first.b = place.b;
        first.s = seq_tiles(place.length, p.window, p.sinks);
        first.hr = static_cast<int>(place.in / first.s.nt);
        first.i = static_cast<int>(place.in - static_cast<long long>(first.hr) * first.s.nt);
        first.end = static_cast<int>(min(static_cast<long long>(first.s.nt), first.i + place.count));
        first.left = place.count - (first.end - first.i);
    }
    // The next row's part of the piece; the caller has checked that tiles are left.
    auto next_row = [&](Cursor& r) {
        if (++r.hr == rows_per_seq) {
            r.hr = 0;
            do {   // sequences without a tile have no part in the list; one with tiles follows, as tiles are left
                if (r.b + 1 >= p.B) {   // unless someone changes the lengths meanwhile
                    r.i = r.end = 0;
                    r.left = 0;
                    return;
                }
                ++r.b;
                r.s = seq_tiles(paged_length(c, p.seq_lens, r.b, p.status), p.window, p.sinks);
            } while (r.s.nt == 0);
        }
        r.i = 0;
        r.end = static_cast<int>(min(static_cast<long long>(r.s.nt), r.left));
        r.left -= r.end;
    };
    auto tile_slot = [&](const SeqTiles& s, int i) { return (i < s.sink_tiles ? i : s.first + i - s.sink_tiles) * kTileKeys; };
    // Which of the 16 slots from j0 on are visible.
    auto visible = [&](const SeqTiles& s, int j0) {
        uint32_t m = j0 + 16 <= s.n ? 0xffffu : (1u << (s.n - j0)) - 1u;
        if (j0 < s.lo) {
            const int sk = p.sinks - j0, lo = s.lo - j0;
            m &= (sk <= 0 ? 0u : sk >= 16 ? 0xffffu : (1u << sk) - 1u) | (lo >= 16 ? 0u : ~((1u << lo) - 1u));
        }
        return m;
    };

    // ---- loader: this warp's tiles, Sh::kStages - 1 ahead of the products
    Cursor ld = first;
    ld.i += warp;
    int ld_pages = 0, ld_k = 32;       // page numbers of this warp's next tiles of the row, one per lane
    bool ld_done = false;
    auto load_next = [&](int stage) {
        while (!ld_done && ld.i >= ld.end) {
            if (ld.left == 0) {
                ld_done = true;
                break;
            }
            next_row(ld);
            ld.i += warp;
            ld_k = 32;
        }
        if (!ld_done) {
            if (ld_k == 32) {   // the page numbers of the warp's next 32 tiles, a lane each
                const int i = ld.i + 4 * lane;
                ld_pages = i < ld.end ? c.table[static_cast<long long>(ld.b) * c.max_pages + (tile_slot(ld.s, i) >> c.page_shift)] : 0;
                if (static_cast<uint32_t>(ld_pages) >= static_cast<uint32_t>(c.n_pages)) {
                    report_paged(p.status, kBadPage, ld.b, ld_pages);
                    ld_pages = -1;
                }
                ld_k = 0;
            }
            const int page = __shfl_sync(0xffffffffu, ld_pages, ld_k);
            ++ld_k;
            const int j0 = tile_slot(ld.s, ld.i);
            const uint32_t vis = page < 0 ? 0u : visible(ld.s, j0);
            if (lane == 0) ring_vis[stage] = vis;   // read behind the barrier that follows the stage's wait
            const int h = ld.hr / p.q_tiles;
            const long long row = (static_cast<long long>(max(page, 0)) * c.Hkv + h) * c.page_size + (j0 & (c.page_size - 1));
            const uint32_t dst = ring + stage * Sh::kStage;
            constexpr int kLanes = Sh::kRow / 16;                     // lanes a row
            const int r0 = lane / kLanes, ch = lane % kLanes;
#pragma unroll
            for (int z = 0; z < 2; ++z) {
                const uint8_t* src = (z ? c.v : c.k) + row * Sh::kRow + r0 * Sh::kRow + ch * 16;
#pragma unroll
                for (int it = 0; it < kTileKeys * kLanes / 32; ++it) {
                    const int r = r0 + it * (32 / kLanes);
                    cp_async16(dst + z * kTileKeys * Sh::kRow + r * Sh::kRow + ((ch ^ (r & 7)) << 4),
                               src + it * (32 / kLanes) * Sh::kRow, (vis >> r) & 1u);
                }
            }
            if (kE4m3 && lane < 8) {
                const float* src = (lane < 4 ? c.k_scale : c.v_scale) + row + (lane & 3) * 4;
                cp_async16(dst + 2 * kTileKeys * Sh::kRow + lane * 16, src, page >= 0);
            }
            ld.i += 4;
        }
        cp_async_commit();   // an empty group where nothing is left, so that the count of groups stays the stages'
    };
#pragma unroll
    for (int s = 0; s < Sh::kStages - 1; ++s) load_next(s);

    // ---- products
    Cursor cur = first;
    int stage = 0;
    while (true) {
        const int h = cur.hr / p.q_tiles, q0 = h * p.group + (cur.hr - h * p.q_tiles) * 8 * NT;   // first query head
        const int heads = min(8 * NT, (h + 1) * p.group - q0);
        // q as the right operand: of k-step ks thread (g, t4) holds head g, two dims and two more; with e4m3 the dims follow
        // the order of a row's bytes: 4 t4 .. 4 t4 + 3.
        uint32_t qf[NT][16];
        float q_mul[NT];   // e4m3: what undoes the power of two of head g
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const bool real = 8 * nt + g < heads;
            const uint32_t* src = reinterpret_cast<const uint32_t*>(p.q + cur.b * p.qs[0] + (q0 + (real ? 8 * nt + g : 0)) * p.qs[1]);
#pragma unroll
            for (int ks = 0; ks < 8; ++ks) {
                qf[nt][2 * ks] = real ? src[ks * 8 + (kE4m3 ? 2 * t4 : t4)] : 0u;
                qf[nt][2 * ks + 1] = real ? src[ks * 8 + (kE4m3 ? 2 * t4 + 1 : t4 + 4)] : 0u;
            }
            if (kE4m3) {
                float most = 0.f;
                auto lo = [](uint32_t x) { return __uint_as_float(x << 16); };
                auto hi = [](uint32_t x) { return __uint_as_float(x & 0xffff0000u); };
#pragma unroll
                for (int x = 0; x < 16; ++x) most = max3(most, fabsf(lo(qf[nt][x])), fabsf(hi(qf[nt][x])));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 1));
                most = fmaxf(most, __shfl_xor_sync(0xffffffffu, most, 2));
                // 14 minus its exponent, within what has a power of two and an inverse; infinities stay what they are
                const int e = most > 0.f && most < INFINITY ? max(-112, min(112, 14 - exponent(most))) : 0;
                const float up = pow2(e);
                q_mul[nt] = pow2(-e);
#pragma unroll
                for (int x = 0; x < 16; ++x) qf[nt][x] = pack_f16x2(lo(qf[nt][x]) * up, hi(qf[nt][x]) * up);
            }
        }
        // The scores' columns are heads 2 t4 and 2 t4 + 1.
        float q_mul2[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int x = 0; x < 2; ++x)
                q_mul2[nt][x] = p.scale_log2 * (kE4m3 ? __shfl_sync(0xffffffffu, q_mul[nt], (2 * t4 + x) * 4) : 1.f);
        float v_ref = 0.f, v_inv = 0.f;   // e4m3: the power of two that V scales are relative to, and 2^7 over it
        float acc[NT][8][4];
        float m[NT][2], l[NT][2];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
            for (int j = 0; j < 8; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) acc[nt][j][e] = 0.f;
            m[nt][0] = m[nt][1] = -INFINITY;
            l[nt][0] = l[nt][1] = 0.f;
        }
        const int row_from = cur.i;
        const bool whole = row_from == 0 && cur.end == cur.s.nt;   // nothing of the row is elsewhere
        for (int i = row_from + warp; i < cur.end; i += 4) {
            load_next(stage == 0 ? Sh::kStages - 1 : stage - 1);
            cp_async_wait<Sh::kStages - 1>();
            __syncwarp();
            const uint32_t sk = ring + stage * Sh::kStage, sv = sk + kTileKeys * Sh::kRow;
            const int j0 = tile_slot(cur.s, i);
            float s[NT][4];
            {
                float s2[NT][2][4];   // two chains
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s2[nt][0][e] = s2[nt][1][e] = 0.f;
                const uint32_t row = sk + (lane & 15) * Sh::kRow;
                const uint32_t hi = lane >> 4, sw = lane & 7;
                if (kE4m3) {
#pragma unroll
                    for (int ci = 0; ci < 4; ++ci) {
                        uint32_t r[4], a[2][4];
                        ldmatrix_x4(r, row + (((2 * ci + hi) ^ sw) << 4));
                        e4m3_to_f16(r[0], a[0][0], a[0][2]);
                        e4m3_to_f16(r[1], a[0][1], a[0][3]);
                        e4m3_to_f16(r[2], a[1][0], a[1][2]);
                        e4m3_to_f16(r[3], a[1][1], a[1][3]);
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) {
                            mma_16816_f16(s2[nt][0], a[0], qf[nt][4 * ci], qf[nt][4 * ci + 1]);
                            mma_16816_f16(s2[nt][1], a[1], qf[nt][4 * ci + 2], qf[nt][4 * ci + 3]);
                        }
                    }
                } else {
#pragma unroll
                    for (int ks = 0; ks < 8; ++ks) {
                        uint32_t a[4];
                        ldmatrix_x4(a, row + (((2 * ks + hi) ^ sw) << 4));
#pragma unroll
                        for (int nt = 0; nt < NT; ++nt) mma_16816(s2[nt][ks & 1], a, qf[nt][2 * ks], qf[nt][2 * ks + 1]);
                    }
                }
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[nt][e] = s2[nt][0][e] + s2[nt][1][e];
            }
            // Elements: (key g, head 2 t4), (g, + 1), (key g + 8, 2 t4), (g + 8, + 1).
            const uint32_t vis = ring_vis[stage];
            float mul[2] = {1.f, 1.f};
            float vs[2] = {1.f, 1.f};
            if (kE4m3) {
                const float* sc = reinterpret_cast<const float*>(smem + (sk - smem_u32(smem)) + 2 * kTileKeys * Sh::kRow);
                mul[0] = sc[g];
                mul[1] = sc[g + 8];
                vs[0] = (vis >> g) & 1u ? sc[16 + g] : 0.f;   // the scales are loaded for all rows, whatever they hold
                vs[1] = (vis >> (g + 8)) & 1u ? sc[24 + g] : 0.f;
                const float most = fmaxf(vs[0], vs[1]);
                if (__any_sync(0xffffffffu, most > v_ref && most < INFINITY)) {
                    float top = most < INFINITY ? most : 0.f;
#pragma unroll
                    for (int sh = 4; sh < 32; sh <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, sh));
                    const int e = max(-119, min(126, exponent(top) + 1));
                    const float down = v_ref * pow2(-e);   // below 1; 0 ahead of the first
                    v_ref = pow2(e);
                    v_inv = pow2(7 - e);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int j = 0; j < 8; ++j)
#pragma unroll
                            for (int x = 0; x < 4; ++x) acc[nt][j][x] *= down;
                }
                vs[0] *= v_inv;
                vs[1] *= v_inv;
            }
            bool over = false;
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[nt][e] = (vis >> (g + 8 * (e >> 1))) & 1u ? s[nt][e] * (kE4m3 ? mul[e >> 1] * q_mul2[nt][e & 1] : q_mul2[nt][e & 1]) : -INFINITY;
                    over = over || s[nt][e] > m[nt][e & 1] + 8.f;
                }
            }
            if (p.scores) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int hq = 8 * nt + 2 * t4 + (e & 1);
                        if (hq < heads)
                            p.scores[(static_cast<long long>(cur.b) * p.Hq + q0 + hq) * p.score_stride + j0 + g + 8 * (e >> 1)] = s[nt][e];
                    }
            }
            if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                    for (int x = 0; x < 2; ++x) {
                        float mx = fmaxf(m[nt][x], fmaxf(s[nt][x], s[nt][x + 2]));
#pragma unroll
                        for (int sh = 4; sh < 32; sh <<= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, sh));
                        const float alpha = mx == -INFINITY ? 1.f : ex2_approx(m[nt][x] - mx);
                        m[nt][x] = mx;
                        l[nt][x] *= alpha;
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            acc[nt][j][x] *= alpha;
                            acc[nt][j][x + 2] *= alpha;
                        }
                    }
            }
            uint32_t pb[NT][2];
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                float e4[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float mm = m[nt][e & 1];
                    e4[e] = ex2_approx(s[nt][e] - (mm == -INFINITY ? 0.f : mm));
                    l[nt][e & 1] += e4[e];
                    if (kE4m3) e4[e] *= vs[e >> 1];
                }
                pb[nt][0] = movmatrix(kE4m3 ? pack_f16x2(e4[0], e4[1]) : pack_bf16x2(e4[0], e4[1]));
                pb[nt][1] = movmatrix(kE4m3 ? pack_f16x2(e4[2], e4[3]) : pack_bf16x2(e4[2], e4[3]));
            }
            if (kE4m3) {
                const uint32_t row = sv + (lane & 15) * Sh::kRow;
                const uint32_t hi = lane >> 4, sw = lane & 7;
#pragma unroll
                for (int ci = 0; ci < 4; ++ci) {
                    uint32_t r[4], a[2][4];
                    ldmatrix_x4_trans(r, row + (((2 * ci + hi) ^ sw) << 4));
                    // bytes: two dims of a key, then of the next; wanted: a dim's two keys
#pragma unroll
                    for (int x = 0; x < 4; ++x) r[x] = __byte_perm(r[x], 0u, 0x3120);
                    e4m3_to_f16(r[0], a[0][0], a[0][1]);
                    e4m3_to_f16(r[1], a[0][2], a[0][3]);
                    e4m3_to_f16(r[2], a[1][0], a[1][1]);
                    e4m3_to_f16(r[3], a[1][2], a[1][3]);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) {
                        mma_16816_f16(acc[nt][2 * ci], a[0], pb[nt][0], pb[nt][1]);
                        mma_16816_f16(acc[nt][2 * ci + 1], a[1], pb[nt][0], pb[nt][1]);
                    }
                }
            } else {
                const uint32_t row = sv + ((lane & 7) + ((lane >> 4) << 3)) * Sh::kRow;
                const uint32_t hi = (lane >> 3) & 1, sw = lane & 7;
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    uint32_t a[4];
                    ldmatrix_x4_trans(a, row + (((2 * j + hi) ^ sw) << 4));
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt) mma_16816(acc[nt][j], a, pb[nt][0], pb[nt][1]);
                }
            }
            __syncwarp();   // the stage may be filled again
            stage = stage + 1 == Sh::kStages ? 0 : stage + 1;
        }

        // The four warps' parts of the row, eight heads at a time: a warp joins two heads, a lane four dims.
        const int row_id = cur.b * rows_per_seq + cur.hr;
        const float back = kE4m3 ? v_ref * 0.0078125f : 1.f;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            if (8 * nt >= heads) break;
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                float sum = l[nt][x];
#pragma unroll
                for (int sh = 4; sh < 32; sh <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, sh);
                if (g == 0)
                    *reinterpret_cast<float2*>(ex_ml + (warp * 8 + 2 * t4 + x) * 2) = make_float2(m[nt][x], sum);
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    float* dst = ex_o + (warp * 8 + 2 * t4 + x) * kOStride + 16 * j;
                    const float a = acc[nt][j][x] * back, b = acc[nt][j][x + 2] * back;
                    if (kE4m3) {
                        *reinterpret_cast<float2*>(dst + 2 * g) = make_float2(a, b);
                    } else {
                        dst[g] = a;
                        dst[g + 8] = b;
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int x = 0; x < 2; ++x) {
                const int hq = 2 * warp + x;
                if (8 * nt + hq >= heads) break;
                float2 ml[4];
                float top = -INFINITY, sum = 0.f;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    ml[w] = *reinterpret_cast<const float2*>(ex_ml + (w * 8 + hq) * 2);
                    top = fmaxf(top, ml[w].x);
                }
                float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float a = part_scale(ml[w].x, top);
                    const float4 v = *reinterpret_cast<const float4*>(ex_o + (w * 8 + hq) * kOStride + 4 * lane);
                    sum = fmaf(a, ml[w].y, sum);
                    o.x = fmaf(a, v.x, o.x);
                    o.y = fmaf(a, v.y, o.y);
                    o.z = fmaf(a, v.z, o.z);
                    o.w = fmaf(a, v.w, o.w);
                }
                if (whole) {
                    const bool some = sum > 0.f || isnan(sum);
                    const float inv = some ? 1.f / sum : 0.f;
                    const long long out = static_cast<long long>(cur.b) * p.Hq + q0 + 8 * nt + hq;
                    reinterpret_cast<uint2*>(p.o)[out * 32 + lane] = some ? make_uint2(pack_bf16x2(o.x * inv, o.y * inv), pack_bf16x2(o.z * inv, o.w * inv))
                                                                          : make_uint2(0u, 0u);
                    if (p.lse && lane == 0) p.lse[out] = some ? (top + log2f(sum)) * kLn2 : -INFINITY;
                } else {
                    const long long slot = (static_cast<long long>(blockIdx.x) + (p.splits > 0 ? 0 : row_id)) * (8 * NT) + 8 * nt + hq;
                    reinterpret_cast<float4*>(p.part_o)[slot * 32 + lane] = o;
                    if (lane == 0) reinterpret_cast<float2*>(p.part_ml)[slot] = make_float2(top, sum);
                }
            }
            __syncthreads();
        }
        if (cur.left == 0) break;
        next_row(cur);
    }
    cp_async_wait<0>();
}

// A row's parts: slots base + first .. base + last; `whole`: there is one, whose CTA wrote the result itself.  No tile: none.
struct RowParts {
    int first, last;
    bool whole;
    long long base;
};
__device__ __forceinline__ RowParts row_parts(const PagedDev& c, const DecodeParams& p, int b, int hr, int nt) {
    const int rows_per_seq = c.Hkv * p.q_tiles;
    const long long row = static_cast<long long>(b) * rows_per_seq + hr;
    if (p.splits > 0) {
        const int per = static_cast<int>(list_piece(nt, p.splits)), last = nt == 0 ? 0 : (nt - 1) / per;
        return {0, last, last == 0, row * p.splits};
    }
    if (nt == 0) return {0, -1, false, row};
    int ahead = 0, all = 0;   // tiles of the sequences before b, and of all
    for (int x = threadIdx.x & 31; x < p.B; x += 32) {
        const int n = seq_tiles(paged_length(c, p.seq_lens, x, p.status), p.window, p.sinks).nt;
        all += n;
        if (x < b) ahead += n;
    }
    ahead = __reduce_add_sync(0xffffffffu, ahead);
    all = __reduce_add_sync(0xffffffffu, all);
    const long long per = list_piece(static_cast<long long>(all) * rows_per_seq, p.n_ctas);
    const long long at = static_cast<long long>(ahead) * rows_per_seq + static_cast<long long>(hr) * nt;
    const int most = p.n_ctas - 1;   // beyond only if someone changes the lengths meanwhile
    const int first = min(most, static_cast<int>(at / per)), last = min(most, static_cast<int>((at + nt - 1) / per));
    return {first, last, first == last, row};
}
// Largest maximum of the parts of a query head; every lane of the warp takes part.
__device__ __forceinline__ float parts_max(const DecodeParams& p, const RowParts& r, long long slot0, int step) {
    float top = -INFINITY;
    for (int x = r.first + (threadIdx.x & 31); x <= r.last; x += 32) top = fmaxf(top, p.part_ml[(slot0 + static_cast<long long>(x) * step) * 2]);
#pragma unroll
    for (int s = 16; s > 0; s >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, s));
    return top;
}
// Joins the parts of the rows that several CTAs share, and gives the rows without a tile their zeros.  One block per row
// and query head; the warps take the parts in turn, a lane four dims.  Latency-bound: a few KB per block, so the
// loads of a warp's parts are independent of one another.  (One block per row with its heads in turn and the sums carried
// from part to part took 11 us for 64 sequences, 24 us for 16 of 8 heads a kv head, 36 us for two long ones.)
template <int NT, int kWarps>
__device__ __forceinline__ void join(const PagedDev& c, const DecodeParams& p, int b, int hr, int hq) {
    __shared__ float4 s_o[kWarps][32];
    __shared__ float s_l[kWarps];
    const int h = hr / p.q_tiles, q0 = h * p.group + (hr - h * p.q_tiles) * 8 * NT;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const SeqTiles s = seq_tiles(paged_length(c, p.seq_lens, b, p.status), p.window, p.sinks);
    const RowParts r = row_parts(c, p, b, hr, s.nt);
    pdl_wait();
    if (r.whole || hq >= min(8 * NT, (h + 1) * p.group - q0)) return;
    const long long slot0 = r.base * (8 * NT) + hq;
    const float top = parts_max(p, r, slot0, 8 * NT);
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
    float l = 0.f;
#pragma unroll 8
    for (int x = r.first + warp; x <= r.last; x += kWarps) {
        const long long slot = slot0 + static_cast<long long>(x) * (8 * NT);
        const float2 ml = reinterpret_cast<const float2*>(p.part_ml)[slot];
        const float4 v = reinterpret_cast<const float4*>(p.part_o)[slot * 32 + lane];
        const float a = part_scale(ml.x, top);
        l = fmaf(a, ml.y, l);
        o.x = fmaf(a, v.x, o.x);
        o.y = fmaf(a, v.y, o.y);
        o.z = fmaf(a, v.z, o.z);
        o.w = fmaf(a, v.w, o.w);
    }
    s_o[warp][lane] = o;
    if (lane == 0) s_l[warp] = l;
    __syncthreads();
    const int d = threadIdx.x;
    if (d >= 128) return;
    const float* so = reinterpret_cast<const float*>(s_o);
    float sum = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
        sum += s_l[w];
        x += so[128 * w + d];
    }
    const bool some = sum > 0.f || isnan(sum);
    const long long out = static_cast<long long>(b) * p.Hq + q0 + hq;
    p.o[out * 128 + d] = __float2bfloat16(some ? x / sum : 0.f);
    if (p.lse && d == 0) p.lse[out] = some ? (top + log2f(sum)) * kLn2 : -INFINITY;
}

// Adds the probabilities to the weights, from the scores and the parts' sums: a block of the join's launch for each stretch of
// kWeighSlots slots.  What does not depend on the sums is under way before they are looked at.  The host does not know the
// lengths: there are blocks, and room for scores, for all that the table has room for (16 sequences of 2049 tokens, 32 heads
// on 8: 34 us with the decode in tables for 2112 slots, 35 for 16384, 65 for 131072).
constexpr int kWeighSlots = 256;
template <int NT, int kWarps>
__device__ __forceinline__ void weigh(const PagedDev& c, const DecodeParams& p, int b, int h, int stretch) {
    __shared__ float s_lse[8 * NT];   // in units of log2
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const SeqTiles s = seq_tiles(paged_length(c, p.seq_lens, b, p.status), p.window, p.sinks);
    const int j0 = stretch * kWeighSlots;
    const RowParts r = j0 < s.n ? row_parts(c, p, b, h, s.nt) : RowParts{0, -1, false, 0};
    const long long q0 = static_cast<long long>(b) * p.Hq + h * p.group;
    constexpr int kSlots = kWarps == 4 ? 2 : 1;   // a thread; with more than 8 warps some have none
    long long row[kSlots];
    float x[kSlots][8 * NT], old[kSlots];
#pragma unroll
    for (int u = 0; u < kSlots; ++u) {
        const int j = j0 + u * 128 + threadIdx.x, end = min(s.n, j0 + kWeighSlots);
        row[u] = j < end ? paged_row(c, b, h, j, p.status) : -1;
    }
    pdl_wait();
    if (j0 >= s.n) return;
#pragma unroll
    for (int u = 0; u < kSlots; ++u) {
        const int j = j0 + u * 128 + threadIdx.x, end = min(s.n, j0 + kWeighSlots);
#pragma unroll
        for (int hq = 0; hq < 8 * NT; ++hq)
            x[u][hq] = j < end && hq < p.group ? p.scores[(q0 + hq) * p.score_stride + j] : -INFINITY;
    }
#pragma unroll
    for (int u = 0; u < kSlots; ++u) old[u] = row[u] >= 0 ? c.weight[row[u]] : 0.f;
    for (int hq = warp; hq < p.group; hq += kWarps) {
        float lse;
        if (r.whole) {
            lse = p.lse[q0 + hq] * kLog2e;
        } else {
            const long long slot0 = r.base * (8 * NT) + hq;
            const float top = parts_max(p, r, slot0, 8 * NT);
            float l = 0.f;
            for (int part = r.first + lane; part <= r.last; part += 32) {
                const float2 ml = reinterpret_cast<const float2*>(p.part_ml)[slot0 + static_cast<long long>(part) * (8 * NT)];
                l = fmaf(part_scale(ml.x, top), ml.y, l);
            }
#pragma unroll
            for (int sh = 16; sh > 0; sh >>= 1) l += __shfl_xor_sync(0xffffffffu, l, sh);
            lse = top + log2f(l);
        }
        // A head without a finite score has no probabilities, as in its output: all differences are to be -inf then.
        if (lane == 0) s_lse[hq] = lse == -INFINITY ? INFINITY : lse;
    }
    __syncthreads();
#pragma unroll
    for (int u = 0; u < kSlots; ++u) {
        if (row[u] < 0) continue;
        float w = 0.f;
#pragma unroll
        for (int hq = 0; hq < 8 * NT; ++hq)
            if (hq < p.group) w += ex2_approx(x[u][hq] - s_lse[hq]);
        c.weight[row[u]] = old[u] + w;
    }
}

// The launch behind the decode kernel, in whose shadow it reads the lengths and tables (that kernel lets it begin only when
// those are there): blockIdx.x = row, blockIdx.y = a query head of it to join, or, behind those, a stretch
// of its slots to weigh.
template <int NT, int kWarps>
__global__ void __launch_bounds__(kWarps * 32) paged_finish_kernel(const PagedDev c, const DecodeParams p, int heads) {
    const int rows_per_seq = c.Hkv * p.q_tiles;
    const int b = blockIdx.x / rows_per_seq, hr = blockIdx.x - b * rows_per_seq;
    if (static_cast<int>(blockIdx.y) < heads) join<NT, kWarps>(c, p, b, hr, blockIdx.y);
    else weigh<NT, kWarps>(c, p, b, hr, blockIdx.y - heads);   // host-checked: one group of query heads, so a row is a kv head
}

int paged_args(const char* who, const fba_paged_t* cache, int B, PagedDev* dev) {
    const char* why = nullptr;
    int code = FBA_ERR_BAD_ARG;
    const auto misaligned = [](const void* x) { return reinterpret_cast<uintptr_t>(x) % 16 != 0; };
    if (!cache || !cache->k || !cache->v || !cache->table) why = "null pointer in the cache";
    else if (B <= 0 || cache->n_pages <= 0 || cache->Hkv <= 0 || cache->max_pages <= 0) why = "non-positive size";
    else if (cache->page_size < 16 || cache->page_size > 256 || (cache->page_size & (cache->page_size - 1)))
        why = "page_size must be 16, 32, 64, 128 or 256";
    else if (cache->e4m3 && (!cache->k_scale || !cache->v_scale)) why = "an e4m3 cache needs k_scale and v_scale";
    else if (!cache->weight != !cache->position) why = "weight and position come together";
    else if (misaligned(cache->k) || misaligned(cache->v) || misaligned(cache->k_scale) || misaligned(cache->v_scale))
        why = "the pools must be 16-byte aligned";
    else if (static_cast<long long>(cache->max_pages) * cache->page_size >= 1 << 30)
        code = FBA_ERR_TOO_LARGE, why = "max_pages * page_size reaches 2^30";
    else if (B > 65535) code = FBA_ERR_TOO_LARGE, why = "more than 65535 sequences";
    if (why) {
        char buf[160];
        snprintf(buf, sizeof(buf), "%s: %s", who, why);
        return set_error(code, buf);
    }
    int shift = 4;
    while ((1 << shift) < cache->page_size) ++shift;
    *dev = PagedDev{static_cast<uint8_t*>(cache->k), static_cast<uint8_t*>(cache->v), cache->e4m3 ? cache->k_scale : nullptr,
                    cache->e4m3 ? cache->v_scale : nullptr, cache->weight, cache->position, cache->table, cache->n_pages,
                    cache->Hkv, cache->page_size, shift, cache->max_pages};
    return FBA_OK;
}

}  // namespace fba

using namespace fba;

extern "C" int fba_paged_append(const fba_paged_t* cache, const void* k, const void* v, const int64_t* k_strides,
                                const int64_t* v_strides, int B, int T, const int32_t* seq_lens, const int32_t* new_lens,
                                const int32_t* positions, int32_t* out_lens, uint32_t* status, void* stream) {
    ProfRange range("fba_paged_append");
    PagedDev c;
    int rc = paged_args("fba_paged_append", cache, B, &c);
    if (rc != FBA_OK) return rc;
    if (!k || !v || !k_strides || !v_strides || !seq_lens || !status)
        return set_error(FBA_ERR_BAD_ARG, "fba_paged_append: null pointer argument");
    if (lens_overlap(out_lens, seq_lens, B) || lens_overlap(out_lens, new_lens, B) || lens_overlap(out_lens, positions, B))
        return set_error(FBA_ERR_BAD_ARG, "fba_paged_append: out_lens must not overlap seq_lens, new_lens or positions");
    if (T <= 0) return set_error(FBA_ERR_BAD_ARG, "fba_paged_append: non-positive size");
    if (static_cast<long long>(T) * c.Hkv > 1 << 30)   // rows, and rows plus a grid's, are counted in 31 bits
        return set_error(FBA_ERR_TOO_LARGE, "fba_paged_append: more than 2^30 rows of a sequence");
    if (reinterpret_cast<uintptr_t>(k) % 16 != 0 || reinterpret_cast<uintptr_t>(v) % 16 != 0)
        return set_error(FBA_ERR_BAD_ARG, "fba_paged_append: k and v must be 16-byte aligned");
    AppendParams p = {static_cast<const __nv_bfloat16*>(k), static_cast<const __nv_bfloat16*>(v), {}, {}, seq_lens, new_lens,
                      positions, out_lens, status, T};
    for (int i = 0; i < 3; ++i) {
        if (k_strides[i] % 8 != 0 || v_strides[i] % 8 != 0)
            return set_error(FBA_ERR_BAD_ARG, "fba_paged_append: strides must be multiples of 8 elements");
        p.ks[i] = k_strides[i];
        p.vs[i] = v_strides[i];
    }
    DeviceGuard guard;
    if ((rc = guard.bind(cache->k)) != FBA_OK) return rc;
    const long long blocks = (static_cast<long long>(T) * c.Hkv + 31) / 32, most = (148 * 16 + B - 1) / B;   // 32 rows a block
    dim3 grid(static_cast<unsigned>(blocks < most ? blocks : most), B);
    auto kernel = cache->e4m3 ? paged_append_kernel<true> : paged_append_kernel<false>;
    return launch_chained(kernel, grid, 256, 0, static_cast<cudaStream_t>(stream), c, p);
}

namespace {
// How a decode call is cut up.
struct DecodePlan {
    int nt, q_tiles, splits, n_ctas, score_stride;   // n_ctas: of the grid
    long long rows;
    uint64_t part_o, part_ml, scores;   // bytes of the workspace, each rounded up to 256
};
DecodePlan decode_plan(int B, int Hq, int Hkv, int page_size, int max_pages, bool e4m3, bool accumulate) {
    DecodePlan d;
    const int group = Hq / Hkv;
    d.nt = group > 8 ? 2 : 1;
    d.q_tiles = (group + 8 * d.nt - 1) / (8 * d.nt);
    d.rows = static_cast<long long>(B) * Hkv * d.q_tiles;
    const long long tiles = static_cast<long long>(max_pages) * page_size / kTileKeys;   // a row has at most
    // Many rows: a CTA per row, or per equal part of a row where that makes four waves of them and leaves parts of 2048 keys.
    // The order in which CTAs end evens out lengths and SMs, and a row in one part needs no join.  Few rows: the list of all
    // tiles in as many pieces as are resident at a time.  Us, list -> rows: 256 sequences of 600 tokens and 8 kv heads 126 ->
    // 100, of 1 - 1000 126 -> 84, 64 of 2048 95 -> 83 (1 part), of 512 - 8192 182 -> 170 (3 parts); e4m3, 64 of 1 - 2048 63 ->
    // 41, of 2048 58 -> 68 (the rule counts two CTAs an SM for both types, though three of e4m3 fit: 512 rows end in a wave
    // that is mostly empty).  Rows that barely fill the chip: 40 sequences of 1500 50 -> 54.  `tiles` is what the table has
    // room for, so the cut, and with it the last bits, follow from its width.
    // (The list in two, three and four waves: 64 sequences of 512 - 8192 183 -> 179, 178, 177; two long e4m3 ones 101 ->
    // 105, 109, 115: a CTA's start and end cost a few us.)
    const long long resident = 148 * (d.nt == 1 && e4m3 ? 3 : 2), four_waves = 4 * 2 * 148;
    const long long most = (tiles + kDecMinTiles - 1) / kDecMinTiles;   // pieces of a row
    d.splits = 0;
    if (tiles <= 2 * kDecMinTiles || d.rows >= four_waves) {
        d.splits = 1;
    } else if (2 * d.rows >= 3 * 2 * 148) {
        const long long want = (four_waves + d.rows - 1) / d.rows, room = tiles / (8 * kDecMinTiles);
        d.splits = static_cast<int>(room < 1 ? 1 : want < room ? want : room);
    }
    const long long pieces = d.splits ? d.rows * d.splits : d.rows * most;
    d.n_ctas = static_cast<int>(d.splits || pieces < resident ? pieces : resident);
    auto up = [](uint64_t n) { return (n + 255) / 256 * 256; };
    const uint64_t slots = d.splits == 1 ? 0 : (d.n_ctas + (d.splits ? 0 : d.rows)) * 8ull * d.nt;
    d.part_o = up(slots * 128 * sizeof(float));
    d.part_ml = up(slots * 2 * sizeof(float));
    d.score_stride = static_cast<int>(tiles * kTileKeys);
    d.scores = accumulate ? up(static_cast<uint64_t>(B) * Hq * d.score_stride * sizeof(float)) : 0;
    return d;
}
template <bool kE4m3, int NT>
int launch_decode(const PagedDev& c, const DecodeParams& p, const DecodePlan& d, cudaStream_t stream) {
    constexpr int smem = DecShape<kE4m3>::kSmem;
    if (cudaFuncSetAttribute(paged_decode_kernel<kE4m3, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
        cudaGetLastError();
        return set_error(FBA_ERR_LAUNCH, "fba_paged_decode: cannot raise the dynamic shared memory limit");
    }
    const unsigned rows = static_cast<unsigned>(d.rows);
    int rc = launch_chained(paged_decode_kernel<kE4m3, NT>, dim3(static_cast<unsigned>(d.n_ctas)), kDecThreads, smem, stream, c, p);
    const int heads = d.splits == 1 ? 0 : p.group < 8 * NT ? p.group : 8 * NT;
    const int stretches = p.scores ? (d.score_stride + kWeighSlots - 1) / kWeighSlots : 0;
    if (rc == FBA_OK && heads + stretches > 0)
        // A row may have many parts where there are few rows: more warps take them then.
        rc = d.splits == 0 && d.n_ctas > 16 * d.rows ? launch_chained(paged_finish_kernel<NT, 16>, dim3(rows, heads + stretches), 512, 0, stream, c, p, heads)
                                    : launch_chained(paged_finish_kernel<NT, 4>, dim3(rows, heads + stretches), 128, 0, stream, c, p, heads);
    return rc;
}
}  // namespace

static int decode_args(const char* who, int B, int Hq, int Hkv, int page_size, int max_pages) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || page_size <= 0 || max_pages <= 0 || Hq % Hkv != 0)
        return set_error(FBA_ERR_BAD_ARG, who);
    if (static_cast<long long>(B) * Hq > 1 << 24) return set_error(FBA_ERR_TOO_LARGE, who);
    if (static_cast<long long>(max_pages) * page_size >= 1 << 30 ||   // tiles of all sequences are counted in 31 bits
        static_cast<long long>(B) * max_pages * page_size / kTileKeys >= 1ll << 31)
        return set_error(FBA_ERR_TOO_LARGE, who);
    return FBA_OK;
}

extern "C" int fba_paged_decode_workspace_bytes(int B, int Hq, int Hkv, int page_size, int max_pages, int e4m3,
                                                int accumulate, uint64_t* bytes) {
    const int rc = decode_args("fba_paged_decode_workspace_bytes: bad size", B, Hq, Hkv, page_size, max_pages);
    if (rc != FBA_OK) return rc;
    if (!bytes) return set_error(FBA_ERR_BAD_ARG, "fba_paged_decode_workspace_bytes: null pointer argument");
    const DecodePlan d = decode_plan(B, Hq, Hkv, page_size, max_pages, e4m3 != 0, accumulate != 0);
    *bytes = d.part_o + d.part_ml + d.scores;
    return FBA_OK;
}

extern "C" int fba_paged_decode(const fba_paged_t* cache, const void* q, const int64_t* q_strides, void* o, float* lse, int B,
                                int Hq, const int32_t* seq_lens, int window, int sinks, float softmax_scale, int accumulate,
                                void* workspace, uint64_t workspace_bytes, uint32_t* status, void* stream_) {
    ProfRange range("fba_paged_decode");
    cudaStream_t stream = static_cast<cudaStream_t>(stream_);
    PagedDev c;
    int rc = paged_args("fba_paged_decode", cache, B, &c);
    if (rc != FBA_OK) return rc;
    if (!q || !q_strides || !o || !seq_lens || !status)
        return set_error(FBA_ERR_BAD_ARG, "fba_paged_decode: null pointer argument");
    rc = decode_args("fba_paged_decode: bad size, or Hq not a multiple of Hkv", B, Hq, c.Hkv, c.page_size, c.max_pages);
    if (rc != FBA_OK) return rc;
    if (window < 0 || sinks < 0) return set_error(FBA_ERR_BAD_ARG, "fba_paged_decode: window and sinks must not be negative");
    if (!(softmax_scale > 0.f) || !(softmax_scale < INFINITY))
        return set_error(FBA_ERR_BAD_ARG, "fba_paged_decode: softmax_scale must be positive and finite");
    const DecodePlan d = decode_plan(B, Hq, c.Hkv, c.page_size, c.max_pages, cache->e4m3 != 0, accumulate != 0);
    if (accumulate && (!c.weight || window != 0 || !lse))
        return set_error(FBA_ERR_BAD_ARG, "fba_paged_decode: accumulation needs a cache with weights, lse, and no window");
    if (accumulate && d.score_stride > 65000 * kWeighSlots)
        return set_error(FBA_ERR_TOO_LARGE, "fba_paged_decode: accumulation takes tables of at most 16.6 million slots");
    if (accumulate && Hq / c.Hkv > 16)
        return set_error(FBA_ERR_BAD_ARG, "fba_paged_decode: accumulation takes at most 16 query heads a kv head");
    if (reinterpret_cast<uintptr_t>(q) % 4 != 0 || q_strides[0] % 2 != 0 || q_strides[1] % 2 != 0)
        return set_error(FBA_ERR_BAD_ARG, "fba_paged_decode: q must be 4-byte aligned, its strides multiples of 2");
    if (reinterpret_cast<uintptr_t>(o) % 8 != 0) return set_error(FBA_ERR_BAD_ARG, "fba_paged_decode: o must be 8-byte aligned");
    const uint64_t need = d.part_o + d.part_ml + d.scores;
    if (need && (!workspace || workspace_bytes < need || reinterpret_cast<uintptr_t>(workspace) % 256 != 0))
        return set_error(FBA_ERR_BAD_ARG,
                         "fba_paged_decode: workspace must be 256-byte aligned, of fba_paged_decode_workspace_bytes() bytes");
    if (d.rows > 0x7fffffffLL) return set_error(FBA_ERR_TOO_LARGE, "fba_paged_decode: more than 2^31 rows");
    DeviceGuard guard;
    if ((rc = guard.bind(cache->k)) != FBA_OK) return rc;

    DecodeParams p = {};
    p.q = static_cast<const __nv_bfloat16*>(q);
    p.qs[0] = q_strides[0];
    p.qs[1] = q_strides[1];
    p.o = static_cast<__nv_bfloat16*>(o);
    p.lse = lse;
    p.seq_lens = seq_lens;
    p.status = status;
    uint8_t* ws = static_cast<uint8_t*>(workspace);
    p.part_o = reinterpret_cast<float*>(ws);
    p.part_ml = reinterpret_cast<float*>(ws + d.part_o);
    p.scores = accumulate ? reinterpret_cast<float*>(ws + d.part_o + d.part_ml) : nullptr;
    p.score_stride = d.score_stride;
    p.B = B;
    p.Hq = Hq;
    p.group = Hq / c.Hkv;
    p.q_tiles = d.q_tiles;
    p.window = window;
    const int cap = c.max_pages * c.page_size;   // below 2^30
    p.sinks = sinks < cap ? sinks : cap;
    p.splits = d.splits;
    p.n_ctas = d.n_ctas;
    p.scale_log2 = softmax_scale * kLog2e;
    if (cache->e4m3) return d.nt == 1 ? launch_decode<true, 1>(c, p, d, stream) : launch_decode<true, 2>(c, p, d, stream);
    return d.nt == 1 ? launch_decode<false, 1>(c, p, d, stream) : launch_decode<false, 2>(c, p, d, stream);
}
