// Accumulated attention weights of a step's keys (gfx950).
//
// For key j and KV head h of a sequence:  mass[j][h] = decay * mass[j][h] + sum over the step's rows r that
// attend j and the query heads a of h's group of  exp(scale q_ra . k_j - lse_ra),  lse_ra the log-sum-exp of
// row r's scores.  Two passes over the keys, K alone: the first leaves (maximum, mass) of every (row, head)
// column over parts of its keys, the second merges a column's parts into its lse and sums the weights of every
// key over the columns - in a fixed order, nothing is added atomically, so the sums do not depend on timing.
// (One pass would have to hold the scores until the lse is known: four bytes of a score and column, written and read.  At
// eight query heads a KV head that is as many as the 68 of a key's MXFP4 codes twice; with fewer heads, or the 256 of a
// bf16 key of 128, it would be less than K again, which a short batch's second pass finds in the last-level cache.)
//
// Both passes are tiles of 16 keys by 16 columns ((row, head) pairs of one KV head; MFMA 16x16x32 with the
// attention kernels' operand types: bf16 on bf16 and MXFP4 pools, f16 on f16 and FP8 pools).  Two forms:
//  - few columns a sequence (decode, verify rows): bound by reading K.  All keys of the step are laid end to end in
//    units of 256 and every workgroup takes one contiguous share, so that it streams; its waves take 64 keys each.  64
//    contexts of 16k to 32k keys of 2 heads of 128 (MXFP4, 212 MB): 46 and 51 us a pass, 4.6 and 4.2 TB/s; eight of 1,548
//    to 28,027: 8.4 and 11.4 us, the launch, the scan and three dependent loads before the first key.
//  - prompt chunks: bound by the exponentials beside the products.  Workgroups take equal shares of blocks of columns
//    (first pass) or keys (second).  512 and 300 rows of 16 heads over 4,608 and 2,001 bf16 keys: 27 and 23 us, and 4.7
//    and 5.0 for the merges.
// Either form serves any step; the host chooses by the rows a sequence has on average.  A step of both kinds pays for it:
// the streaming form's second pass shares out keys, whose sequences' column blocks differ, and the other form's blocks are
// mostly empty for a sequence of one row.
#include <algorithm>
#include <type_traits>

#include "common.hpp"
#include "launch.hpp"

namespace lia {

constexpr uint32_t kMassThreads = 256;
constexpr uint32_t kMassSeqs = kMassThreads; // sequences of one scan, one a thread
constexpr uint32_t kUnit = 256;              // keys of a unit: 64 a wave
constexpr uint32_t kBlockCols = 256;         // prompt chunks: columns of a block of the first pass, 64 a wave
constexpr uint32_t kBlockKeys = 512;         // ... keys of a block of the second pass, 128 a wave
constexpr uint32_t kNoBlock = 0xffffffffu;
constexpr uint32_t kStatLead = 3, kSumLead = 6; // ... units that beginning a block costs, in either pass

struct MassParams {
    const void *q, *kc, *k_scales;
    const uint32_t *cu, *positions, *sequences, *pages;
    float *mass;
    // (maximum, mass) of a column over a part of its keys.  Few columns: [slot][16 NT], a slot for each share's part
    // of a column block; prompt chunks: [share][2][kBlockCols], the block it ends and the one it begins.
    float2 *stats;
    uint32_t slots;     // few columns: slots there are
    float *lse;         // prompt chunks: [h][columns], log2 of the mass over all keys, a sequence's from column_base()
    uint4 *queries;     // ... [h][columns / 16][D / 32][64]: their operands, a lane's 16 bytes each
    float *sums;        // ... [share][2][keys], as stats, of the second pass
    uint4 *begun[2];    // ... [share]: the block it begins and another ends, for either pass
    uint32_t hq, hkv, group, group_magic, stride, page_shift, pool_pages, n_seqs, n_rows, columns;
    float scale_log2, decay;
    int q_f32, fresh;
};

// A sequence of the step.
struct MassSeq {
    uint32_t r0, rows, p0, trow; // first packed row, rows, the first one's position, table row
    uint32_t n, cols;            // keys, columns of a KV head
};

// The scan of a launch: up to kMassSeqs sequences and the exclusive sums of three counts of each, by every workgroup
// itself (a list made by a launch of its own would cost more than the two dependent loads it saves).
struct MassScan {
    uint32_t items[kMassSeqs + 1], units[kMassSeqs + 1], blocks[kMassSeqs + 1];
    uint32_t r0[kMassSeqs], rows[kMassSeqs], p0[kMassSeqs], trow[kMassSeqs];
    uint32_t wave[3][8];
};

// Sequences first .. first + count - 1; counts(s): a sequence's three.
template <uint32_t THREADS, class F>
__device__ __forceinline__ void mass_scan(const MassParams &p, MassScan &sc, uint32_t first, uint32_t count, F &&counts) {
    const uint32_t t = threadIdx.x, lane = t & 63, w = t >> 6;
    uint3 a = make_uint3(0, 0, 0);
    if (t < count) {
        MassSeq s;
        s.r0 = p.cu[first + t];
        s.rows = s.r0 < p.n_rows ? min(p.cu[first + t + 1] - s.r0, p.n_rows - s.r0) : 0; // (none outside the step)
        s.p0 = s.rows ? p.positions[s.r0] : 0;
        s.trow = s.rows ? p.sequences[s.r0] : 0;
        s.n = s.rows ? s.p0 + s.rows : 0;
        s.cols = s.rows * p.group;
        sc.r0[t] = s.r0; sc.rows[t] = s.rows; sc.p0[t] = s.p0; sc.trow[t] = s.trow;
        if (s.rows) a = counts(s);
    }
    uint3 sum = a;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t x = __shfl_up(sum.x, off), y = __shfl_up(sum.y, off), z = __shfl_up(sum.z, off);
        if (lane >= (uint32_t)off) { sum.x += x; sum.y += y; sum.z += z; }
    }
    if (lane == 63) { sc.wave[0][w] = sum.x; sc.wave[1][w] = sum.y; sc.wave[2][w] = sum.z; }
    __syncthreads();
    for (uint32_t i = 0; i < w; i++) { sum.x += sc.wave[0][i]; sum.y += sc.wave[1][i]; sum.z += sc.wave[2][i]; }
    if (t < kMassSeqs) { sc.items[t] = sum.x - a.x; sc.units[t] = sum.y - a.y; sc.blocks[t] = sum.z - a.z; }
    if (t == THREADS - 1) { sc.items[kMassSeqs] = sum.x; sc.units[kMassSeqs] = sum.y; sc.blocks[kMassSeqs] = sum.z; }
    __syncthreads();
}

// The sequence that owns item `it` (the last whose items start at or before it), wave-uniform.
__device__ __forceinline__ uint32_t owner_of(const uint32_t *starts, uint32_t it) {
    uint32_t n = 0;
#pragma unroll
    for (uint32_t i = 0; i < kMassSeqs / 64; i++)
        n += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(starts[64 * i + (threadIdx.x & 63)] <= it));
    return n - 1;
}

__device__ __forceinline__ MassSeq seq_of(const MassParams &p, const MassScan &sc, uint32_t b) {
    MassSeq s;
    s.r0 = uniform(sc.r0[b]); s.rows = uniform(sc.rows[b]); s.p0 = uniform(sc.p0[b]); s.trow = uniform(sc.trow[b]);
    s.n = s.p0 + s.rows;
    s.cols = s.rows * p.group;
    return s;
}

template <int D, int KVT>
struct KTile {
    static constexpr bool MB = KVT == LIA_BF16 || KVT == LIA_FP4; // operand type
    static constexpr int KT = D / 32;
    static constexpr uint32_t ROW = KVT == LIA_FP4 ? D / 2 : KVT == LIA_FP8_E4M3 ? D : 2 * D; // bytes of a key's head
    static constexpr int WORDS = ROW / 16; // words a lane holds of a 16-key tile
    static constexpr uint32_t LDS = ROW >= 64 ? 16 * ROW : 0;
    uint32_t w[WORDS];
    uint32_t s; // FP4: the lane's block scale; FP8: the page scale's bits
};

// First dim of a lane's eight elements of k step ks (K and Q alike).
template <int D, int KVT>
__device__ __forceinline__ uint32_t dim_of(int ks, uint32_t g) {
    if constexpr (KVT == LIA_FP4) return (D / 4) * g + 8 * ks;
    if constexpr (KVT == LIA_FP8_E4M3) return 64 * (ks >> 1) + 16 * g + 8 * (ks & 1);
    return 32 * ks + 8 * g;
}

// Loads 16 keys from key t0 of a sequence (page: the physical page of t0's logical page; keys at or past n, and pages
// outside the pool, read as zeros).  Lanes take the tile's bytes in order, and operands() turns them through LDS: loaded as an
// operand holds them, every lane of four reads another key's row, which costs the L1 four lookups for one (16 keys of 256
// bytes: 64 clocks a load, and what bounded the first pass over a chunk of prompt rows, 40 us for 20).
template <int D, int KVT>
__device__ __forceinline__ void load_tile(const MassParams &p, KTile<D, KVT> &k, uint32_t t0, uint32_t n,
                                          uint32_t page, uint32_t h) {
    using T = KTile<D, KVT>;
    const uint32_t lane = lane_id(), g = lane >> 4, li = lane & 15, P = 1u << p.page_shift;
    const uint32_t off = t0 & (P - 1);
    const uint32_t live = page < p.pool_pages && t0 < n ? min(n - t0, P - off) : 0u;
    constexpr bool FP4 = KVT == LIA_FP4;
    const uint32_t row = FP4 ? T::ROW : p.hkv * T::ROW; // from key to key
    const uint64_t at = FP4 ? (((uint64_t)page * p.hkv + h) * P + off) * row
                            : ((uint64_t)page * P + off) * row + (uint64_t)h * T::ROW;
    // (a descriptor from the head's first byte: the last live key's head ends inside it)
    const __amdgpu_buffer_rsrc_t r = make_rsrc((const uint8_t *)p.kc + at, live ? (live - 1) * row + T::ROW : 0u);
    if constexpr (T::LDS == 0) { // (512 bytes a tile)
        const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)(li * T::ROW + 8 * g), 0, 0));
        k.w[0] = x.x; k.w[1] = x.y;
    } else {
#pragma unroll
        for (int q = 0; q < T::WORDS / 4; q++) {
            const uint32_t o = 1024 * q + 16 * lane;
            const u32x4 x = buffer_load16(r, o / T::ROW * row + o % T::ROW);
            k.w[4 * q] = x.x; k.w[4 * q + 1] = x.y; k.w[4 * q + 2] = x.z; k.w[4 * q + 3] = x.w;
        }
    }
    k.s = 0;
    if constexpr (FP4) {
        const __amdgpu_buffer_rsrc_t rs = make_rsrc((const uint8_t *)p.k_scales + at / 16, live * (D / 32));
        k.s = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(rs, (int)(li * (D / 32) + (D == 128 ? g : g >> 1)), 0, 0);
    }
    if constexpr (KVT == LIA_FP8_E4M3) {
        const __amdgpu_buffer_rsrc_t rs = make_rsrc((const float *)p.k_scales + ((uint64_t)page * p.hkv + h), live ? 4u : 0u);
        k.s = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(rs, 0, 0, 0);
    }
}

// A tile's operands: lane (g, li) of step ks holds key li's dims dim_of(ks, g) .. +7.  lds: this wave's own, its 16-byte
// pieces at positions that keep the 16 keys of a piece in different banks.
template <int D, int KVT>
__device__ __forceinline__ void operands(const KTile<D, KVT> &k, uint8_t *lds, u32x4 (&a)[D / 32]) {
    using T = KTile<D, KVT>;
    constexpr int KT = D / 32;
    const uint32_t lane = lane_id(), g = lane >> 4, li = lane & 15;
    if constexpr (T::LDS == 0) {
#pragma unroll
        for (int ks = 0; ks < KT; ks++) a[ks] = e2m1x8_to_bf16x8(k.w[ks], u2f(k.s << 23));
    } else {
        constexpr uint32_t PIECES = T::ROW / 16, ROWS = 16 / PIECES; // ... of a key, and keys of 256 bytes
        auto place = [](uint32_t key, uint32_t piece) { return key * T::ROW + 16 * (piece ^ (key / ROWS % PIECES)); };
#pragma unroll
        for (int q = 0; q < T::WORDS / 4; q++) {
            const uint32_t o = 64 * q + lane;
            *(u32x4 *)(lds + place(o / PIECES, o % PIECES)) =
                u32x4{k.w[4 * q], k.w[4 * q + 1], k.w[4 * q + 2], k.w[4 * q + 3]};
        }
#pragma unroll
        for (int q = 0; q < T::WORDS / 4; q++) {
            const u32x4 x = *(const u32x4 *)(lds + place(li, 4 * q + g));
            if constexpr (KVT == LIA_FP4) {
#pragma unroll
                for (int ks = 0; ks < KT; ks++) a[ks] = e2m1x8_to_bf16x8(x[ks], u2f(k.s << 23));
            } else if constexpr (KVT == LIA_FP8_E4M3) {
                a[2 * q] = e4m3x8_to_f16x8(u32x2{x.x, x.y});
                a[2 * q + 1] = e4m3x8_to_f16x8(u32x2{x.z, x.w});
            } else {
                a[q] = x;
            }
        }
    }
}
template <int D, int KVT>
constexpr uint32_t kTileLds = KTile<D, KVT>::LDS ? KTile<D, KVT>::LDS : 16;

// What a tile's scores are multiplied by.
template <int D, int KVT>
__device__ __forceinline__ float score_scale(const MassParams &p, const KTile<D, KVT> &k) {
    return KVT == LIA_FP8_E4M3 ? u2f(uniform(f2u(p.scale_log2 * u2f(k.s)))) : p.scale_log2; // (uniform)
}

__device__ __forceinline__ uint32_t div_group(const MassParams &p, uint32_t col) {
    return p.group == 1 ? col : __umulhi(col, p.group_magic);
}

// Query operands of NT tiles of 16 columns from col0 of a sequence: the lane's column li, dims dim_of(ks, g) .. +7 (past the
// last column that one's again: of zeros, a key that holds an infinity would make NaNs where the column's weight is 0).  All loads are issued before any is converted: a latency each would be what a segment costs.
template <int D, int KVT, int NT>
__device__ __forceinline__ void load_queries(const MassParams &p, const MassSeq &s, uint32_t h, uint32_t col0,
                                             u32x4 (&out)[NT][D / 32]) {
    constexpr bool MB = KTile<D, KVT>::MB;
    constexpr int KT = D / 32;
    const uint32_t g = lane_id() >> 4, li = lane_id() & 15, qb = p.q_f32 ? 4 : 2;
    const __amdgpu_buffer_rsrc_t r = make_rsrc(p.q, p.n_rows * p.hq * D * qb);
    uint32_t at[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) {
        const uint32_t col = min(col0 + 16 * n + li, s.cols - 1), ri = div_group(p, col);
        at[n] = ((s.r0 + ri) * p.hq + h * p.group + col - ri * p.group) * D * qb;
    }
    if (p.q_f32) {
        f32x4 x[NT][KT][2];
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int ks = 0; ks < KT; ks++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    x[n][ks][e] = __builtin_bit_cast(f32x4, buffer_load16(r, at[n] + dim_of<D, KVT>(ks, g) * 4 + 16 * e));
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int ks = 0; ks < KT; ks++) {
                const f32x4 a = x[n][ks][0], b = x[n][ks][1];
                out[n][ks] = u32x4{pack2<MB>(a.x, a.y), pack2<MB>(a.z, a.w), pack2<MB>(b.x, b.y), pack2<MB>(b.z, b.w)};
            }
        return;
    }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int ks = 0; ks < KT; ks++) out[n][ks] = buffer_load16(r, at[n] + dim_of<D, KVT>(ks, g) * 2);
    if constexpr (!MB) {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int ks = 0; ks < KT; ks++)
#pragma unroll
                for (int e = 0; e < 4; e++)
                    out[n][ks][e] = pack2<MB>(bf16_to_f32(out[n][ks][e] & 0xffffu), bf16_to_f32(out[n][ks][e] >> 16));
    }
}

// Pages of a key range: lane i holds the page of logical page base + i.
struct MassPages {
    const uint32_t *table;
    uint32_t limit, base, page;
};
__device__ __forceinline__ void pages_at(MassPages &w, uint32_t base) {
    w.base = base;
    w.page = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(make_rsrc(w.table, w.limit * 4), (int)((base + lane_id()) * 4), 0, 0);
}
// ... moved on where it does not reach logical page `last` (uniform).
__device__ __forceinline__ void pages_reach(MassPages &w, uint32_t from, uint32_t last) {
    if (last - w.base >= 64) {
        pages_at(w, from);
        asm volatile("" : "+v"(w.page)); // waited for here, not wherever a page is used (and with it for all loads)
    }
}
__device__ __forceinline__ uint32_t page_of(const MassPages &w, uint32_t logical) {
    return (uint32_t)__builtin_amdgcn_readlane((int)w.page, (int)((logical - w.base) & 63));
}

// A wave's running (maximum, mass) of 16 NT columns: per lane its own reference in the maximum's place, near its first keys'
// scores.  It need not be the maximum: the masses are floats, and what a reference below it costs is range, not bits.  It is
// raised when four keys' masses pass 2^64 (2^27 of them still sum below 2^128).
template <int NT>
struct MassState {
    bool begun;       // every lane has a reference for each of its columns (uniform)
    uint32_t lim[NT]; // live keys of the column
    float m[NT], thr[NT], l[NT];
};

// Scores of N tiles, tile i's keys 4g .. 4g+3 (from t0[i]) against column tile nt[i]: one check of all of them for a raised
// reference, so that the tiles' chains of instructions run side by side.
template <int N, int NT>
__device__ __forceinline__ void mass_scores(MassState<NT> &st, const f32x4 (&x)[N], const float (&ss)[N],
                                            const uint32_t (&t0)[N], const int (&col)[N], uint32_t hi, bool masked) {
    const uint32_t g = lane_id() >> 4;
    float e[N][4];
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int i = 0; i < 4; i++) e[n][i] = __builtin_fmaf(x[n][i], ss[n], -st.m[col[n]]);
    if (!masked && st.begun) {
        float sum[N], top = 0.0f;
#pragma unroll
        for (int n = 0; n < N; n++) {
            sum[n] = (fast_exp2(e[n][0]) + fast_exp2(e[n][1])) + (fast_exp2(e[n][2]) + fast_exp2(e[n][3]));
            top = fmaxf(top, sum[n]);
        }
        if (!__builtin_amdgcn_ballot_w64(top > 0x1p64f)) {
#pragma unroll
            for (int n = 0; n < N; n++) st.l[col[n]] += sum[n];
            return;
        }
    }
    { // a raised reference (rare), or masked keys
        float mx[NT];
#pragma unroll
        for (int c = 0; c < NT; c++) mx[c] = -INFINITY;
        if (masked) {
#pragma unroll
            for (int n = 0; n < N; n++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (t0[n] + 4 * g + i >= min(st.lim[col[n]], hi)) e[n][i] = -INFINITY;
        }
#pragma unroll
        for (int n = 0; n < N; n++)
            mx[col[n]] = fmaxf(mx[col[n]], fmaxf(fmaxf(e[n][0], e[n][1]), fmaxf(e[n][2], e[n][3])));
#pragma unroll
        for (int c = 0; c < NT; c++) {
            const float up = mx[c] > st.thr[c] ? mx[c] : 0.0f;
            st.l[c] *= st.thr[c] == -INFINITY ? 0.0f : fast_exp2(-up); // (up may be far below 0 at first)
            st.m[c] += up;
            if (mx[c] > st.thr[c]) st.thr[c] = 8.0f;
#pragma unroll
            for (int n = 0; n < N; n++)
                if (col[n] == c) {
#pragma unroll
                    for (int i = 0; i < 4; i++) e[n][i] -= up;
                }
        }
        bool wait = false;
#pragma unroll
        for (int c = 0; c < NT; c++) wait |= st.thr[c] != 8.0f;
        st.begun = __builtin_amdgcn_ballot_w64(wait) == 0;
    }
#pragma unroll
    for (int n = 0; n < N; n++)
        st.l[col[n]] += (fast_exp2(e[n][0]) + fast_exp2(e[n][1])) + (fast_exp2(e[n][2]) + fast_exp2(e[n][3]));
}

// The wave's columns from col0 of a sequence: limits and queries.
template <int D, int KVT, int NT>
__device__ __forceinline__ void mass_begin(const MassParams &p, const MassSeq &s, uint32_t h, uint32_t col0,
                                           MassState<NT> &st, u32x4 (&q)[NT][D / 32]) {
    const uint32_t li = lane_id() & 15;
    st.begun = false;
    load_queries<D, KVT, NT>(p, s, h, col0, q);
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const uint32_t col = col0 + 16 * nt + li;
        st.lim[nt] = col < s.cols ? s.p0 + div_group(p, col) + 1 : 0;
        st.m[nt] = 0.0f; st.l[nt] = 0.0f; st.thr[nt] = -INFINITY;
    }
}

// (maximum, mass) of the wave's columns over its lanes; -inf and 0 without a live key.
template <int NT>
__device__ __forceinline__ void mass_end(const MassState<NT> &st, int nt, float &M, float &L) {
    M = rows_max(st.l[nt] != 0.0f ? st.m[nt] : -INFINITY);
    L = rows_sum(st.l[nt] != 0.0f ? st.l[nt] * fast_exp2(st.m[nt] - M) : 0.0f);
}

// Keys [t, hi) in steps of `step`, 64 at a time, in four tiles: a tile's registers take the keys a step further as soon as
// its operands are out of them.  tile(j, operands, score scale) for each, then done(t).
template <int D, int KVT, class F, class G>
__device__ __forceinline__ void mass_stream(const MassParams &p, MassPages &w, uint32_t t, uint32_t hi, uint32_t step,
                                            uint32_t h, uint8_t *lds, F &&tile, G &&done) {
    constexpr int KT = D / 32;
    KTile<D, KVT> k[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        load_tile<D, KVT>(p, k[j], t + 16 * j, hi, page_of(w, (t + 16 * j) >> p.page_shift), h);
        __builtin_amdgcn_sched_barrier(0); // in this order, so that the first tile's use waits for its loads alone
    }
#pragma unroll 1
    for (; t < hi; t += step) {
        pages_reach(w, (t + step) >> p.page_shift, (t + step + 63) >> p.page_shift);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t t1 = t + step + 16 * j;
            const float ss = score_scale(p, k[j]);
            u32x4 a[KT];
            operands<D, KVT>(k[j], lds, a);
            load_tile<D, KVT>(p, k[j], t1, hi, page_of(w, t1 >> p.page_shift), h);
            tile(t + 16 * j, j, a, ss);
        }
        done(t);
    }
}

// The first pass over keys [t, hi): NT = 1 scores its four key tiles together, NT = 4 each key tile's four column tiles
// (at most `tiles` of them are the sequence's: the others' queries are zeros).
template <int D, int KVT, int NT>
__device__ __forceinline__ void mass_first(const MassParams &p, MassPages &w, uint32_t t, uint32_t hi, uint32_t step,
                                           uint32_t h, uint8_t *lds, const u32x4 (&q)[NT][D / 32], MassState<NT> &st,
                                           uint32_t free_hi) {
    constexpr bool MB = KTile<D, KVT>::MB;
    f32x4 x[4];
    float ss[4];
    mass_stream<D, KVT>(
        p, w, t, hi, step, h, lds,
        [&](uint32_t t0, int j, const u32x4 (&a)[D / 32], float scale) {
            if constexpr (NT == 1) {
                x[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                ss[j] = scale;
#pragma unroll
                for (int ks = 0; ks < D / 32; ks++) x[j] = mfma16x16x32<MB>(a[ks], q[0][ks], x[j]);
            } else {
                const float s4[4] = {scale, scale, scale, scale};
                const uint32_t t4[4] = {t0, t0, t0, t0};
                const int c4[4] = {0, 1, 2, 3};
#pragma unroll
                for (int c = 0; c < 4; c++) x[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int ks = 0; ks < D / 32; ks++)
#pragma unroll
                    for (int c = 0; c < 4; c++) x[c] = mfma16x16x32<MB>(a[ks], q[c][ks], x[c]);
                mass_scores<4, 4>(st, x, s4, t4, c4, hi, t0 + 16 > min(free_hi, hi));
            }
        },
        [&](uint32_t t0) {
            if constexpr (NT == 1) {
                const uint32_t t4[4] = {t0, t0 + 16, t0 + 32, t0 + 48};
                const int c4[4] = {0, 0, 0, 0};
                mass_scores<4, 1>(st, x, ss, t4, c4, hi, t0 + 64 > min(free_hi, hi));
            }
        });
}

__device__ __forceinline__ MassPages pages_for(const MassParams &p, const MassSeq &s) {
    const uint32_t pages = (s.n + (1u << p.page_shift) - 1) >> p.page_shift;
    return MassPages{p.pages + (size_t)s.trow * p.stride, min(pages, p.stride), 0, 0};
}

// Key `key` takes x: into its decayed weight, or (again) into what this call has given it already.
__device__ __forceinline__ void mass_add(const MassParams &p, const MassPages &w, const MassSeq &s, uint32_t h, uint32_t key,
                                         float x, bool again = false) {
    if (key >= s.n || (key >> p.page_shift) >= w.limit) return;
    const uint32_t page = w.table[key >> p.page_shift];
    if (page >= p.pool_pages) return;
    float *out = p.mass + (((size_t)page * p.hkv + h) << p.page_shift) + (key & ((1u << p.page_shift) - 1));
    if (again) *out += x;
    else *out = p.decay == 0.0f || (p.fresh && key >= s.p0) ? x : __builtin_fmaf(p.decay, *out, x);
}

// ------------------------------------------------------------------ few columns a sequence

// Workgroups of a streaming pass a CU, as many as its registers hold: with 64 columns a block two, with 16 four on MXFP4 pools
// and three on the others, whose tiles are four and two times as many registers.
template <int KVT, int NT>
constexpr uint32_t kFewPerCU = NT > 1 ? 2 : KVT == LIA_FP4 ? 4 : 3;

// Share w of `units` over G workgroups (G <= units, so that none is empty; further workgroups have none), and the share
// that owns a unit.
__device__ __forceinline__ uint32_t share_lo(uint32_t w, uint32_t units, uint32_t G) {
    return w < G ? (uint32_t)((uint64_t)w * units / G) : units;
}
__device__ __forceinline__ uint32_t share_of(uint32_t unit, uint32_t units, uint32_t G) {
    return (uint32_t)((((uint64_t)unit + 1) * G - 1) / units);
}

// A sequence's counts: units of its KV heads (the second pass's items), units of its column blocks of 16 NT columns (the
// first pass's), and those blocks.
template <int NT>
__device__ __forceinline__ uint3 few_counts(const MassParams &p, const MassSeq &s) {
    const uint32_t per = (s.n + kUnit - 1) / kUnit, blocks = p.hkv * ((s.cols + 16 * NT - 1) / (16 * NT));
    return make_uint3(p.hkv * per, blocks * per, blocks);
}

// First pass.  A share's part of a column block has slot (share + the block's index), unique as both only grow.
template <int D, int KVT, int NT>
__global__ __launch_bounds__(kMassThreads, (kFewPerCU<KVT, NT>)) void few_stats_kernel(MassParams p) {
    __shared__ MassScan sc;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kMassThreads / 64][kTileLds<D, KVT>];
    __shared__ float s_m[4][16 * NT], s_l[4][16 * NT];
    const uint32_t t_ = threadIdx.x, lane = t_ & 63, g = lane >> 4, li = lane & 15, G = gridDim.x;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(t_ >> 6));
    uint32_t base = 0; // slots of the scans before
    for (uint32_t first = 0; first < p.n_seqs; first += kMassSeqs) {
        mass_scan<kMassThreads>(p, sc, first, min(p.n_seqs - first, kMassSeqs),
                                [&](const MassSeq &s) { return few_counts<NT>(p, s); });
        const uint32_t units = uniform(sc.units[kMassSeqs]), shares = min(G, units);
        const uint32_t end = share_lo(blockIdx.x + 1, units, shares);
        for (uint32_t u = share_lo(blockIdx.x, units, shares); u < end;) {
            const uint32_t bi = owner_of(sc.units, u);
            const MassSeq s = seq_of(p, sc, bi);
            const uint32_t per = (s.n + kUnit - 1) / kUnit, rel = u - uniform(sc.units[bi]);
            const uint32_t block = rel / per, k0 = rel - block * per, k1 = min(per, k0 + (end - u));
            const uint32_t cbs = (s.cols + 16 * NT - 1) / (16 * NT), h = block / cbs, col0 = (block - h * cbs) * 16 * NT;
            MassPages w = pages_for(p, s);
            const uint32_t lo = k0 * kUnit + 64 * wave, hi = min(k1 * kUnit, s.n);
            pages_at(w, lo >> p.page_shift);
            MassState<NT> st;
            u32x4 q[NT][D / 32];
            mass_begin<D, KVT, NT>(p, s, h, col0, st, q);
            const uint32_t free_hi = s.p0 + div_group(p, col0) + 1;
            mass_first<D, KVT, NT>(p, w, lo, hi, kUnit, h, lds[wave], q, st, free_hi);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                float M, L;
                mass_end<NT>(st, nt, M, L);
                if (g == 0) { s_m[wave][16 * nt + li] = M; s_l[wave][16 * nt + li] = L; }
            }
            lds_barrier();
            const uint32_t slot = base + blockIdx.x + uniform(sc.blocks[bi]) + block;
            if (t_ < 16 * NT && slot < p.slots) {
                float M = -INFINITY, L = 0.0f;
#pragma unroll
                for (int v = 0; v < 4; v++)
                    if (s_l[v][t_] != 0.0f) M = fmaxf(M, s_m[v][t_]);
#pragma unroll
                for (int v = 0; v < 4; v++)
                    if (s_l[v][t_] != 0.0f) L += s_l[v][t_] * fast_exp2(s_m[v][t_] - M);
                p.stats[(size_t)slot * 16 * NT + t_] = make_float2(M, L);
            }
            lds_barrier();
            u += k1 - k0;
        }
        base += G + uniform(sc.blocks[kMassSeqs]);
        __syncthreads(); // the scan is rewritten
    }
}

// Second pass: 64 keys a wave (K as the B operand: lane (g, li) of tile j holds key 16j + li against columns 4g ..
// 4g+3 of a column tile), a column block of 16 NT columns at a time, whose lse all threads merge from the first pass's slots
// when a segment begins.  Sequences of more columns go over their segment once a block and add to what the blocks
// before left (a lane meets its own keys again).
template <int D, int KVT, int NT>
__global__ __launch_bounds__(kMassThreads, (kFewPerCU<KVT, NT>)) void few_sums_kernel(MassParams p, uint32_t stat_groups) {
    constexpr int KT = D / 32;
    constexpr uint32_t COLS = 16 * NT, PARTS = kMassThreads / COLS, BATCH = 4;
    __shared__ MassScan sc;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kMassThreads / 64][kTileLds<D, KVT>];
    __shared__ __attribute__((aligned(16))) float s_lse[COLS];
    __shared__ float s_m[PARTS][COLS], s_l[PARTS][COLS];
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15, G = gridDim.x;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    uint32_t base = 0;
    for (uint32_t first = 0; first < p.n_seqs; first += kMassSeqs) {
        mass_scan<kMassThreads>(p, sc, first, min(p.n_seqs - first, kMassSeqs),
                                [&](const MassSeq &s) { return few_counts<NT>(p, s); });
        const uint32_t items = uniform(sc.items[kMassSeqs]), stat_units = uniform(sc.units[kMassSeqs]);
        const uint32_t shares = min(G, items), stat_shares = min(stat_groups, stat_units);
        const uint32_t end = share_lo(blockIdx.x + 1, items, shares);
        for (uint32_t u = share_lo(blockIdx.x, items, shares); u < end;) {
            const uint32_t bi = owner_of(sc.items, u);
            const MassSeq s = seq_of(p, sc, bi);
            const uint32_t per = (s.n + kUnit - 1) / kUnit, rel = u - uniform(sc.items[bi]);
            const uint32_t h = rel / per, k0 = rel - h * per, k1 = min(per, k0 + (end - u));
            const uint32_t cbs = (s.cols + COLS - 1) / COLS;
            const uint32_t lo = k0 * kUnit + 64 * wave, hi = min(k1 * kUnit, s.n);
            u += k1 - k0;
#pragma unroll 1
            for (uint32_t cb = 0; cb < cbs; cb++) {
                const uint32_t col0 = cb * COLS;
                MassPages w = pages_for(p, s);
                pages_at(w, lo >> p.page_shift);
                u32x4 q[NT][KT];
                load_queries<D, KVT, NT>(p, s, h, col0, q);
                {
                    const uint32_t c = threadIdx.x % COLS, part = threadIdx.x / COLS, id = h * cbs + cb;
                    const uint32_t x0 = uniform(sc.units[bi]) + id * per, w0 = share_of(x0, stat_units, stat_shares);
                    const uint32_t parts = share_of(x0 + per - 1, stat_units, stat_shares) - w0 + 1;
                    const uint32_t slot0 = base + w0 + uniform(sc.blocks[bi]) + id;
                    float M = -INFINITY, L = 0.0f;
                    for (uint32_t i = part; i < parts; i += PARTS * BATCH) {
                        float2 x[BATCH];
#pragma unroll
                        for (uint32_t k = 0; k < BATCH; k++)
                            x[k] = p.stats[(size_t)min(slot0 + min(i + PARTS * k, parts - 1), p.slots - 1) * COLS + c];
                        float nm = M;
#pragma unroll
                        for (uint32_t k = 0; k < BATCH; k++)
                            if (i + PARTS * k < parts && x[k].y != 0.0f) nm = fmaxf(nm, x[k].x);
                        if (L != 0.0f) L *= fast_exp2(M - nm);
                        M = nm;
#pragma unroll
                        for (uint32_t k = 0; k < BATCH; k++)
                            if (i + PARTS * k < parts && x[k].y != 0.0f) L += x[k].y * fast_exp2(x[k].x - M);
                    }
                    s_m[part][c] = M;
                    s_l[part][c] = L;
                    lds_barrier();
                    if (threadIdx.x < COLS) {
                        M = -INFINITY; L = 0.0f;
#pragma unroll
                        for (uint32_t v = 0; v < PARTS; v++)
                            if (s_l[v][c] != 0.0f) M = fmaxf(M, s_m[v][c]);
#pragma unroll
                        for (uint32_t v = 0; v < PARTS; v++)
                            if (s_l[v][c] != 0.0f) L += s_l[v][c] * fast_exp2(s_m[v][c] - M);
                        s_lse[c] = col0 + c < s.cols ? M + __builtin_amdgcn_logf(L) : INFINITY; // log2; no column: weight 0
                    }
                    lds_barrier();
                }
                const uint32_t free_hi = s.p0 + div_group(p, col0) + 1; // live for all of the block's columns
                const bool pad = s.cols - col0 < COLS;                  // columns that are none
                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                // a tile's weights, summed over the lane's columns; hidden: some pair is, or a column is none
                auto weigh = [&](uint32_t t0, int nt, const f32x4 &x, float ss, auto hidden) {
                    const f32x4 lse = *(const f32x4 *)&s_lse[16 * nt + 4 * g];
                    float e[4];
#pragma unroll
                    for (int i = 0; i < 4; i++) e[i] = fast_exp2(__builtin_fmaf(x[i], ss, -lse[i]));
                    if constexpr (hidden) {
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const uint32_t col = col0 + 16 * nt + 4 * g + i;
                            if (col >= s.cols || t0 + li > s.p0 + div_group(p, col)) e[i] = 0.0f;
                        }
                    }
                    return (e[0] + e[1]) + (e[2] + e[3]);
                };
                f32x4 x[4];
                float sss[4];
                mass_stream<D, KVT>(
                    p, w, lo, hi, kUnit, h, lds[wave],
                    [&](uint32_t t0, int j, const u32x4 (&b)[KT], float ss) {
                        if constexpr (NT == 1) {
                            x[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
                            sss[j] = ss;
#pragma unroll
                            for (int ks = 0; ks < KT; ks++) x[j] = mfma16x16x32<KTile<D, KVT>::MB>(q[0][ks], b[ks], x[j]);
                        } else {
#pragma unroll
                            for (int c = 0; c < NT; c++) x[c] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                            for (int ks = 0; ks < KT; ks++)
#pragma unroll
                                for (int c = 0; c < NT; c++) x[c] = mfma16x16x32<KTile<D, KVT>::MB>(q[c][ks], b[ks], x[c]);
                            if (pad || t0 + 16 > free_hi) {
#pragma unroll
                                for (int c = 0; c < NT; c++) acc[j] += weigh(t0, c, x[c], ss, std::true_type{});
                            } else {
#pragma unroll
                                for (int c = 0; c < NT; c++) acc[j] += weigh(t0, c, x[c], ss, std::false_type{});
                            }
                        }
                    },
                    [&](uint32_t t0) { // the wave's 64 keys
                        if constexpr (NT == 1) {
                            if (t0 + 64 > free_hi) {
#pragma unroll
                                for (int j = 0; j < 4; j++) acc[j] = weigh(t0 + 16 * j, 0, x[j], sss[j], std::true_type{});
                            } else {
#pragma unroll
                                for (int j = 0; j < 4; j++) acc[j] = weigh(t0 + 16 * j, 0, x[j], sss[j], std::false_type{});
                            }
                        }
                        float mine = 0.0f;
#pragma unroll
                        for (int i = 0; i < 4; i++) {
                            const float y = rows_sum(acc[i]);
                            if (g == (uint32_t)i) mine = y;
                            acc[i] = 0.0f;
                        }
                        mass_add(p, w, s, h, t0 + lane, mine, cb > 0);
                    });
                lds_barrier(); // the lse is rewritten
            }
        }
        base += stat_groups + uniform(sc.blocks[kMassSeqs]);
        __syncthreads(); // the scan is rewritten
    }
}

// ------------------------------------------------------------------ prompt chunks

// Columns are padded so that a sequence's begin at a multiple of 16.
__device__ __forceinline__ uint32_t column_base(const MassParams &p, const MassSeq &s, uint32_t b) {
    return 16 * (s.r0 * p.group / 16 + b);
}

// Both passes go over blocks of a KV head in units of equal work, laid end to end over heads and sequences; every workgroup
// takes one contiguous share.  A block within a share is finished by it; of others it leaves its part, at most two: of the
// block it enters the share in (0) and of the one it leaves it in (1).  The share that begins a block notes it, and a
// small kernel merges the parts in the shares' order.  A block is charged a lead of further units for what a share spends
// before its first tile and after its last, so that shares of two blocks end with the others: 512 and 300 rows of 16 heads
// over 4,608 and 2,001 bf16 keys, shares of 5 units and of 11, took 60.0 us with leads of 0, 57.5 of 1 and 3, 55.8 of 2 and
// 6, 55.2 of 3 and 6, 55.0 of 4 and 12.

// The block of `blocks` (up to 2^24: there are none of more than 2^23, 512 keys each) that owns unit rel, units before a
// block given by before() (which grows), wave-uniform.
template <class F>
__device__ __forceinline__ uint32_t block_of(uint32_t blocks, uint32_t rel, F &&before) {
    uint32_t lo = 0;
    for (uint32_t stride = blocks > 262144 ? 262144 : blocks > 4096 ? 4096 : blocks > 64 ? 64 : 1; stride; stride >>= 6) {
        const uint32_t i = lo + lane_id() * stride;
        lo += ((uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(i < blocks && before(i) <= rel)) - 1) * stride;
    }
    return lo;
}

// First pass: blocks of 256 columns in units of 64 keys.  Block i has units up to its last row's position and at most one more:
// ceil(p0 / 64) + ceil(4 (i + 1) / group).  Units of the first n blocks, leads and all.
__device__ __forceinline__ uint32_t stat_units(const MassParams &p, const MassSeq &s, uint32_t n) {
    const uint32_t G = p.group, a = div_group(p, n), r = n - a * G;
    uint32_t full = 0, rest = 0; // of a period of `group` blocks
#pragma unroll
    for (uint32_t k = 0; k < 4; k++) {
        const uint32_t from = k * G / 4;
        full += G - from;
        rest += r > from ? r - from : 0;
    }
    const uint32_t tri = a & 1 ? a * ((a - 1) / 2) : a / 2 * (a - 1); // a (a - 1) / 2 (modulo 2^32, as the rest)
    return ((s.p0 + 63) / 64 + kStatLead) * n + a * full + 4 * G * tri + 4 * a * r + rest;
}
__device__ __forceinline__ uint32_t stat_blocks(const MassSeq &s) { return (s.cols + kBlockCols - 1) / kBlockCols; }

template <int D, int KVT>
__global__ __launch_bounds__(kMassThreads, 2) void chunk_stats_kernel(MassParams p) {
    constexpr int NT = 4;
    __shared__ MassScan sc;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kMassThreads / 64][kTileLds<D, KVT>];
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15, G = gridDim.x;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    uint32_t share = blockIdx.x; // ... of this scan's
    for (uint32_t first = 0; first < p.n_seqs; first += kMassSeqs, share += G) {
        mass_scan<kMassThreads>(p, sc, first, min(p.n_seqs - first, kMassSeqs), [&](const MassSeq &s) {
            return make_uint3(p.hkv * stat_units(p, s, stat_blocks(s)), 0, 0);
        });
        const uint32_t units = uniform(sc.items[kMassSeqs]), shares = min(G, units);
        const uint32_t end = share_lo(blockIdx.x + 1, units, shares);
        uint4 begun = make_uint4(kNoBlock, 0, 0, 0);
        for (uint32_t u = share_lo(blockIdx.x, units, shares); u < end;) {
            const uint32_t bi = owner_of(sc.items, u);
            const MassSeq s = seq_of(p, sc, bi);
            const uint32_t blocks = stat_blocks(s), head = stat_units(p, s, blocks);
            uint32_t rel = u - uniform(sc.items[bi]);
            const uint32_t h = rel / head;
            rel -= h * head;
            const uint32_t cb = block_of(blocks, rel, [&](uint32_t i) { return stat_units(p, s, i); });
            const uint32_t b0 = stat_units(p, s, cb), len = stat_units(p, s, cb + 1) - b0;
            const uint32_t take = min(b0 + len - rel, end - u), last_share = share_of(u - (rel - b0) + len - 1, units, shares);
            const uint32_t k0 = max(rel - b0, kStatLead) - kStatLead, k1 = max(rel - b0 + take, kStatLead) - kStatLead;
            u += take;
            if (k1 == 0) continue; // of the lead alone
            const uint32_t col0 = cb * kBlockCols + wave * 64, c0 = column_base(p, s, first + bi) + cb * kBlockCols;
            const bool whole = k0 == 0 && k1 + kStatLead == len;
            if (col0 < s.cols) {
                // keys past the wave's last row's position are no column's
                const uint32_t last = s.p0 + div_group(p, min(col0 + 63, s.cols - 1)) + 1;
                const uint32_t lo = k0 * 64, hi = min(k1 * 64, last);
                MassPages w = pages_for(p, s);
                pages_at(w, lo >> p.page_shift);
                MassState<NT> st;
                u32x4 q[NT][D / 32];
                mass_begin<D, KVT, NT>(p, s, h, col0, st, q);
                if (k0 == 0) { // for the second pass
                    uint4 *out = p.queries + ((size_t)h * p.columns + c0 + wave * 64) / 16 * (D / 32) * 64 + lane;
#pragma unroll
                    for (int nt = 0; nt < NT; nt++)
                        if (col0 + 16 * nt < s.cols) {
#pragma unroll
                            for (int ks = 0; ks < D / 32; ks++)
                                out[(nt * (D / 32) + ks) * 64] = make_uint4(q[nt][ks].x, q[nt][ks].y, q[nt][ks].z, q[nt][ks].w);
                        }
                }
                const uint32_t free_hi = s.p0 + div_group(p, col0) + 1;
                mass_first<D, KVT, NT>(p, w, lo, hi, 64, h, lds[wave], q, st, free_hi);
                float *lse = p.lse + (size_t)h * p.columns + c0 + wave * 64;
                float2 *part = p.stats + ((size_t)share * 2 + (k0 == 0)) * kBlockCols + wave * 64;
#pragma unroll
                for (int nt = 0; nt < NT; nt++) {
                    float M, L;
                    mass_end<NT>(st, nt, M, L);
                    const uint32_t c = 16 * nt + li;
                    if (g == 0 && col0 + c < s.cols) {
                        if (whole) lse[c] = M + __builtin_amdgcn_logf(L); // log2
                        else part[c] = make_float2(M, L);
                    }
                }
            }
            if (k0 == 0 && !whole)
                begun = make_uint4(h, c0, min(s.cols - cb * kBlockCols, kBlockCols), last_share);
        }
        if (threadIdx.x == 0) p.begun[0][share] = begun;
        __syncthreads(); // the scan is rewritten
    }
}

// The lse of the blocks that several shares have parts of, a thread a column.
__global__ __launch_bounds__(kBlockCols) void chunk_lse_kernel(MassParams p, uint32_t G) {
    constexpr uint32_t BATCH = 8;
    const uint4 b = p.begun[0][blockIdx.x];
    const uint32_t c = threadIdx.x;
    if (b.x == kNoBlock || c >= b.z) return;
    const uint32_t parts = b.w - blockIdx.x % G + 1;
    const float2 *x = p.stats + (size_t)blockIdx.x * 2 * kBlockCols + c; // the first part is in the share's second place
    float M = -INFINITY, L = 0.0f;
    for (uint32_t i = 0; i < parts; i += BATCH) {
        float2 v[BATCH];
#pragma unroll
        for (uint32_t k = 0; k < BATCH; k++) {
            const uint32_t n = min(i + k, parts - 1);
            v[k] = x[(size_t)(n ? 2 * n : 1) * kBlockCols];
            if (i + k >= parts) v[k].y = 0.0f;
        }
        float nm = M;
#pragma unroll
        for (uint32_t k = 0; k < BATCH; k++)
            if (v[k].y != 0.0f) nm = fmaxf(nm, v[k].x);
        if (L != 0.0f) L *= fast_exp2(M - nm);
        M = nm;
#pragma unroll
        for (uint32_t k = 0; k < BATCH; k++)
            if (v[k].y != 0.0f) L += v[k].y * fast_exp2(v[k].x - M);
    }
    p.lse[(size_t)b.x * p.columns + b.y + c] = M + __builtin_amdgcn_logf(L); // log2
}

// Second pass: blocks of 512 keys in units of 16 columns.  Block i begins at the unit that holds the first column that attends
// its first key, floor((512 i - p0) group / 16).
constexpr uint32_t kBlockSkip = kBlockKeys / 16; // ... units a block later, by the group
__device__ __forceinline__ uint32_t sum_first(const MassParams &p, const MassSeq &s, uint32_t i) {
    const uint32_t y = (s.p0 * p.group + 15) / 16, x = i * kBlockSkip * p.group;
    return x > y ? x - y : 0;
}
// Units of the first n blocks, leads and all.
__device__ __forceinline__ uint32_t sum_units(const MassParams &p, const MassSeq &s, uint32_t n) {
    const uint32_t y = (s.p0 * p.group + 15) / 16, from = div_group(p, y / kBlockSkip) + 1; // first block that skips units
    auto tri = [](uint32_t a) { return a & 1 ? a * ((a - 1) / 2) : a / 2 * (a - 1); };
    uint32_t x = ((s.cols + 15) / 16 + kSumLead) * n;
    if (n > from) x -= kBlockSkip * p.group * (tri(n) - tri(from)) - y * (n - from);
    return x;
}

// Every wave holds its 128 keys' operands in registers and goes over the share's column tiles; the next tile's queries,
// which the four waves read together, are on their way.
template <int D, int KVT>
__global__ __launch_bounds__(kMassThreads, 2) void chunk_sums_kernel(MassParams p) {
    constexpr int KT = D / 32, TILES = 8;
    constexpr uint32_t KEYS = 16 * TILES;
    __shared__ MassScan sc;
    __shared__ __attribute__((aligned(16))) uint8_t lds[kMassThreads / 64][kTileLds<D, KVT>];
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15, G = gridDim.x;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    uint32_t own = blockIdx.x;
    for (uint32_t first = 0; first < p.n_seqs; first += kMassSeqs, own += G) {
        mass_scan<kMassThreads>(p, sc, first, min(p.n_seqs - first, kMassSeqs), [&](const MassSeq &s) {
            return make_uint3(p.hkv * sum_units(p, s, (s.n + kBlockKeys - 1) / kBlockKeys), 0, 0);
        });
        const uint32_t units = uniform(sc.items[kMassSeqs]), shares = min(G, units);
        const uint32_t stop = share_lo(blockIdx.x + 1, units, shares);
        uint4 begun = make_uint4(kNoBlock, 0, 0, 0);
        for (uint32_t u = share_lo(blockIdx.x, units, shares); u < stop;) {
            const uint32_t bi = owner_of(sc.items, u);
            const MassSeq s = seq_of(p, sc, bi);
            const uint32_t blocks = (s.n + kBlockKeys - 1) / kBlockKeys, head = sum_units(p, s, blocks);
            uint32_t rel = u - uniform(sc.items[bi]);
            const uint32_t h = rel / head;
            rel -= h * head;
            const uint32_t kb = block_of(blocks, rel, [&](uint32_t i) { return sum_units(p, s, i); });
            const uint32_t b0 = sum_units(p, s, kb), len = sum_units(p, s, kb + 1) - b0;
            const uint32_t take = min(b0 + len - rel, stop - u), last_share = share_of(u - (rel - b0) + len - 1, units, shares);
            const uint32_t j0 = max(rel - b0, kSumLead) - kSumLead, j1 = max(rel - b0 + take, kSumLead) - kSumLead;
            const uint32_t t = kb * kBlockKeys + wave * KEYS;
            const bool whole = j0 == 0 && j1 + kSumLead == len;
            u += take;
            if (j1 == 0) continue; // of the lead alone
            if (j0 == 0 && !whole) begun = make_uint4(first + bi, h, kb * kBlockKeys, last_share);
            if (t >= s.n) continue; // (no barrier in the loop)
            MassPages w = pages_for(p, s);
            pages_at(w, t >> p.page_shift);
            const uint32_t from = sum_first(p, s, kb), end = from + j1;
            uint32_t nt = from + j0;
            const uint32_t c0 = column_base(p, s, first + bi);
            const __amdgpu_buffer_rsrc_t rq = make_rsrc(p.queries + ((size_t)h * p.columns + c0) / 16 * KT * 64,
                                                        (s.cols + 15) / 16 * KT * 1024);
            const __amdgpu_buffer_rsrc_t rl = make_rsrc(p.lse + (size_t)h * p.columns + c0, (s.cols + 15) / 16 * 64);
            auto query = [&](uint32_t tile, u32x4 (&q)[KT], f32x4 &lse) {
#pragma unroll
                for (int ks = 0; ks < KT; ks++) q[ks] = buffer_load16(rq, (tile * KT + ks) * 1024 + lane * 16);
                lse = __builtin_bit_cast(f32x4, buffer_load16(rl, tile * 64 + g * 16));
            };
            u32x4 q[KT], qn[KT], b[TILES][KT];
            float ss[TILES], acc[TILES];
            f32x4 lse, lsen;
            query(nt, q, lse);
            {
                KTile<D, KVT> k[TILES];
#pragma unroll
                for (int j = 0; j < TILES; j++)
                    load_tile<D, KVT>(p, k[j], t + 16 * j, s.n, page_of(w, (t + 16 * j) >> p.page_shift), h);
#pragma unroll
                for (int j = 0; j < TILES; j++) {
                    ss[j] = score_scale(p, k[j]);
                    operands<D, KVT>(k[j], lds[wave], b[j]);
                    acc[j] = 0.0f;
                    __builtin_amdgcn_sched_barrier(0);
                }
            }
#pragma unroll 1
            for (; nt < end; nt++) {
                query(nt + 1, qn, lsen);
                const bool masked = t + KEYS > s.p0 + div_group(p, 16 * nt) + 1 || 16 * nt + 16 > s.cols;
                uint32_t lim[4];
                if (masked) {
#pragma unroll
                    for (int i = 0; i < 4; i++) {
                        const uint32_t col = 16 * nt + 4 * g + i;
                        lim[i] = col < s.cols ? s.p0 + div_group(p, col) + 1 : 0;
                    }
                }
                // Two tiles' products are on their way while the exponentials of the two before are summed.
                auto tiles = [&](auto hidden) { // (two bodies: a branch in each tile would keep them apart)
                    f32x4 x[2][2];
                    auto products = [&](int j) {
#pragma unroll
                        for (int i = 0; i < 2; i++) x[j / 2 & 1][i] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int ks = 0; ks < KT; ks++)
#pragma unroll
                            for (int i = 0; i < 2; i++)
                                x[j / 2 & 1][i] = mfma16x16x32<KTile<D, KVT>::MB>(q[ks], b[j + i][ks], x[j / 2 & 1][i]);
                    };
                    products(0);
#pragma unroll
                    for (int j = 0; j < TILES; j += 2) {
                        if (j + 2 < TILES) products(j + 2);
                        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
                        for (int i = 0; i < 2; i++) {
                            float e[4];
#pragma unroll
                            for (int c = 0; c < 4; c++)
                                e[c] = fast_exp2(__builtin_fmaf(x[j / 2 & 1][i][c], ss[j + i], -lse[c]));
                            if constexpr (hidden) {
#pragma unroll
                                for (int c = 0; c < 4; c++)
                                    if (t + 16 * (j + i) + li >= lim[c]) e[c] = 0.0f;
                            }
                            acc[j + i] += (e[0] + e[1]) + (e[2] + e[3]);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
                };
                if (masked) tiles(std::true_type{});
                else tiles(std::false_type{});
#pragma unroll
                for (int ks = 0; ks < KT; ks++) q[ks] = qn[ks];
                lse = lsen;
            }
#pragma unroll
            for (int i = 0; i < TILES / 4; i++) { // lane (g, li): key 16 g + li of these 64
                float mine = 0.0f;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float y = rows_sum(acc[4 * i + j]);
                    if (g == (uint32_t)j) mine = y;
                }
                if (whole) mass_add(p, w, s, h, t + 64 * i + lane, mine);
                else p.sums[((size_t)own * 2 + (j0 == 0)) * kBlockKeys + wave * KEYS + 64 * i + lane] = mine;
            }
        }
        if (threadIdx.x == 0) p.begun[1][own] = begun;
        __syncthreads(); // the scan is rewritten
    }
}

// The sums of the blocks that several shares have parts of, a thread a key.
__global__ __launch_bounds__(kBlockKeys) void chunk_add_kernel(MassParams p, uint32_t G) {
    constexpr uint32_t BATCH = 8;
    const uint4 b = p.begun[1][blockIdx.x];
    if (b.x == kNoBlock) return;
    MassSeq s;
    s.r0 = p.cu[b.x];
    s.rows = min(p.cu[b.x + 1] - s.r0, p.n_rows - s.r0);
    s.p0 = p.positions[s.r0];
    s.trow = p.sequences[s.r0];
    s.n = s.p0 + s.rows;
    s.cols = s.rows * p.group;
    if (b.z + threadIdx.x >= s.n) return; // (waves of no keys leave no parts)
    const uint32_t parts = b.w - blockIdx.x % G + 1;
    const float *x = p.sums + (size_t)blockIdx.x * 2 * kBlockKeys + threadIdx.x;
    float sum = 0.0f;
    for (uint32_t i = 0; i < parts; i += BATCH) {
        float v[BATCH];
#pragma unroll
        for (uint32_t k = 0; k < BATCH; k++) {
            const uint32_t n = min(i + k, parts - 1);
            v[k] = x[(size_t)(n ? 2 * n : 1) * kBlockKeys];
        }
#pragma unroll
        for (uint32_t k = 0; k < BATCH; k++)
            if (i + k < parts) sum += v[k];
    }
    mass_add(p, pages_for(p, s), s, b.y, b.z + threadIdx.x, sum);
}

// ------------------------------------------------------------------ host side

struct MassLaunch {
    uint32_t cus, scans;
    uint64_t few_units; // an upper bound, from the configuration's context
    bool chunks, narrow;
};

template <int D, int KVT, int NT>
static hipError_t launch_few(const MassParams &p, const MassLaunch &n, hipStream_t s) {
    const uint32_t G = (uint32_t)std::min<uint64_t>(std::max<uint64_t>(n.few_units, 1), kFewPerCU<KVT, NT> * n.cus);
    const hipError_t e = launch<few_stats_kernel<D, KVT, NT>>(dim3(G), dim3(kMassThreads), 0, s, p);
    if (e != hipSuccess) return e;
    return launch<few_sums_kernel<D, KVT, NT>>(dim3(G), dim3(kMassThreads), 0, s, p, G);
}

template <int D, int KVT>
static hipError_t launch_weights(const MassParams &p, const MassLaunch &n, hipStream_t s) {
    if (!n.chunks) return n.narrow ? launch_few<D, KVT, 1>(p, n, s) : launch_few<D, KVT, 4>(p, n, s);
    const uint32_t G = 2 * n.cus; // what the CUs hold
    hipError_t e = launch<chunk_stats_kernel<D, KVT>>(dim3(G), dim3(kMassThreads), 0, s, p);
    if (e == hipSuccess) e = launch<chunk_lse_kernel>(dim3(G * n.scans), dim3(kBlockCols), 0, s, p, G);
    if (e == hipSuccess) e = launch<chunk_sums_kernel<D, KVT>>(dim3(G), dim3(kMassThreads), 0, s, p);
    if (e == hipSuccess) e = launch<chunk_add_kernel>(dim3(G * n.scans), dim3(kBlockKeys), 0, s, p, G);
    return e;
}

template <int D>
static hipError_t launch_weights_kv(int kv, const MassParams &p, const MassLaunch &n, hipStream_t s) {
    if (kv == LIA_BF16) return launch_weights<D, LIA_BF16>(p, n, s);
    if (kv == LIA_F16) return launch_weights<D, LIA_F16>(p, n, s);
    if (kv == LIA_FP4) return launch_weights<D, LIA_FP4>(p, n, s);
    return launch_weights<D, LIA_FP8_E4M3>(p, n, s);
}

static uint32_t mass_cus() {
    const uint32_t c = device_cus();
    return c ? c : 256;
}

static uint64_t mass_scans(uint64_t n_seqs) { return (n_seqs + kMassSeqs - 1) / kMassSeqs; }

// Slots of the streaming form's first pass in blocks of `cols` columns: one a share and scan, one a column block.
static uint64_t few_slots(const lia_attention_config *c, uint64_t cols) {
    const uint64_t group = c->num_q_heads / c->num_kv_heads;
    return mass_scans(c->max_seqs) * 4 * mass_cus() +
           (uint64_t)c->num_kv_heads * ((uint64_t)c->max_rows * group / cols + c->max_seqs);
}

// Workspace: either form's arrays.
static uint64_t mass_bytes(const lia_attention_config *c) {
    const uint64_t columns = (uint64_t)c->max_rows * (c->num_q_heads / c->num_kv_heads), hkv = c->num_kv_heads;
    const uint64_t share = 2 * (kBlockCols * sizeof(float2) + kBlockKeys * sizeof(float) + sizeof(uint4));
    const uint64_t padded = (columns + 16 * (uint64_t)c->max_seqs + 15) / 16 * 16;
    const uint64_t chunks = mass_scans(c->max_seqs) * 2 * mass_cus() * share + padded * hkv * (2 * c->head_dim + sizeof(float));
    const uint64_t narrow = few_slots(c, 16) * 16 * sizeof(float2), wide = few_slots(c, 64) * 64 * sizeof(float2);
    return std::max(chunks, std::max(narrow, wide));
}

} // namespace lia

using namespace lia;

static int validate_weights(const lia_attention_config *c) {
    if (!c) return LIA_E_ARG;
    if (c->num_kv_heads == 0 || c->num_q_heads == 0 || c->num_q_heads % c->num_kv_heads) return LIA_E_ARG;
    if (c->num_q_heads / c->num_kv_heads > 32) return LIA_E_UNSUPPORTED;
    if (c->head_dim != 64 && c->head_dim != 128) return LIA_E_UNSUPPORTED;
    if (c->page_size < 16 || (c->page_size & (c->page_size - 1))) return LIA_E_UNSUPPORTED;
    if (c->q_dtype != LIA_F32 && c->q_dtype != LIA_BF16) return LIA_E_UNSUPPORTED;
    if (c->kv_dtype != LIA_F16 && c->kv_dtype != LIA_BF16 && c->kv_dtype != LIA_FP8_E4M3 && c->kv_dtype != LIA_FP4)
        return LIA_E_UNSUPPORTED;
    if (c->stride == 0 || c->max_seqs == 0 || c->max_rows == 0 || c->max_context == 0) return LIA_E_ARG;
    if (!(c->scale > 0.0f) || !(c->scale < INFINITY)) return LIA_E_ARG;
    // the queries are read through one 32-bit buffer range, a page through another
    if ((uint64_t)c->max_rows * c->num_q_heads * c->head_dim * 4 >= (1ull << 31) ||
        (uint64_t)c->page_size * c->num_kv_heads * c->head_dim * 2 >= (1ull << 31))
        return LIA_E_UNSUPPORTED;
    // Units of work are counted in 32 bits, those of a scan's sequences together, and so are keys (of up to a block or a
    // step past the last) and a key's columns.  (By the bounds above, no product below reaches 2^64.)
    const uint64_t keys = std::min<uint64_t>(c->max_context, (uint64_t)c->stride * c->page_size);
    const uint64_t heads = c->num_kv_heads, group = c->num_q_heads / c->num_kv_heads, columns = c->max_rows * group;
    const uint64_t seqs = std::min<uint64_t>(c->max_seqs, kMassSeqs);
    const uint64_t chunks = std::min<uint64_t>(seqs, c->max_rows / 16); // (16 rows and more a sequence)
    // few columns: 256 keys by 16 columns
    const uint64_t few = heads * (seqs + columns / 16) * (keys / 256 + 1);
    // prompt chunks, blocks of 256 columns: units of 64 keys up to the block's last row's position - those before the rows and
    // those of rows rounded up apart, and up to four more where the block is not full - and the lead
    const uint64_t stats = heads * (chunks + columns / 256) * (keys / 64 + 7 + kStatLead);
    // ... and blocks of 512 keys: units of 16 columns and the lead
    const uint64_t sums = heads * ((1 + kSumLead) * chunks + columns / 16) * (keys / 512 + 1);
    // slots and padded columns
    const uint64_t places = std::max(few_slots(c, 16), columns + 16 * (uint64_t)c->max_seqs + 16);
    if (std::max(std::max(few, stats), std::max(sums, places)) >= (1ull << 32) || (keys + 1024) * group >= (1ull << 32))
        return LIA_E_UNSUPPORTED;
    return LIA_OK;
}

extern "C" size_t lia_attention_weights_workspace_bytes(const lia_attention_config *c) {
    return validate_weights(c) == LIA_OK ? (size_t)mass_bytes(c) : 0;
}

extern "C" int lia_attention_weights(const lia_attention_config *c, uint32_t n_seqs, uint32_t n_rows,
                                     const uint32_t *cu_seqlens, const uint32_t *positions,
                                     const uint32_t *sequences, const uint32_t *pages, const void *q,
                                     const void *kc, const float *k_scales, float decay, int32_t fresh,
                                     float *mass, void *workspace, size_t workspace_bytes, lia_stream_t stream) {
    if (const int st = validate_weights(c)) return st;
    if (n_seqs == 0 || n_seqs > c->max_seqs || n_rows == 0 || n_rows > c->max_rows) return LIA_E_ARG;
    if (!cu_seqlens || !positions || !sequences || !pages || !q || !kc || !mass || !workspace) return LIA_E_ARG;
    if ((c->kv_dtype == LIA_FP8_E4M3 || c->kv_dtype == LIA_FP4) && !k_scales) return LIA_E_ARG;
    if (!(decay >= 0.0f) || !(decay < INFINITY)) return LIA_E_ARG;
    if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)workspace) & 15) return LIA_E_ALIGN;
    if ((uintptr_t)mass & 3) return LIA_E_ALIGN;
    if (workspace_bytes < mass_bytes(c)) return LIA_E_WORKSPACE;
    const uint32_t group = c->num_q_heads / c->num_kv_heads;
    MassParams p;
    p.q = q; p.kc = kc; p.k_scales = k_scales;
    p.cu = cu_seqlens; p.positions = positions; p.sequences = sequences; p.pages = pages;
    p.mass = mass;
    const uint32_t cus = mass_cus();
    // Prompt chunks: 16 and more rows a sequence on average (the prefill kernel's batches).  Below, column blocks of 16
    // where sequences have no more on average (decode), else of 64, which read their keys once for four blocks.
    MassLaunch n;
    n.cus = cus;
    n.scans = (uint32_t)mass_scans(n_seqs);
    n.chunks = n_rows >= 16 * n_seqs;
    n.narrow = n_rows * group <= 16 * n_seqs;
    const uint64_t context = c->max_context, heads = c->num_kv_heads;
    n.few_units = heads * (n_seqs + (uint64_t)n_rows * group / (n.narrow ? 16 : 64)) * ((context + kUnit - 1) / kUnit);
    p.columns = (n_rows * group + 16 * n_seqs + 15) / 16 * 16;
    const uint64_t shares = 2 * (uint64_t)cus * n.scans;
    p.stats = (float2 *)workspace;
    p.slots = (uint32_t)few_slots(c, n.narrow ? 16 : 64);
    p.begun[0] = (uint4 *)(p.stats + shares * 2 * kBlockCols);
    p.begun[1] = p.begun[0] + shares;
    p.sums = (float *)(p.begun[1] + shares);
    p.lse = p.sums + shares * 2 * kBlockKeys;
    p.queries = (uint4 *)(p.lse + heads * p.columns);
    p.hq = c->num_q_heads; p.hkv = c->num_kv_heads; p.group = group;
    p.group_magic = group > 1 ? (uint32_t)((1ull << 32) / group) + 1 : 0; // floor(col / group) for col < 2^27
    p.stride = c->stride;
    p.page_shift = (uint32_t)__builtin_ctz(c->page_size);
    p.pool_pages = c->pool_pages;
    p.n_seqs = n_seqs; p.n_rows = n_rows;
    p.scale_log2 = c->scale * 1.4426950408889634f;
    p.decay = decay;
    p.q_f32 = c->q_dtype == LIA_F32;
    p.fresh = fresh != 0;
    hipStream_t st = (hipStream_t)stream;
    const hipError_t e = c->head_dim == 128 ? launch_weights_kv<128>(c->kv_dtype, p, n, st)
                                            : launch_weights_kv<64>(c->kv_dtype, p, n, st);
    return e == hipSuccess ? LIA_OK : LIA_E_HIP;
}
