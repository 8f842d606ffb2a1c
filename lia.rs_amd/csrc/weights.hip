// Accumulated attention weights of a step's keys (gfx950).
//
// For key j and KV head h of a sequence:  mass[j][h] = decay * mass[j][h] + sum over the step's rows r that
// attend j and the query heads a of h's group of  exp(scale q_ra . k_j - lse_ra),  lse_ra the log-sum-exp of
// row r's scores.  Two passes over the keys, K alone: the first leaves (maximum, mass) of every (row, head)
// column over each split of the keys, the second merges a column's splits into its lse and sums the weights
// of every key over the columns - each key by one wave, in one order, so nothing is added atomically and the
// sums do not depend on timing.
//
// Both are S^T = K Q^T tiles of 16 keys by 16 columns ((row, head) pairs of one KV head; MFMA 16x16x32 with the
// attention kernels' operand types: bf16 on bf16 and MXFP4 pools, f16 on f16 and FP8 pools).  A sequence of up to
// kFewColumns columns (decode, verify rows) is bound by reading K: its keys are divided over the waves, 64
// at a time.  More columns (prompt chunks) are bound by the exponentials beside the products: the waves of a
// workgroup walk the same keys, each with columns of its own.
#include "common.hpp"
#include "launch.hpp"

namespace lia {

constexpr uint32_t kFewColumns = 64;
constexpr uint32_t kMassSeqs = 1024;  // sequences of one scan
constexpr uint32_t kMassThreads = 256;

struct MassParams {
    const void *q, *kc, *k_scales;
    const uint32_t *cu, *positions, *sequences, *pages;
    float *mass;
    float2 *stats;          // per sequence, KV head and split: (maximum, mass) of every column
    uint32_t capacity;      // entries of stats
    uint32_t hq, hkv, group, group_magic, stride, page_shift, pool_pages, n_seqs, n_rows;
    float scale_log2, decay;
    int q_f32, fresh;
};

// A sequence of the step and how its keys are split.
struct MassSeq {
    uint32_t r0, p0, n, cols, trow; // first packed row and its position, keys, columns of a KV head, table row
    bool many;
    uint32_t split, splits;         // keys of a split, splits
};

__device__ __forceinline__ MassSeq mass_seq(const MassParams &p, uint32_t b) {
    MassSeq s;
    s.r0 = p.cu[b];
    const uint32_t rows = p.cu[b + 1] - s.r0;
    s.cols = rows * p.group;
    s.many = s.cols > kFewColumns;
    s.p0 = rows ? p.positions[s.r0] : 0;
    s.trow = rows ? p.sequences[s.r0] : 0;
    s.n = rows ? s.p0 + rows : 0;
    // at most 64 splits of 512 keys and more (few columns), 32 of 1,024 and more (many)
    s.split = s.many ? 1024 * ((s.n + 32767) / 32768) : max(512u, ((s.n + 63) / 64 + 255) / 256 * 256);
    s.splits = (s.n + s.split - 1) / s.split;
    return s;
}

// Work items of a sequence in the two passes.
__device__ __forceinline__ uint32_t stat_items(const MassParams &p, const MassSeq &s) {
    return p.hkv * s.splits * (s.many ? (s.cols + 255) / 256 : 1u);
}
__device__ __forceinline__ uint32_t sum_items(const MassParams &p, const MassSeq &s) {
    return s.n ? p.hkv * (s.many ? (s.n + 63) / 64 : (s.n + 255) / 256) : 0u;
}

template <int D, int KVT>
struct KTile {
    static constexpr bool MB = KVT == LIA_BF16 || KVT == LIA_FP4; // operand type
    static constexpr int KT = D / 32;
    // bytes a lane holds of a 16-key tile: D/4 elements
    static constexpr int WORDS = KVT == LIA_FP4 ? D / 32 : KVT == LIA_FP8_E4M3 ? D / 16 : D / 8;
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
// outside the pool, read as zeros).
template <int D, int KVT>
__device__ __forceinline__ void load_tile(const MassParams &p, KTile<D, KVT> &k, uint32_t t0, uint32_t n,
                                          uint32_t page, uint32_t h) {
    const uint32_t lane = lane_id(), g = lane >> 4, li = lane & 15, P = 1u << p.page_shift;
    const uint32_t off = t0 & (P - 1);
    const uint32_t live = page < p.pool_pages && t0 < n ? min(n - t0, P - off) : 0u;
    if constexpr (KVT == LIA_FP4) {
        const uint64_t at = (((uint64_t)page * p.hkv + h) * P + off) * (D / 2);
        const __amdgpu_buffer_rsrc_t r = make_rsrc((const uint8_t *)p.kc + at, live * (D / 2));
        const __amdgpu_buffer_rsrc_t rs = make_rsrc((const uint8_t *)p.k_scales + at / 16, live * (D / 32));
        const uint32_t o = li * (D / 2) + g * (D / 8);
        if constexpr (D == 128) {
            const u32x4 x = buffer_load16(r, o);
            k.w[0] = x.x; k.w[1] = x.y; k.w[2] = x.z; k.w[3] = x.w;
        } else {
            const u32x2 x = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)o, 0, 0));
            k.w[0] = x.x; k.w[1] = x.y;
        }
        k.s = (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(rs, (int)(li * (D / 32) + (D == 128 ? g : g >> 1)), 0, 0);
    } else {
        constexpr uint32_t EB = KVT == LIA_FP8_E4M3 ? 1 : 2;
        const uint32_t row = p.hkv * D * EB;
        const uint64_t at = ((uint64_t)page * P + off) * row + (uint64_t)h * D * EB;
        // (a descriptor from the head's first byte: the last live key's head ends inside it)
        const __amdgpu_buffer_rsrc_t r = make_rsrc((const uint8_t *)p.kc + at, live ? (live - 1) * row + D * EB : 0u);
#pragma unroll
        for (int q = 0; q < KTile<D, KVT>::WORDS / 4; q++) {
            const u32x4 x = buffer_load16(r, li * row + 64 * q + 16 * g);
            k.w[4 * q] = x.x; k.w[4 * q + 1] = x.y; k.w[4 * q + 2] = x.z; k.w[4 * q + 3] = x.w;
        }
        k.s = 0;
        if constexpr (KVT == LIA_FP8_E4M3) {
            if (live) k.s = f2u(((const float *)p.k_scales)[(size_t)page * p.hkv + h]); // (uniform)
        }
    }
}

template <int D, int KVT>
__device__ __forceinline__ u32x4 operand(const KTile<D, KVT> &k, int ks) {
    if constexpr (KVT == LIA_FP4) return e2m1x8_to_bf16x8(k.w[ks], u2f(k.s << 23));
    if constexpr (KVT == LIA_FP8_E4M3) {
        return e4m3x8_to_f16x8(u32x2{k.w[2 * ks], k.w[2 * ks + 1]});
    } else {
        return u32x4{k.w[4 * ks], k.w[4 * ks + 1], k.w[4 * ks + 2], k.w[4 * ks + 3]};
    }
}

// What a tile's scores are multiplied by.
template <int D, int KVT>
__device__ __forceinline__ float score_scale(const MassParams &p, const KTile<D, KVT> &k) {
    return KVT == LIA_FP8_E4M3 ? p.scale_log2 * u2f(k.s) : p.scale_log2;
}

// Query operand of the 16-column tile's column col (li's): dims dim_of(ks, g) .. +7.
template <int D, int KVT>
__device__ __forceinline__ void load_query(const MassParams &p, uint32_t row, uint32_t head, bool valid,
                                           u32x4 (&out)[D / 32]) {
    constexpr bool MB = KTile<D, KVT>::MB;
    const uint32_t g = lane_id() >> 4, qb = p.q_f32 ? 4 : 2;
    const __amdgpu_buffer_rsrc_t r = make_rsrc(p.q, p.n_rows * p.hq * D * qb);
#pragma unroll
    for (int ks = 0; ks < D / 32; ks++) {
        const uint32_t off = valid ? ((row * p.hq + head) * D + dim_of<D, KVT>(ks, g)) * qb : 0x80000000u;
        float x[8];
        if (p.q_f32) {
            const f32x4 a = __builtin_bit_cast(f32x4, buffer_load16(r, off));
            const f32x4 b = __builtin_bit_cast(f32x4, buffer_load16(r, off + 16));
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
            x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        } else {
            const u32x4 w = buffer_load16(r, off);
            if constexpr (MB) {
                out[ks] = w;
                continue;
            }
#pragma unroll
            for (int e = 0; e < 4; e++) {
                x[2 * e] = bf16_to_f32(w[e] & 0xffffu);
                x[2 * e + 1] = bf16_to_f32(w[e] >> 16);
            }
        }
        out[ks] = u32x4{pack2<MB>(x[0], x[1]), pack2<MB>(x[2], x[3]), pack2<MB>(x[4], x[5]), pack2<MB>(x[6], x[7])};
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
__device__ __forceinline__ uint32_t page_of(MassPages &w, uint32_t logical) {
    if (logical - w.base >= 64) pages_at(w, logical); // (uniform)
    return (uint32_t)__builtin_amdgcn_readlane((int)w.page, (int)((logical - w.base) & 63));
}

// The scan of a launch: exclusive sums of the sequences' items and stats in LDS, by every workgroup itself.
struct MassScan {
    uint32_t items[kMassSeqs + 1], stats[kMassSeqs + 1];
};

// Sequences first .. first + count - 1; `base`: stats before them.
template <bool SUM>
__device__ __forceinline__ void mass_scan(const MassParams &p, MassScan &sc, uint32_t first, uint32_t count,
                                          uint32_t base) {
    __shared__ uint32_t wa[kMassThreads / 64], wb[kMassThreads / 64], run[2];
    const uint32_t t = threadIdx.x;
    if (t == 0) { run[0] = 0; run[1] = base; }
    __syncthreads();
    for (uint32_t i = 0; i < count; i += kMassThreads) {
        uint32_t a = 0, b = 0;
        if (i + t < count) {
            const MassSeq s = mass_seq(p, first + i + t);
            a = SUM ? sum_items(p, s) : stat_items(p, s);
            b = p.hkv * s.splits * s.cols;
        }
        const uint32_t a0 = a, b0 = b;
        block_scan2(a, b, wa, wb);
        if (i + t < count) {
            sc.items[i + t] = run[0] + a - a0;
            sc.stats[i + t] = run[1] + b - b0;
        }
        __syncthreads();
        if (t == kMassThreads - 1) { run[0] += a; run[1] += b; }
        __syncthreads();
    }
    if (t == 0) { sc.items[count] = run[0]; sc.stats[count] = run[1]; }
    __syncthreads();
}

// Last index a of arr[0 .. n) (ascending, arr[0] <= v) with arr[a] <= v.
__device__ __forceinline__ uint32_t owner(const uint32_t *arr, uint32_t n, uint32_t v) {
    uint32_t a = 0, e = n;
#pragma unroll 1
    while (a + 1 < e) {
        const uint32_t mid = (a + e) >> 1;
        if (arr[mid] <= v) a = mid; else e = mid;
    }
    return a;
}

__device__ __forceinline__ uint32_t div_group(const MassParams &p, uint32_t col) {
    return p.group == 1 ? col : __umulhi(col, p.group_magic);
}

// First pass: (maximum, mass) of 64 columns a wave over the item's keys, online, the reference raised only when
// some lane's score passes it by 2^8; merged over the lanes, and over the waves where these divide the keys.
template <int D, int KVT>
__global__ __launch_bounds__(kMassThreads, 2) void weight_stats_kernel(MassParams p) {
    constexpr int NT = 4, KT = D / 32;
    __shared__ MassScan sc;
    __shared__ float s_m[4][64], s_l[4][64];
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    uint32_t base = 0;
    for (uint32_t first = 0; first < p.n_seqs; first += kMassSeqs) {
        const uint32_t count = min(p.n_seqs - first, kMassSeqs);
        mass_scan<false>(p, sc, first, count, base);
        base = sc.stats[count];
        if (base > p.capacity) return; // metadata beyond the configuration: no work (uniform)
        const uint32_t items = sc.items[count];
        for (uint32_t it = blockIdx.x; it < items; it += gridDim.x) {
            const uint32_t bi = uniform(owner(sc.items, count, it));
            const MassSeq s = mass_seq(p, first + bi);
            uint32_t x = it - sc.items[bi];
            const uint32_t h = x % p.hkv;
            x /= p.hkv;
            const uint32_t split = x % s.splits, block = x / s.splits;
            const uint32_t col0 = s.many ? block * 256 + wave * 64 : 0;
            const uint32_t lo = split * s.split;
            // keys past the wave's last row's position are no column's
            const uint32_t last_col = min(col0 + 63, s.cols - 1);
            const uint32_t last = col0 < s.cols ? s.p0 + div_group(p, last_col) + 1 : 0;
            const uint32_t hi = min(min(lo + s.split, s.n), last);
            const uint32_t free_hi = s.p0 + div_group(p, col0) + 1; // live for all of its columns
            const uint32_t step = s.many ? 64 : 256;
            const int tiles = col0 < s.cols ? (int)min((s.cols - col0 + 15) / 16, (uint32_t)NT) : 0;
            u32x4 q[NT][KT];
            uint32_t lim[NT];
            float m[NT], thr[NT], l[NT];
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const uint32_t col = col0 + 16 * nt + li, ri = div_group(p, col);
                const bool valid = col < s.cols;
                lim[nt] = valid ? s.p0 + ri + 1 : 0;
                if (nt < tiles) load_query<D, KVT>(p, s.r0 + ri, h * p.group + col - ri * p.group, valid, q[nt]);
                m[nt] = 0.0f; l[nt] = 0.0f; thr[nt] = -INFINITY;
            }
            MassPages w{p.pages + (size_t)s.trow * p.stride, min((s.n + (1u << p.page_shift) - 1) >> p.page_shift, p.stride)};
            uint32_t t = lo + (s.many ? 0 : 64 * wave);
            pages_at(w, t >> p.page_shift);
            KTile<D, KVT> k[4];
#pragma unroll
            for (int j = 0; j < 4; j++) load_tile<D, KVT>(p, k[j], t + 16 * j, hi, page_of(w, (t + 16 * j) >> p.page_shift), h);
#pragma unroll 1
            for (; t < hi; t += step) {
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t t0 = t + 16 * j;
                    const float ss = score_scale(p, k[j]);
                    u32x4 a[KT];
#pragma unroll
                    for (int ks = 0; ks < KT; ks++) a[ks] = operand(k[j], ks);
                    load_tile<D, KVT>(p, k[j], t0 + step, hi, page_of(w, (t0 + step) >> p.page_shift), h);
                    if (t0 >= hi) continue;
                    const bool masked = t0 + 16 > min(free_hi, hi);
#pragma unroll
                    for (int nt = 0; nt < NT; nt++) {
                        if (nt >= tiles) continue; // uniform
                        f32x4 sc4 = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int ks = 0; ks < KT; ks++) sc4 = mfma16x16x32<KTile<D, KVT>::MB>(a[ks], q[nt][ks], sc4);
                        float e[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) e[i] = __builtin_fmaf(sc4[i], ss, -m[nt]);
                        if (masked) {
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                if (t0 + 4 * g + i >= min(lim[nt], hi)) e[i] = -INFINITY;
                        }
                        const float mx = fmaxf(fmaxf(e[0], e[1]), fmaxf(e[2], e[3]));
                        if (__builtin_amdgcn_ballot_w64(mx > thr[nt])) {
                            if (mx > thr[nt]) { // per lane: its own reference
                                l[nt] *= fast_exp2(-mx);
                                m[nt] += mx;
                                thr[nt] = 8.0f;
#pragma unroll
                                for (int i = 0; i < 4; i++) e[i] -= mx;
                            }
                        }
                        l[nt] += (fast_exp2(e[0]) + fast_exp2(e[1])) + (fast_exp2(e[2]) + fast_exp2(e[3]));
                    }
                }
            }
            // the lanes of a column, then (keys divided over the waves) the waves
#pragma unroll
            for (int nt = 0; nt < NT; nt++) {
                const float M = rows_max(l[nt] != 0.0f ? m[nt] : -INFINITY);
                const float L = rows_sum(l[nt] != 0.0f ? l[nt] * fast_exp2(m[nt] - M) : 0.0f);
                if (g == 0) { s_m[wave][16 * nt + li] = M; s_l[wave][16 * nt + li] = L; }
            }
            float2 *out = p.stats + sc.stats[bi] + ((size_t)h * s.splits + split) * s.cols;
            if (s.many) {
                // (a wave reads what it wrote itself)
                const uint32_t col = col0 + lane;
                if (col < s.cols) out[col] = make_float2(s_m[wave][lane], s_l[wave][lane]);
            } else {
                lds_barrier();
                if (wave == 0 && lane < s.cols) {
                    float M = -INFINITY, L = 0.0f;
#pragma unroll
                    for (int v = 0; v < 4; v++)
                        if (s_l[v][lane] != 0.0f) M = fmaxf(M, s_m[v][lane]);
#pragma unroll
                    for (int v = 0; v < 4; v++)
                        if (s_l[v][lane] != 0.0f) L += s_l[v][lane] * fast_exp2(s_m[v][lane] - M);
                    out[lane] = make_float2(M, L);
                }
                lds_barrier();
            }
        }
        __syncthreads(); // the scan is rewritten
    }
}

// log2-sum-exp2 of column col of a (sequence, KV head) from its splits (li's column; the four lane rows share
// the splits).
__device__ __forceinline__ float column_lse(const float2 *stats, uint32_t splits, uint32_t cols, uint32_t col) {
    const uint32_t g = lane_id() >> 4, c = min(col, cols - 1);
    float M = -INFINITY, L = 0.0f;
    for (uint32_t s0 = 0; s0 < splits; s0 += 8) {
        float2 x[2];
#pragma unroll
        for (int i = 0; i < 2; i++) x[i] = stats[(size_t)min(s0 + 4 * i + g, splits - 1) * cols + c];
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if (s0 + 4 * i + g >= splits || x[i].y == 0.0f) continue;
            const float nm = fmaxf(M, x[i].x);
            L = L * fast_exp2(M - nm) + x[i].y * fast_exp2(x[i].x - nm); // (M = -inf: 0)
            M = nm;
        }
    }
    const float all = rows_max(M);
    const float sum = rows_sum(L != 0.0f ? L * fast_exp2(M - all) : 0.0f);
    return all + __builtin_amdgcn_logf(sum); // log2
}

// Sum over the 16 lanes of a row, in every one of them.
__device__ __forceinline__ float lanes_sum(float x) {
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) x += shfl_xor(x, o);
    return x;
}

// Second pass: 64 keys a wave, their K in registers, against column tile after column tile.
template <int D, int KVT>
__global__ __launch_bounds__(kMassThreads, 2) void weight_sums_kernel(MassParams p) {
    constexpr int KT = D / 32;
    __shared__ MassScan sc;
    __shared__ float part[4][64];
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t P = 1u << p.page_shift;
    uint32_t base = 0;
    for (uint32_t first = 0; first < p.n_seqs; first += kMassSeqs) {
        const uint32_t count = min(p.n_seqs - first, kMassSeqs);
        mass_scan<true>(p, sc, first, count, base);
        base = sc.stats[count];
        if (base > p.capacity) return;
        const uint32_t items = sc.items[count];
        for (uint32_t it = blockIdx.x; it < items; it += gridDim.x) {
            const uint32_t bi = uniform(owner(sc.items, count, it));
            const MassSeq s = mass_seq(p, first + bi);
            const uint32_t x = it - sc.items[bi], h = x % p.hkv, kb = x / p.hkv;
            const uint32_t t = s.many ? kb * 64 : kb * 256 + 64 * wave;
            const float2 *stats = p.stats + sc.stats[bi] + (size_t)h * s.splits * s.cols;
            MassPages w{p.pages + (size_t)s.trow * p.stride, min((s.n + P - 1) >> p.page_shift, p.stride)};
            f32x4 acc[4];
#pragma unroll
            for (int j = 0; j < 4; j++) acc[j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
            if (t < s.n) { // uniform
                pages_at(w, t >> p.page_shift);
                KTile<D, KVT> k[4];
                float ss[4];
                u32x4 a[4][KT];
#pragma unroll
                for (int j = 0; j < 4; j++) load_tile<D, KVT>(p, k[j], t + 16 * j, s.n, page_of(w, (t + 16 * j) >> p.page_shift), h);
                // columns of rows before the first key attend none of these
                const uint32_t from = t > s.p0 ? (t - s.p0) * p.group / 16 : 0, all = (s.cols + 15) / 16;
                uint32_t nt = s.many ? from + wave : from;
                const uint32_t stride = s.many ? 4 : 1;
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    ss[j] = score_scale(p, k[j]);
#pragma unroll
                    for (int ks = 0; ks < KT; ks++) a[j][ks] = operand(k[j], ks);
                }
#pragma unroll 1
                for (; nt < all; nt += stride) {
                    const uint32_t col = 16 * nt + li, ri = div_group(p, col);
                    const bool valid = col < s.cols;
                    u32x4 q[KT];
                    load_query<D, KVT>(p, s.r0 + ri, h * p.group + col - ri * p.group, valid, q);
                    const float lse = column_lse(stats, s.splits, s.cols, col);
                    const uint32_t lim = valid ? s.p0 + ri + 1 : 0;
                    const bool masked = t + 64 > s.p0 + div_group(p, 16 * nt) + 1 || 16 * nt + 16 > s.cols;
#pragma unroll
                    for (int j = 0; j < 4; j++) {
                        f32x4 sc4 = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int ks = 0; ks < KT; ks++) sc4 = mfma16x16x32<KTile<D, KVT>::MB>(a[j][ks], q[ks], sc4);
                        float e[4];
#pragma unroll
                        for (int i = 0; i < 4; i++) e[i] = fast_exp2(__builtin_fmaf(sc4[i], ss[j], -lse));
                        if (masked) {
#pragma unroll
                            for (int i = 0; i < 4; i++)
                                if (t + 16 * j + 4 * g + i >= lim) e[i] = 0.0f;
                        }
#pragma unroll
                        for (int i = 0; i < 4; i++) acc[j][i] += e[i];
                    }
                }
            }
            // sum over the columns of a tile; lane (g, li) then keeps key 16 (li/4) + 4g + li%4 of the 64
            float mine = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const float y = lanes_sum(acc[j][i]);
                    if (li == 4 * (uint32_t)j + i) mine = y;
                }
            uint32_t key = 16 * (li >> 2) + 4 * g + (li & 3);
            if (s.many) {
                part[wave][key] = mine;
                lds_barrier();
                key = lane;
                mine = (part[0][lane] + part[1][lane]) + (part[2][lane] + part[3][lane]);
                lds_barrier();
                if (wave != 0) continue;
            }
            const uint32_t at = t + key;
            if (at < s.n && (at >> p.page_shift) < w.limit) {
                const uint32_t page = w.table[at >> p.page_shift];
                if (page < p.pool_pages) {
                    float *out = p.mass + (((size_t)page * p.hkv + h) << p.page_shift) + (at & (P - 1));
                    *out = p.decay == 0.0f || (p.fresh && at >= s.p0) ? mine : __builtin_fmaf(p.decay, *out, mine);
                }
            }
        }
        __syncthreads(); // the scan is rewritten
    }
}

template <int D, int KVT>
static hipError_t launch_weights(const MassParams &p, uint32_t n_a, uint32_t n_b, hipStream_t s) {
    hipError_t e = launch<weight_stats_kernel<D, KVT>>(dim3(n_a), dim3(kMassThreads), 0, s, p);
    if (e == hipSuccess) e = launch<weight_sums_kernel<D, KVT>>(dim3(n_b), dim3(kMassThreads), 0, s, p);
    return e;
}

template <int D>
static hipError_t launch_weights_kv(int kv, const MassParams &p, uint32_t n_a, uint32_t n_b, hipStream_t s) {
    if (kv == LIA_BF16) return launch_weights<D, LIA_BF16>(p, n_a, n_b, s);
    if (kv == LIA_F16) return launch_weights<D, LIA_F16>(p, n_a, n_b, s);
    if (kv == LIA_FP4) return launch_weights<D, LIA_FP4>(p, n_a, n_b, s);
    return launch_weights<D, LIA_FP8_E4M3>(p, n_a, n_b, s);
}

// Entries of the statistics a configuration's largest step needs: 64 splits of the columns of sequences of few
// (at most kFewColumns of a KV head each), 32 of the others', fewer where the context is short.
static uint64_t stats_entries(const lia_attention_config *c) {
    const uint64_t group = c->num_q_heads / c->num_kv_heads, hkv = c->num_kv_heads;
    const uint64_t cols = (uint64_t)c->max_rows * group;
    const uint64_t few = (uint64_t)c->max_seqs * kFewColumns < cols ? (uint64_t)c->max_seqs * kFewColumns : cols;
    const uint64_t a = c->max_context > 512 * 64 ? 64 : (c->max_context + 511) / 512;
    const uint64_t b = c->max_context > 1024 * 32 ? 32 : (c->max_context + 1023) / 1024;
    return hkv * (few * (a ? a : 1) + cols * (b ? b : 1));
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
    // the queries are read through one 32-bit buffer range, a page through another; a step's statistics are indexed
    // in 32 bits
    if ((uint64_t)c->max_rows * c->num_q_heads * c->head_dim * 4 >= (1ull << 31) ||
        (uint64_t)c->page_size * c->num_kv_heads * c->head_dim * 2 >= (1ull << 31) || stats_entries(c) >= (1ull << 31))
        return LIA_E_UNSUPPORTED;
    return LIA_OK;
}

extern "C" size_t lia_attention_weights_workspace_bytes(const lia_attention_config *c) {
    return validate_weights(c) == LIA_OK ? (size_t)stats_entries(c) * sizeof(float2) : 0;
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
    const uint64_t entries = stats_entries(c);
    if (workspace_bytes < entries * sizeof(float2)) return LIA_E_WORKSPACE;
    const uint32_t group = c->num_q_heads / c->num_kv_heads;
    MassParams p;
    p.q = q; p.kc = kc; p.k_scales = k_scales;
    p.cu = cu_seqlens; p.positions = positions; p.sequences = sequences; p.pages = pages;
    p.mass = mass;
    p.stats = (float2 *)workspace;
    p.capacity = (uint32_t)entries;
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
    uint32_t cus = device_cus();
    if (!cus) cus = 256;
    // a workgroup an item, up to a few on every CU (they take further items in turn)
    const uint64_t few = (uint64_t)n_seqs * p.hkv, context = c->max_context;
    const uint64_t a = few * ((context + 511) / 512) + (uint64_t)n_rows * c->num_q_heads / 256 * ((context + 1023) / 1024);
    const uint64_t b = few * ((context + 63) / 64);
    const uint32_t n_a = (uint32_t)(a < 2ull * cus ? a : 2ull * cus), n_b = (uint32_t)(b < 4ull * cus ? b : 4ull * cus);
    const hipError_t e = c->head_dim == 128 ? launch_weights_kv<128>(c->kv_dtype, p, n_a, n_b, (hipStream_t)stream)
                                            : launch_weights_kv<64>(c->kv_dtype, p, n_a, n_b, (hipStream_t)stream);
    return e == hipSuccess ? LIA_OK : LIA_E_HIP;
}
