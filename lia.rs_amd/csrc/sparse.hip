// Attention over selected pages of a paged KV pool (gfx950): summaries of full pages, the selection of pages for each row and
// KV head by their summaries, and the attention over the selection.
#include "common.hpp"
#include "launch.hpp"
#include "rows.hpp"

#include <algorithm>

namespace lia {

typedef __attribute__((ext_vector_type(4))) int i32x4;

// Exponent field of the unit of 8-bit codes whose largest magnitude has the bits `top`: that magnitude's, less 6 - its code
// is then 64 to 127.5 -, and never a subnormal unit.
__device__ __forceinline__ uint32_t unit_field(uint32_t top) { return max(top >> 23, 7u) - 6; }

// x / 2^(field - 127) as a code within +-127, rounded to nearest even (exact until then).
__device__ __forceinline__ int code_of(float x, uint32_t field) {
    const float y = __builtin_rintf(x * u2f((254u - field) << 23));
    return (int)fminf(fmaxf(y, -127.0f), 127.0f);
}

__device__ __forceinline__ uint32_t pack_codes(int a, int b, int c, int d) {
    return (uint32_t)(a & 255) | (uint32_t)(b & 255) << 8 | (uint32_t)(c & 255) << 16 | (uint32_t)d << 24;
}

// ------------------------------------------------------------------ page summaries

// One wave per slot and KV head; waves whose slot does not end its page leave.  A lane holds eight channels, the lanes
// of a key's row side by side, so that a load covers whole rows; what the lanes of a channel found is joined by lane moves.
// A step's launch is two loads that wait for each other (the slot, its page): 1.3 us of eight rows, 3.8 of 812 that end 51
// pages.  Whole pools are read at 4.3-4.9 TB/s (8 heads of 128, bf16 pages of 16 keys), 5.9 (of 256).
template <int D, int KVT>
__global__ __launch_bounds__(256) void summary_kernel(uint32_t n, uint32_t hkv, uint32_t page_shift, uint32_t pool_pages,
                                                      const uint32_t *slots, const void *kc, const void *k_scales,
                                                      int8_t *codes, float *scales) {
    constexpr uint32_t PER = D / 8, ROWS = 64 / PER; // lanes of a row, rows of a load
    const uint32_t w = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (w >= n) return;
    const uint32_t slot = slots[w / hkv], h = w % hkv, P = 1u << page_shift, page = slot >> page_shift;
    if ((slot & (P - 1)) != P - 1 || page >= pool_pages || slot == kNone) return;
    const uint32_t lane = threadIdx.x & 63, e = lane % PER * 8, row = lane / PER;
    float hi[8], lo[8];
    bool odd = false;
#pragma unroll
    for (int j = 0; j < 8; j++) { hi[j] = -INFINITY; lo[j] = INFINITY; }
#pragma unroll 4
    for (uint32_t t = 0; t < P; t += ROWS) { // (pages hold 16 keys at least)
        float x[8];
        values8<KVT>(kc, k_scales, (page << page_shift) + t + row, page_shift, hkv, h, D, e, x);
#pragma unroll
        for (int j = 0; j < 8; j++) {
            odd |= !(fabsf(x[j]) < INFINITY);
            hi[j] = fmaxf(hi[j], x[j]);
            lo[j] = fminf(lo[j], x[j]);
        }
    }
    auto larger = [](float a, float b) { return fmaxf(a, b); };
    auto lower = [](uint32_t a, uint32_t b) { return f2u(fminf(u2f(a), u2f(b))); };
    auto higher = [](uint32_t a, uint32_t b) { return f2u(fmaxf(u2f(a), u2f(b))); };
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
        if constexpr (PER == 8) { // (two rows of keys to 16 lanes: row_ror:8)
            hi[j] = fmaxf(hi[j], dpp<0x128>(hi[j]));
            lo[j] = fminf(lo[j], dpp<0x128>(lo[j]));
        }
        hi[j] = u2f(rows_all<true>(f2u(hi[j]), higher));
        lo[j] = u2f(rows_all<true>(f2u(lo[j]), lower));
        top = fmaxf(top, fmaxf(fabsf(hi[j]), fabsf(lo[j])));
    }
    top = group_all<PER>(top, larger);
    const bool bad = __builtin_amdgcn_ballot_w64(odd) != 0;
    const uint32_t field = unit_field(f2u(top));
    const size_t at = (size_t)page * hkv + h;
    if (row == 0) {
        int a[8], b[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            a[j] = bad ? 0 : code_of(hi[j], field);
            b[j] = bad ? 0 : code_of(lo[j], field);
        }
        int8_t *to = codes + at * 2 * D + e;
        *(u32x2 *)to = u32x2{pack_codes(a[0], a[1], a[2], a[3]), pack_codes(a[4], a[5], a[6], a[7])};
        *(u32x2 *)(to + D) = u32x2{pack_codes(b[0], b[1], b[2], b[3]), pack_codes(b[4], b[5], b[6], b[7])};
    }
    if (lane == 0) scales[at] = bad ? INFINITY : u2f(field << 23);
}

// ------------------------------------------------------------------ page scores

struct SelectPagesParams {
    const uint32_t *cu, *positions, *sequences, *pages;
    const void *q;
    const int8_t *codes;
    const float *scales;
    float *scores; // [row][kv head][span]
    uint32_t *selected, *counts;
    uint32_t n_seqs, n_rows, hq, hkv, group, pad_shift, rows; // pad_shift: log2 of the columns that a row's heads take
    uint32_t stride, span, page_shift, pool_pages;      // span: pages of the longest row
    uint32_t budget, first, recent, q_f32;
};

__device__ __forceinline__ uint32_t live_rows(const uint32_t *cu, uint32_t n_seqs, uint32_t n_rows) {
    return min(cu[n_seqs], n_rows);
}
__device__ __forceinline__ uint32_t row_pages(uint32_t position, uint32_t page_shift, uint32_t span) {
    return min((position >> page_shift) + 1, span); // (no overflow: pages hold 16 keys at least)
}

// A tile is p.rows consecutive packed rows (a power of two), each with its group's heads as columns of a matrix product: 16 CT
// columns in all.  Lane i < p.rows of every wave holds row i.
struct TileRows {
    uint32_t first, live;  // first row, live rows
    uint32_t pos, seq;     // this lane's
    uint64_t runs;         // rows that begin a run: consecutive positions of one sequence
};
__device__ __forceinline__ TileRows tile_rows(const SelectPagesParams &p, uint32_t tile) {
    TileRows x;
    const uint32_t lane = threadIdx.x & 63;
    x.first = tile * p.rows;
    const uint32_t r = min(x.first + min(lane, p.rows - 1), p.n_rows - 1);
    x.pos = p.positions[r];
    x.seq = p.sequences[r];
    const uint32_t total = live_rows(p.cu, p.n_seqs, p.n_rows);
    x.live = x.first < total ? min(p.rows, total - x.first) : 0;
    const uint32_t was = (uint32_t)__shfl_up((int)x.pos, 1), of = (uint32_t)__shfl_up((int)x.seq, 1);
    x.runs = __builtin_amdgcn_ballot_w64(lane < x.live && (lane == 0 || of != x.seq || was + 1 != x.pos));
    return x;
}
__device__ __forceinline__ uint32_t from_lane(uint32_t x, uint32_t lane) {
    return (uint32_t)__builtin_amdgcn_readlane((int)x, (int)lane);
}

// Bytes of a column's codes in LDS: its positive part, then its negative one (rows apart by 16 bytes more, so that the 16
// columns of an operand's read lie in different banks).
template <int D>
constexpr uint32_t kColumn = 2 * D + 16;

template <int D, int CT>
struct __attribute__((aligned(16))) ColumnCodes {
    int8_t codes[16 * CT * kColumn<D>];
    float unit[16 * CT]; // NaN: no column, and a product that no maximum takes
};

// The columns' queries as codes: D / 8 neighbouring lanes a column.  (Rows that are not live are read all the same, so that
// the queries are on their way beside the rows' positions; their columns' scores go nowhere.)
template <int D, int CT, int THREADS>
__device__ __forceinline__ void column_codes(const SelectPagesParams &p, uint32_t first, uint32_t h, ColumnCodes<D, CT> &to) {
    constexpr uint32_t PER = D / 8, N = 16 * CT * PER;
#pragma unroll
    for (uint32_t i0 = 0; i0 < N; i0 += THREADS) {
        const uint32_t i = i0 + threadIdx.x;
        if (i >= N) break; // (whole waves)
        const uint32_t m = i / PER, e = i % PER * 8, row = m >> p.pad_shift, head = m & ((1u << p.pad_shift) - 1);
        const bool valid = row < p.rows && first + row < p.n_rows && head < p.group;
        const size_t from = ((size_t)(first + (valid ? row : 0)) * p.hq + h * p.group + (valid ? head : 0)) * D + e;
        float x[8], top = 0.0f;
        if (p.q_f32) load8<0>(p.q, from, x);
        else load8<2>(p.q, from, x);
#pragma unroll
        for (int j = 0; j < 8; j++) top = fmaxf(top, fabsf(x[j]));
        top = group_all<PER>(top, [](float a, float b) { return fmaxf(a, b); });
        const uint32_t field = unit_field(f2u(top));
        int up[8], down[8];
#pragma unroll
        for (int j = 0; j < 8; j++) {
            const int v = code_of(x[j], field);
            up[j] = max(v, 0);
            down[j] = min(v, 0);
        }
        int8_t *at = to.codes + m * kColumn<D> + e;
        *(u32x2 *)at = u32x2{pack_codes(up[0], up[1], up[2], up[3]), pack_codes(up[4], up[5], up[6], up[7])};
        *(u32x2 *)(at + D) = u32x2{pack_codes(down[0], down[1], down[2], down[3]), pack_codes(down[4], down[5], down[6], down[7])};
        if (e == 0) to.unit[m] = valid ? u2f(field << 23) : __builtin_nanf("");
    }
    __syncthreads();
}

// A wave's operand: columns' codes and the units of the columns that this lane's results belong to.
template <int D, int CT>
struct Columns {
    i32x4 a[CT][D / 32];
    float u[CT][4];
    __device__ __forceinline__ void load(const ColumnCodes<D, CT> &from) {
        const uint32_t lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
#pragma unroll
        for (int c = 0; c < CT; c++) {
#pragma unroll
            for (int s = 0; s < D / 32; s++) a[c][s] = *(const i32x4 *)(from.codes + (16 * c + li) * kColumn<D> + 64 * s + 16 * g);
#pragma unroll
            for (int i = 0; i < 4; i++) u[c][i] = from.unit[16 * c + 4 * g + i];
        }
    }
};

// A wave's 16 pages in LDS, from where they are read as operands (rows apart by 16 bytes more, as the columns').
template <int D>
using PageStage = int8_t[16 * kColumn<D>];

// Scores of pages [base, base + 64) of one table for a wave's columns: put(row of the tile, page, score).  A page is 2 D + 4
// bytes a KV head, 1/32 of its bf16 keys and values, and 64 of them are on their way at once.  A = the
// queries' codes, their positive part against the largest values and their negative part against the smallest, B = the
// pages' codes; both operands hold 16 bytes a lane of the same 64, so the products add up over the head whatever their
// order within it, and exactly, in 32-bit integers.  The pages are loaded in memory's order, a page's lanes side by side, and
// turned through LDS: loaded as operands, neighbouring lanes would read different pages, a look-up of the L1 each (a chunk of
// 812 rows on 16k and 9k keys, both with the picks: 90 us so, 31 as they lie).
// page: entry base + lane of the table, kNone past the pages that count.
template <int D, int CT, class PUT>
__device__ __forceinline__ void score_pages(const SelectPagesParams &p, const Columns<D, CT> &q, uint32_t page, uint32_t base,
                                            uint32_t h, PageStage<D> &stage, PUT &&put) {
    constexpr int KS = D / 32, PER = D / 8, LOADS = D / 32; // lanes of a page, loads of 16 pages
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
    const bool held = page < p.pool_pages;
    const uint32_t mine = (held ? page : 0) * p.hkv + h; // (the host bounds the pool's heads to 2^32)
    const int8_t *codes = p.codes + 16 * (lane % PER);
    i32x4 raw[4][LOADS];
#pragma unroll
    for (int k = 0; k < 4; k++)
#pragma unroll
        for (int j = 0; j < LOADS; j++) {
            const uint32_t of = (uint32_t)__shfl((int)mine, 16 * k + (64 / PER) * j + (int)(lane / PER));
            raw[k][j] = *(const i32x4 *)(codes + (uint64_t)of * (2 * D));
        }
    const float scale = held ? p.scales[mine] : 0.0f; // (0: pages outside the pool score 0)
#pragma unroll
    for (int k = 0; k < 4; k++) {
        i32x4 b[KS];
#pragma unroll
        for (int j = 0; j < LOADS; j++)
            *(i32x4 *)(stage + ((64 / PER) * j + lane / PER) * kColumn<D> + 16 * (lane % PER)) = raw[k][j];
#pragma unroll
        for (int s = 0; s < KS; s++) b[s] = *(const i32x4 *)(stage + li * kColumn<D> + 64 * s + 16 * g);
        const float sc = __shfl(scale, 16 * k + (int)li);
        const uint32_t to = base + 16 * k + li;
        float best[CT][4];
#pragma unroll
        for (int c = 0; c < CT; c++) {
            i32x4 sum = i32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < KS; s++) sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(q.a[c][s], b[s], sum, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; i++) best[c][i] = (float)sum[i] * q.u[c][i];
        }
        // (rounding keeps the order, so the largest product times the page's unit is the largest of the scores)
        auto out = [&](uint32_t row, float x) {
            put(row, to, (sc < INFINITY ? x * sc : INFINITY) + 0.0f);
        };
        if (CT == 1 && p.pad_shift < 2) { // groups of one or two heads: four or two rows a lane
            if (p.pad_shift == 0) {
#pragma unroll
                for (int i = 0; i < 4; i++) out(4 * g + i, best[0][i]);
            } else {
                out(2 * g, fmaxf(best[0][0], best[0][1]));
                out(2 * g + 1, fmaxf(best[0][2], best[0][3]));
            }
            continue;
        }
#pragma unroll
        for (int c = 0; c < CT; c++) {
            float z = fmaxf(fmaxf(best[c][0], best[c][1]), fmaxf(best[c][2], best[c][3]));
            auto larger = [](uint32_t a, uint32_t b) { return f2u(fmaxf(u2f(a), u2f(b))); };
            if (p.pad_shift >= 4) z = u2f(rows_all<true>(f2u(z), larger));
            else if (p.pad_shift == 3) z = u2f(rows_all<false>(f2u(z), larger));
            best[c][0] = z;
            if (p.pad_shift == 5) { // 32 columns a row: two tiles
                if (!(c & 1)) continue;
                z = fmaxf(z, best[c & ~1][0]);
            }
            if ((4 * g & ((1u << p.pad_shift) - 1)) == 0) out((16 * c + 4 * g) >> p.pad_shift, z);
        }
    }
}

// Pages that the scores choose among in a run of rows: [lo, hi) of its last row's, none where that keeps all its pages.
__device__ __forceinline__ bool run_pages(const SelectPagesParams &p, uint32_t last_pos, uint32_t &lo, uint32_t &hi) {
    const uint32_t n = row_pages(last_pos, p.page_shift, p.span);
    lo = p.first;
    hi = n - p.recent;
    return n > p.budget;
}

// ------------------------------------------------------------------ page selection

constexpr uint32_t kPickBins = 1024, kPickDirect = 64;

template <int THREADS>
struct PickShared {
    uint32_t hist[kPickBins], red[2 * THREADS / 64], bin, above, in, listed;
    uint64_t list[kPickDirect], last;
};

// The k0 best of c > k0 candidates with the scores get(i), in ascending order behind out[first .. ): a workgroup's work.  A
// candidate is a pair (score's place in the floats' total order, counted from the lowest candidate's; pages from the last
// candidate), and the last kept one is found from the top: ten bits of the pair at a time, beginning at the highest
// bit in which the scores differ, until the digit's bin holds 64 candidates at most, which are ranked directly.  Pairs
// are distinct, so the kept ones are those not below it, and equal scores go by the lower page.  The time is that of its
// barriers, some twelve: 4 us for 2,000 candidates of four waves.
template <int THREADS, class GET>
__device__ __forceinline__ void pick_pages(PickShared<THREADS> &sh, uint32_t c, uint32_t k0, uint32_t first, uint32_t *out,
                                           GET &&get) {
    constexpr uint32_t WAVES = THREADS / 64, BINS = kPickBins / THREADS, ROWS = 8, SEG = THREADS * ROWS;
    const uint32_t t = threadIdx.x, lane = t & 63;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(t >> 6));
    // a segment's candidates in registers, a run of 64 ROWS a wave, 64 a row; more than one are loaded anew for each pass
    const uint32_t segments = (c + SEG - 1) / SEG;
    uint32_t v[ROWS];
    auto place = [&](uint32_t seg, uint32_t x) { return seg * SEG + (wave * ROWS + x) * 64 + lane; };
    auto load = [&](uint32_t seg) {
#pragma unroll
        for (uint32_t x = 0; x < ROWS; x++) {
            const uint32_t b = f2u(get(min(place(seg, x), c - 1)));
            v[x] = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
        }
    };
    auto waves_before = [&] { // of sh.red: every load at once
        uint32_t sum = 0;
#pragma unroll
        for (uint32_t w = 0; w < WAVES; w++) sum += w < wave ? sh.red[w] : 0;
        return sum;
    };
    uint32_t low = 0xffffffffu, high = 0;
    for (uint32_t seg = 0; seg < segments; seg++) {
        load(seg);
#pragma unroll
        for (uint32_t x = 0; x < ROWS; x++) {
            low = min(low, v[x]);
            high = max(high, v[x]);
        }
    }
    auto lower = [](uint32_t a, uint32_t b) { return min(a, b); };
    auto higher = [](uint32_t a, uint32_t b) { return max(a, b); };
    low = rows_all<true>(group_all<16>(low, lower), lower);
    high = rows_all<true>(group_all<16>(high, higher), higher);
    if (lane == 0) { sh.red[2 * wave] = low; sh.red[2 * wave + 1] = high; }
#pragma unroll
    for (uint32_t i = 0; i < BINS; i++) sh.hist[t + i * THREADS] = 0;
    if (t == 0) sh.listed = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t w = 0; w < WAVES; w++) { low = min(low, sh.red[2 * w]); high = max(high, sh.red[2 * w + 1]); }
    // the pair: the score's place above the lowest one's (d), then c - 1 - page (e); digits of d first, of e where all of d is
    // known.  known and found: the bits of each that the digits have given.
    const uint32_t range = high - low;
    auto d_of = [&](uint32_t x) { return v[x] - low; };
    auto e_of = [&](uint32_t seg, uint32_t x) { return c - 1 - place(seg, x); };
    uint32_t d_bits = range ? 32 - (uint32_t)__builtin_clz(range) : 0, e_bits = 32 - (uint32_t)__builtin_clz(c - 1); // (c > 1)
    uint32_t d_known = 0, d_found = 0, e_known = 0, e_found = 0;
    auto fits = [&](uint32_t seg, uint32_t x) {
        return (d_of(x) & d_known) == d_found && (e_of(seg, x) & e_known) == e_found && place(seg, x) < c;
    };
    uint32_t k = k0, many = c;
    bool again = false;
    while (many > kPickDirect && many > k) { // (uniform)
        const bool of_d = d_bits > 0;
        const uint32_t bits = of_d ? d_bits : e_bits, shift = bits > 10 ? bits - 10 : 0, mask = (1u << (bits - shift)) - 1;
        if (again) {
#pragma unroll
            for (uint32_t i = 0; i < BINS; i++) sh.hist[t + i * THREADS] = 0;
            __syncthreads();
        }
        again = true;
        for (uint32_t seg = 0; seg < segments; seg++) {
            if (segments > 1) load(seg);
#pragma unroll
            for (uint32_t x = 0; x < ROWS; x++)
                if (fits(seg, x)) atomicAdd(&sh.hist[(of_d ? d_of(x) : e_of(seg, x)) >> shift & mask], 1u);
        }
        __syncthreads();
        uint32_t own[BINS], sum = 0; // BINS bins a thread, the t-th from the top
#pragma unroll
        for (uint32_t i = 0; i < BINS; i++) { own[i] = sh.hist[kPickBins - 1 - t * BINS - i]; sum += own[i]; }
        const uint32_t upto = wave_scan(sum);
        if (lane == 63) sh.red[wave] = upto;
        __syncthreads();
        uint32_t over = upto - sum + waves_before();
        if (over < k && k <= over + sum) {
#pragma unroll
            for (uint32_t i = 0; i < BINS; i++) {
                if (over < k && k <= over + own[i]) {
                    sh.bin = kPickBins - 1 - t * BINS - i;
                    sh.above = over;
                    sh.in = own[i];
                }
                over += own[i];
            }
        }
        __syncthreads();
        (of_d ? d_found : e_found) |= sh.bin << shift;
        (of_d ? d_known : e_known) |= mask << shift;
        (of_d ? d_bits : e_bits) = shift;
        k -= sh.above;
        many = sh.in;
    }
    // the lowest kept pair: every one of the last bin's, or its k-th from the top
    uint32_t d_last = d_found, e_last = e_found;
    if (many > k) {
        for (uint32_t seg = 0; seg < segments; seg++) {
            if (segments > 1) load(seg);
#pragma unroll
            for (uint32_t x = 0; x < ROWS; x++)
                if (fits(seg, x)) sh.list[atomicAdd(&sh.listed, 1u)] = (uint64_t)d_of(x) << 32 | e_of(seg, x);
        }
        __syncthreads();
        constexpr uint32_t SHARE = THREADS / kPickDirect; // neighbouring lanes rank one of them
        const uint32_t mine = t / SHARE, part = t % SHARE * (kPickDirect / SHARE);
        const uint64_t y = sh.list[mine];
        uint32_t rank = 0;
#pragma unroll
        for (uint32_t i = 0; i < kPickDirect / SHARE; i++) rank += part + i < many && sh.list[part + i] > y;
        rank = group_all<SHARE>(rank, [](uint32_t a, uint32_t b) { return a + b; });
        if (mine < many && rank + 1 == k) sh.last = y;
        __syncthreads();
        d_last = (uint32_t)(sh.last >> 32);
        e_last = (uint32_t)sh.last;
    }
    uint32_t at = first;
    for (uint32_t seg = 0; seg < segments; seg++) {
        if (segments > 1) load(seg);
        uint64_t keep[ROWS];
        uint32_t count = 0;
#pragma unroll
        for (uint32_t x = 0; x < ROWS; x++) {
            const uint32_t d = d_of(x);
            keep[x] = __builtin_amdgcn_ballot_w64(place(seg, x) < c && (d > d_last || (d == d_last && e_of(seg, x) >= e_last)));
            count += (uint32_t)__builtin_popcountll(keep[x]);
        }
        if (lane == 0) sh.red[wave] = count;
        __syncthreads();
        uint32_t to = at + waves_before();
#pragma unroll
        for (uint32_t w = 0; w < WAVES; w++) at += sh.red[w];
        __syncthreads(); // (the shared memory is free again)
#pragma unroll
        for (uint32_t x = 0; x < ROWS; x++) {
            if (keep[x] >> lane & 1)
                out[to + __builtin_amdgcn_mbcnt_hi((uint32_t)(keep[x] >> 32), __builtin_amdgcn_mbcnt_lo((uint32_t)keep[x], 0))] =
                    first + place(seg, x);
            to += (uint32_t)__builtin_popcountll(keep[x]);
        }
    }
}

// One row's and KV head's list: all its pages, or the first and the recent ones and those picked by get(candidate).
template <int THREADS, class GET>
__device__ __forceinline__ void write_pages(const SelectPagesParams &p, PickShared<THREADS> &sh, uint32_t r, uint32_t h,
                                            uint32_t pos, GET &&get) {
    const uint32_t n = row_pages(pos, p.page_shift, p.span), t = threadIdx.x;
    uint32_t *out = p.selected + ((size_t)r * p.hkv + h) * p.budget;
    if (h == 0 && t == 0) p.counts[r] = min(n, p.budget);
    if (n <= p.budget) {
        for (uint32_t i = t; i < p.budget; i += THREADS) out[i] = i < n ? i : kNone;
        return;
    }
    const uint32_t k0 = p.budget - p.first - p.recent; // kept of the candidates
    for (uint32_t i = t; i < p.first; i += THREADS) out[i] = i;
    for (uint32_t i = t; i < p.recent; i += THREADS) out[p.first + k0 + i] = n - p.recent + i;
    if (k0) pick_pages<THREADS>(sh, n - p.first - p.recent, k0, p.first, out, get);
}

constexpr uint32_t kPickThreads = 256, kChooseThreads = 1024, kChooseSpan = 12288; // (48 KiB of LDS for the scores, the rest 79)

// Scores and selection of one row and KV head: sixteen waves score 64 pages each in turn, four pick.  64 rows of 2 KV heads
// over 1,000 to 2,000 pages each take 18.3 us for the 51 MB of summaries (7 at the rate of a large read): they are 128
// workgroups, so half of the compute units read nothing, and a workgroup reads its table in two trips before its pick.
template <int D>
__global__ __launch_bounds__(kChooseThreads) void page_choose_kernel(SelectPagesParams p) {
    extern __shared__ float scores[]; // [span]
    __shared__ ColumnCodes<D, 1> columns;
    __shared__ PickShared<kPickThreads> sh;
    __shared__ __attribute__((aligned(16))) PageStage<D> stages[kChooseThreads / 64];
    const uint32_t r = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 63;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t pos = p.positions[r], seq = p.sequences[r], total = live_rows(p.cu, p.n_seqs, p.n_rows);
    column_codes<D, 1, kChooseThreads>(p, r, h, columns);
    if (r >= total) return;
    uint32_t lo, hi;
    if (run_pages(p, pos, lo, hi)) {
        Columns<D, 1> q;
        q.load(columns);
        const uint32_t *table = p.pages + (size_t)seq * p.stride;
        uint32_t base = (lo & ~63u) + 64 * wave;
        uint32_t page = base + lane < hi ? table[base + lane] : kNone;
        for (; base < hi; base += kChooseThreads) {
            const uint32_t then = base + kChooseThreads + lane;
            const uint32_t next = then < hi ? table[then] : kNone;
            score_pages<D, 1>(p, q, page, base, h, stages[wave], [&](uint32_t row, uint32_t at, float x) {
                if (row == 0 && at < hi) scores[at] = x;
            });
            page = next;
        }
        __syncthreads();
    }
    if (threadIdx.x >= kPickThreads) return; // (a pick by all sixteen waves takes no less time)
    write_pages<kPickThreads>(p, sh, r, h, pos, [&](uint32_t x) { return scores[p.first + x]; });
}

// The same in two launches, so that many workgroups share a long table or a chunk's: scores of kScorePages pages (four tiles of
// columns, whose codes take as long as 64 pages a wave: twice as many, 30.9 us so 29.4 with the picks for 812 rows) ...
// Eight rows of 2 KV heads over up to 2,000 pages: 5.3 us, two loads in turn and the products; 812 rows: 16.8 us for
// 5.8 G multiply-adds in 8 bits, held up by turning the codes through LDS.
constexpr uint32_t kScorePages = 256;
constexpr uint32_t score_pages_of(int ct) { return ct == 4 ? 2 * kScorePages : kScorePages; }

template <int D, int CT>
__global__ __launch_bounds__(256) void page_score_kernel(SelectPagesParams p) {
    constexpr uint32_t PAGES = score_pages_of(CT);
    __shared__ ColumnCodes<D, CT> columns;
    __shared__ __attribute__((aligned(16))) PageStage<D> stages[4];
    const uint32_t h = blockIdx.y, lane = threadIdx.x & 63, begin = blockIdx.z * PAGES;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const TileRows rows = tile_rows(p, blockIdx.x);
    auto run_of = [&](uint64_t runs, uint32_t &i0, uint32_t &i1, uint32_t &hi) { // the next run, if it needs these pages
        uint32_t lo;
        i0 = (uint32_t)__builtin_ctzll(runs);
        runs &= runs - 1;
        i1 = runs ? (uint32_t)__builtin_ctzll(runs) : rows.live;
        return run_pages(p, from_lane(rows.pos, i1 - 1), lo, hi) && begin < hi && begin + PAGES > lo;
    };
    uint32_t i0, i1, hi;
    bool any = false; // (the same in every wave)
    for (uint64_t runs = rows.runs; runs; runs &= runs - 1) any |= run_of(runs, i0, i1, hi);
    if (!any) return;
    column_codes<D, CT, 256>(p, rows.first, h, columns);
    Columns<D, CT> q;
    q.load(columns);
    for (uint64_t runs = rows.runs; runs; runs &= runs - 1) {
        if (!run_of(runs, i0, i1, hi)) continue;
        const uint32_t *table = p.pages + (size_t)from_lane(rows.seq, i0) * p.stride;
        const uint32_t end = min(begin + PAGES, hi);
        uint32_t base = begin + 64 * wave;
        uint32_t page = base + lane < end ? table[base + lane] : kNone;
        for (; base < end; base += 256) {
            const uint32_t then = base + 256 + lane, next = then < end ? table[then] : kNone;
            score_pages<D, CT>(p, q, page, base, h, stages[wave], [&](uint32_t row, uint32_t at, float x) {
                if (row - i0 < i1 - i0 && at < end) p.scores[((size_t)(rows.first + row) * p.hkv + h) * p.span + at] = x;
            });
            page = next;
        }
    }
}

// ... and the picks, of scores read into LDS once: 5.7 us for 16 lists, 10 us for 1,624 of 1,050 pages.
constexpr uint32_t kPickHeld = 4096; // candidates that a workgroup keeps in LDS

__global__ __launch_bounds__(kPickThreads) void page_pick_kernel(SelectPagesParams p) {
    __shared__ PickShared<kPickThreads> sh;
    __shared__ float held[kPickHeld];
    const uint32_t r = blockIdx.x, h = blockIdx.y;
    const uint32_t pos = p.positions[r];
    if (r >= live_rows(p.cu, p.n_seqs, p.n_rows)) return;
    const uint32_t n = row_pages(pos, p.page_shift, p.span);
    const float *from = p.scores + ((size_t)r * p.hkv + h) * p.span + p.first;
    if (n <= p.budget || n - p.first - p.recent > kPickHeld) {
        write_pages<kPickThreads>(p, sh, r, h, pos, [&](uint32_t x) { return from[x]; });
        return;
    }
    const uint32_t c = n - p.first - p.recent;
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < c; i += kPickThreads) held[i] = from[i];
    __syncthreads();
    write_pages<kPickThreads>(p, sh, r, h, pos, [&](uint32_t x) { return held[x]; });
}

// ------------------------------------------------------------------ attention over selected pages

struct SelectedParams {
    const uint32_t *cu, *positions, *sequences, *pages, *selected, *counts;
    const void *q, *kc, *vc, *k_scales, *v_scales;
    void *out;
    float *part_o;   // [unit][part][head of the group][D]: unnormalised sums
    float2 *part_ml; // [unit][part][head]: reference (log2), mass
    uint32_t n_seqs, n_rows, hq, hkv, group, stride, page_shift, pool_pages, budget;
    uint32_t parts, per, q_f32, out_f32; // per: chunks of 32 keys a part
    float scale_log2;
};

// 16 keys of an FP8 or MXFP4 pool's plane in registers.  FP8 rows lie as in memory: PIECES lanes side by side hold a key's head,
// 16 bytes each, and LOADS loads the 16 keys; put() writes them as rows of bf16 values (exactly; the page's scale is the
// caller's) into LDS, from where both products' operands are read: loaded as operands, neighbouring lanes would read
// different keys, a look-up of the L1 each (812 rows of 64 bf16 pages of 16 keys: 109 us so, 59 as they lie).  MXFP4 rows,
// a quarter as long as bf16 ones and a head's keys one run, are loaded as the first product's operand: lane (g, li) holds
// D / 4 elements of key li, and K goes no way through LDS.
template <int D, bool FP4>
struct Tile {
    static constexpr uint32_t ROW = FP4 ? D / 2 : D; // bytes of a key's head
    static constexpr uint32_t PIECES = FP4 ? 4 : ROW / 16, KEYS = 64 / PIECES;
    static constexpr int LOADS = 16 / KEYS, WORDS = ROW / PIECES / 4;
    uint32_t w[LOADS][WORDS];
    uint32_t s; // MXFP4: the block's scale

    // The key (of 16) and the piece of it that load i of this lane holds.
    static __device__ __forceinline__ uint32_t key(int i) {
        const uint32_t lane = threadIdx.x & 63;
        return FP4 ? lane & 15 : lane / PIECES + i * KEYS;
    }
    static __device__ __forceinline__ uint32_t piece() { return FP4 ? (threadIdx.x & 63) >> 4 : threadIdx.x & (PIECES - 1); }
    // Byte of load i's piece from the tile's first key's head; step: heads between keys.  (Uniform bases, one offset a lane
    // and load.)
    static __device__ __forceinline__ uint32_t offset(int i, uint32_t step) { return key(i) * step * ROW + 4 * WORDS * piece(); }
    // first: byte of the tile's first key's head in the plane.
    __device__ __forceinline__ void load(const void *plane, const void *scales, uint64_t first, const uint32_t (&at)[LOADS]) {
        const uint8_t *from = (const uint8_t *)plane + first;
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            if constexpr (WORDS == 4) {
                const u32x4 x = *(const u32x4 *)(from + at[i]);
                w[i][0] = x.x; w[i][1] = x.y; w[i][2] = x.z; w[i][3] = x.w;
            } else {
                const u32x2 x = *(const u32x2 *)(from + at[i]);
                w[i][0] = x.x; w[i][1] = x.y;
            }
        }
        if constexpr (FP4) s = ((const uint8_t *)scales + first / 16)[at[0] / 16]; // (a head's keys lie together)
    }
    // Operand ks of the first product (MXFP4).
    __device__ __forceinline__ u32x4 operand(int ks) const { return e2m1x8_to_bf16x8(w[0][ks], u2f(s << 23)); }
    // Keys from `limit` on as zeros.
    __device__ __forceinline__ void clear_from(uint32_t limit) {
#pragma unroll
        for (int i = 0; i < LOADS; i++) {
            if (key(i) < limit) continue;
#pragma unroll
            for (int j = 0; j < WORDS; j++) w[i][j] = 0;
            s = 0;
        }
    }
    // Into 16 rows of a stage from byte `to`, STRIDE bytes apart.  at: this lane's first chunk's byte (at_of).
    static constexpr uint32_t CHUNKS = FP4 ? WORDS : 2; // of a piece
    template <uint32_t STRIDE>
    static __device__ __forceinline__ uint32_t at_of() { return key(0) * STRIDE + 16 * CHUNKS * piece(); }
    template <uint32_t STRIDE>
    __device__ __forceinline__ void put(uint8_t *to) const {
#pragma unroll
        for (int i = 0; i < LOADS; i++)
#pragma unroll
            for (uint32_t j = 0; j < CHUNKS; j++) {
                u32x4 x;
                if constexpr (FP4) x = operand(j);
                else x = e4m3x8_to_bf16x8(w[i][2 * j], w[i][2 * j + 1]);
                *(u32x4 *)(to + i * KEYS * STRIDE + 16 * j) = x;
            }
    }
};

// Bytes between staged rows: more than a row by 16 for K, whose operands are read 16 rows at a chunk, and by 32 for V, whose
// transposed reads take 32 bytes of each of 8 rows at once, so that the rows read together lie in different banks.
template <int D>
constexpr uint32_t kStrideK = 2 * D + 16;
template <int D>
constexpr uint32_t kStrideV = 2 * D + 32;

// 16-bit tiles straight from memory into LDS: a load moves KEYS keys' heads, 1 KiB, lane by lane behind each other, so the
// rows of a load cannot be apart, and lanes load the 16-byte piece that is to stand in their place: piece ^ turn(key) of
// the row, loads 32 bytes further apart than they are long, so that the rows that an operand's or a transposed read takes
// together lie in different banks.  Loads end at the keys that the row attends: the places of the others become zeros.
template <int D>
struct Direct {
    static constexpr uint32_t ROW = 2 * D, PIECES = ROW / 16, KEYS = 64 / PIECES, STRIDE = 1024 + 32;
    static constexpr int LOADS = 16 / KEYS;                           // of a tile of 16 keys
    static constexpr uint32_t TILE = LOADS * STRIDE, STAGE = 2 * TILE; // bytes of a tile, of a plane's chunk
    static __device__ __forceinline__ uint32_t turn(uint32_t key) { // (of a load's; even, so pairs of pieces stay together)
        return D == 128 ? 4 * (key & 3) : 2 * (key >> 1 & 3);
    }
    static __device__ __forceinline__ uint32_t row(uint32_t key) { return key / KEYS * STRIDE + key % KEYS * ROW; }
    // Byte of load i's piece from the tile's first key's head; step: heads between keys.
    static __device__ __forceinline__ uint32_t offset(int i, uint32_t step) {
        const uint32_t lane = threadIdx.x & 63, key = lane / PIECES;
        return (key + i * KEYS) * step * ROW + 16 * (lane % PIECES ^ turn(key));
    }
    // bytes: of the tile's keys that count.
    static __device__ __forceinline__ void load(const void *plane, uint64_t first, uint32_t bytes,
                                                const uint32_t (&at)[LOADS], uint8_t *to) {
        const __amdgpu_buffer_rsrc_t r = make_rsrc((const uint8_t *)plane + first, bytes);
#pragma unroll
        for (int i = 0; i < LOADS; i++)
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void *)(to + i * STRIDE), 16,
                                                     (int)at[i], 0, 0, 0);
    }
};

// One row's selected keys of one KV head, or a part of them: its waves take chunks of 32 keys of the list in turn and merge
// through LDS at the end.  S^T = K Q^T; K and V go through the wave's LDS, V's transposed reads giving keys side by side;
// softmax in the log2 domain with a reference that is raised when a score passes it by 8.  Queries are rounded to the
// operands' 16 bits, and so are the weights, since the products take no others at their rate; the mass is summed of the
// rounded weights, so that a rounding common to both sides of the fraction cancels in part; on FP8 pools the weights above
// the line are rounded with V's scale in them, which differs between the pages of a product, so nothing does.  Mass and
// outputs are summed in f32.  Relative to 64 bits, bf16 outputs (which alone are 1.7e-3 off): bf16 and MXFP4 pools 2.1e-3,
// FP8 2.4e-3, f16 1.7e-3.
// 16-bit pools are loaded into the stages directly (8 rows and 2 KV heads of 512 keys 8.0 us through registers, 7.1 so; 64 of
// 1,024 15.0 and 14.6; head_dim 64 9.6 and 8.7); K's stage takes the next chunk once its operands are read, V's
// once its are.  The others are converted on their way, and share one stage between K and V.
// A decode row reads its keys once, so HBM bounds many rows and latency few: 64 rows of 2 KV heads and 2,048 FP8 keys
// take 15.6-16.4 us for 67 MB (9.3 at the rate of a large read; 2.6 us go before the first key, 1.7 after the last), 16 of
// 1,024 bf16 keys 6.3.  Rows of a chunk read the same pages again from the L2: 812 of 1,024 keys, 850 MB in 57-59 us,
// 15 TB/s; the 512 workgroups that a chip holds at once take a chunk's chain of loads, products and softmax in turn.  Two chunks in flight a wave, or two or eight waves, were no faster.
// MXFP4's registers are held to three waves a SIMD (96 rows 11.6 us, with two 11.9); FP8's are three's as they come.
template <int D, int NT, int KVT, int WAVES>
__global__ __launch_bounds__(64 * WAVES, KVT == LIA_FP4 && NT == 1 ? 3 : 2) void selected_kernel(SelectedParams p) {
    constexpr bool FP8 = KVT == LIA_FP8_E4M3, FP4 = KVT == LIA_FP4, DIRECT = !FP8 && !FP4, BF = KVT != LIA_F16;
    using T = Tile<D, FP4>;
    using S = Direct<D>;
    constexpr int KT = D / 32, DT = D / 16;
    constexpr uint32_t ROW = DIRECT ? S::ROW : T::ROW;
    constexpr uint32_t STAGE = DIRECT ? S::STAGE : 32 * kStrideV<D>, COLS = 16 * NT, SK = kStrideK<D>, SV = kStrideV<D>;
    __shared__ __attribute__((aligned(16))) uint8_t stages[WAVES * STAGE], v_stages[DIRECT ? WAVES * STAGE : 16];
    __shared__ float s_m[WAVES][COLS], s_l[WAVES][COLS];
    const uint32_t r = blockIdx.x, hk = blockIdx.y, part = blockIdx.z;
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t shift = p.page_shift;
    const uint32_t *picked = p.selected + ((size_t)r * p.hkv + hk) * p.budget;
    // everything that waits for nothing, at once: the row, the wave's first 64 entries of the list, the queries
    const uint32_t begin = part * p.per; // chunks of the list (the host bounds budget << shift)
    uint32_t base = 32 * (begin + wave) >> shift;
    uint32_t w_sel = base + lane < p.budget ? picked[base + lane] : kNone;
    const uint32_t pos = p.positions[r], listed = p.counts[r], seq = p.sequences[r];
    const uint32_t total = live_rows(p.cu, p.n_seqs, p.n_rows);
    u32x4 q[NT][KT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const uint32_t col = 16 * nt + li;
        const size_t at = ((size_t)r * p.hq + hk * p.group + min(col, p.group - 1)) * D;
#pragma unroll
        for (int ks = 0; ks < KT; ks++) {
            const uint32_t dim = FP4 ? D / 4 * g + 8 * ks : 32 * ks + 8 * g; // as the first product takes them
            float x[8];
            if (p.q_f32) load8<0>(p.q, at + dim, x);
            else load8<2>(p.q, at + dim, x);
            q[nt][ks] = u32x4{pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]), pack2<BF>(x[4], x[5]), pack2<BF>(x[6], x[7])};
        }
    }
    if (r >= total) return;
    const uint32_t count = min(listed, p.budget);
    const uint32_t *table = p.pages + (size_t)seq * p.stride;
    const uint32_t end = min(begin + p.per, ((count << shift) + 31) / 32);
    const size_t unit = (size_t)r * p.hkv + hk, rec = unit * p.parts + part;
    if (p.parts > 1 && begin >= end) { // (uniform) nothing here: a record without mass
        if (threadIdx.x < p.group) p.part_ml[rec * p.group + threadIdx.x] = make_float2(0.0f, 0.0f);
        return;
    }
    float m[NT], thr[NT];
    f32x4 l[NT], o[NT][DT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        m[nt] = 0.0f;
        thr[nt] = -INFINITY;
        l[nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int n = 0; n < DT; n++) o[nt][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    }
    // 64 entries of the list from `base`, one a lane: the keys that the row attends, the byte of the page's first key's head
    // (page 0's in the place of a page outside the pool) and the page's scales
    uint32_t w_limit = 0, w_lo = 0, w_hi = 0;
    float w_ks = 1.0f, w_vs = 1.0f;
    uint64_t w_held = 0;
    const uint32_t step = FP4 ? 1 : p.hkv; // heads between keys
    auto window = [&] {
        const bool live = base + lane < count && w_sel < p.stride && w_sel <= pos >> shift;
        uint32_t page = live ? table[w_sel] : kNone;
        const bool held = page < p.pool_pages;
        page = held ? page : 0;
        const uint64_t at = (FP4 ? ((uint64_t)page * p.hkv + hk) << shift : ((uint64_t)page << shift) * p.hkv + hk) * ROW;
        w_lo = (uint32_t)at;
        w_hi = (uint32_t)(at >> 32);
        w_limit = live ? min(pos - (w_sel << shift) + 1, 1u << shift) : 0u;
        w_held = __builtin_amdgcn_ballot_w64(held);
        if constexpr (FP8) {
            w_ks = ((const float *)p.k_scales)[(size_t)page * p.hkv + hk];
            w_vs = ((const float *)p.v_scales)[(size_t)page * p.hkv + hk];
        }
    };
    struct Chunk {
        T k[2], v[2];         // (16-bit pools: on their way to LDS instead)
        uint64_t first[2];    // byte of the tile's first key's head
        uint32_t limit[2];    // keys of the tile that the row attends
        bool held[2];
        float ks[2], vs[2];
    };
    Chunk x;
    constexpr int LOADS = DIRECT ? S::LOADS : T::LOADS;
    uint32_t offsets[LOADS];
#pragma unroll
    for (int i = 0; i < LOADS; i++) {
        if constexpr (DIRECT) offsets[i] = S::offset(i, step);
        else offsets[i] = T::offset(i, step);
    }
    auto place = [&](uint32_t c) {
        if (((32 * c + 16) >> shift) - base >= 64) {
            base = 32 * c >> shift;
            w_sel = base + lane < p.budget ? picked[base + lane] : kNone;
            window();
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint32_t key = 32 * c + 16 * j;
            const int i = (int)((key >> shift) - base);
            const uint32_t off = key & ((1u << shift) - 1);
            x.limit[j] = (uint32_t)min(max(__builtin_amdgcn_readlane((int)w_limit, i) - (int)off, 0), 16);
            x.held[j] = w_held >> i & 1;
            if constexpr (FP8) {
                x.ks[j] = u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(w_ks), i));
                x.vs[j] = u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(w_vs), i));
            }
            const uint64_t lo = (uint32_t)__builtin_amdgcn_readlane((int)w_lo, i), hi = (uint32_t)__builtin_amdgcn_readlane((int)w_hi, i);
            x.first[j] = (hi << 32 | lo) + off * (step * ROW); // (the host bounds a page's bytes)
        }
    };
    uint8_t *const stage = stages + wave * STAGE, *const v_stage = DIRECT ? v_stages + wave * STAGE : stage;
    // Loads of the chunk that was placed; where it has no keys, as many all the same, so that a wait can count them.
    auto fetch_k = [&](uint8_t *__restrict__ stage) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if constexpr (DIRECT)
                S::load(p.kc, x.first[j], x.held[j] ? x.limit[j] * step * S::ROW : 0, offsets, stage + j * S::TILE);
            else x.k[j].load(p.kc, p.k_scales, x.first[j], offsets);
        }
    };
    auto fetch_v = [&](uint8_t *__restrict__ v_stage) {
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if constexpr (DIRECT)
                S::load(p.vc, x.first[j], x.held[j] ? x.limit[j] * step * S::ROW : 0, offsets, v_stage + j * S::TILE);
            else x.v[j].load(p.vc, p.v_scales, x.first[j], offsets);
        }
    };
    // this lane's bytes in the stage: what it writes of K and V, K's operand (row li) and V's transposed read (row 4g + li / 4)
    uint8_t *const k_to = stage + T::template at_of<SK>(), *const v_to = stage + T::template at_of<SV>();
    const uint8_t *const k_from = stage + li * SK + 16 * g, *const v_from = stage + (4 * g + li / 4) * SV + 8 * (li & 3);
    uint32_t k_at[KT], v_at[DT]; // the same of direct stages, whose pieces are turned
    if constexpr (DIRECT) {
        const uint32_t v_row = 4 * g + li / 4;
#pragma unroll
        for (int i = 0; i < KT; i++) k_at[i] = S::row(li) + 16 * ((4 * i + g) ^ S::turn(li % S::KEYS));
#pragma unroll
        for (int n = 0; n < DT; n++)
            v_at[n] = S::row(v_row) + 16 * ((2 * n + (li & 3) / 2) ^ S::turn(v_row % S::KEYS)) + 8 * (li & 1);
    }
    uint32_t c = begin + wave;
    if (c < end) {
        window();
        place(c);
        fetch_k(stage);
        fetch_v(v_stage);
    }
    // (direct stages as arguments that do not alias: reads of one then wait for its own loads alone)
    auto chunk = [&](uint8_t *__restrict__ k_stage, uint8_t *__restrict__ v_stage) __attribute__((always_inline)) {
        const uint32_t lim[2] = {x.limit[0], x.limit[1]};
        float kf[2], vf[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            kf[j] = FP8 ? p.scale_log2 * x.ks[j] : p.scale_log2;
            vf[j] = FP8 ? x.vs[j] : 1.0f;
            if constexpr (!DIRECT)
                if (lim[j] < 16 || !x.held[j]) { // (uniform) slots without a key may hold anything
                    x.k[j].clear_from(x.held[j] ? lim[j] : 0);
                    x.v[j].clear_from(x.held[j] ? lim[j] : 0);
                    if (!x.held[j]) { kf[j] = p.scale_log2; vf[j] = 1.0f; }
                }
        }
        u32x4 a[2][KT];
        if constexpr (DIRECT) {
            wait_vmcnt<2 * LOADS>(); // K has come, V may be on its way
            asm volatile("" ::: "memory");
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < KT; i++) a[j][i] = *(const u32x4 *)(k_stage + k_at[i] + j * S::TILE);
        }
        // every operand of K is on its way before V takes its place (LDS keeps a wave's order), and the next chunk's loads are
        // issued as soon as this one's registers are written
        if constexpr (!DIRECT && !FP4) {
#pragma unroll
            for (int j = 0; j < 2; j++) x.k[j].template put<SK>(k_to + j * 16 * SK);
        }
        if constexpr (!DIRECT) {
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < KT; i++) {
                    if constexpr (FP4) a[j][i] = x.k[j].operand(i);
                    else a[j][i] = *(const u32x4 *)(k_from + j * 16 * SK + 64 * i);
                }
#pragma unroll
            for (int j = 0; j < 2; j++) x.v[j].template put<SV>(v_to + j * 16 * SV);
        }
        __builtin_amdgcn_sched_barrier(0);
        if constexpr (DIRECT) {
            if (c + WAVES < end) place(c + WAVES);
            else x.held[0] = x.held[1] = false;
            __builtin_amdgcn_s_waitcnt(0xC07F); // lgkmcnt(0): K's operands are read
            asm volatile("" ::: "memory");
            fetch_k(k_stage);
        } else if (c + WAVES < end) {
            place(c + WAVES);
            fetch_k(stage);
            fetch_v(stage);
        }
        __builtin_amdgcn_sched_barrier(0);
        f32x4 s[2][NT];
#pragma unroll
        for (int nt = 0; nt < NT; nt++) s[0][nt] = s[1][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int i = 0; i < KT; i++)
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int nt = 0; nt < NT; nt++) s[j][nt] = mfma16x16x32<BF>(a[j][i], q[nt][i], s[j][nt]);
        asm volatile("" ::: "memory"); // (the stage is read back through a builtin)
        // V^T: d rows 16 n .. +15, keys {4g .. 4g+3, 16+4g .. 16+4g+3} as P^T holds them
        u32x4 vt[DT];
        if constexpr (DIRECT) wait_vmcnt<2 * LOADS>(); // V has come, the next K may be on its way
        asm volatile("" ::: "memory");
#pragma unroll
        for (int n = 0; n < DT; n++) {
            const uint8_t *a0p = DIRECT ? v_stage + v_at[n] : v_from + 32 * n, *a1p = a0p + (DIRECT ? S::TILE : 16 * SV);
            const s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(a0p));
            const s16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(a1p));
            const u32x2 b0 = __builtin_bit_cast(u32x2, a0), b1 = __builtin_bit_cast(u32x2, a1);
            vt[n] = u32x4{b0.x, b0.y, b1.x, b1.y};
        }
        asm volatile("" ::: "memory"); // (the next chunk's staging stays behind these reads)
        u32x4 pb[NT], pl[NT]; // weights times V's scale, weights
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float e[2][4];
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    e[j][i] = __builtin_fmaf(s[j][nt][i], kf[j], -m[nt]);
                }
            if (lim[0] + lim[1] < 32) { // (uniform)
#pragma unroll
                for (int j = 0; j < 2; j++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        if (4 * g + i >= lim[j]) e[j][i] = -INFINITY;
            }
            float mx = fmaxf(fmaxf(fmaxf(e[0][0], e[0][1]), fmaxf(e[0][2], e[0][3])),
                             fmaxf(fmaxf(e[1][0], e[1][1]), fmaxf(e[1][2], e[1][3])));
            if (__builtin_amdgcn_ballot_w64(mx > thr[nt])) { // (uniform, rare after the first chunk)
                mx = rows_max(mx);
                if (mx > thr[nt]) { // the same in the four lanes of the column
                    // before the first key there is nothing to scale, and a score far below 0 would make of it 0 times infinity
                    const float f = thr[nt] == -INFINITY ? 0.0f : fast_exp2(-mx);
                    l[nt] *= f;
#pragma unroll
                    for (int n = 0; n < DT; n++) o[nt][n] *= f;
                    m[nt] += mx;
                    thr[nt] = 8.0f;
#pragma unroll
                    for (int j = 0; j < 2; j++)
#pragma unroll
                        for (int i = 0; i < 4; i++) e[j][i] -= mx;
                }
            }
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) e[j][i] = fast_exp2(e[j][i]);
            pl[nt] = u32x4{pack2<BF>(e[0][0], e[0][1]), pack2<BF>(e[0][2], e[0][3]), pack2<BF>(e[1][0], e[1][1]),
                           pack2<BF>(e[1][2], e[1][3])};
            pb[nt] = pl[nt];
            if constexpr (FP8)
                pb[nt] = u32x4{pack2<BF>(e[0][0] * vf[0], e[0][1] * vf[0]), pack2<BF>(e[0][2] * vf[0], e[0][3] * vf[0]),
                               pack2<BF>(e[1][0] * vf[1], e[1][1] * vf[1]), pack2<BF>(e[1][2] * vf[1], e[1][3] * vf[1])};
            const uint32_t one = BF ? 0x3F803F80u : 0x3C003C00u;
            l[nt] = mfma16x16x32<BF>(u32x4{one, one, one, one}, pl[nt], l[nt]);
        }
        if constexpr (DIRECT) {
            __builtin_amdgcn_s_waitcnt(0xC07F); // lgkmcnt(0): V's operands are read
            asm volatile("" ::: "memory");
            fetch_v(v_stage);
            __builtin_amdgcn_sched_barrier(0);
        }
#pragma unroll
        for (int n = 0; n < DT; n++)
#pragma unroll
            for (int nt = 0; nt < NT; nt++) o[nt][n] = mfma16x16x32<BF>(vt[n], pb[nt], o[nt][n]);
    };
#pragma unroll 1
    for (; c < end; c += WAVES) chunk(stage, v_stage);
    if constexpr (DIRECT) { // the last (empty) loads' zeros have come before the stages hold sums
        wait_vmcnt<0>();
        asm volatile("" ::: "memory");
    }
    // the waves' columns merged: each leaves its sums as they are, and takes the others' by their references
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const uint32_t col = 16 * nt + li;
        f32x4 *box = (f32x4 *)stage;
        if (nt) lds_barrier(); // the stages are free again
#pragma unroll
        for (int n = 0; n < DT; n++) box[n * 64 + lane] = o[nt][n];
        if (g == 0) {
            s_m[wave][col] = m[nt];
            s_l[wave][col] = l[nt][0];
        }
        lds_barrier();
        float M = -INFINITY, L = 0.0f, f[WAVES];
#pragma unroll
        for (int w = 0; w < WAVES; w++)
            if (s_l[w][col] != 0.0f) M = fmaxf(M, s_m[w][col]);
#pragma unroll
        for (int w = 0; w < WAVES; w++) {
            const float lw = s_l[w][col];
            f[w] = lw != 0.0f ? fast_exp2(s_m[w][col] - M) : 0.0f;
            L = __builtin_fmaf(lw, f[w], L);
        }
        if (col < p.group) {
            const float inv = L > 0.0f ? 1.0f / L : 0.0f;
#pragma unroll
            for (int n = 0; n < DT; n += WAVES) {
                const uint32_t d0 = 16 * (n + wave) + 4 * g;
                f32x4 x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int w = 0; w < WAVES; w++) x += ((const f32x4 *)(stages + w * STAGE))[(n + wave) * 64 + lane] * f[w];
                if (p.parts > 1) {
                    *(f32x4 *)(p.part_o + (rec * p.group + col) * D + d0) = x;
                } else {
                    x *= inv;
                    const size_t at = ((size_t)r * p.hq + hk * p.group + col) * D + d0;
                    if (p.out_f32) *(f32x4 *)((float *)p.out + at) = x;
                    else *(u32x2 *)((uint16_t *)p.out + at) = u32x2{pack2<true>(x.x, x.y), pack2<true>(x.z, x.w)};
                }
            }
            if (p.parts > 1 && wave == 0 && g == 0)
                p.part_ml[rec * p.group + col] = make_float2(M == -INFINITY ? 0.0f : M, L);
        }
    }
}

// The parts of a row's head joined: a wave for each, whose lanes hold the parts' masses and then four elements of every
// 256 / D-th part (64 parts at most).  What it reads is small: 3-4 us are a launch and two loads in turn.
template <int D>
__global__ __launch_bounds__(256) void selected_join_kernel(SelectedParams p) {
    constexpr uint32_t QUADS = D / 4, SHARE = 64 / QUADS;
    const uint32_t i = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t lane = threadIdx.x & 63, head = i % p.hq, r = i / p.hq;
    if (r >= p.n_rows) return;
    const uint32_t total = live_rows(p.cu, p.n_seqs, p.n_rows);
    const uint32_t hk = head / p.group, col = head % p.group;
    const size_t rec = ((size_t)r * p.hkv + hk) * p.parts;
    const uint32_t share = lane / QUADS, d0 = lane % QUADS * 4;
    constexpr uint32_t FLIGHT = 4; // loads on their way
    f32x4 y[FLIGHT];
    auto sums = [&](uint32_t w0) {
#pragma unroll
        for (uint32_t j = 0; j < FLIGHT; j++)
            y[j] = *(const f32x4 *)(p.part_o + ((rec + min(w0 + j * SHARE + share, p.parts - 1)) * p.group + col) * D + d0);
    };
    sums(0);
    const float2 ml = lane < p.parts ? p.part_ml[(rec + lane) * p.group + col] : make_float2(0.0f, 0.0f);
    const float M = rows_max(group_all<16>(ml.y != 0.0f ? ml.x : -INFINITY, [](float a, float b) { return fmaxf(a, b); }));
    const float f = ml.y != 0.0f ? fast_exp2(ml.x - M) : 0.0f;
    const float L = rows_sum(group_all<16>(ml.y * f, [](float a, float b) { return a + b; }));
    f32x4 x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t w0 = 0;;) {
#pragma unroll
        for (uint32_t j = 0; j < FLIGHT; j++) {
            const uint32_t w = w0 + j * SHARE + share;
            const float fw = __shfl(f, (int)min(w, 63u));
            if (w < p.parts && fw != 0.0f) x += y[j] * fw; // (a part without mass wrote no sums)
        }
        w0 += FLIGHT * SHARE;
        if (w0 >= p.parts) break;
        sums(w0);
    }
#pragma unroll
    for (uint32_t o = QUADS; o < 64; o <<= 1)
#pragma unroll
        for (int e = 0; e < 4; e++) x[e] += shfl_xor(x[e], (int)o);
    if (r >= total || share) return;
    x *= L > 0.0f ? 1.0f / L : 0.0f;
    const size_t at = ((size_t)r * p.hq + head) * D + d0;
    if (p.out_f32) *(f32x4 *)((float *)p.out + at) = x;
    else *(u32x2 *)((uint16_t *)p.out + at) = u32x2{pack2<true>(x.x, x.y), pack2<true>(x.z, x.w)};
}

} // namespace lia

using namespace lia;

extern "C" int lia_page_summaries(const lia_kv_layout *L, uint32_t rows, const uint32_t *slots, const void *kc,
                                  const float *k_scales, int8_t *codes, float *scales, lia_stream_t stream) {
    if (!L || !slots || !kc || !codes || !scales) return LIA_E_ARG;
    if (L->num_kv_heads == 0) return LIA_E_ARG;
    if (L->page_size < 16 || (L->page_size & (L->page_size - 1))) return LIA_E_UNSUPPORTED;
    if (L->head_dim != 64 && L->head_dim != 128) return LIA_E_UNSUPPORTED;
    if (L->dtype != LIA_F16 && L->dtype != LIA_BF16 && L->dtype != LIA_FP8_E4M3 && L->dtype != LIA_FP4)
        return LIA_E_UNSUPPORTED;
    if ((L->dtype == LIA_FP8_E4M3 || L->dtype == LIA_FP4) && !k_scales) return LIA_E_ARG;
    if (((uintptr_t)kc | (uintptr_t)codes) & 15) return LIA_E_ALIGN;
    if (((uintptr_t)scales | (uintptr_t)slots) & 3) return LIA_E_ALIGN;
    const uint64_t n = (uint64_t)rows * L->num_kv_heads;
    if (n >= (1ull << 26) - 256) return LIA_E_ARG; // (a wave each: 2^32 threads)
    if (rows == 0) return LIA_OK;
    hipError_t e;
#define LIA_SUMMARY(D, KVT)                                                                                            \
    e = launch<summary_kernel<D, KVT>>(dim3((uint32_t)((n + 3) / 4)), dim3(256), 0, (hipStream_t)stream, (uint32_t)n,  \
                                       L->num_kv_heads, (uint32_t)__builtin_ctz(L->page_size), L->pool_pages, slots,   \
                                       kc, (const void *)k_scales, codes, scales)
#define LIA_SUMMARY_D(KVT) do { if (L->head_dim == 128) LIA_SUMMARY(128, KVT); else LIA_SUMMARY(64, KVT); } while (0)
    switch (L->dtype) {
    case LIA_F16: LIA_SUMMARY_D(LIA_F16); break;
    case LIA_BF16: LIA_SUMMARY_D(LIA_BF16); break;
    case LIA_FP8_E4M3: LIA_SUMMARY_D(LIA_FP8_E4M3); break;
    default: LIA_SUMMARY_D(LIA_FP4); break;
    }
#undef LIA_SUMMARY_D
#undef LIA_SUMMARY
    return e == hipSuccess ? LIA_OK : LIA_E_HIP;
}

// The geometry that both calls over selected pages share.
static int validate_pages(const lia_attention_config *c) {
    if (!c) return LIA_E_ARG;
    if (c->num_kv_heads == 0 || c->num_q_heads == 0 || c->num_q_heads % c->num_kv_heads) return LIA_E_ARG;
    if (c->num_q_heads / c->num_kv_heads > 32 || c->num_kv_heads > 65535) return LIA_E_UNSUPPORTED;
    if (c->head_dim != 64 && c->head_dim != 128) return LIA_E_UNSUPPORTED;
    if (c->page_size < 16 || (c->page_size & (c->page_size - 1))) return LIA_E_UNSUPPORTED;
    if (c->q_dtype != LIA_F32 && c->q_dtype != LIA_BF16) return LIA_E_UNSUPPORTED;
    if (c->stride == 0 || c->max_seqs == 0 || c->max_rows == 0 || c->max_context == 0) return LIA_E_ARG;
    if (c->pool_pages == 0) return LIA_E_ARG; // page 0 is read in the place of others
    if ((uint64_t)c->pool_pages * c->num_kv_heads >= 1ull << 32) return LIA_E_UNSUPPORTED;
    if (c->max_rows >= 1u << 22) return LIA_E_UNSUPPORTED; // (workgroups of 1,024 threads a row)
    if ((uint64_t)c->max_rows * c->num_q_heads >= (1ull << 32) / (c->head_dim / 4) - 256) return LIA_E_UNSUPPORTED;
    return LIA_OK;
}

// Pages of the longest row.
static uint32_t page_span(const lia_attention_config *c) {
    const uint64_t n = ((uint64_t)c->max_context + c->page_size - 1) / c->page_size;
    return n < c->stride ? (uint32_t)n : c->stride;
}

static int validate_select(const lia_attention_config *c) {
    if (const int st = validate_pages(c)) return st;
    // workgroups of 256 pages are the grid's third extent
    if (page_span(c) > 65535ull * kScorePages) return LIA_E_UNSUPPORTED;
    return LIA_OK;
}

static uint64_t select_bytes(const lia_attention_config *c) {
    return (uint64_t)c->max_rows * c->num_kv_heads * page_span(c) * sizeof(float);
}

extern "C" size_t lia_page_select_workspace_bytes(const lia_attention_config *c) {
    return validate_select(c) == LIA_OK ? (size_t)select_bytes(c) : 0;
}

template <int D>
static hipError_t launch_scores(int ct, dim3 grid, hipStream_t s, const SelectPagesParams &p) {
    if (ct == 1) return launch<page_score_kernel<D, 1>>(grid, dim3(256), 0, s, p);
    if (ct == 2) return launch<page_score_kernel<D, 2>>(grid, dim3(256), 0, s, p);
    return launch<page_score_kernel<D, 4>>(grid, dim3(256), 0, s, p);
}

extern "C" int lia_page_select(const lia_attention_config *c, uint32_t n_seqs, uint32_t n_rows, const uint32_t *cu_seqlens,
                               const uint32_t *positions, const uint32_t *sequences, const uint32_t *pages, const void *q,
                               const int8_t *codes, const float *scales, uint32_t budget, uint32_t first, uint32_t recent,
                               uint32_t *selected, uint32_t *counts, void *workspace, size_t workspace_bytes,
                               lia_stream_t stream) {
    if (const int st = validate_select(c)) return st;
    if (n_seqs == 0 || n_seqs > c->max_seqs || n_rows == 0 || n_rows > c->max_rows) return LIA_E_ARG;
    if (!cu_seqlens || !positions || !sequences || !pages || !q || !codes || !scales || !selected || !counts || !workspace)
        return LIA_E_ARG;
    if (recent == 0 || (uint64_t)first + recent > budget) return LIA_E_ARG;
    if (((uintptr_t)q | (uintptr_t)codes | (uintptr_t)workspace) & 15) return LIA_E_ALIGN;
    if (((uintptr_t)scales | (uintptr_t)selected | (uintptr_t)counts) & 3) return LIA_E_ALIGN;
    if (workspace_bytes < select_bytes(c)) return LIA_E_WORKSPACE;
    const uint32_t group = c->num_q_heads / c->num_kv_heads, span = page_span(c);
    uint32_t pad = 0;
    while (1u << pad < group) pad++;
    // Rows of a tile: as many as there are columns for, and as a sequence has on average.  Prompt chunks (16 rows and
    // more a sequence) of groups of three heads and more share the pages' codes among four tiles of columns, which pays
    // once narrower tiles are six workgroups a compute unit (512 rows of groups of 8 and 2 KV heads, of 512 pages: 22.2 us
    // so, 20.7 narrow; of 1,024: 24.1 and 27.7; 2,048 of them 49.8 and 69.6; 16 of them 19.8 and 14.3).
    uint32_t rows = 1, tiles = n_rows;
    auto widen = [&](uint32_t columns) {
        rows = columns >> pad;
        while (rows > 1 && (uint64_t)n_seqs * (rows / 2) >= n_rows) rows /= 2;
        tiles = (n_rows + rows - 1) / rows;
    };
    int ct = group > 16 ? 2 : 1;
    widen(16 * ct);
    if (group > 2 && n_rows >= 16ull * n_seqs &&
        (uint64_t)tiles * c->num_kv_heads * ((span + kScorePages - 1) / kScorePages) >= 1536)
        widen(16 * (ct = 4));
    const SelectPagesParams p{cu_seqlens, positions, sequences, pages, q, codes, scales, (float *)workspace, selected, counts,
                              n_seqs, n_rows, c->num_q_heads, c->num_kv_heads, group, pad, rows, c->stride, span,
                              (uint32_t)__builtin_ctz(c->page_size), c->pool_pages, budget, first, recent,
                              c->q_dtype == LIA_F32};
    hipStream_t s = (hipStream_t)stream;
    hipError_t e = hipSuccess;
    // One launch for single rows where tables are short or workgroups many, each of which keeps a compute unit busy with its
    // table.  With the summaries' launch, in one and in two: 16 rows and heads of 1,024 pages 12.2 us and 12.1, of 512 10.6
    // and 11.9, of 2,048 15.8 and 12.4; 128 of 2,048 21.3 and 25.4, 64 of them 19.5 and 17.3.  Tiles of two rows took
    // longer in one launch nearly everywhere (8 sequences of 1,024 pages 15.4 and 13.0, 64 of them 18.2 and 17.7).
    // Pages are counted by the configuration, the host knows no step's; where that is far above the step's own, the form is
    // that of the longer tables (64 prompt rows over 1,000 pages 14.8 us, 20.5 configured for 8,192; 64 rows over 1,000
    // to 2,000 19.6, 24.4 for 16,384; 8 rows, 16 and 812 prompt rows the same).
    if (ct == 1 && rows == 1 && span <= kChooseSpan && (span <= 1024 || (uint64_t)n_rows * c->num_kv_heads >= 128)) {
        const dim3 grid(n_rows, c->num_kv_heads), block(kChooseThreads);
        const uint32_t bytes = span * (uint32_t)sizeof(float);
        e = c->head_dim == 128 ? launch<page_choose_kernel<128>>(grid, block, bytes, s, p)
                               : launch<page_choose_kernel<64>>(grid, block, bytes, s, p);
        return e == hipSuccess ? LIA_OK : LIA_E_HIP;
    }
    if (span > budget) { // (else every row keeps all its pages)
        const dim3 grid(tiles, c->num_kv_heads, (span + score_pages_of(ct) - 1) / score_pages_of(ct));
        e = c->head_dim == 128 ? launch_scores<128>(ct, grid, s, p) : launch_scores<64>(ct, grid, s, p);
    }
    if (e == hipSuccess) e = launch<page_pick_kernel>(dim3(n_rows, c->num_kv_heads), dim3(kPickThreads), 0, s, p);
    return e == hipSuccess ? LIA_OK : LIA_E_HIP;
}

static int validate_selected(const lia_attention_config *c, uint32_t budget) {
    if (const int st = validate_pages(c)) return st;
    if (c->out_dtype != LIA_F32 && c->out_dtype != LIA_BF16) return LIA_E_UNSUPPORTED;
    if (c->kv_dtype != LIA_F16 && c->kv_dtype != LIA_BF16 && c->kv_dtype != LIA_FP8_E4M3 && c->kv_dtype != LIA_FP4)
        return LIA_E_UNSUPPORTED;
    if (!(c->scale > 0.0f) || !(c->scale < INFINITY)) return LIA_E_ARG;
    if ((uint64_t)c->page_size * c->num_kv_heads * c->head_dim * 2 >= 1ull << 31) return LIA_E_UNSUPPORTED; // bytes of a page
    if (budget == 0 || (uint64_t)budget * c->page_size >= (1ull << 31)) return LIA_E_ARG;
    return LIA_OK;
}

// Workgroups that share a row and KV head: as many as give the chip a workgroup a compute unit, each with a chunk for every
// wave, where a list is long enough to be worth the launch that joins them.  Chunks up to which a list stays whole, and the
// times on either side, whole and shared, in us over three inputs in turn (head_dim 128, 8 heads a KV head):
//   16-bit: 24 up to 32 rows and heads (32 of them: 768 keys 9.5 and 9.8, 1,024 11.0 and 10.7), 40 up to 128 (64: 1,024 keys
//     11.4 and 12.7, 1,536 15.4 and 14.9; 66: 4,096 keys 52 and 32; 128: 1,024 keys 15.5 and 18.2, 1,536 25.8 and 23.9, 16,384
//     221 and 190); keys of head_dim 64 are half as long, and above 64 rows and heads it is 64 (128: 2,048 keys 16.6 and
//     18.7, 4,096 40 and 30);
//   FP8, whose chunks take longer: 12 up to 64 (32: 512 keys 8.5 and 8.0; 64: 9.2 and 9.2), 20 up to 128 (66: 768 keys
//     11.8 and 10.9; 128: 768 keys 12.1 and 12.5, 1,024 14.4 and 13.7, 16,384 170 and 104);
//   MXFP4: 16 up to 64 (64: 512 keys 7.5 and 8.2, 768 9.4 and 9.3), 24 up to 128 (128: 768 keys 10.3 and 11.1, 1,024
//     11.9 and 11.8, 16,384 133 and 82).
// More rows and heads stay whole.  16-bit lists gain little there (130, in three parts: 1,024 keys 15.5 and 18.8, 4,096 63 and
// 61, 16,384 222 and 207); FP8 and MXFP4 lists would gain from 2,048 keys on (130: 23.9 and 20.6, 19.2 and 15.4; 192, in
// two: 27.9 and 27.1, 19.5 and 18.8; of 16,384 keys 193 and 161, 141 and 98), for records of twice this workspace.
constexpr uint32_t kSelectedFill = 256, kSelectedWaves = 4;
static uint32_t selected_parts(const lia_attention_config *c, uint32_t n_rows, uint32_t budget) {
    const uint64_t units = (uint64_t)n_rows * c->num_kv_heads, chunks = ((uint64_t)budget * c->page_size + 31) / 32;
    const bool few = units <= kSelectedFill / 4;
    uint64_t whole;
    if (c->kv_dtype == LIA_FP8_E4M3) whole = few ? 12 : 20;
    else if (c->kv_dtype == LIA_FP4) whole = few ? 16 : 24;
    else whole = units <= kSelectedFill / 8 ? 24 : few || c->head_dim == 128 ? 40 : 64;
    if (units > kSelectedFill / 2 || chunks <= whole) return 1;
    return (uint32_t)std::min<uint64_t>(std::min(kSelectedFill / units, (chunks + kSelectedWaves - 1) / kSelectedWaves), 64);
}

// Records of the step that has most.
static uint64_t selected_bytes(const lia_attention_config *c) {
    return (uint64_t)kSelectedFill * (c->num_q_heads / c->num_kv_heads) * (c->head_dim * sizeof(float) + sizeof(float2));
}

extern "C" size_t lia_selected_attention_workspace_bytes(const lia_attention_config *c, uint32_t budget) {
    return validate_selected(c, budget) == LIA_OK ? (size_t)selected_bytes(c) : 0;
}

template <int D, int NT>
static hipError_t launch_selected(int kv, dim3 grid, hipStream_t s, const SelectedParams &p) {
    const dim3 block(64 * kSelectedWaves);
    if (kv == LIA_BF16) return launch<selected_kernel<D, NT, LIA_BF16, kSelectedWaves>>(grid, block, 0, s, p);
    if (kv == LIA_F16) return launch<selected_kernel<D, NT, LIA_F16, kSelectedWaves>>(grid, block, 0, s, p);
    if (kv == LIA_FP4) return launch<selected_kernel<D, NT, LIA_FP4, kSelectedWaves>>(grid, block, 0, s, p);
    return launch<selected_kernel<D, NT, LIA_FP8_E4M3, kSelectedWaves>>(grid, block, 0, s, p);
}

extern "C" int lia_selected_attention(const lia_attention_config *c, uint32_t n_seqs, uint32_t n_rows,
                                      const uint32_t *cu_seqlens, const uint32_t *positions, const uint32_t *sequences,
                                      const uint32_t *pages, const void *q, const void *kc, const void *vc,
                                      const float *k_scales, const float *v_scales, uint32_t budget,
                                      const uint32_t *selected, const uint32_t *counts, void *workspace,
                                      size_t workspace_bytes, void *out, lia_stream_t stream) {
    if (const int st = validate_selected(c, budget)) return st;
    if (n_seqs == 0 || n_seqs > c->max_seqs || n_rows == 0 || n_rows > c->max_rows) return LIA_E_ARG;
    if (!cu_seqlens || !positions || !sequences || !pages || !q || !kc || !vc || !selected || !counts || !workspace || !out)
        return LIA_E_ARG;
    if ((c->kv_dtype == LIA_FP8_E4M3 || c->kv_dtype == LIA_FP4) && (!k_scales || !v_scales)) return LIA_E_ARG;
    if (((uintptr_t)q | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)workspace | (uintptr_t)out) & 15) return LIA_E_ALIGN;
    if (((uintptr_t)selected | (uintptr_t)counts) & 3) return LIA_E_ALIGN;
    if (workspace_bytes < selected_bytes(c)) return LIA_E_WORKSPACE;
    const uint32_t group = c->num_q_heads / c->num_kv_heads, parts = selected_parts(c, n_rows, budget);
    SelectedParams p{cu_seqlens, positions, sequences, pages, selected, counts, q, kc, vc, k_scales, v_scales, out,
                     (float *)workspace, nullptr, n_seqs, n_rows, c->num_q_heads, c->num_kv_heads, group, c->stride,
                     (uint32_t)__builtin_ctz(c->page_size), c->pool_pages, budget, parts,
                     (uint32_t)((((uint64_t)budget * c->page_size + 31) / 32 + parts - 1) / parts), c->q_dtype == LIA_F32,
                     c->out_dtype == LIA_F32, c->scale * 1.4426950408889634f};
    p.part_ml = (float2 *)(p.part_o + (uint64_t)kSelectedFill * group * c->head_dim);
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid(n_rows, c->num_kv_heads, parts);
    hipError_t e;
    if (c->head_dim == 128)
        e = group > 16 ? launch_selected<128, 2>(c->kv_dtype, grid, s, p) : launch_selected<128, 1>(c->kv_dtype, grid, s, p);
    else
        e = group > 16 ? launch_selected<64, 2>(c->kv_dtype, grid, s, p) : launch_selected<64, 1>(c->kv_dtype, grid, s, p);
    if (e == hipSuccess && parts > 1) {
        const dim3 join((n_rows * c->num_q_heads + 3) / 4);
        e = c->head_dim == 128 ? launch<selected_join_kernel<128>>(join, dim3(256), 0, s, p)
                               : launch<selected_join_kernel<64>>(join, dim3(256), 0, s, p);
    }
    return e == hipSuccess ? LIA_OK : LIA_E_HIP;
}
