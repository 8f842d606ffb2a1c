// Attention over selected pages of a paged KV pool (gfx950): summaries of full pages, the selection of pages for each row and
// KV head by their summaries, and the attention over the selection.
#include "common.hpp"
#include "launch.hpp"
#include "rows.hpp"

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
// of a key's row side by side, so that a load covers whole rows.
template <int D, int KVT>
__global__ __launch_bounds__(256) void summary_kernel(uint32_t n, uint32_t hkv, uint32_t page_shift, uint32_t pool_pages,
                                                      const uint32_t *slots, const void *kc, const void *k_scales,
                                                      int8_t *codes, float *scales) {
    constexpr uint32_t PER = D / 8, ROWS = 64 / PER; // lanes of a row, rows of a load
    const uint32_t w = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (w >= n) return;
    const uint32_t slot = slots[w / hkv], h = w % hkv, P = 1u << page_shift, page = slot >> page_shift;
    if ((slot & (P - 1)) != P - 1 || page >= pool_pages) return;
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
    float top = 0.0f;
#pragma unroll
    for (int j = 0; j < 8; j++) {
#pragma unroll
        for (uint32_t o = PER; o < 64; o <<= 1) {
            hi[j] = fmaxf(hi[j], shfl_xor(hi[j], (int)o));
            lo[j] = fminf(lo[j], shfl_xor(lo[j], (int)o));
        }
        top = fmaxf(top, fmaxf(fabsf(hi[j]), fabsf(lo[j])));
    }
#pragma unroll
    for (uint32_t o = 1; o < PER; o <<= 1) top = fmaxf(top, shfl_xor(top, (int)o));
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
    uint32_t n_seqs, n_rows, hq, hkv, group, pad_shift; // pad_shift: log2 of the columns that a row's heads take
    uint32_t stride, span, page_shift, pool_pages;      // span: pages of the longest row
    uint32_t budget, first, recent, q_f32;
};

__device__ __forceinline__ uint32_t live_rows(const uint32_t *cu, uint32_t n_seqs, uint32_t n_rows) {
    return min(cu[n_seqs], n_rows);
}
__device__ __forceinline__ uint32_t row_pages(uint32_t position, uint32_t page_shift, uint32_t span) {
    return min((position >> page_shift) + 1, span); // (no overflow: pages hold 16 keys at least)
}

constexpr uint32_t kScorePages = 256; // pages of a workgroup, 64 a wave

// Scores of 64 pages a wave for the 16 CT columns of a tile of rows: consecutive rows of one sequence, each with its
// group's heads as columns.  A = the queries' codes, their positive part against the largest values and their negative part
// against the smallest, B = the pages' codes; both operands hold 16 bytes a lane of the same 64, so the products add up over
// the head whatever their order within it, and exactly, in 32-bit integers.
template <int D, int CT>
__global__ __launch_bounds__(256) void page_score_kernel(SelectPagesParams p) {
    constexpr int KS = D / 64; // k steps of each part
    const uint32_t r0 = blockIdx.x, h = blockIdx.y, lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    const uint32_t total = live_rows(p.cu, p.n_seqs, p.n_rows);
    if (r0 >= total) return;
    const uint32_t rows = (16u * CT) >> p.pad_shift; // rows of a tile: those whose positions share a multiple of it
    const uint32_t pos0 = p.positions[r0], seq = p.sequences[r0];
    if (r0 > 0 && (pos0 & (rows - 1)) && p.sequences[r0 - 1] == seq && p.positions[r0 - 1] + 1 == pos0) return;
    bool in = lane < rows && r0 + lane < total && (pos0 & (rows - 1)) + lane < rows;
    if (in) in = p.sequences[r0 + lane] == seq && p.positions[r0 + lane] == pos0 + lane;
    const uint64_t ins = __builtin_amdgcn_ballot_w64(in);
    const uint32_t nrows = ~ins ? (uint32_t)__builtin_ctzll(~ins) : 64u;
    const uint32_t n = row_pages(pos0 + nrows - 1, p.page_shift, p.span);
    if (n <= p.budget) return; // every row keeps all its pages
    const uint32_t lo = p.first, hi = n - p.recent, base = blockIdx.z * kScorePages + wave * 64;
    if (base >= hi || base + 64 <= lo) return;
    const uint32_t at = base + lane;
    const uint32_t page = at < hi ? p.pages[(size_t)seq * p.stride + at] : kNone;
    const bool held = page < p.pool_pages;
    const uint32_t mine = held ? page : 0;
    const float scale = held ? p.scales[(size_t)mine * p.hkv + h] : 0.0f; // (0: pages outside the pool score 0)
    i32x4 b[4][2 * KS];
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const uint32_t pg = (uint32_t)__shfl((int)mine, 16 * k + (int)li);
        const int8_t *from = p.codes + ((size_t)pg * p.hkv + h) * (2 * D) + 16 * g;
#pragma unroll
        for (int s = 0; s < 2 * KS; s++) b[k][s] = *(const i32x4 *)(from + 64 * s);
    }
    i32x4 a[CT][2 * KS];
    float u[CT][4]; // units of the columns that this lane's results belong to, 0 where there is none
#pragma unroll
    for (int c = 0; c < CT; c++) {
        const uint32_t m = 16 * c + li, row = m >> p.pad_shift, head = m & ((1u << p.pad_shift) - 1);
        const bool valid = row < nrows && head < p.group;
        const size_t from = ((size_t)(r0 + (valid ? row : 0)) * p.hq + h * p.group + (valid ? head : 0)) * D + 16 * g;
        float x[KS][16], top = 0.0f;
#pragma unroll
        for (int s = 0; s < KS; s++) {
#pragma unroll
            for (int e = 0; e < 16; e += 8) {
                float y[8];
                if (p.q_f32) load8<0>(p.q, from + 64 * s + e, y);
                else load8<2>(p.q, from + 64 * s + e, y);
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    x[s][e + j] = y[j];
                    top = fmaxf(top, fabsf(y[j]));
                }
            }
        }
        const uint32_t field = unit_field(f2u(rows_max(top)));
#pragma unroll
        for (int s = 0; s < KS; s++) {
#pragma unroll
            for (int w = 0; w < 4; w++) {
                int up[4], down[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int v = code_of(x[s][4 * w + j], field);
                    up[j] = max(v, 0);
                    down[j] = min(v, 0);
                }
                a[c][s][w] = (int)pack_codes(up[0], up[1], up[2], up[3]);
                a[c][KS + s][w] = (int)pack_codes(down[0], down[1], down[2], down[3]);
            }
        }
        const float unit = valid ? u2f(field << 23) : 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++) u[c][i] = __shfl(unit, 4 * (int)g + i);
    }
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const float sc = __shfl(scale, 16 * k + (int)li);
        const uint32_t to = base + 16 * k + li;
        const bool write = to >= lo && to < hi;
        float best[CT][4];
#pragma unroll
        for (int c = 0; c < CT; c++) {
            i32x4 sum = i32x4{0, 0, 0, 0};
#pragma unroll
            for (int s = 0; s < 2 * KS; s++) sum = __builtin_amdgcn_mfma_i32_16x16x64_i8(a[c][s], b[k][s], sum, 0, 0, 0);
#pragma unroll
            for (int i = 0; i < 4; i++) best[c][i] = u[c][i] > 0.0f ? (float)sum[i] * u[c][i] : -INFINITY;
        }
        // (rounding keeps the order, so the largest product times the page's unit is the largest of the scores)
        auto put = [&](uint32_t row, float x) {
            if (write && row < nrows)
                p.scores[((size_t)(r0 + row) * p.hkv + h) * p.span + to] = (sc < INFINITY ? x * sc : INFINITY) + 0.0f;
        };
#pragma unroll
        for (int c = 0; c < CT; c++) {
            if (p.pad_shift == 0) {
#pragma unroll
                for (int i = 0; i < 4; i++) put(16 * c + 4 * g + i, best[c][i]);
                continue;
            }
            const float x = fmaxf(best[c][0], best[c][1]), y = fmaxf(best[c][2], best[c][3]);
            if (p.pad_shift == 1) {
                put(8 * c + 2 * g, x);
                put(8 * c + 2 * g + 1, y);
                continue;
            }
            float z = fmaxf(x, y);
            if (p.pad_shift >= 3) z = fmaxf(z, shfl_xor(z, 16));
            if (p.pad_shift >= 4) z = fmaxf(z, shfl_xor(z, 32));
            if (p.pad_shift == 5) { // 32 columns a row: two tiles
                best[c][0] = z;
                if (c & 1) {
                    z = fmaxf(z, best[c - (c & 1)][0]);
                    if (g == 0) put(c / 2, z);
                }
                continue;
            }
            if ((g & ((1u << (p.pad_shift - 2)) - 1)) == 0) put((16 * c + 4 * g) >> p.pad_shift, z);
        }
    }
}

// ------------------------------------------------------------------ page selection

constexpr uint32_t kPickBins = 1024, kPickDirect = 64;

// One workgroup per row and KV head.  A candidate is a pair (score's place in the floats' total order, counted from the lowest
// candidate's; pages from the last candidate), and the last kept one is found from the top: ten bits of the pair at a time,
// beginning at the highest bit in which the scores differ, until the digit's bin holds 64 candidates at most, which are
// ranked directly.  Pairs are distinct, so the kept ones are those not below it, and equal scores go by the lower page.
template <int THREADS, int ROWS>
__global__ __launch_bounds__(THREADS) void page_pick_kernel(SelectPagesParams p) {
    constexpr uint32_t WAVES = THREADS / 64, SEG = THREADS * ROWS, BINS = kPickBins / THREADS > 0 ? kPickBins / THREADS : 1;
    __shared__ uint32_t hist[kPickBins], red[2 * WAVES], bin_s, above_s, in_s, listed;
    __shared__ uint64_t list[kPickDirect], last_s;
    const uint32_t r = blockIdx.x, h = blockIdx.y, t = threadIdx.x, lane = t & 63;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(t >> 6));
    if (r >= live_rows(p.cu, p.n_seqs, p.n_rows)) return;
    const uint32_t n = row_pages(p.positions[r], p.page_shift, p.span);
    uint32_t *out = p.selected + ((size_t)r * p.hkv + h) * p.budget;
    if (h == 0 && t == 0) p.counts[r] = min(n, p.budget);
    if (n <= p.budget) {
        for (uint32_t i = t; i < p.budget; i += THREADS) out[i] = i < n ? i : kNone;
        return;
    }
    const uint32_t k0 = p.budget - p.first - p.recent, c = n - p.first - p.recent; // kept of the candidates; c > k0
    for (uint32_t i = t; i < p.first; i += THREADS) out[i] = i;
    for (uint32_t i = t; i < p.recent; i += THREADS) out[p.first + k0 + i] = n - p.recent + i;
    if (k0 == 0) return;
    const float *scores = p.scores + ((size_t)r * p.hkv + h) * p.span + p.first;
    const uint32_t segments = (c + SEG - 1) / SEG;
    uint32_t v[ROWS];
    auto place = [&](uint32_t seg, uint32_t x) { return seg * SEG + (wave * ROWS + x) * 64 + lane; };
    auto load = [&](uint32_t seg) {
#pragma unroll
        for (uint32_t x = 0; x < ROWS; x++) {
            const uint32_t b = f2u(scores[min(place(seg, x), c - 1)]);
            v[x] = b ^ ((b >> 31) ? 0xffffffffu : 0x80000000u);
        }
    };
    uint32_t low = 0xffffffffu, high = 0;
    for (uint32_t seg = 0; seg < segments; seg++) {
        load(seg);
#pragma unroll
        for (uint32_t x = 0; x < ROWS; x++) { low = min(low, v[x]); high = max(high, v[x]); }
    }
#pragma unroll
    for (int o = 32; o; o >>= 1) {
        low = min(low, (uint32_t)__shfl_xor((int)low, o));
        high = max(high, (uint32_t)__shfl_xor((int)high, o));
    }
    if (lane == 0) { red[2 * wave] = low; red[2 * wave + 1] = high; }
    __syncthreads();
    for (uint32_t w = 0; w < WAVES; w++) { low = min(low, red[2 * w]); high = max(high, red[2 * w + 1]); }
    // the pair: the score above the lowest one, then c - 1 - page in as many bits as that takes
    const uint32_t page_bits = 32 - (uint32_t)__builtin_clz(c - 1), range = high - low; // (c > 1)
    auto pair = [&](uint32_t seg, uint32_t x) { return (uint64_t)(v[x] - low) << page_bits | (c - 1 - place(seg, x)); };
    uint32_t bits = page_bits + (range ? 32 - (uint32_t)__builtin_clz(range) : 0);
    uint64_t found = 0, known = bits >= 64 ? 0ull : ~0ull << bits; // the bits above are 0 in every pair
    uint32_t k = k0, many = c;
    while (many > kPickDirect && many > k) {
        const uint32_t shift = bits > 10 ? bits - 10 : 0, width = bits - shift;
        __syncthreads();
        for (uint32_t i = t; i < kPickBins; i += THREADS) hist[i] = 0;
        __syncthreads();
        for (uint32_t seg = 0; seg < segments; seg++) {
            if (segments > 1) load(seg);
#pragma unroll
            for (uint32_t x = 0; x < ROWS; x++) {
                const uint64_t y = pair(seg, x);
                if (place(seg, x) < c && (y & known) == found)
                    atomicAdd(&hist[(uint32_t)(y >> shift) & ((1u << width) - 1)], 1u);
            }
        }
        __syncthreads();
        uint32_t own[BINS], sum = 0; // thread t: BINS bins, the t-th from the top
        if (t < kPickBins / BINS) {
#pragma unroll
            for (uint32_t i = 0; i < BINS; i++) { own[i] = hist[kPickBins - 1 - t * BINS - i]; sum += own[i]; }
        }
        uint32_t upto = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint32_t y = (uint32_t)__shfl_up((int)upto, o);
            if (lane >= (uint32_t)o) upto += y;
        }
        if (lane == 63) red[wave] = upto;
        __syncthreads();
        uint32_t over = upto - sum;
        for (uint32_t w = 0; w < wave; w++) over += red[w];
        if (t < kPickBins / BINS && over < k && k <= over + sum) {
#pragma unroll
            for (uint32_t i = 0; i < BINS; i++) {
                if (over < k && k <= over + own[i]) {
                    bin_s = kPickBins - 1 - t * BINS - i;
                    above_s = over;
                    in_s = own[i];
                }
                over += own[i];
            }
        }
        __syncthreads();
        found |= (uint64_t)bin_s << shift;
        known |= (uint64_t)((1u << width) - 1) << shift;
        k -= above_s;
        many = in_s;
        bits = shift;
    }
    // the lowest kept pair: every one of the last bin's, or its k-th from the top
    uint64_t last = found;
    if (many > k) {
        if (t == 0) listed = 0;
        __syncthreads();
        for (uint32_t seg = 0; seg < segments; seg++) {
            if (segments > 1) load(seg);
#pragma unroll
            for (uint32_t x = 0; x < ROWS; x++) {
                const uint64_t y = pair(seg, x);
                if (place(seg, x) < c && (y & known) == found) list[atomicAdd(&listed, 1u)] = y;
            }
        }
        __syncthreads();
        if (t < many) {
            const uint64_t y = list[t];
            uint32_t rank = 1;
            for (uint32_t i = 0; i < many; i++) rank += list[i] > y;
            if (rank == k) last_s = y;
        }
        __syncthreads();
        last = last_s;
    }
    uint32_t before = p.first;
    for (uint32_t seg = 0; seg < segments; seg++) {
        if (segments > 1) load(seg);
        uint64_t keep[ROWS];
        uint32_t count = 0;
#pragma unroll
        for (uint32_t x = 0; x < ROWS; x++) {
            keep[x] = __builtin_amdgcn_ballot_w64(place(seg, x) < c && pair(seg, x) >= last);
            count += (uint32_t)__builtin_popcountll(keep[x]);
        }
        __syncthreads();
        if (lane == 0) red[wave] = count;
        __syncthreads();
        uint32_t at = before;
        for (uint32_t w = 0; w < WAVES; w++) {
            if (w < wave) at += red[w];
            before += red[w];
        }
#pragma unroll
        for (uint32_t x = 0; x < ROWS; x++) {
            if (keep[x] >> lane & 1)
                out[at + (uint32_t)__builtin_popcountll(keep[x] & ((1ull << lane) - 1))] = p.first + place(seg, x);
            at += (uint32_t)__builtin_popcountll(keep[x]);
        }
    }
}

// ------------------------------------------------------------------ attention over selected pages

struct SelectedParams {
    const uint32_t *cu, *positions, *sequences, *pages, *selected, *counts;
    const void *q, *kc, *vc, *k_scales, *v_scales;
    void *out;
    float *part_o;   // [unit][part][head of the group][D]: unnormalised sums
    float2 *part_ml; // [unit][part][head]: reference (log2), mass
    uint32_t n_seqs, n_rows, hq, hkv, group, stride, page_shift, pool_pages, budget;
    uint32_t parts, q_f32, out_f32;
    float scale_log2;
};

// How a pool type's tiles of 16 keys lie in registers: lane (g, li) holds D / 4 elements of key li, in pieces of eight
// that are one operand each.  dim(ks): the first element of piece ks.
template <int D, int KVT>
struct Tile {
    static constexpr bool F16 = KVT == LIA_F16, FP8 = KVT == LIA_FP8_E4M3, FP4 = KVT == LIA_FP4;
    static constexpr int KT = D / 32, DT = D / 16;
    static constexpr int WORDS = FP4 ? D / 32 : FP8 ? D / 16 : D / 8;
    uint32_t w[WORDS], s;

    static __device__ __forceinline__ uint32_t dim(uint32_t g, int ks) {
        if constexpr (FP4) return D / 4 * g + 8 * ks;
        else if constexpr (FP8) return 64 * (ks / 2) + 16 * g + 8 * (ks % 2);
        else return 32 * ks + 8 * g;
    }
    // row: the key's head, counted in heads over the plane
    __device__ __forceinline__ void load(const void *plane, const void *scales, size_t row, uint32_t g) {
        if constexpr (FP4) {
            const uint8_t *from = (const uint8_t *)plane + row * (D / 2) + g * (D / 8);
            if constexpr (D == 128) {
                const u32x4 a = *(const u32x4 *)from;
                w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
            } else {
                const u32x2 a = *(const u32x2 *)from;
                w[0] = a.x; w[1] = a.y;
            }
            s = ((const uint8_t *)scales)[row * (D / 32) + (D == 128 ? g : g >> 1)];
        } else {
            const uint8_t *from = (const uint8_t *)plane + row * (FP8 ? D : 2 * D) + 16 * g;
#pragma unroll
            for (int i = 0; i < WORDS / 4; i++) {
                const u32x4 a = *(const u32x4 *)(from + 64 * i);
                w[4 * i] = a.x; w[4 * i + 1] = a.y; w[4 * i + 2] = a.z; w[4 * i + 3] = a.w;
            }
        }
    }
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < WORDS; i++) w[i] = 0;
        s = 0;
    }
    // Piece ks as eight 16-bit values, exactly (FP8 and MXFP4: bf16; the page's scale of FP8 codes is the caller's).
    __device__ __forceinline__ u32x4 piece(int ks) const {
        if constexpr (FP4) {
            return e2m1x8_to_bf16x8(w[ks], u2f(s << 23));
        } else if constexpr (FP8) {
            typedef __attribute__((ext_vector_type(2))) __bf16 b2;
            const uint32_t x = w[2 * ks], y = w[2 * ks + 1];
            return u32x4{__builtin_bit_cast(uint32_t, (b2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, false)),
                         __builtin_bit_cast(uint32_t, (b2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(x, 1.0f, true)),
                         __builtin_bit_cast(uint32_t, (b2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.0f, false)),
                         __builtin_bit_cast(uint32_t, (b2)__builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(y, 1.0f, true))};
        } else {
            return u32x4{w[4 * ks], w[4 * ks + 1], w[4 * ks + 2], w[4 * ks + 3]};
        }
    }
};

constexpr int kSelWaves = 4;

// Swizzle of the 16-byte chunks of a staged row of V: rows that a transposed read serves together lie in different banks.
template <int D>
__device__ __forceinline__ uint32_t sel_swizzle(uint32_t row) { return D == 128 ? 2 * (row & 7) : 2 * ((row >> 1) & 1); }

// One row's selected keys of one KV head, or a part of them: its waves take every fourth chunk of 32 keys of the list and
// merge through LDS at the end.  S^T = K Q^T with K's operands straight from memory; V goes through the wave's LDS, whose
// transposed reads give keys side by side; softmax in the log2 domain with a reference that is raised when a score passes it
// by 8.
template <int D, int NT, int KVT>
__global__ __launch_bounds__(64 * kSelWaves, NT == 1 ? 3 : 2) void selected_kernel(SelectedParams p) {
    using T = Tile<D, KVT>;
    constexpr bool BF = !T::F16;
    constexpr int KT = T::KT, DT = T::DT;
    constexpr uint32_t STAGE = 32 * D, COLS = 16 * NT;
    __shared__ __attribute__((aligned(16))) uint16_t stages[kSelWaves * STAGE];
    __shared__ float s_m[kSelWaves][COLS], s_l[kSelWaves][COLS];
    const uint32_t r = blockIdx.x, hk = blockIdx.y, part = blockIdx.z;
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (r >= live_rows(p.cu, p.n_seqs, p.n_rows)) return;
    const uint32_t shift = p.page_shift, pos = p.positions[r];
    const uint32_t count = min(p.counts[r], p.budget);
    const uint32_t *table = p.pages + (size_t)p.sequences[r] * p.stride;
    const uint32_t *picked = p.selected + ((size_t)r * p.hkv + hk) * p.budget;
    const uint32_t keys = count << shift, chunks = (keys + 31) / 32; // (the host bounds budget << shift)
    const uint32_t per = (chunks + p.parts - 1) / p.parts;
    const uint32_t begin = min(part * per, chunks), end = min(begin + per, chunks);
    const size_t unit = (size_t)r * p.hkv + hk, rec = unit * p.parts + part;
    if (p.parts > 1 && begin == end) { // (uniform) nothing here: a record without mass
        if (threadIdx.x < p.group) p.part_ml[rec * p.group + threadIdx.x] = make_float2(0.0f, 0.0f);
        return;
    }
    u32x4 q[NT][KT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const uint32_t col = 16 * nt + li;
        const size_t at = ((size_t)r * p.hq + hk * p.group + min(col, p.group - 1)) * D;
#pragma unroll
        for (int ks = 0; ks < KT; ks++) {
            float x[8];
            if (p.q_f32) load8<0>(p.q, at + T::dim(g, ks), x);
            else load8<2>(p.q, at + T::dim(g, ks), x);
            q[nt][ks] = u32x4{pack2<BF>(x[0], x[1]), pack2<BF>(x[2], x[3]), pack2<BF>(x[4], x[5]), pack2<BF>(x[6], x[7])};
        }
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
    // 64 entries of the list from `base`, one a lane: first key, page (0 in the place of one outside the pool) and scales
    uint32_t base = begin * 32 >> shift, w_key = 0, w_page = 0;
    float w_ks = 1.0f, w_vs = 1.0f;
    uint64_t w_live = 0, w_held = 0;
    auto window = [&](uint32_t from) {
        base = from;
        const uint32_t i = from + lane;
        const uint32_t sel = i < count ? picked[i] : kNone;
        const bool live = sel < p.stride && sel <= pos >> shift;
        const uint32_t page = live ? table[sel] : kNone;
        const bool held = page < p.pool_pages;
        w_key = sel << shift;
        w_page = held ? page : 0;
        w_live = __builtin_amdgcn_ballot_w64(live);
        w_held = __builtin_amdgcn_ballot_w64(held);
        if constexpr (T::FP8) {
            w_ks = ((const float *)p.k_scales)[(size_t)w_page * p.hkv + hk];
            w_vs = ((const float *)p.v_scales)[(size_t)w_page * p.hkv + hk];
        }
    };
    T k[2], v[2];
    uint32_t limit[2]; // keys of the tile that the row attends
    bool held[2];
    float ks_of[2], vs_of[2];
    auto fetch = [&](uint32_t c) {
        if (((32 * c + 16) >> shift) - base >= 64) window(32 * c >> shift);
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint32_t key = 32 * c + 16 * j;
            const int i = (int)((key >> shift) - base);
            const uint32_t off = key & ((1u << shift) - 1);
            const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)w_key, i) + off;
            const uint32_t page = (uint32_t)__builtin_amdgcn_readlane((int)w_page, i);
            limit[j] = (w_live >> i & 1) && first <= pos ? min(pos - first + 1, 16u) : 0u;
            held[j] = w_held >> i & 1;
            if constexpr (T::FP8) {
                ks_of[j] = u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(w_ks), i));
                vs_of[j] = u2f((uint32_t)__builtin_amdgcn_readlane((int)f2u(w_vs), i));
            }
            const size_t row = T::FP4 ? (((size_t)page * p.hkv + hk) << shift) + off + li
                                      : (((size_t)page << shift) + off + li) * p.hkv + hk;
            v[j].load(p.vc, p.v_scales, row, g);
            k[j].load(p.kc, p.k_scales, row, g);
        }
    };
    uint16_t *stage = stages + wave * STAGE;
    const uint32_t r0 = 4 * g + li / 4; // a transposed read's row
    const uint32_t vb = r0 * 2 * D + 16 * ((li & 3) >> 1) + 8 * (li & 1) + 16 * sel_swizzle<D>(r0);
    uint32_t c = begin + wave;
    if (c < end) {
        window(32 * c >> shift);
        fetch(c);
    }
#pragma unroll 1
    for (; c < end; c += kSelWaves) {
        const uint32_t lim[2] = {limit[0], limit[1]};
        float kf[2], vf[2];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            kf[j] = T::FP8 ? p.scale_log2 * ks_of[j] : p.scale_log2;
            vf[j] = T::FP8 ? vs_of[j] : 1.0f;
            if (lim[j] < 16 || !held[j]) { // (uniform) slots without a key may hold anything
                if (li >= lim[j] || !held[j]) { k[j].clear(); v[j].clear(); }
                if (!held[j]) { kf[j] = p.scale_log2; vf[j] = 1.0f; }
            }
        }
        f32x4 s[2][NT];
#pragma unroll
        for (int j = 0; j < 2; j++) {
            const uint32_t row = 16 * j + li;
#pragma unroll
            for (int i = 0; i < KT; i++)
                *(u32x4 *)((uint8_t *)stage + row * 2 * D + 16 * ((T::dim(g, i) / 8) ^ sel_swizzle<D>(row))) = v[j].piece(i);
        }
#pragma unroll
        for (int j = 0; j < 2; j++) {
#pragma unroll
            for (int nt = 0; nt < NT; nt++) s[j][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < KT; i++) {
                const u32x4 a = k[j].piece(i);
#pragma unroll
                for (int nt = 0; nt < NT; nt++) s[j][nt] = mfma16x16x32<BF>(a, q[nt][i], s[j][nt]);
            }
        }
        asm volatile("" ::: "memory"); // (the stage is read back through a builtin)
        if (c + kSelWaves < end) fetch(c + kSelWaves);
        u32x4 pb[NT], pl[NT]; // weights times V's scale, weights
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            float e[2][4];
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    e[j][i] = __builtin_fmaf(s[j][nt][i], kf[j], -m[nt]);
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
            if constexpr (T::FP8)
                pb[nt] = u32x4{pack2<BF>(e[0][0] * vf[0], e[0][1] * vf[0]), pack2<BF>(e[0][2] * vf[0], e[0][3] * vf[0]),
                               pack2<BF>(e[1][0] * vf[1], e[1][1] * vf[1]), pack2<BF>(e[1][2] * vf[1], e[1][3] * vf[1])};
            const uint32_t one = BF ? 0x3F803F80u : 0x3C003C00u;
            l[nt] = mfma16x16x32<BF>(u32x4{one, one, one, one}, pl[nt], l[nt]);
        }
        // V^T: d rows 16 n .. +15, keys {4g .. 4g+3, 16+4g .. 16+4g+3} as P^T holds them
#pragma unroll
        for (int n = 0; n < DT; n++) {
            const uint8_t *a0p = (const uint8_t *)stage + (vb ^ (32 * n)), *a1p = a0p + 32 * D;
            const s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(a0p));
            const s16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(a1p));
            const u32x2 b0 = __builtin_bit_cast(u32x2, a0), b1 = __builtin_bit_cast(u32x2, a1);
#pragma unroll
            for (int nt = 0; nt < NT; nt++) o[nt][n] = mfma16x16x32<BF>(u32x4{b0.x, b0.y, b1.x, b1.y}, pb[nt], o[nt][n]);
        }
        asm volatile("" ::: "memory"); // (the next chunk's staging stays behind these reads)
    }
    // the waves' columns merged
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        if (g == 0) {
            s_m[wave][16 * nt + li] = m[nt];
            s_l[wave][16 * nt + li] = l[nt][0];
        }
    }
    lds_barrier();
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const uint32_t col = 16 * nt + li;
        float M = -INFINITY, L = 0.0f, mine = 0.0f;
#pragma unroll
        for (int w = 0; w < kSelWaves; w++)
            if (s_l[w][col] != 0.0f) M = fmaxf(M, s_m[w][col]);
#pragma unroll
        for (int w = 0; w < kSelWaves; w++) {
            const float lw = s_l[w][col], f = lw != 0.0f ? fast_exp2(s_m[w][col] - M) : 0.0f;
            L = __builtin_fmaf(lw, f, L);
            if (w == (int)wave) mine = f;
        }
        f32x4 *box = (f32x4 *)stage;
#pragma unroll
        for (int n = 0; n < DT; n++) box[n * 64 + lane] = o[nt][n] * mine;
        lds_barrier();
        if (col < p.group) {
            const float inv = L > 0.0f ? 1.0f / L : 0.0f;
#pragma unroll
            for (int n = 0; n < DT; n += kSelWaves) {
                const uint32_t d0 = 16 * (n + wave) + 4 * g;
                f32x4 x = ((const f32x4 *)stages)[(n + wave) * 64 + lane];
#pragma unroll
                for (int w = 1; w < kSelWaves; w++) x += ((const f32x4 *)(stages + w * STAGE))[(n + wave) * 64 + lane];
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
        if (nt + 1 < NT) lds_barrier(); // the stages are free again
    }
}

// The parts of a row's head joined: one thread per four elements.
template <int D>
__global__ __launch_bounds__(256) void selected_join_kernel(SelectedParams p) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x, quads = D / 4;
    const uint32_t d0 = i % quads * 4, head = i / quads % p.hq, r = i / quads / p.hq;
    if (r >= live_rows(p.cu, p.n_seqs, p.n_rows)) return;
    const uint32_t hk = head / p.group, col = head % p.group;
    const size_t rec = ((size_t)r * p.hkv + hk) * p.parts;
    float M = -INFINITY, L = 0.0f;
    for (uint32_t w = 0; w < p.parts; w++) {
        const float2 ml = p.part_ml[(rec + w) * p.group + col];
        if (ml.y != 0.0f) M = fmaxf(M, ml.x);
    }
    f32x4 x = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    for (uint32_t w = 0; w < p.parts; w++) {
        const float2 ml = p.part_ml[(rec + w) * p.group + col];
        if (ml.y == 0.0f) continue;
        const float f = fast_exp2(ml.x - M);
        L = __builtin_fmaf(ml.y, f, L);
        x += *(const f32x4 *)(p.part_o + ((rec + w) * p.group + col) * D + d0) * f;
    }
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
    if (n >= 1ull << 26) return LIA_E_ARG; // (a wave each)
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
    const SelectPagesParams p{cu_seqlens, positions, sequences, pages, q, codes, scales, (float *)workspace, selected, counts,
                              n_seqs, n_rows, c->num_q_heads, c->num_kv_heads, group, pad, c->stride, span,
                              (uint32_t)__builtin_ctz(c->page_size), c->pool_pages, budget, first, recent,
                              c->q_dtype == LIA_F32};
    hipStream_t s = (hipStream_t)stream;
    hipError_t e = hipSuccess;
    if (span > budget) { // (else every row keeps all its pages)
        // prompt chunks: four tiles of columns share the pages' codes
        const int ct = n_rows >= 16ull * n_seqs ? 4 : group > 16 ? 2 : 1;
        const dim3 grid(n_rows, c->num_kv_heads, (span + kScorePages - 1) / kScorePages);
        e = c->head_dim == 128 ? launch_scores<128>(ct, grid, s, p) : launch_scores<64>(ct, grid, s, p);
    }
    if (e != hipSuccess) return LIA_E_HIP;
    const dim3 grid(n_rows, c->num_kv_heads);
    e = span <= 2048 ? launch<page_pick_kernel<256, 8>>(grid, dim3(256), 0, s, p)
                     : launch<page_pick_kernel<1024, 8>>(grid, dim3(1024), 0, s, p);
    return e == hipSuccess ? LIA_OK : LIA_E_HIP;
}

static int validate_selected(const lia_attention_config *c, uint32_t budget) {
    if (const int st = validate_pages(c)) return st;
    if (c->out_dtype != LIA_F32 && c->out_dtype != LIA_BF16) return LIA_E_UNSUPPORTED;
    if (c->kv_dtype != LIA_F16 && c->kv_dtype != LIA_BF16 && c->kv_dtype != LIA_FP8_E4M3 && c->kv_dtype != LIA_FP4)
        return LIA_E_UNSUPPORTED;
    if (!(c->scale > 0.0f) || !(c->scale < INFINITY)) return LIA_E_ARG;
    if (budget == 0 || (uint64_t)budget * c->page_size >= (1ull << 31)) return LIA_E_ARG;
    return LIA_OK;
}

// Workgroups that share a row and KV head: as many as fill the chip twice, each with a chunk for every wave.
constexpr uint32_t kSelectedFill = 512;
static uint32_t selected_parts(const lia_attention_config *c, uint32_t n_rows, uint32_t budget) {
    const uint64_t units = (uint64_t)n_rows * c->num_kv_heads, chunks = ((uint64_t)budget * c->page_size + 31) / 32;
    const uint64_t want = (kSelectedFill + units - 1) / units, most = (chunks + kSelWaves - 1) / kSelWaves;
    return (uint32_t)(want < most ? want : most);
}

// Records of the step that has most: fewer units than fill the chip, shared until they do.
static uint64_t selected_bytes(const lia_attention_config *c) {
    return 2ull * kSelectedFill * (c->num_q_heads / c->num_kv_heads) * (c->head_dim * sizeof(float) + sizeof(float2));
}

extern "C" size_t lia_selected_attention_workspace_bytes(const lia_attention_config *c, uint32_t budget) {
    return validate_selected(c, budget) == LIA_OK ? (size_t)selected_bytes(c) : 0;
}

template <int D, int NT>
static hipError_t launch_selected(int kv, dim3 grid, hipStream_t s, const SelectedParams &p) {
    const dim3 block(64 * kSelWaves);
    if (kv == LIA_BF16) return launch<selected_kernel<D, NT, LIA_BF16>>(grid, block, 0, s, p);
    if (kv == LIA_F16) return launch<selected_kernel<D, NT, LIA_F16>>(grid, block, 0, s, p);
    if (kv == LIA_FP4) return launch<selected_kernel<D, NT, LIA_FP4>>(grid, block, 0, s, p);
    return launch<selected_kernel<D, NT, LIA_FP8_E4M3>>(grid, block, 0, s, p);
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
                     (uint32_t)__builtin_ctz(c->page_size), c->pool_pages, budget, parts, c->q_dtype == LIA_F32,
                     c->out_dtype == LIA_F32, c->scale * 1.4426950408889634f};
    p.part_ml = (float2 *)(p.part_o + 2ull * kSelectedFill * group * c->head_dim);
    hipStream_t s = (hipStream_t)stream;
    const dim3 grid(n_rows, c->num_kv_heads, parts);
    hipError_t e;
    if (c->head_dim == 128)
        e = group > 16 ? launch_selected<128, 2>(c->kv_dtype, grid, s, p) : launch_selected<128, 1>(c->kv_dtype, grid, s, p);
    else
        e = group > 16 ? launch_selected<64, 2>(c->kv_dtype, grid, s, p) : launch_selected<64, 1>(c->kv_dtype, grid, s, p);
    if (e == hipSuccess && parts > 1) {
        const uint32_t n = n_rows * c->num_q_heads * (c->head_dim / 4);
        e = c->head_dim == 128 ? launch<selected_join_kernel<128>>(dim3((n + 255) / 256), dim3(256), 0, s, p)
                               : launch<selected_join_kernel<64>>(dim3((n + 255) / 256), dim3(256), 0, s, p);
    }
    return e == hipSuccess ? LIA_OK : LIA_E_HIP;
}
