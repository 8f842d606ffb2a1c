// Eviction of keys from the paged KV pool by a weight per key and KV head (gfx950): the selection of the keys that
// stay, and their move to the front of the sequence.
#include "common.hpp"
#include "launch.hpp"

namespace lia {

constexpr uint32_t kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;

struct SelectParams {
    const uint32_t *rows, *lengths, *pages; // per sequence: table row, keys
    uint32_t stride, page_shift, pool_pages, hkv, budget, recent;
    const float *mass;                      // [page][kv head][page_size]
    uint32_t *kept, *counts;                // [sequence][kv head][budget], [sequence]
};

// Floats as whole numbers in their IEEE total order.
__device__ __forceinline__ uint32_t order_of(uint32_t bits) {
    return bits ^ ((bits >> 31) ? 0xffffffffu : 0x80000000u);
}

// One workgroup selects the keys of one sequence and KV head: the last min(recent, budget) and the heaviest of
// the others, ties to the lower index, in ascending order.  The k-th heaviest is found by its digits, 11, 11 and
// 10 bits from the top: a histogram of the keys that share the digits found so far, and the bin that holds the
// k-th.  Each wave owns a run of consecutive keys, 64 a row, ROWS rows of them held in registers (the rest
// is read again), so the kept keys come out in order with one scan of sixteen counts.
template <int ROWS>
__global__ __launch_bounds__(kSelectThreads) void select_kernel(SelectParams p) {
    constexpr uint32_t kBins = 2048;
    __shared__ uint32_t hist[kBins], w_sum[kSelectWaves], w_more[kSelectWaves], w_same[kSelectWaves], s_bin, s_above;
    const uint32_t t = threadIdx.x, lane = t & 63;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(t >> 6));
    const uint32_t b = blockIdx.x / p.hkv, h = blockIdx.x % p.hkv;
    const uint32_t P = 1u << p.page_shift;
    const uint32_t n = (uint32_t)min((uint64_t)p.lengths[b], (uint64_t)p.stride << p.page_shift);
    uint32_t *out = p.kept + ((size_t)b * p.hkv + h) * p.budget;
    if (h == 0 && t == 0) p.counts[b] = min(n, p.budget);
    if (n <= p.budget) {
        for (uint32_t i = t; i < p.budget; i += kSelectThreads) out[i] = i < n ? i : kNone;
        return;
    }
    const uint32_t r = min(p.recent, p.budget), c = n - r; // candidates 0 .. c-1, of which k stay
    uint32_t k = p.budget - r;
    for (uint32_t i = t; i < r; i += kSelectThreads) out[k + i] = c + i;
    if (k == 0) return;
    const uint32_t *table = p.pages + (size_t)p.rows[b] * p.stride;
    const uint32_t rows = (c + kSelectThreads - 1) / kSelectThreads; // per wave
    const uint32_t first = wave * rows * 64 + lane;
    auto fetch = [&](uint32_t i) { // (keys past the candidates: any entry, never used)
        i = min(i, c - 1);
        const uint32_t page = table[i >> p.page_shift];
        const float m = page < p.pool_pages ? p.mass[(((size_t)page * p.hkv + h) << p.page_shift) + (i & (P - 1))] : 0.0f;
        return order_of(f2u(m));
    };
    uint32_t u[ROWS];
#pragma unroll
    for (int x = 0; x < ROWS; x++) u[x] = (uint32_t)x < rows ? fetch(first + 64 * x) : 0u;
    // f(key index, order) for every key of the wave, in order; all lanes call it (inside: index < c)
    auto sweep = [&](auto &&f) {
#pragma unroll
        for (int x = 0; x < ROWS; x++)
            if ((uint32_t)x < rows) f(first + 64 * x, u[x]);
        for (uint32_t x = ROWS; x < rows; x += 8) {
            uint32_t v[8];
#pragma unroll
            for (int y = 0; y < 8; y++) v[y] = fetch(first + 64 * min(x + y, rows - 1));
#pragma unroll
            for (int y = 0; y < 8; y++)
                if (x + y < rows) f(first + 64 * (x + y), v[y]);
        }
    };
    uint32_t found = 0, known = 0; // the digits found, and their mask
#pragma unroll 1
    for (int pass = 0; pass < 3; pass++) {
        const uint32_t shift = pass == 0 ? 21 : pass == 1 ? 10 : 0, bins = pass == 2 ? 1024 : 2048;
        hist[t] = 0;
        hist[t + 1024] = 0;
        __syncthreads();
        sweep([&](uint32_t i, uint32_t v) {
            const bool in = i < c && (v & known) == found;
            const uint64_t all = __builtin_amdgcn_ballot_w64(in);
            if (!all) return;
            // the lanes of the first lane's bin add once (masses of 0 are many); the others one by one
            const uint32_t d = (v >> shift) & (bins - 1), lead = (uint32_t)__builtin_ctzll(all);
            const uint32_t dl = (uint32_t)__builtin_amdgcn_readlane((int)d, (int)lead);
            const uint64_t same = __builtin_amdgcn_ballot_w64(in && d == dl);
            if (lane == lead) atomicAdd(&hist[dl], (uint32_t)__builtin_popcountll(same));
            if (in && d != dl) atomicAdd(&hist[d], 1u);
        });
        __syncthreads();
        // keys in the bins above, from the top: thread t owns the t-th pair from the top
        const uint32_t b1 = bins - 1 - 2 * t, b0 = bins - 2 - 2 * t; // (t < bins / 2)
        const uint32_t h1 = t < bins / 2 ? hist[b1] : 0, h0 = t < bins / 2 ? hist[b0] : 0;
        uint32_t sum = h0 + h1;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const uint32_t y = __shfl_up(sum, off);
            if (lane >= (uint32_t)off) sum += y;
        }
        if (lane == 63) w_sum[wave] = sum;
        __syncthreads();
        uint32_t above = sum - h0 - h1;
        for (uint32_t w = 0; w < wave; w++) above += w_sum[w];
        if (above < k && k <= above + h1) { s_bin = b1; s_above = above; }
        else if (above + h1 < k && k <= above + h1 + h0) { s_bin = b0; s_above = above + h1; }
        __syncthreads();
        found |= s_bin << shift;
        known |= (bins - 1) << shift;
        k -= s_above;
    }
    // every key above `found` stays, and the first k of those equal to it
    uint32_t more = 0, same = 0;
    sweep([&](uint32_t i, uint32_t v) {
        more += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(i < c && v > found));
        same += (uint32_t)__builtin_popcountll(__builtin_amdgcn_ballot_w64(i < c && v == found));
    });
    if (lane == 0) { w_more[wave] = more; w_same[wave] = same; }
    __syncthreads();
    more = same = 0;
    for (uint32_t w = 0; w < wave; w++) { more += w_more[w]; same += w_same[w]; }
    const uint64_t before = (1ull << lane) - 1;
    sweep([&](uint32_t i, uint32_t v) {
        const uint64_t a = __builtin_amdgcn_ballot_w64(i < c && v > found);
        const uint64_t e = __builtin_amdgcn_ballot_w64(i < c && v == found);
        const uint32_t eq = same + (uint32_t)__builtin_popcountll(e & before);
        const uint32_t at = more + (uint32_t)__builtin_popcountll(a & before) + min(eq, k);
        if (i < c && (v > found || (v == found && eq < k))) out[at] = i;
        more += (uint32_t)__builtin_popcountll(a);
        same += (uint32_t)__builtin_popcountll(e);
    });
}

// What a compaction moves of a key's head: `planes` runs of memory of 64 << x bytes or less.
struct MovePlane {
    uint8_t *base;
    uint32_t row_shift;   // log2 of the units of one key's head that this piece moves
    uint32_t unit;        // bytes of a unit: 16, 4 or 2
    uint32_t head_major;  // [page][kv head][page_size] (else [page][page_size][kv head])
    uint32_t row_units;   // units of a key's head in the plane
    uint32_t piece;       // first unit of the piece
};
constexpr uint32_t kMaxMoves = 16;
struct MoveParams {
    const uint32_t *rows, *pages, *to, *kept, *counts;
    uint32_t stride, page_shift, pool_pages, hkv, budget, n_moves;
    MovePlane move[kMaxMoves];
};

constexpr uint32_t kMoveThreads = 1024, kMoveUnits = 8;

// One workgroup moves one piece of one sequence's and KV head's kept keys, in runs of as many keys as its threads
// hold in registers: a run is loaded whole before any of it is written, and the runs go up.  Key i comes from
// kept[i] >= i, so a run overwrites no key that a later run reads, and the destination may be the source's pages.
template <typename T>
__device__ __forceinline__ void move_piece(const MoveParams &p, const MovePlane &m, uint32_t b, uint32_t h) {
    const uint32_t count = min(p.counts[b], p.budget), P = 1u << p.page_shift;
    const uint32_t *kept = p.kept + ((size_t)b * p.hkv + h) * p.budget;
    const size_t row = (size_t)p.rows[b] * p.stride;
    const uint32_t units = count << m.row_shift; // (the host bounds budget << row_shift)
    T *plane = (T *)m.base;
    auto place = [&](const uint32_t *table, uint32_t key) -> size_t { // first unit of a key's head, or -1
        if ((key >> p.page_shift) >= p.stride) return ~(size_t)0;
        const uint32_t page = table[row + (key >> p.page_shift)], off = key & (P - 1);
        if (page >= p.pool_pages) return ~(size_t)0;
        const size_t at = m.head_major ? (((size_t)page * p.hkv + h) << p.page_shift) + off
                                       : (((size_t)page << p.page_shift) + off) * p.hkv + h;
        return at * m.row_units + m.piece;
    };
    for (uint32_t x0 = 0; x0 < units; x0 += kMoveThreads * kMoveUnits) {
        T v[kMoveUnits];
        size_t dst[kMoveUnits];
#pragma unroll
        for (uint32_t k = 0; k < kMoveUnits; k++) {
            const uint32_t x = x0 + k * kMoveThreads + threadIdx.x;
            dst[k] = ~(size_t)0;
            if (x >= units) continue;
            const uint32_t i = x >> m.row_shift, part = x & ((1u << m.row_shift) - 1);
            const size_t from = place(p.pages, kept[i]), to = place(p.to, i);
            if (from == ~(size_t)0 || to == ~(size_t)0 || from == to) continue;
            v[k] = plane[from + part];
            dst[k] = to + part;
        }
        __builtin_amdgcn_s_waitcnt(0); // every load of the run has come back
        __syncthreads();
#pragma unroll
        for (uint32_t k = 0; k < kMoveUnits; k++)
            if (dst[k] != ~(size_t)0) plane[dst[k]] = v[k];
    }
}

__global__ __launch_bounds__(kMoveThreads) void compact_kernel(MoveParams p) {
    const MovePlane m = p.move[blockIdx.y];
    const uint32_t b = blockIdx.x / p.hkv, h = blockIdx.x % p.hkv;
    if (m.unit == 16) move_piece<u32x4>(p, m, b, h);
    else if (m.unit == 4) move_piece<uint32_t>(p, m, b, h);
    else move_piece<uint16_t>(p, m, b, h);
}

} // namespace lia

using namespace lia;

static int validate_layout(const lia_kv_layout *L) {
    if (!L) return LIA_E_ARG;
    if (L->num_kv_heads == 0 || L->page_size == 0 || (L->page_size & (L->page_size - 1))) return LIA_E_ARG;
    return LIA_OK;
}

extern "C" int lia_kv_select(const lia_kv_layout *L, uint32_t n_seqs, const uint32_t *table_rows,
                             const uint32_t *lengths, const uint32_t *pages, uint32_t stride, uint32_t budget,
                             uint32_t recent, const float *mass, uint32_t *kept, uint32_t *counts,
                             lia_stream_t stream) {
    if (const int st = validate_layout(L)) return st;
    if (!table_rows || !lengths || !pages || !mass || !kept || !counts || stride == 0 || budget == 0) return LIA_E_ARG;
    if (((uintptr_t)mass | (uintptr_t)kept | (uintptr_t)counts) & 3) return LIA_E_ALIGN;
    if ((uint64_t)n_seqs * L->num_kv_heads >= (1ull << 31)) return LIA_E_ARG;
    if (n_seqs == 0) return LIA_OK;
    const SelectParams p{table_rows, lengths, pages, stride, (uint32_t)__builtin_ctz(L->page_size), L->pool_pages,
                         L->num_kv_heads, budget, recent, mass, kept, counts};
    const dim3 grid(n_seqs * L->num_kv_heads), block(kSelectThreads);
    hipStream_t s = (hipStream_t)stream;
    const hipError_t e = (uint64_t)stride * L->page_size <= 8 * kSelectThreads
                             ? launch<select_kernel<8>>(grid, block, 0, s, p)
                             : launch<select_kernel<32>>(grid, block, 0, s, p);
    return e == hipSuccess ? LIA_OK : LIA_E_HIP;
}

extern "C" int lia_kv_compact(const lia_kv_layout *L, uint32_t n_seqs, const uint32_t *table_rows,
                              const uint32_t *pages, const uint32_t *to_pages, uint32_t stride, uint32_t budget,
                              const uint32_t *kept, const uint32_t *counts, void *kc, void *vc, float *k_scales,
                              float *v_scales, float *mass, lia_stream_t stream) {
    if (const int st = validate_layout(L)) return st;
    if (!table_rows || !pages || !to_pages || !kept || !counts || !kc || !vc || stride == 0 || budget == 0) return LIA_E_ARG;
    if (L->dtype != LIA_F16 && L->dtype != LIA_BF16 && L->dtype != LIA_FP4) return LIA_E_UNSUPPORTED;
    if (L->head_dim != 64 && L->head_dim != 128) return LIA_E_UNSUPPORTED;
    const bool fp4 = L->dtype == LIA_FP4;
    if (fp4 && (!k_scales || !v_scales)) return LIA_E_ARG;
    if (((uintptr_t)kc | (uintptr_t)vc) & 15) return LIA_E_ALIGN;
    if (fp4 && (((uintptr_t)k_scales | (uintptr_t)v_scales) & 3)) return LIA_E_ALIGN;
    if ((uintptr_t)mass & 3) return LIA_E_ALIGN;
    if ((uint64_t)n_seqs * L->num_kv_heads >= (1ull << 31) || budget >= (1u << 28)) return LIA_E_ARG;
    if (n_seqs == 0) return LIA_OK;
    MoveParams p{table_rows, pages, to_pages, kept, counts, stride, (uint32_t)__builtin_ctz(L->page_size),
                 L->pool_pages, L->num_kv_heads, budget, 0, {}};
    const uint32_t row = fp4 ? L->head_dim / 32 : L->head_dim / 8; // 16-byte units of a key's head
    for (void *plane : {kc, vc})
        for (uint32_t u = 0; u < row; u += 4) {
            const uint32_t w = row - u < 4 ? row - u : 4;
            p.move[p.n_moves++] = MovePlane{(uint8_t *)plane, (uint32_t)__builtin_ctz(w), 16, fp4, row, u};
        }
    if (fp4) {
        const uint32_t sb = L->head_dim / 32; // 4 or 2 scale bytes of a key's head, one unit
        for (void *plane : {(void *)k_scales, (void *)v_scales})
            p.move[p.n_moves++] = MovePlane{(uint8_t *)plane, 0, sb, 1, 1, 0};
    }
    if (mass) p.move[p.n_moves++] = MovePlane{(uint8_t *)mass, 0, 4, 1, 1, 0};
    const hipError_t e = launch<compact_kernel>(dim3(n_seqs * L->num_kv_heads, p.n_moves), dim3(kMoveThreads), 0,
                                                (hipStream_t)stream, p);
    return e == hipSuccess ? LIA_OK : LIA_E_HIP;
}
