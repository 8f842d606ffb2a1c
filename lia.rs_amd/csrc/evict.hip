// Eviction of keys from the paged KV pool by a weight per key and KV head (gfx950): the selection of the keys that
// stay, and their move to the front of the sequence.
#include "common.hpp"
#include "launch.hpp"

namespace lia {

constexpr uint32_t kSelectThreads = 1024, kSelectWaves = kSelectThreads / 64;
constexpr uint32_t kSelectRows = 8;                             // rows of 64 keys a wave holds in registers
constexpr uint32_t kSegment = kSelectThreads * kSelectRows;     // keys of a workgroup
constexpr uint32_t kBins = 2048;

struct SelectParams {
    const uint32_t *rows, *lengths, *pages; // per sequence: table row, keys
    uint32_t stride, page_shift, pool_pages, hkv, budget, recent;
    const float *mass;                      // [page][kv head][page_size]
    uint32_t *kept, *counts;                // [sequence][kv head][budget], [sequence]
    // sequences of more than kSegment candidates: [sequence and head][digit][segment][bin] counts of a segment's keys, and
    // [sequence and head][digit] the digits found before it with the keys still to take
    uint16_t *hist;
    uint2 *state;
    uint32_t segments;
};

// Floats as whole numbers in their IEEE total order.
__device__ __forceinline__ uint32_t order_of(uint32_t bits) {
    return bits ^ ((bits >> 31) ? 0xffffffffu : 0x80000000u);
}

// The digits of the k-th heaviest key are found from the top, 11, 11 and 10 bits: shift and bins of digit d.
__device__ __forceinline__ uint32_t digit_shift(int d) { return d == 0 ? 21 : d == 1 ? 10 : 0; }
__device__ __forceinline__ uint32_t digit_bins(int d) { return d == 2 ? 1024 : 2048; }

struct SelectShared {
    uint32_t hist[kBins], sum[kSelectWaves], more[kSelectWaves], same[kSelectWaves], bin, above, in;
};

// A sequence and KV head: keys, those kept for being recent, candidates, and how many of these stay.
struct SelectSeq {
    uint32_t n, recent, c, k;
    const uint32_t *table;
    uint32_t *out;
};
__device__ __forceinline__ SelectSeq select_seq(const SelectParams &p, uint32_t b, uint32_t h) {
    SelectSeq s;
    const uint64_t held = (uint64_t)p.stride << p.page_shift; // keys a table row holds
    s.n = p.lengths[b] < held ? p.lengths[b] : (uint32_t)held;
    s.recent = min(p.recent, p.budget);
    s.c = s.n - min(s.recent, s.n);
    s.k = s.n <= p.budget ? 0 : p.budget - s.recent; // 0: nothing to choose
    s.table = p.pages + (size_t)p.rows[b] * p.stride;
    s.out = p.kept + ((size_t)b * p.hkv + h) * p.budget;
    return s;
}

// A workgroup's candidates from key `first`: wave w holds a run of 64 kSelectRows of them, 64 a row.
struct SelectKeys {
    uint32_t first, u[kSelectRows]; // this lane's first key; row x's is 64 x further
};
__device__ __forceinline__ SelectKeys select_keys(const SelectParams &p, const SelectSeq &s, uint32_t h, uint32_t first) {
    SelectKeys k;
    k.first = first + (threadIdx.x >> 6) * 64 * kSelectRows + (threadIdx.x & 63);
    uint32_t page[kSelectRows];
#pragma unroll
    for (uint32_t x = 0; x < kSelectRows; x++) page[x] = s.table[min(k.first + 64 * x, s.c - 1) >> p.page_shift];
#pragma unroll
    for (uint32_t x = 0; x < kSelectRows; x++) { // (keys past the candidates: any entry, never used)
        const uint32_t off = min(k.first + 64 * x, s.c - 1) & ((1u << p.page_shift) - 1);
        const float m = page[x] < p.pool_pages ? p.mass[(((size_t)page[x] * p.hkv + h) << p.page_shift) + off] : 0.0f;
        k.u[x] = order_of(f2u(m));
    }
    return k;
}

// Counts the keys that share the digits found (known: their mask) by digit d, into the workgroup's bins.
__device__ __forceinline__ void select_count(SelectShared &sh, const SelectSeq &s, const SelectKeys &keys, int d,
                                             uint32_t found, uint32_t known) {
    const uint32_t lane = threadIdx.x & 63, shift = digit_shift(d), bins = digit_bins(d);
    sh.hist[threadIdx.x] = 0;
    sh.hist[threadIdx.x + 1024] = 0;
    __syncthreads();
#pragma unroll
    for (uint32_t x = 0; x < kSelectRows; x++) {
        const uint32_t v = keys.u[x];
        const bool in = keys.first + 64 * x < s.c && (v & known) == found;
        const uint64_t all = __builtin_amdgcn_ballot_w64(in);
        if (!all) continue;
        // the lanes of the first lane's bin add once (weights of 0 are many); the others one by one
        const uint32_t bin = (v >> shift) & (bins - 1), lead = (uint32_t)__builtin_ctzll(all);
        const uint32_t first = (uint32_t)__builtin_amdgcn_readlane((int)bin, (int)lead);
        const uint64_t same = __builtin_amdgcn_ballot_w64(in && bin == first);
        if (lane == lead) atomicAdd(&sh.hist[first], (uint32_t)__builtin_popcountll(same));
        if (in && bin != first) atomicAdd(&sh.hist[bin], 1u);
    }
    __syncthreads();
}

// The bin that holds the k-th key from the top: thread t brings the counts of the t-th pair of bins from the top (high:
// of the upper one).  Afterwards sh.bin, sh.above (keys in the bins above it) and sh.in (keys in it) say it.
__device__ __forceinline__ void select_bin(SelectShared &sh, uint32_t bins, uint32_t high, uint32_t low, uint32_t k) {
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6;
    uint32_t sum = high + low;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const uint32_t y = __shfl_up(sum, off);
        if (lane >= (uint32_t)off) sum += y;
    }
    if (lane == 63) sh.sum[wave] = sum;
    __syncthreads();
    uint32_t above = sum - high - low;
    for (uint32_t w = 0; w < wave; w++) above += sh.sum[w];
    if (above < k && k <= above + high) {
        sh.bin = bins - 1 - 2 * t; sh.above = above; sh.in = high;
    } else if (above + high < k && k <= above + high + low) {
        sh.bin = bins - 2 - 2 * t; sh.above = above + high; sh.in = low;
    }
    __syncthreads();
}

// Writes the workgroup's kept keys in ascending order: all above `found` (of the digits known), and the first k of the
// sequence equal to it; more and same: such keys before the workgroup's.
__device__ __forceinline__ void select_write(SelectShared &sh, const SelectSeq &s, const SelectKeys &keys, uint32_t found,
                                             uint32_t known, uint32_t k, uint32_t more, uint32_t same) {
    const uint32_t lane = threadIdx.x & 63;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    uint64_t over[kSelectRows], at[kSelectRows];
    uint32_t a = 0, e = 0;
#pragma unroll
    for (uint32_t x = 0; x < kSelectRows; x++) {
        const bool in = keys.first + 64 * x < s.c;
        const uint32_t v = keys.u[x] & known;
        over[x] = __builtin_amdgcn_ballot_w64(in && v > found);
        at[x] = __builtin_amdgcn_ballot_w64(in && v == found);
        a += (uint32_t)__builtin_popcountll(over[x]);
        e += (uint32_t)__builtin_popcountll(at[x]);
    }
    if (lane == 0) { sh.more[wave] = a; sh.same[wave] = e; }
    __syncthreads();
    for (uint32_t w = 0; w < wave; w++) { more += sh.more[w]; same += sh.same[w]; }
    const uint64_t before = (1ull << lane) - 1;
#pragma unroll
    for (uint32_t x = 0; x < kSelectRows; x++) {
        const uint32_t eq = same + (uint32_t)__builtin_popcountll(at[x] & before);
        const uint32_t to = more + (uint32_t)__builtin_popcountll(over[x] & before) + min(eq, k);
        if ((over[x] >> lane & 1) || ((at[x] >> lane & 1) && eq < k)) s.out[to] = keys.first + 64 * x;
        more += (uint32_t)__builtin_popcountll(over[x]);
        same += (uint32_t)__builtin_popcountll(at[x]);
    }
}

// The selection.  Up to kSegment candidates of a sequence and head are one workgroup's, whole: it counts digit after
// digit, and ends early where a bin's keys all stay.  With more, every workgroup of this first launch counts its
// segment's first digits, select_step_kernel's launches find a digit each and count the next, and the last writes: one
// workgroup on one compute unit took 235 us for two sequences of 128k keys and eight heads, most of it instructions; the
// four launches take 33 (7.8, 7.4, 6.8 and 11.2), a chain of loads, counts and sums each.  16 sequences of 2k to 8k
// keys and two heads: 12 us on 32 workgroups, two or three digits in turn.
__global__ __launch_bounds__(kSelectThreads) void select_kernel(SelectParams p) {
    __shared__ SelectShared sh;
    const uint32_t t = threadIdx.x, b = blockIdx.x / p.hkv, h = blockIdx.x % p.hkv, seg = blockIdx.y;
    const SelectSeq s = select_seq(p, b, h);
    if (seg == 0) {
        if (h == 0 && t == 0) p.counts[b] = min(s.n, p.budget);
        if (s.n <= p.budget) {
            for (uint32_t i = t; i < p.budget; i += kSelectThreads) s.out[i] = i < s.n ? i : kNone;
        } else {
            for (uint32_t i = t; i < s.recent; i += kSelectThreads) s.out[s.k + i] = s.c + i;
        }
    }
    if (s.k == 0 || seg * kSegment >= s.c) return;
    const SelectKeys keys = select_keys(p, s, h, seg * kSegment);
    if (s.c > kSegment) {
        select_count(sh, s, keys, 0, 0, 0);
        uint32_t *to = (uint32_t *)(p.hist + (((size_t)blockIdx.x * 3) * p.segments + seg) * kBins);
        to[t] = sh.hist[2 * t] | sh.hist[2 * t + 1] << 16; // (a segment's counts are below 2^16)
        return;
    }
    uint32_t found = 0, known = 0, k = s.k;
#pragma unroll 1
    for (int d = 0; d < 3; d++) {
        const uint32_t bins = digit_bins(d);
        select_count(sh, s, keys, d, found, known);
        const bool mine = t < bins / 2;
        select_bin(sh, bins, mine ? sh.hist[bins - 1 - 2 * t] : 0, mine ? sh.hist[bins - 2 - 2 * t] : 0, k);
        found |= sh.bin << digit_shift(d);
        known |= (bins - 1) << digit_shift(d);
        k -= sh.above;
        if (k == sh.in) break; // (uniform) every key of the bin stays
    }
    select_write(sh, s, keys, found, known, k, 0, 0);
}

// Digit d - 1 of the sequences of several segments, from all their counts; then this segment's counts of digit d, or
// (d = 3) its kept keys, behind those of the segments before it, which their counts give.
template <int DIGIT>
__global__ __launch_bounds__(kSelectThreads) void select_step_kernel(SelectParams p) {
    __shared__ SelectShared sh;
    const uint32_t t = threadIdx.x, lane = t & 63, wave = t >> 6;
    const uint32_t b = blockIdx.x / p.hkv, h = blockIdx.x % p.hkv, seg = blockIdx.y;
    const SelectSeq s = select_seq(p, b, h);
    if (s.k == 0 || s.c <= kSegment || seg * kSegment >= s.c) return;
    const uint32_t segments = (s.c + kSegment - 1) / kSegment, bins = digit_bins(DIGIT - 1);
    const uint32_t *hist = (const uint32_t *)(p.hist + (size_t)blockIdx.x * 3 * p.segments * kBins); // pairs of bins
    uint2 *state = p.state + (size_t)blockIdx.x * 3;
    const uint2 was = DIGIT == 1 ? make_uint2(0, s.k) : state[DIGIT - 1];
    const SelectKeys keys = select_keys(p, s, h, seg * kSegment);
    auto pair = [&](int d, uint32_t g, uint32_t i) { // counts of bins 2i and 2i + 1 of a segment
        const uint32_t x = hist[((size_t)d * p.segments + g) * (kBins / 2) + i];
        return make_uint2(x & 0xffffu, x >> 16);
    };
    const uint32_t mine = bins / 2 - 1 - t; // the t-th pair from the top
    uint32_t high = 0, low = 0;
    if (t < bins / 2) {
        for (uint32_t g0 = 0; g0 < segments; g0 += 8) {
            uint2 x[8];
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) x[i] = pair(DIGIT - 1, min(g0 + i, segments - 1), mine);
#pragma unroll
            for (uint32_t i = 0; i < 8; i++)
                if (g0 + i < segments) { low += x[i].x; high += x[i].y; }
        }
    }
    select_bin(sh, bins, high, low, was.y);
    const uint32_t found = was.x | sh.bin << digit_shift(DIGIT - 1), k = was.y - sh.above;
    if constexpr (DIGIT < 3) {
        if (seg == 0 && t == 0) state[DIGIT] = make_uint2(found, k);
        const uint32_t known = ~0u << digit_shift(DIGIT - 1);
        __syncthreads(); // the bins are used again
        select_count(sh, s, keys, DIGIT, found, known);
        uint32_t *to = (uint32_t *)(p.hist + (((size_t)blockIdx.x * 3 + DIGIT) * p.segments + seg) * kBins);
        to[t] = sh.hist[2 * t] | sh.hist[2 * t + 1] << 16;
    } else {
        // keys above and equal to `found` in the segments before
        uint32_t more = 0, same = 0;
#pragma unroll 1
        for (int d = 0; d < 3; d++) {
            const uint32_t at = found >> digit_shift(d) & (digit_bins(d) - 1);
            if (t >= digit_bins(d) / 2 || 2 * t + 1 < at) continue;
            for (uint32_t g0 = 0; g0 < seg; g0 += 8) {
                uint2 x[8];
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) x[i] = pair(d, min(g0 + i, segments - 1), t);
#pragma unroll
                for (uint32_t i = 0; i < 8; i++) {
                    if (g0 + i >= seg) continue;
                    more += (2 * t > at ? x[i].x : 0) + (2 * t + 1 > at ? x[i].y : 0);
                    if (d == 2) same += (2 * t == at ? x[i].x : 0) + (2 * t + 1 == at ? x[i].y : 0);
                }
            }
        }
#pragma unroll
        for (int o = 32; o; o >>= 1) {
            more += (uint32_t)__shfl_xor((int)more, o);
            same += (uint32_t)__shfl_xor((int)same, o);
        }
        __syncthreads();
        if (lane == 0) { sh.more[wave] = more; sh.same[wave] = same; }
        __syncthreads();
        more = same = 0;
        for (uint32_t w = 0; w < kSelectWaves; w++) { more += sh.more[w]; same += sh.same[w]; }
        __syncthreads(); // (select_write's counts take their place)
        select_write(sh, s, keys, found, ~0u, k, more, same);
    }
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

constexpr uint32_t kMoveThreads = 512, kMoveUnits = 8, kMoveRun = kMoveThreads * kMoveUnits;

// A workgroup moves one piece of one sequence's and KV head's kept keys, in runs of as many keys as its threads hold in
// registers.  Where a destination page is the source's (in place), one workgroup moves all runs, each loaded whole
// before any of it is written, and upwards: key i comes from kept[i] >= i, so a run overwrites no key that a later
// run reads.  Else the runs are apart and gridDim.z workgroups share them: 8,192 keys of two sequences and 8 bf16 heads of
// 128, 134 MB read and written, take 38 us (3.5 TB/s; a head's row of 256 bytes comes from a place of its own).
template <typename T>
__device__ __forceinline__ void move_piece(const MoveParams &p, const MovePlane &m, uint32_t b, uint32_t h, bool apart) {
    const uint32_t count = min(p.counts[b], p.budget), P = 1u << p.page_shift;
    const uint32_t *kept = p.kept + ((size_t)b * p.hkv + h) * p.budget;
    const size_t row = (size_t)p.rows[b] * p.stride;
    const uint32_t units = count << m.row_shift; // (the host bounds budget << row_shift)
    T *plane = (T *)m.base;
    auto unit_of = [&](uint32_t page, uint32_t key) -> size_t { // first unit of a key's head
        const uint32_t off = key & (P - 1);
        const size_t at = m.head_major ? (((size_t)page * p.hkv + h) << p.page_shift) + off
                                       : (((size_t)page << p.page_shift) + off) * p.hkv + h;
        return at * m.row_units + m.piece;
    };
    const uint32_t step = apart ? kMoveRun * gridDim.z : kMoveRun;
    for (uint32_t x0 = apart ? blockIdx.z * kMoveRun : 0; x0 < units; x0 += step) {
        // every index, then every page, then every unit of the run (clamped, so that none waits for another)
        T v[kMoveUnits];
        uint32_t from[kMoveUnits], src[kMoveUnits], dst[kMoveUnits];
        bool ok[kMoveUnits];
#pragma unroll
        for (uint32_t k = 0; k < kMoveUnits; k++)
            from[k] = kept[min(x0 + k * kMoveThreads + threadIdx.x, units - 1) >> m.row_shift];
#pragma unroll
        for (uint32_t k = 0; k < kMoveUnits; k++) {
            const uint32_t x = x0 + k * kMoveThreads + threadIdx.x, i = min(x, units - 1) >> m.row_shift;
            const uint32_t a = from[k] >> p.page_shift, c = i >> p.page_shift;
            ok[k] = x < units && a < p.stride && c < p.stride;
            src[k] = p.pages[row + min(a, p.stride - 1)];
            dst[k] = p.to[row + min(c, p.stride - 1)];
        }
#pragma unroll
        for (uint32_t k = 0; k < kMoveUnits; k++) {
            const uint32_t x = x0 + k * kMoveThreads + threadIdx.x;
            ok[k] &= src[k] < p.pool_pages && dst[k] < p.pool_pages && (src[k] != dst[k] || from[k] != x >> m.row_shift);
            if (ok[k]) v[k] = plane[unit_of(src[k], from[k]) + (x & ((1u << m.row_shift) - 1))];
        }
        if (!apart) {
            __builtin_amdgcn_s_waitcnt(0); // every load of the run has come back
            __syncthreads();
        }
#pragma unroll
        for (uint32_t k = 0; k < kMoveUnits; k++) {
            const uint32_t x = x0 + k * kMoveThreads + threadIdx.x;
            if (ok[k]) plane[unit_of(dst[k], x >> m.row_shift) + (x & ((1u << m.row_shift) - 1))] = v[k];
        }
    }
}

__global__ __launch_bounds__(kMoveThreads) void compact_kernel(MoveParams p) {
    const MovePlane m = p.move[blockIdx.y];
    const uint32_t b = blockIdx.x / p.hkv, h = blockIdx.x % p.hkv;
    bool apart = p.pages != p.to;
    if (apart) { // (uniform) another table: do any of its pages stay?
        const uint32_t pages = min((min(p.counts[b], p.budget) + (1u << p.page_shift) - 1) >> p.page_shift, p.stride);
        const size_t row = (size_t)p.rows[b] * p.stride;
        bool same = false;
        for (uint32_t i = threadIdx.x; i < pages; i += kMoveThreads) same |= p.pages[row + i] == p.to[row + i];
        apart = !__syncthreads_or(same);
    }
    if (!apart && blockIdx.z) return;
    if (m.unit == 16) move_piece<u32x4>(p, m, b, h, apart);
    else if (m.unit == 4) move_piece<uint32_t>(p, m, b, h, apart);
    else move_piece<uint16_t>(p, m, b, h, apart);
}

} // namespace lia

using namespace lia;

static int validate_layout(const lia_kv_layout *L) {
    if (!L) return LIA_E_ARG;
    if (L->num_kv_heads == 0 || L->page_size == 0 || (L->page_size & (L->page_size - 1))) return LIA_E_ARG;
    return LIA_OK;
}

// Segments of the longest sequence a table holds; more than one take a workspace.
static uint64_t select_segments(const lia_kv_layout *L, uint32_t stride) {
    return ((uint64_t)stride * L->page_size + kSegment - 1) / kSegment;
}

extern "C" size_t lia_kv_select_workspace_bytes(const lia_kv_layout *L, uint32_t n_seqs, uint32_t stride) {
    if (validate_layout(L) || stride == 0) return 0;
    const uint64_t g = select_segments(L, stride), heads = (uint64_t)n_seqs * L->num_kv_heads;
    return g > 1 ? (size_t)(heads * 3 * (g * kBins * sizeof(uint16_t) + sizeof(uint2))) : 0;
}

extern "C" int lia_kv_select(const lia_kv_layout *L, uint32_t n_seqs, const uint32_t *table_rows,
                             const uint32_t *lengths, const uint32_t *pages, uint32_t stride, uint32_t budget,
                             uint32_t recent, const float *mass, uint32_t *kept, uint32_t *counts,
                             void *workspace, size_t workspace_bytes, lia_stream_t stream) {
    if (const int st = validate_layout(L)) return st;
    if (!table_rows || !lengths || !pages || !mass || !kept || !counts || stride == 0 || budget == 0) return LIA_E_ARG;
    if (((uintptr_t)mass | (uintptr_t)kept | (uintptr_t)counts) & 3) return LIA_E_ALIGN;
    const uint64_t segments = select_segments(L, stride);
    if ((uint64_t)n_seqs * L->num_kv_heads >= (1ull << 31) || segments > 65535) return LIA_E_ARG;
    if (n_seqs == 0) return LIA_OK;
    const size_t need = lia_kv_select_workspace_bytes(L, n_seqs, stride);
    if (need && (!workspace || workspace_bytes < need)) return LIA_E_WORKSPACE;
    if (need && ((uintptr_t)workspace & 15)) return LIA_E_ALIGN;
    const size_t heads = (size_t)n_seqs * L->num_kv_heads;
    SelectParams p{table_rows, lengths, pages, stride, (uint32_t)__builtin_ctz(L->page_size), L->pool_pages,
                   L->num_kv_heads, budget, recent, mass, kept, counts, (uint16_t *)workspace, nullptr, (uint32_t)segments};
    p.state = (uint2 *)(p.hist + heads * 3 * segments * kBins);
    const dim3 grid((uint32_t)heads, (uint32_t)segments), block(kSelectThreads);
    hipStream_t s = (hipStream_t)stream;
    hipError_t e = launch<select_kernel>(grid, block, 0, s, p);
    if (e == hipSuccess && segments > 1) e = launch<select_step_kernel<1>>(grid, block, 0, s, p);
    if (e == hipSuccess && segments > 1) e = launch<select_step_kernel<2>>(grid, block, 0, s, p);
    if (e == hipSuccess && segments > 1) e = launch<select_step_kernel<3>>(grid, block, 0, s, p);
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
    if ((uint64_t)n_seqs * L->num_kv_heads >= (1ull << 31) || budget >= (1u << 27)) return LIA_E_ARG;
    if (n_seqs == 0) return LIA_OK;
    MoveParams p{table_rows, pages, to_pages, kept, counts, stride, (uint32_t)__builtin_ctz(L->page_size),
                 L->pool_pages, L->num_kv_heads, budget, 0, {}};
    const uint32_t row = fp4 ? L->head_dim / 32 : L->head_dim / 8; // 16-byte units of a key's head
    // in place a head's row goes in pieces of 64 bytes, a workgroup each, since one workgroup moves all runs of a piece;
    // to another table whole, so that lines are read and written once (8,192 keys of 128 bf16 elements of 16 heads, both
    // planes: 49 us in pieces)
    const uint32_t piece = pages == to_pages && row > 4 ? 4 : row;
    for (void *plane : {kc, vc})
        for (uint32_t u = 0; u < row; u += piece)
            p.move[p.n_moves++] = MovePlane{(uint8_t *)plane, (uint32_t)__builtin_ctz(piece), 16, fp4, row, u};
    if (fp4) {
        const uint32_t sb = L->head_dim / 32; // 4 or 2 scale bytes of a key's head, one unit
        for (void *plane : {(void *)k_scales, (void *)v_scales})
            p.move[p.n_moves++] = MovePlane{(uint8_t *)plane, 0, sb, 1, 1, 0};
    }
    if (mass) p.move[p.n_moves++] = MovePlane{(uint8_t *)mass, 0, 4, 1, 1, 0};
    // runs shared by as many workgroups as fill the chip four times (where they are apart)
    const uint64_t groups = (uint64_t)n_seqs * L->num_kv_heads * p.n_moves;
    const uint64_t runs = ((uint64_t)budget * piece + kMoveRun - 1) / kMoveRun, want = (1024 + groups - 1) / groups;
    const uint32_t z = pages == to_pages ? 1u : (uint32_t)(runs < want ? runs : want);
    const hipError_t e = launch<compact_kernel>(dim3(n_seqs * L->num_kv_heads, p.n_moves, z), dim3(kMoveThreads), 0,
                                                (hipStream_t)stream, p);
    return e == hipSuccess ? LIA_OK : LIA_E_HIP;
}
