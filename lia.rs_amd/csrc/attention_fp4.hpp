// Attention over MXFP4 pools (gfx950): the decode kernel and the prefill kernel's staging.
//
// Included by attention.hip, whose plan, units, ranges, split records and combine kernels serve these
// pools too.  A key and its value are (D/2 + D/32) bytes each: 136 bytes at head_dim 128 where a 16-bit
// pool holds 512, so a decode step reads a quarter of the memory and each byte carries four times the
// arithmetic.
#pragma once

namespace lia {

template <int D>
struct F4 {
    static constexpr int WAVES = 4;
    static constexpr int THREADS = 64 * WAVES;
    static constexpr int ROW = D / 2;         // code bytes of a key's head
    static constexpr int SROW = D / 32;       // its scales
    static constexpr int LW = D / 32;         // code words a lane loads of a 16-key tile
    static constexpr int KT = D / 32;         // k steps of S^T = K Q^T
    static constexpr int DT = D / 16;         // 16-dim tiles of O
    static constexpr int STAGE = 32 * D;      // bf16 elements of a wave's staged V chunk
};

// Window of 64 logical pages from `first` (one per lane: byte offset of the head's codes in the plane, live
// code bytes) from page ids already loaded.  Table entries outside the pool have no live keys.
__device__ __forceinline__ void window_fp4(const AttnParams &p, WideWindow &w, uint32_t page, uint32_t first,
                                           uint32_t tlim, uint32_t hk, uint32_t row) {
    const uint32_t shift = p.page_shift, P = 1u << shift;
    const uint64_t off = ((uint64_t)page * p.hkv + hk) * ((uint64_t)P * row);
    const uint32_t pstart = (first + lane_id()) << shift;
    w.base = first;
    w.off_lo = (uint32_t)off;
    w.off_hi = (uint32_t)(off >> 32);
    w.bytes = page < p.pool_pages && tlim > pstart ? min(tlim - pstart, P) * row : 0u;
}

__device__ __forceinline__ uint32_t window_pages(const uint32_t *table, uint32_t first, uint32_t limit) {
    return (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(make_rsrc(table, limit * 4),
                                                          (int)((first + lane_id()) * 4), 0, 0);
}

__device__ __forceinline__ uint32_t load_scale(__amdgpu_buffer_rsrc_t r, uint32_t off) {
    return (uint8_t)__builtin_amdgcn_raw_buffer_load_b8(r, (int)off, 0, 0);
}

__device__ __forceinline__ float scale_of(uint32_t s) { return u2f(s << 23); } // (as the conversions read it)

// A 32-key chunk of one plane in registers.  Lane (g, li) of tile j holds key 16j + li, dims D/4 g .. +D/4-1 (at
// head_dim 128 one whole block and its scale), so a tile is one contiguous run of memory.
template <int D>
struct F4Chunk {
    uint32_t w[2][F4<D>::LW], s[2];
};

// The tiles of a chunk: byte offset of their codes in a plane, and whether their page lies in the pool.
struct F4Tiles {
    uint64_t off[2];
    bool in[2];
};

// Window of 64 logical pages from `first`, one per lane: byte offset of the head's codes (page 0's for a page outside the
// pool, whose registers are cleared afterwards; the host refuses pools without pages), and the lanes whose page lies in the
// pool.
struct F4Window {
    uint32_t base, off_lo, off_hi;
    uint64_t in;
};
__device__ __forceinline__ void window_f4(const AttnParams &p, F4Window &w, uint32_t page, uint32_t first, uint32_t hk,
                                          uint32_t row) {
    const bool in = page < p.pool_pages;
    const uint64_t off = ((uint64_t)(in ? page : 0) * p.hkv + hk) * ((uint64_t)row << p.page_shift);
    w.base = first;
    w.off_lo = (uint32_t)off;
    w.off_hi = (uint32_t)(off >> 32);
    w.in = __builtin_amdgcn_ballot_w64(in);
}

template <int D>
__device__ __forceinline__ F4Tiles tiles_f4(const AttnParams &p, const F4Window &w, uint32_t t) {
    F4Tiles r;
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const uint32_t t0 = t + 16 * j;
        const int rel = (int)(((t0 >> p.page_shift) - w.base) & 63);
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)w.off_lo, rel);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)w.off_hi, rel);
        r.off[j] = (((uint64_t)hi << 32) | lo) + (t0 & ((1u << p.page_shift) - 1)) * F4<D>::ROW;
        r.in[j] = w.in >> rel & 1;
    }
    return r;
}

// Loads a chunk of a plane.  A page is read to its end whatever keys it holds: what lies past the range's last key - a
// former owner's rows, or memory that was never written - is cleared before it is used.
template <int D>
__device__ __forceinline__ void load_f4(F4Chunk<D> &c, const uint8_t *codes, const uint8_t *scales, const F4Tiles &x,
                                        uint32_t code_off, uint32_t scale_off) {
#pragma unroll
    for (int j = 0; j < 2; j++) {
        const uint8_t *from = codes + x.off[j];
        if constexpr (D == 128) {
            const u32x4 a = __builtin_nontemporal_load((const u32x4 *)(from + code_off));
            c.w[j][0] = a.x; c.w[j][1] = a.y; c.w[j][2] = a.z; c.w[j][3] = a.w;
        } else {
            const u32x2 a = __builtin_nontemporal_load((const u32x2 *)(from + code_off));
            c.w[j][0] = a.x; c.w[j][1] = a.y;
        }
        c.s[j] = scales[x.off[j] / 16 + scale_off];
    }
}

template <int D, int NT>
struct F4State {
    u32x4 qr[NT][F4<D>::KT]; // queries: lane (g, col) holds dims D/4 g + 8s .. +7 of k step s
    uint32_t lo, hi, lim[NT]; // the range; per column the live keys from its first
    uint32_t free_lo, free_hi;
    float m[NT], thr[NT];
    f32x4 l[NT];             // the mass, in every row of the tile
    f32x4 o[NT][F4<D>::DT];
};

// The queries from byte at[nt] (one type for all, chosen once: a choice at each load would wait for each).
template <int D, int NT>
__device__ __forceinline__ void load_queries_f4(const AttnParams &p, const uint32_t (&at)[NT],
                                                u32x4 (&q)[NT][F4<D>::KT]) {
    constexpr int KT = F4<D>::KT;
    const __amdgpu_buffer_rsrc_t r = make_rsrc(p.q, p.n_rows * p.hq * D * (p.q_f32 ? 4 : 2));
    if (p.q_f32) {
        f32x4 x[NT][KT][2];
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int ks = 0; ks < KT; ks++)
#pragma unroll
                for (int e = 0; e < 2; e++)
                    x[nt][ks][e] = __builtin_bit_cast(f32x4, buffer_load16(r, at[nt] + 32 * ks + 16 * e));
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int ks = 0; ks < KT; ks++) {
                const f32x4 a = x[nt][ks][0], b = x[nt][ks][1];
                q[nt][ks] = u32x4{pack2<true>(a.x, a.y), pack2<true>(a.z, a.w), pack2<true>(b.x, b.y),
                                  pack2<true>(b.z, b.w)};
            }
    } else {
#pragma unroll
        for (int nt = 0; nt < NT; nt++)
#pragma unroll
            for (int ks = 0; ks < KT; ks++) q[nt][ks] = buffer_load16(r, at[nt] + 16 * ks);
    }
}

// Scales from 253 on make infinities of large codes, and 255 NaNs: a weight of 0, which is what a hidden key has, would not
// cancel these in the products of a tile.  Their blocks are looked for by the scale.
__device__ __forceinline__ bool may_overflow(uint32_t s) { return s >= 253; }

// Row i of tile `tile` of O takes x in the columns that attend the key (counted from the range's first).
template <int D, int NT>
__device__ __forceinline__ void add_to(f32x4 (&o)[NT][F4<D>::DT], const uint32_t (&lim)[NT], uint32_t key, uint32_t tile,
                                       int i, float x) {
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        const float a = key < lim[nt] ? x : 0.0f;
#pragma unroll
        for (int n = 0; n < F4<D>::DT; n++) o[nt][n][i] += n == (int)tile ? a : 0.0f;
    }
    __builtin_amdgcn_sched_barrier(0); // (one row at a time: few registers)
}

// The infinities and NaNs among a block's 32 staged values (key: counted from the range's first, row: of the stage) go to the
// columns that attend the key, and zeros take their place in the stage.
template <int D, int NT>
__device__ __forceinline__ void settle(f32x4 (&o)[NT][F4<D>::DT], const uint32_t (&lim)[NT], uint16_t *stage,
                                       uint32_t key, uint32_t row, uint32_t block) {
    const uint32_t g = lane_id() >> 4;
#pragma unroll
    for (int m = 0; m < 2; m++) { // (the 16 lanes of a g read and write the same four values)
        const uint32_t tile = 2 * block + m, at = row * 2 * D + 16 * ((2 * tile + (g >> 1)) ^ swz_v<D>(row)) + 8 * (g & 1);
        u32x2 *const from = (u32x2 *)((uint8_t *)stage + at);
        u32x2 x = *from;
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t h = x[i / 2] >> (16 * (i & 1)) & 0xffffu;
            const bool finite = (h & 0x7f80u) != 0x7f80u;
            add_to<D, NT>(o, lim, key, tile, i, finite ? 0.0f : bf16_to_f32(h));
            if (!finite) x[i / 2] &= i & 1 ? 0x0000ffffu : 0xffff0000u;
        }
        *from = x;
    }
    asm volatile("" ::: "memory"); // (the stage is read back through a builtin)
}

// One chunk: scores, online softmax (log2 domain, a lazily raised reference as in the 16-bit kernels),
// O^T += V^T P^T.  K's codes become bf16 operands in registers; V's are staged as bf16 rows in this wave's
// LDS and read back transposed.  Codes times their scale are bf16 values exactly, so with bf16 queries
// only the weights are rounded (bf16, by up to 2^-8 of each, as a bf16 output is); f32 queries are rounded to
// bf16 as well, whatever the output's type, since the products have operands of one 16-bit type.  The mass sums
// the same rounded weights.  next() loads the next chunk as soon as the operands are out of the registers, and the loads
// pass under the rest of this one (at one place, so that the number of loads in flight is known at every wait).  in:
// whether the chunk's tiles lie in the pool.
template <int D, int NT, class NEXT>
__device__ __forceinline__ void compute_f4(const AttnParams &p, F4Chunk<D> &k, F4Chunk<D> &v, const bool (&in)[2],
                                           uint32_t t, F4State<D, NT> &st, uint16_t *stage, NEXT &&next) {
    using F = F4<D>;
    const uint32_t lane = lane_id(), g = lane >> 4, li = lane & 15;
    // LDS byte offsets of V's staging writes (row li, chunk LW g + w at position ^ swz, i.e. ^ 16 w; row 16 + li
    // swizzles alike) and of its transposed reads (tile n at ^ 32 n).  Opaque, so that every chunk takes its
    // dozen addresses from these two registers instead of holding them all across the loop.
    uint32_t wb = li * 2 * D + 16 * ((F::LW * g) ^ swz_v<D>(li));
    const uint32_t r0 = 4 * g + li / 4;
    uint32_t vb = r0 * 2 * D + 16 * ((li & 3) >> 1) + 8 * (li & 1) + 16 * swz_v<D>(r0);
    asm volatile("" : "+v"(wb), "+v"(vb));
    if (!(in[0] && in[1]) || t + 32 > st.hi) { // (uniform, and rare) keys outside the pool and past the range are zeros
#pragma unroll
        for (int j = 0; j < 2; j++) {
            if (in[j] && t + 16 * j + li < st.hi) continue;
#pragma unroll
            for (int w = 0; w < F::LW; w++) k.w[j][w] = v.w[j][w] = 0;
            k.s[j] = v.s[j] = 0;
        }
    }
    uint64_t odd[2]; // lanes whose block may hold infinities or NaNs
#pragma unroll
    for (int j = 0; j < 2; j++) {
        odd[j] = __builtin_amdgcn_ballot_w64(may_overflow(v.s[j]));
        if constexpr (D == 64) odd[j] &= 0x0000ffff0000ffffull; // (a block is two lanes')
#pragma unroll
        for (int w = 0; w < F::LW; w++)
            *(u32x4 *)((uint8_t *)stage + (wb ^ (16 * w)) + j * 32 * D) = e2m1x8_to_bf16x8(v.w[j][w], scale_of(v.s[j]));
    }
    __builtin_amdgcn_sched_barrier(0); // (V's conversions before K's: their registers are not held together)
    f32x4 s[2][NT];
#pragma unroll
    for (int j = 0; j < 2; j++) {
#pragma unroll
        for (int nt = 0; nt < NT; nt++) s[j][nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int ks = 0; ks < F::KT; ks++) {
            const u32x4 a = e2m1x8_to_bf16x8(k.w[j][ks], scale_of(k.s[j]));
#pragma unroll
            for (int nt = 0; nt < NT; nt++) s[j][nt] = mfma16x16x32<true>(a, st.qr[nt][ks], s[j][nt]);
        }
    }
    __builtin_amdgcn_sched_barrier(0);
    next();
    __builtin_amdgcn_sched_barrier(0);
    const bool masked = !(t >= st.free_lo && t + 32 <= st.free_hi);
    u32x4 pb[NT];
#pragma unroll
    for (int nt = 0; nt < NT; nt++) {
        float e[2][4];
#pragma unroll
        for (int j = 0; j < 2; j++)
#pragma unroll
            for (int i = 0; i < 4; i++) e[j][i] = __builtin_fmaf(s[j][nt][i], p.scale_log2, -st.m[nt]);
        if (masked) {
#pragma unroll
            for (int j = 0; j < 2; j++)
#pragma unroll
                for (int i = 0; i < 4; i++)
                    if (t + 16 * j + 4 * g + i - st.lo >= st.lim[nt]) e[j][i] = -INFINITY;
        }
        float mx = fmaxf(fmaxf(fmaxf(e[0][0], e[0][1]), fmaxf(e[0][2], e[0][3])),
                         fmaxf(fmaxf(e[1][0], e[1][1]), fmaxf(e[1][2], e[1][3])));
        if (__builtin_amdgcn_ballot_w64(mx > st.thr[nt])) { // wave-uniform: rare after the first chunk
            mx = rows_max(mx);
            if (mx > st.thr[nt]) { // the same in the 4 lanes of the column
                // before the first live key there is nothing to scale, and a score far below 0 would
                // make of it 0 times infinity
                const float factor = st.thr[nt] == -INFINITY ? 0.0f : fast_exp2(-mx);
                st.l[nt] *= factor;
#pragma unroll
                for (int n = 0; n < F::DT; n++) st.o[nt][n] *= factor;
                st.m[nt] += mx;
                st.thr[nt] = 8.0f;
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
        pb[nt] = u32x4{pack2<true>(e[0][0], e[0][1]), pack2<true>(e[0][2], e[0][3]),
                       pack2<true>(e[1][0], e[1][1]), pack2<true>(e[1][2], e[1][3])};
        const u32x4 ones = u32x4{0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u};
        st.l[nt] = mfma16x16x32<true>(ones, pb[nt], st.l[nt]);
    }
    if constexpr (NT > 1) __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int j = 0; j < 2; j++) {
        while (odd[j]) { // (uniform, and rare)
            const uint32_t b = (uint32_t)__builtin_ctzll(odd[j]), row = 16 * j + (b & 15);
            odd[j] &= odd[j] - 1;
            settle<D, NT>(st.o, st.lim, stage, t + row - st.lo, row, D == 128 ? b >> 4 : b >> 5);
        }
    }
    // V^T operand: d rows 16n .. +15, k slots = keys {4g .. 4g+3, 16+4g .. 16+4g+3} (as P^T holds them)
#pragma unroll
    for (int n = 0; n < F::DT; n++) {
        const uint8_t *a0p = (const uint8_t *)stage + (vb ^ (32 * n)), *a1p = a0p + 32 * D;
        const s16x4 a0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(a0p));
        const s16x4 a1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4 *)(a1p));
        const u32x2 b0 = __builtin_bit_cast(u32x2, a0), b1 = __builtin_bit_cast(u32x2, a1);
        const u32x4 vt = u32x4{b0.x, b0.y, b1.x, b1.y};
#pragma unroll
        for (int nt = 0; nt < NT; nt++) st.o[nt][n] = mfma16x16x32<true>(vt, pb[nt], st.o[nt][n]);
    }
}

// The decode kernel: a workgroup takes the plan's block range as attention_kernel does, but its waves
// share nothing while they walk it - wave w takes every fourth 32-key chunk over the full head_dim, the
// next chunk's loads in flight under the current one's arithmetic - and merge their columns through LDS
// when a unit ends, so a range leaves one record however many waves walked it.  Bound by HBM on a full
// server's step (64 contexts of 16k to 32k keys of 2 heads of 128, 424 MB: 76 us with the plan and the combine,
// 5.6 TB/s); on eight contexts (26 MB) 10 to 11 us, by the trips to memory before a range's first key and after
// its last; on the verify rows of 32 sequences (73 MB) 24 us, at two waves a SIMD.  K from registers and V through LDS: the
// operand of V^T needs keys side by side that memory has a row apart.  A second chunk in flight a wave
// spilled registers (11.2 -> 13.2 us on eight contexts).
template <int D, int NT>
__global__ __launch_bounds__(F4<D>::THREADS, NT == 1 ? 3 : 2) void attention_fp4_kernel(AttnParams p) {
    using F = F4<D>;
    constexpr uint32_t COLS = 16 * NT;
    __shared__ __attribute__((aligned(16))) uint16_t stages[F::WAVES * F::STAGE];
    __shared__ float s_m[F::WAVES][COLS], s_l[F::WAVES][COLS];
    const WorkDesc wd = p.work[blockIdx.x];
    const uint32_t lane = threadIdx.x & 63, g = lane >> 4, li = lane & 15;
    const uint32_t wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    uint16_t *stage = stages + wave * F::STAGE;
    const uint32_t code_off = li * F::ROW + g * (D / 8);
    const uint32_t scale_off = li * F::SROW + (D == 128 ? g : g >> 1);
    const uint32_t shift = p.page_shift;
    uint32_t u = wd.unit, lo = wd.lo;
    const uint32_t hi = wd.hi;
    bool first = true;
    // the plan guarantees a unit covers every block of a non-empty range
    while (lo < hi) {
        UnitDesc ud;
        if (first) ud = wd.first;
        else ud = p.units[u];
        first = false;
        const uint32_t bs = ud.block_start, uend = bs + ud.nblocks;
        if (uend <= lo) { u++; continue; }
        const uint32_t seg_end = min(hi, uend);
        const uint32_t hk = uniform(unit_head(ud)), nrows = unit_rows(ud), ncols = nrows * p.group;
        const uint32_t *table = uniform_ptr(p.pages + (size_t)ud.table_row * p.stride);
        const uint32_t kend = ud.kend, kcache = ud.kcache, cb = ud.cblocks, pos0 = kend - nrows;
        auto key_of = [&](uint32_t i) { return i < cb ? 32 * i : min(kcache + 32 * (i - cb), kend); };
        const uint32_t r_lo = uniform(key_of(lo - bs)), r_hi = uniform(min(key_of(seg_end - bs), kend));
        const uint32_t page_limit = (r_hi + (1u << shift) - 1) >> shift;
        uint32_t t = (r_lo & ~31u) + 32 * wave;
        // the window's pages, and the next window's on their way
        const uint32_t first_page = (r_lo & ~31u) >> shift;
        uint32_t pages_now = window_pages(table, first_page, page_limit);
        uint32_t pages_next = window_pages(table, first_page + 64, page_limit);

        F4State<D, NT> st;
        st.lo = r_lo;
        st.hi = r_hi;
        const int w0 = (int)min(pos0 + 1, r_hi) - (int)r_lo;
        st.free_lo = r_lo;
        st.free_hi = r_lo + (w0 > 0 ? (uint32_t)w0 : 0u);
        uint32_t qat[NT]; // first byte of the lane's queries (out of range: zeros)
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const uint32_t col = nt * 16 + li;
            const bool valid = col < ncols;
            const uint32_t ri = valid ? col / p.group : 0;
            const int w = (int)min(pos0 + ri + 1, r_hi) - (int)r_lo;
            st.lim[nt] = valid && w > 0 ? (uint32_t)w : 0u;
            qat[nt] = valid ? (((ud.rowbeg + ri) * p.hq + hk * p.group + col % p.group) * D + (D / 4) * g) * (p.q_f32 ? 4 : 2)
                            : 0x80000000u;
            st.m[nt] = 0.0f;
            st.thr[nt] = -INFINITY;
            st.l[nt] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int n = 0; n < F::DT; n++) st.o[nt][n] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        }
        load_queries_f4<D, NT>(p, qat, st.qr);
        F4Window win;
        window_f4(p, win, pages_now, first_page, hk, F::ROW);
        auto reach = [&](uint32_t at) { // the window that holds the chunk's pages
            if ((at >> shift) - win.base >= 64) {
                window_f4(p, win, pages_next, win.base + 64, hk, F::ROW);
                pages_next = window_pages(table, win.base + 64, page_limit);
            }
        };
        constexpr uint32_t STEP = 32 * F::WAVES;
        const uint8_t *kc = (const uint8_t *)p.kc, *vc = (const uint8_t *)p.vc;
        const uint8_t *ksc = (const uint8_t *)p.k_scales, *vsc = (const uint8_t *)p.v_scales;
        if (t < r_hi) {
            F4Chunk<D> k, v;
            F4Tiles x = tiles_f4<D>(p, win, t);
            load_f4<D>(v, vc, vsc, x, code_off, scale_off);
            load_f4<D>(k, kc, ksc, x, code_off, scale_off);
#pragma unroll 1
            for (; t < r_hi; t += STEP) {
                const bool in[2] = {x.in[0], x.in[1]};
                const uint32_t tn = t + STEP;
                const bool more = tn < r_hi; // uniform
                if (more) {
                    reach(tn);
                    x = tiles_f4<D>(p, win, tn);
                }
                compute_f4<D, NT>(p, k, v, in, t, st, stage, [&] {
                    if (!more) return;
                    load_f4<D>(v, vc, vsc, x, code_off, scale_off);
                    load_f4<D>(k, kc, ksc, x, code_off, scale_off);
                });
            }
        }
        // merge the waves' columns (from an opaque lane, so that nothing of it is held over the loop above)
        uint32_t elane = threadIdx.x & 63;
        asm volatile("" : "+v"(elane));
        const uint32_t eg = elane >> 4, eli = elane & 15;
        const bool whole = lo == bs && seg_end == uend;
        const uint32_t rec = (wd.flags >> 8) + u;
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            if (eg == 0) {
                s_m[wave][nt * 16 + eli] = st.m[nt];
                s_l[wave][nt * 16 + eli] = st.l[nt][0];
            }
        }
        lds_barrier();
#pragma unroll
        for (int nt = 0; nt < NT; nt++) {
            const uint32_t col = nt * 16 + eli;
            float M = -INFINITY, L = 0.0f, mine = 0.0f;
#pragma unroll
            for (int w = 0; w < F::WAVES; w++)
                if (s_l[w][col] != 0.0f) M = fmaxf(M, s_m[w][col]);
#pragma unroll
            for (int w = 0; w < F::WAVES; w++) {
                const float lw = s_l[w][col], f = lw != 0.0f ? fast_exp2(s_m[w][col] - M) : 0.0f;
                L = __builtin_fmaf(lw, f, L);
                if (w == (int)wave) mine = f;
            }
            f32x4 *box = (f32x4 *)stage;
#pragma unroll
            for (int n = 0; n < F::DT; n++) box[n * 64 + elane] = st.o[nt][n] * mine;
            lds_barrier();
            if (col < ncols) {
                const uint32_t row = ud.rowbeg + col / p.group, head = hk * p.group + col % p.group;
                const float inv = L > 0.0f ? 1.0f / L : 0.0f;
#pragma unroll
                for (int n = 0; n < F::DT; n += F::WAVES) {
                    const uint32_t d0 = 16 * (n + wave) + 4 * eg;
                    f32x4 v = ((const f32x4 *)stages)[(n + wave) * 64 + elane];
#pragma unroll
                    for (int w = 1; w < F::WAVES; w++)
                        v += ((const f32x4 *)(stages + w * F::STAGE))[(n + wave) * 64 + elane];
                    if (!whole) {
                        *(f32x4 *)(p.part_o + ((size_t)rec * COLS + col) * D + d0) = v;
                    } else {
                        v *= inv;
                        const size_t at = ((size_t)row * p.hq + head) * D + d0;
                        if (p.out_f32) *(f32x4 *)((float *)p.out + at) = v;
                        else *(u32x2 *)((uint16_t *)p.out + at) = u32x2{pack2<true>(v.x, v.y), pack2<true>(v.z, v.w)};
                    }
                }
                if (!whole && wave == 0 && eg == 0) {
                    p.part_ml[((size_t)rec * COLS + col) * 2] = M == -INFINITY ? 0.0f : M;
                    p.part_ml[((size_t)rec * COLS + col) * 2 + 1] = L;
                }
            }
            lds_barrier(); // the stages (and s_m, s_l) are free again
        }
        lo = seg_end;
        u++;
    }
}

// ------------------------------------------------------------------ the prefill kernel's staging
//
// A thread loads one eighth of a key's codes (8 bytes at head_dim 128) of K and of V with their scales,
// one step before it writes them, converted to bf16, into the stages that 16-bit pools load straight into
// LDS; everything after the stages is the bf16 pools' code, and what bounds it bounds this: four chunks of
// 300 to 1,500 rows of 32 heads over 0 to 6,000 cached keys take 155 us, on a bf16 pool 164.
template <int D>
struct F4Share {
    uint32_t k[D / 64], v[D / 64], ks, vs;
};

template <int W>
__device__ __forceinline__ void load_words(uint32_t (&x)[W], __amdgpu_buffer_rsrc_t r, uint32_t off) {
    if constexpr (W == 2) {
        const u32x2 a = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(r, (int)off, 0, 0));
        x[0] = a.x; x[1] = a.y;
    } else {
        x[0] = (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(r, (int)off, 0, 0);
    }
}

template <int D>
__device__ __forceinline__ void wide_issue_fp4(const AttnParams &p, uint32_t t, const WideWindow &w,
                                               uint32_t tlim, uint32_t wave, F4Share<D> &r) {
    using F = F4<D>;
    const uint32_t shift = p.page_shift, P = 1u << shift, lane = lane_id();
    const uint32_t t0 = t + 16 * (wave >> 1);           // the wave's tile: its keys 8 (wave % 2) .. +7
    const WideTile tile = wide_tile(w, t0, shift, tlim);
    const uint32_t sh = (t0 & (P - 1)) * F::ROW;
    const uint32_t nb = tile.bytes ? tile.bytes - sh : 0u;
    const uint64_t off = tile.off + sh;
    const uint32_t key = 8 * (wave & 1) + lane / 8, piece = lane & 7;
    const uint32_t co = key * F::ROW + piece * (D / 16), so = key * F::SROW + piece * F::SROW / 8;
    load_words<D / 64>(r.k, make_rsrc((const uint8_t *)p.kc + off, nb), co);
    load_words<D / 64>(r.v, make_rsrc((const uint8_t *)p.vc + off, nb), co);
    r.ks = load_scale(make_rsrc((const uint8_t *)p.k_scales + off / 16, nb / 16), so);
    r.vs = load_scale(make_rsrc((const uint8_t *)p.v_scales + off / 16, nb / 16), so);
}

// The infinities and NaNs of a stage's V, which are staged as zeros (as settle() leaves them, since a hidden key's weight of
// 0 would not cancel them): the threads that have some, one bit each, and such a thread's elements, two bits each (1:
// infinity, 2: its negative, 3: NaN).
struct F4Odd {
    uint64_t threads[4];
    uint32_t which[256];
};

// Returns the wave's threads that may have some.
template <int D>
__device__ __forceinline__ uint64_t wide_commit_fp4(const F4Share<D> &r, uint32_t wave, uint16_t *kst, uint16_t *vst) {
    const uint32_t lane = lane_id(), key = 8 * wave + lane / 8, piece = lane & 7;
#pragma unroll
    for (int w = 0; w < D / 64; w++) {
        const uint32_t chunk = (D / 64) * piece + w;
        *(u32x4 *)(kst + key * D + ((chunk ^ swz_k<D>(key)) * 8)) = e2m1x8_to_bf16x8(r.k[w], scale_of(r.ks));
        *(u32x4 *)(vst + key * D + ((chunk ^ swz_v<D>(key)) * 8)) = e2m1x8_to_bf16x8(r.v[w], scale_of(r.vs));
    }
    return __builtin_amdgcn_ballot_w64(may_overflow(r.vs));
}

template <int D>
__device__ __forceinline__ void odd_zeros(uint64_t some, uint32_t wave, uint16_t *vst, F4Odd &odd) {
    const uint32_t lane = lane_id(), key = 8 * wave + lane / 8, piece = lane & 7;
    if (lane == 0) odd.threads[wave] = some;
    if (!some) return; // (uniform)
    uint32_t which = 0;
#pragma unroll 1
    for (int i = 0; i < D / 8; i++) { // this thread's elements again, one by one
        uint16_t *const at = vst + key * D + (((D / 64) * piece + i / 8) ^ swz_v<D>(key)) * 8 + (i & 7);
        const uint32_t h = *at;
        if ((h & 0x7f80u) != 0x7f80u) continue;
        which |= ((h & 0x7fu) ? 3u : h >> 15 ? 2u : 1u) << (2 * i);
        *at = 0;
    }
    odd.which[64 * wave + lane] = which;
}

// ... to the columns that attend their key (counted from the range's first): a piece is D / 8 dims, one tile of O or half of one.
template <int D, int NT>
__device__ __forceinline__ void settle_piece(f32x4 (&o)[NT][F4<D>::DT], const uint32_t (&lim)[NT], uint32_t which,
                                             uint32_t key, uint32_t piece) {
    const uint32_t g = lane_id() >> 4, tile = D == 128 ? piece : piece >> 1;
    const uint32_t mine = D == 128 ? which >> (8 * g) : (g >> 1) == (piece & 1) ? which >> (8 * (g & 1)) : 0u;
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t x = mine >> (2 * i) & 3;
        add_to<D, NT>(o, lim, key, tile, i, x == 0 ? 0.0f : x == 3 ? __builtin_nanf("") : x == 2 ? -INFINITY : INFINITY);
    }
}

// Keys [s_lo, s_hi) of an MXFP4 pool into the running state (the steps of wide_range_fp8).  Returns whether a block of V that
// the workgroup staged may hold infinities or NaNs: without ODD the state is then of no use.  (With a
// branch a step for what hardly any pool holds, the batch above takes 160.0 us for 155.4.)
template <int D, bool ODD>
__device__ __forceinline__ bool wide_range_fp4(const AttnParams &p, const uint32_t *table, uint32_t s_lo,
                                               uint32_t s_hi, uint32_t hk, uint32_t wave, bool active,
                                               WState<D, LIA_FP4> &st, uint16_t *const (&st_k)[4],
                                               uint16_t *const (&st_v)[4], uint32_t free_lo, uint32_t free_hi) {
    constexpr int NS = kWideStages;
    __shared__ F4Odd odd[ODD ? NS : 1];
    __shared__ uint32_t any[4];
    const uint32_t shift = p.page_shift;
    const uint32_t page_limit = (s_hi + (1u << shift) - 1) >> shift;
    const float one[2] = {1.0f, 1.0f};
    uint64_t some = 0;
    for (uint32_t wbeg = s_lo & ~31u; wbeg < s_hi;) {
        const uint32_t wend = min(s_hi, ((wbeg >> shift) + 64) << shift);
        WideWindow win;
        window_fp4(p, win, window_pages(table, wbeg >> shift, page_limit), wbeg >> shift, wend, hk, F4<D>::ROW);
        F4Share<D> r;
        // every wave finished the previous window's chunks before their stages are refilled
        lds_barrier();
        auto commit = [&](int stage) {
            const uint64_t now = wide_commit_fp4<D>(r, wave, st_k[stage], st_v[stage]);
            if constexpr (ODD) odd_zeros<D>(now, wave, st_v[stage], odd[stage]);
            some |= now;
        };
        wide_issue_fp4<D>(p, wbeg, win, wend, wave, r);
        commit(0);
        wide_issue_fp4<D>(p, wbeg + 32, win, wend, wave, r);
        for (uint32_t t = wbeg;; t += 32 * NS) {
#pragma unroll
            for (int c = 0; c < NS; c++) {
                const uint32_t tc = t + 32 * c;
                lds_barrier(); // chunk tc is in its stage; chunk tc - 32 is retired
                commit((c + 1) % NS); // chunk tc + 32
                wide_issue_fp4<D>(p, tc + 64, win, wend, wave, r);
                if (active)
                    wide_compute<D, LIA_FP4>(p, tc, st, st_k[c], st_v[c], !(tc >= free_lo && tc + 32 <= free_hi), one,
                                             one);
                if constexpr (ODD) {
                    const uint32_t word = ((const uint32_t *)odd[c].threads)[lane_id() & 7];
#pragma unroll 1
                    for (uint32_t i = 0; i < 8 && active; i++) { // word i: threads 32 i .. +31, four keys
                        uint32_t x = (uint32_t)__builtin_amdgcn_readlane((int)word, (int)i);
#pragma unroll 1
                        for (; x; x &= x - 1) {
                            const uint32_t b = (uint32_t)__builtin_ctz(x);
                            settle_piece<D, WCfg<D>::NTW>(st.o, st.lim, uniform(odd[c].which[32 * i + b]),
                                                          tc + 4 * i + b / 8 - st.lo, b & 7);
                        }
                    }
                }
                if (tc + 32 >= wend) goto window_done;
            }
        }
    window_done:
        wbeg = wend;
    }
    if constexpr (ODD) return true;
    if (lane_id() == 0) any[wave] = some != 0;
    lds_barrier(); // (the next range's first is before it is written again)
    return uniform(any[0] | any[1] | any[2] | any[3]) != 0;
}

} // namespace lia
