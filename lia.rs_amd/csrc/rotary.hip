// The position rotation's table from given frequencies, and projections on their way into the step: queries and keys
// normalised for each head and rotated, keys and values appended to the paged pool (gfx950).
#include "common.hpp"
#include "launch.hpp"
#include "rows.hpp"

namespace lia {

// cos and sin of a - k pi/2 for whole k, and k mod 4.  The reduction is in double (pi/2 in two parts under fused
// multiply-adds: what it loses of an angle below 2^32 is under 2^-50), the rest of at most pi/4 and what its rounding to
// float left of it in float: the Taylor series to x^9 and x^10 (the next terms are below 2^-27 of the value there).
__device__ __forceinline__ void sincos_of(double angle, float &c, float &s) {
    const double k = rint(angle * 0.63661977236758134);
    double r = __builtin_fma(-k, 1.5707963267948966, angle);
    r = __builtin_fma(-k, 6.123233995736766e-17, r);
    const float x = (float)r, lo = (float)(r - (double)x), y = x * x;
    float sp = 1.0f / 362880, cp = -1.0f / 3628800;
    sp = __builtin_fmaf(sp, y, -1.0f / 5040);
    sp = __builtin_fmaf(sp, y, 1.0f / 120);
    sp = __builtin_fmaf(sp, y, -1.0f / 6);
    cp = __builtin_fmaf(cp, y, 1.0f / 40320);
    cp = __builtin_fmaf(cp, y, -1.0f / 720);
    cp = __builtin_fmaf(cp, y, 1.0f / 24);
    cp = __builtin_fmaf(cp, y, -0.5f);
    const float sx = __builtin_fmaf(x * y, sp, x + lo), cx = __builtin_fmaf(y, cp, __builtin_fmaf(-x, lo, 1.0f));
    const double q = k - 4.0 * floor(k * 0.25);
    const bool odd = q == 1.0 || q == 3.0;
    c = odd ? sx : cx;
    s = odd ? cx : sx;
    if (q == 1.0 || q == 2.0) c = -c;
    if (q >= 2.0) s = -s;
}

// Table [rows][half][2] of attention * {cos, sin}(positions[r] * frequencies[i]): a thread per row and two columns, so that
// a store is 16 bytes.  Angles are products in double, which hold a position's turn exactly enough at any length (in float
// the angle of position 100,000 is off by 4e-3).  Small tables are a launch and two loads in turn: 1.4 us for 8 rows of 32
// pairs, 2.7 for 4,096 of 64; 65,536 rows are written at 3.6 TB/s.
__global__ __launch_bounds__(256) void rope_table_kernel(uint32_t n, uint32_t pairs, const uint32_t *positions,
                                                         const double *frequencies, float attention, float *out) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= n) return;
    const uint32_t r = i / pairs, c = i - r * pairs;
    const double at = (double)positions[r];
    float4 v;
    sincos_of(at * frequencies[2 * c], v.x, v.y);
    sincos_of(at * frequencies[2 * c + 1], v.z, v.w);
    ((float4 *)out)[i] = make_float4(v.x * attention, v.y * attention, v.z * attention, v.w * attention);
}

struct RotateParams {
    uint32_t n, pieces, per_shift, hq, hkv, rot, interleaved; // n: eights of the step; per_shift: log2 of a head's
    size_t in_stride;                                         // elements between rows
    const uint32_t *positions, *sequences, *pages, *slot_mapping;
    uint32_t stride, page_shift, pool_pages;
    const float *table;
    const void *q_weight, *k_weight, *input;
    int weight_kind, query_bf16;
    float eps;
    void *query, *kc, *vc;
    void *k_scales, *v_scales;
};

// One thread holds eight elements of a head.  A head's threads are neighbours: they add up its squares by lane exchanges,
// and a rotated half finds the other half's eight in the lane rot / 16 away: every element is read once and written once, in
// 16-byte pieces, and nothing between.  4,096 bf16 rows of 32 + 2 x 8 heads of 128, 102 MB: 27.5 us over eight inputs in
// turn, 3.7 TB/s (a copy of as many bytes 22), 22.5 over one that stays in the last-level cache.  8 rows 3.6 us: a launch
// and three loads in turn, the input beside the slot, the weights behind the head's kind, the table behind the norm.
template <int SRC, int KVT>
__global__ __launch_bounds__(256) void rotate_kernel(RotateParams p) {
    const uint32_t i = blockIdx.x * 256 + threadIdx.x;
    if (i >= p.n) return; // (whole heads)
    const uint32_t r = i / p.pieces, e = i - r * p.pieces, per = 1u << p.per_shift;
    const uint32_t h = e >> p.per_shift, t = e & (per - 1);
    float x[8];
    load8<SRC>(p.input, r * p.in_stride + (size_t)e * 8, x);
    uint32_t slot = kNone;
    if (h >= p.hq)
        slot = row_slot(r, p.slot_mapping, p.positions, p.sequences, p.pages, p.stride, p.page_shift, p.pool_pages);
    const bool value = h >= p.hq + p.hkv;
    if (!value) {
        const void *weight = h < p.hq ? p.q_weight : p.k_weight;
        if (weight) {
            float w[8], sum = 0.0f;
            if (p.weight_kind == 0) load8<0>(weight, t * 8, w);
            else if (p.weight_kind == 1) load8<1>(weight, t * 8, w);
            else load8<2>(weight, t * 8, w);
#pragma unroll
            for (int j = 0; j < 8; j++) sum = __builtin_fmaf(x[j], x[j], sum);
            auto add = [](float a, float b) { return a + b; };
            sum = per == 16 ? group_all<16>(sum, add) : group_all<8>(sum, add);
            const float f = 1.0f / sqrtf(sum / (float)(8 * per) + p.eps);
#pragma unroll
            for (int j = 0; j < 8; j++) x[j] *= f * w[j];
        }
        const uint32_t half = p.rot / 2;
        if (t * 8 < p.rot) {
            if (p.interleaved) {
                const float4 *cs = (const float4 *)(p.table + ((size_t)r * half + t * 4) * 2);
                const float4 a = cs[0], b = cs[1];
                const float c[4] = {a.x, a.z, b.x, b.z}, s[4] = {a.y, a.w, b.y, b.w};
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float u = x[2 * j], v = x[2 * j + 1];
                    x[2 * j] = __builtin_fmaf(u, c[j], -(v * s[j]));
                    x[2 * j + 1] = __builtin_fmaf(v, c[j], u * s[j]);
                }
            } else {
                const bool upper = t * 8 >= half;
                const uint32_t at = t * 8 - (upper ? half : 0);
                const float4 *cs = (const float4 *)(p.table + ((size_t)r * half + at) * 2);
                const int from = (int)(threadIdx.x & 63) + (upper ? -(int)(half / 8) : (int)(half / 8));
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const float4 a = cs[j]; // {c, s, c, s}
                    const float u = __shfl(x[2 * j], from), v = __shfl(x[2 * j + 1], from);
                    x[2 * j] = __builtin_fmaf(x[2 * j], a.x, upper ? u * a.y : -(u * a.y));
                    x[2 * j + 1] = __builtin_fmaf(x[2 * j + 1], a.z, upper ? v * a.w : -(v * a.w));
                }
            }
        }
    }
    if (h < p.hq) {
        const size_t to = ((size_t)r * p.hq + h) * (8 * per) + t * 8;
        if (p.query_bf16) put8<2>(p.query, to, x);
        else put8<0>(p.query, to, x);
        return;
    }
    if (slot == kNone) return;
    const uint32_t kh = h - p.hq - (value ? p.hkv : 0);
    void *pool = value ? p.vc : p.kc, *scales = value ? p.v_scales : p.k_scales;
    if constexpr (KVT == LIA_FP4) {
        const size_t b = mxfp4_block(slot, p.page_shift, p.hkv, kh, 8 * per, t * 8);
        store8_fp4((uint8_t *)pool, (uint8_t *)scales, b, t, x);
    } else {
        Divisor d{};
        if constexpr (KVT == LIA_FP8_E4M3)
            d = divisor(append_scale((float *)scales, (size_t)(slot >> p.page_shift) * p.hkv + kh));
        store8<KVT>(pool, (((size_t)slot * p.hkv + kh) * per + t) * 8, x, d);
    }
}

} // namespace lia

using namespace lia;

extern "C" int lia_rope_table(uint32_t rows, uint32_t rotary_dim, const uint32_t *positions, const double *frequencies,
                              float attention, float *table, lia_stream_t stream) {
    if (!positions || !frequencies || !table) return LIA_E_ARG;
    if (rotary_dim == 0 || rotary_dim % 4) return LIA_E_UNSUPPORTED;
    if (((uintptr_t)table & 15) || ((uintptr_t)frequencies & 7) || ((uintptr_t)positions & 3)) return LIA_E_ALIGN;
    if (rows == 0) return LIA_OK;
    const uint64_t n = (uint64_t)rows * (rotary_dim / 4);
    if (n >= (1ull << 32) - 256) return LIA_E_ARG;
    const hipError_t e = launch<rope_table_kernel>(dim3((uint32_t)((n + 255) / 256)), dim3(256), 0, (hipStream_t)stream,
                                                   (uint32_t)n, rotary_dim / 4, positions, frequencies, attention, table);
    return e == hipSuccess ? LIA_OK : LIA_E_HIP;
}

template <int SRC>
static hipError_t launch_rotate(int kv, dim3 grid, hipStream_t s, const RotateParams &p) {
    if (kv == LIA_F16) return launch<rotate_kernel<SRC, LIA_F16>>(grid, dim3(256), 0, s, p);
    if (kv == LIA_BF16) return launch<rotate_kernel<SRC, LIA_BF16>>(grid, dim3(256), 0, s, p);
    if (kv == LIA_FP8_E4M3) return launch<rotate_kernel<SRC, LIA_FP8_E4M3>>(grid, dim3(256), 0, s, p);
    return launch<rotate_kernel<SRC, LIA_FP4>>(grid, dim3(256), 0, s, p);
}

extern "C" int lia_qk_norm_rope_kv_append(const lia_kv_layout *L, uint32_t num_q_heads, uint32_t rows,
                                          const uint32_t *positions, const uint32_t *sequences, const uint32_t *pages,
                                          uint32_t stride, const uint32_t *slot_mapping, uint32_t rotary_dim,
                                          int32_t interleaved, const float *table, const void *q_weight,
                                          const void *k_weight, int32_t weight_dtype, float eps, const void *input,
                                          int32_t input_dtype, size_t input_stride, void *query, int32_t query_dtype,
                                          void *kc, void *vc, float *k_scales, float *v_scales, lia_stream_t stream) {
    if (!L || !input || !query || !kc || !vc) return LIA_E_ARG;
    if (L->num_kv_heads == 0 || num_q_heads == 0) return LIA_E_ARG;
    if (L->page_size == 0 || (L->page_size & (L->page_size - 1))) return LIA_E_ARG;
    if (L->head_dim != 64 && L->head_dim != 128) return LIA_E_UNSUPPORTED;
    if (L->dtype != LIA_F16 && L->dtype != LIA_BF16 && L->dtype != LIA_FP8_E4M3 && L->dtype != LIA_FP4)
        return LIA_E_UNSUPPORTED;
    if (rotary_dim % 16 || rotary_dim > L->head_dim) return LIA_E_UNSUPPORTED;
    if (query_dtype != LIA_F32 && query_dtype != LIA_BF16) return LIA_E_UNSUPPORTED;
    const int src = src_kind_of(input_dtype), wk = src_kind_of(weight_dtype);
    if (src < 0 || ((q_weight || k_weight) && wk < 0)) return LIA_E_UNSUPPORTED;
    if (rotary_dim && !table) return LIA_E_ARG;
    if ((q_weight || k_weight) && !(eps >= 0.0f && eps < INFINITY)) return LIA_E_ARG;
    if (!slot_mapping && (!positions || !sequences || !pages || stride == 0)) return LIA_E_ARG;
    if ((L->dtype == LIA_FP8_E4M3 || L->dtype == LIA_FP4) && (!k_scales || !v_scales)) return LIA_E_ARG;
    if (((uintptr_t)input | (uintptr_t)query | (uintptr_t)kc | (uintptr_t)vc | (uintptr_t)table | (uintptr_t)q_weight |
         (uintptr_t)k_weight) & 15)
        return LIA_E_ALIGN;
    const uint64_t heads = (uint64_t)num_q_heads + 2ull * L->num_kv_heads;
    if (heads > (1u << 24)) return LIA_E_ARG;
    if (input_stride < heads * L->head_dim) return LIA_E_ARG;
    if (input_stride % 8) return LIA_E_ALIGN;
    if (rows == 0) return LIA_OK;
    const uint64_t pieces = heads * (L->head_dim / 8), n = rows * pieces;
    if (n >= (1ull << 32) - 256 || rows * (uint64_t)input_stride >= (1ull << 60)) return LIA_E_ARG;
    const RotateParams p{(uint32_t)n, (uint32_t)pieces, L->head_dim == 128 ? 4u : 3u, num_q_heads, L->num_kv_heads,
                         rotary_dim, interleaved != 0, input_stride, positions, sequences, pages, slot_mapping, stride,
                         (uint32_t)__builtin_ctz(L->page_size), L->pool_pages, table, q_weight, k_weight, input, wk,
                         query_dtype == LIA_BF16, eps, query, kc, vc, k_scales, v_scales};
    const dim3 grid((uint32_t)((n + 255) / 256));
    hipStream_t s = (hipStream_t)stream;
    const hipError_t e = src == 0 ? launch_rotate<0>(L->dtype, grid, s, p) : src == 1 ? launch_rotate<1>(L->dtype, grid, s, p)
                                                                           : launch_rotate<2>(L->dtype, grid, s, p);
    return e == hipSuccess ? LIA_OK : LIA_E_HIP;
}
