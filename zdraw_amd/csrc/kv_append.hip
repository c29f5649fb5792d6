// Cache append: new key (and query) rows normalised, rotated and rounded on their way, value rows rounded, keys and
// values written where the request's cache (its pages) has their place.
//
//     y = x rsqrt(mean(x^2) + eps) w                      (with norm weights)
//     z = y cos_p + turn(y) sin_p                          (with a rotation; p = the token's position)
// where turn takes (y0, y1) to (-y1, y0) on adjacent pairs, or on the pairs (y_i, y_{i+64}). Sums and products in f32,
// one rounding to the cache's type at the end.
//
// Bound by bytes: every row is read once and written once, 16 lanes a row with 8 elements each. A group of lanes takes
// SLOTS rows of one token (query, key and value heads side by side), so that the token's table rows, place and page are
// looked up once for all of them and their loads are in flight together. 16384 tokens, 24 heads, f32 rows to bf16: 750 MB in
// 159 us, 4.7 TB/s; 2080 tokens, 32 and 8 heads, 16-bit: 51 MB in 14.6 us.
#include "attn_device.hpp"
#include "masked_kernel.h"

namespace zdraw {
namespace app {

template <typename TIn, typename TOut, int SLOTS>
__global__ void __launch_bounds__(256) kv_append_kernel(const AppendArgs a) {
    touch_args<sizeof(AppendArgs)>();
    const int lane16 = (int)threadIdx.x & 15;
    const int d0 = lane16 * 8;
    const int slots = a.heads + 2 * a.kv_heads;
    const int chunks = (slots + SLOTS - 1) / SLOTS;
    const unsigned group = blockIdx.x * 16u + (threadIdx.x >> 4); // (rows are fewer than 2^31)
    const unsigned token = group / (unsigned)chunks;
    const int slot0 = (int)(group - token * (unsigned)chunks) * SLOTS;
    const int req = (int)(token / (unsigned)a.tokens);
    const int tok = (int)(token - (unsigned)req * (unsigned)a.tokens);
    if (req >= a.requests) return;

    Raw8<TIn> raw[SLOTS];
#pragma unroll
    for (int i = 0; i < SLOTS; i++) {
        const int s = min(slot0 + i, slots - 1);
        const char* const p = s < a.heads ? a.q + (int64_t)req * a.q_s[0] + (int64_t)tok * a.q_s[1] + (int64_t)s * a.q_s[2]
                              : s < a.heads + a.kv_heads
                                  ? a.k + (int64_t)req * a.k_s[0] + (int64_t)tok * a.k_s[1] + (int64_t)(s - a.heads) * a.k_s[2]
                                  : a.v + (int64_t)req * a.v_s[0] + (int64_t)tok * a.v_s[1] + (int64_t)(s - a.heads - a.kv_heads) * a.v_s[2];
        raw[i] = ld_raw8<TIn>(reinterpret_cast<const TIn*>(p) + d0, true);
    }
    const unsigned start = a.starts[req];
    const unsigned count = a.counts ? a.counts[req] : (unsigned)a.tokens;
    if ((unsigned)tok >= count) return;
    // a row past the cache's room, or on a page that the pool does not have, is not kept
    const unsigned long long at = (unsigned long long)start + (unsigned)tok;
    bool kept = at < (unsigned long long)a.capacity;
    int64_t page = req, row = (int64_t)(kept ? at : 0);
    if (a.table) {
        const unsigned pg = a.table[(int64_t)req * a.table_ld + (row >> a.page_shift)];
        kept = kept && pg < (unsigned)a.pages;
        page = pg;
        row &= a.page_mask;
    }
    f32x4 c[2], sn[2];
    if (a.rotation != 0) {
        const unsigned long long last = (unsigned long long)a.rope_rows - 1, want = at + a.position_base;
        const int64_t r = (int64_t)(want < last ? want : last) * D + d0;
        c[0] = *reinterpret_cast<const f32x4*>(a.cos_t + r);
        c[1] = *reinterpret_cast<const f32x4*>(a.cos_t + r + 4);
        sn[0] = *reinterpret_cast<const f32x4*>(a.sin_t + r);
        sn[1] = *reinterpret_cast<const f32x4*>(a.sin_t + r + 4);
    }
#pragma unroll
    for (int i = 0; i < SLOTS; i++) {
        const int s = slot0 + i;
        if (s >= slots) break;
        const bool is_q = s < a.heads, is_v = s >= a.heads + a.kv_heads;
        float x[8];
        unpack8(raw[i], x);
        if (!is_v) { // (uniform over the row's 16 lanes)
            const float* const w = is_q ? a.q_w : a.k_w;
            if (w) {
                float ss = 0.f;
#pragma unroll
                for (int j = 0; j < 8; j++) ss += x[j] * x[j];
                ss = row_group_sum<16>(ss);
                const float inv = rsqrtf(ss * (1.0f / D) + a.eps);
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = x[j] * inv * w[d0 + j];
            }
            if (a.rotation != 0) {
                float y[8];
#pragma unroll
                for (int j = 0; j < 8; j++) {
                    if (a.rotation == 1) {
                        y[j] = j & 1 ? x[j - 1] : -x[j + 1];
                    } else { // dims 64 apart: lanes 8 apart (row_ror 8)
                        const float o = __uint_as_float(__builtin_amdgcn_update_dpp(0u, __float_as_uint(x[j]), 0x128, 0xF, 0xF, true));
                        y[j] = lane16 < 8 ? -o : o;
                    }
                }
#pragma unroll
                for (int j = 0; j < 8; j++) x[j] = x[j] * c[j >> 2][j & 3] + y[j] * sn[j >> 2][j & 3];
            }
        }
        u32x4 out;
        if constexpr (std::is_same<TOut, f16_t>::value) {
            f32x8 t;
#pragma unroll
            for (int j = 0; j < 8; j++) t[j] = x[j];
            out = __builtin_bit_cast(u32x4, __builtin_convertvector(t, f16x8));
        } else {
            out = pack_bf16x8(x);
        }
        char* p;
        if (is_q) p = a.qo + (int64_t)req * a.qo_s[0] + (int64_t)tok * a.qo_s[1] + (int64_t)s * a.qo_s[2];
        else if (!is_v) p = a.ck + page * a.ck_s[0] + row * a.ck_s[1] + (int64_t)(s - a.heads) * a.ck_s[2];
        else p = a.cv + page * a.cv_s[0] + row * a.cv_s[1] + (int64_t)(s - a.heads - a.kv_heads) * a.cv_s[2];
        if (is_q || kept) *reinterpret_cast<u32x4*>(p + 16 * lane16) = out;
    }
}

template <typename TIn, typename TOut>
hipError_t launch(const AppendArgs& a, hipStream_t stream) {
    const int slots = a.heads + 2 * a.kv_heads;
    const long long tokens = (long long)a.requests * a.tokens;
    constexpr int S = 4;
    const bool many = tokens * slots >= 65536;
    const long long groups = tokens * (many ? (slots + S - 1) / S : slots);
    const dim3 grid((unsigned)((groups + 15) / 16)), block(256);
    if (many) kv_append_kernel<TIn, TOut, S><<<grid, block, 0, stream>>>(a);
    else kv_append_kernel<TIn, TOut, 1><<<grid, block, 0, stream>>>(a);
    return hipGetLastError();
}

} // namespace app

hipError_t launch_kv_append(const AppendArgs& a, hipStream_t stream) {
    if (a.dtype == kF16) {
        if (a.in_dtype == kF32) return app::launch<float, f16_t>(a, stream);
        if (a.in_dtype == kF16) return app::launch<f16_t, f16_t>(a, stream);
        return app::launch<bf16_t, f16_t>(a, stream);
    }
    if (a.in_dtype == kF32) return app::launch<float, bf16_t>(a, stream);
    if (a.in_dtype == kF16) return app::launch<f16_t, bf16_t>(a, stream);
    return app::launch<bf16_t, bf16_t>(a, stream);
}

} // namespace zdraw
