// Attention whose rows see one range of keys each: causal and prefix rows, packed documents, and the rows of many
// requests over one shared prefix and their own cached keys.
//
// Row i of a sequence sees keys lo_i <= j < hi_i, and
//     s_ij = scale q_i.k_j,   s_ij = cap tanh(s_ij / cap) if capped,   s_ij -= slope |pos_i - j| if biased
//     o_i  = sum_j exp(s_ij) v_j / sum_j exp(s_ij)
// in one pass over the keys with a running reference point. Every mask offered here is such a range, so a tile of rows
// walks the union of its rows' ranges and looks at single keys only in the blocks that some row's border crosses.
//
//   * Rows are (token, query head of a key head's group): the heads that share keys share their loads, and one token of
//     a group of eight fills a quarter of a matrix instruction instead of a thirty-second.
//   * S^T = K Q^T on 32 x 32 x 16 matrix instructions: a lane owns one row, its reductions stay in the lane but for one
//     exchange, and its exponentials are the B operand of O^T += V^T P^T as they stand.
//   * Key blocks of 32 go from global memory straight into LDS; K chunks swizzled by row, V chunks by row & 3, V^T read
//     with the transposing LDS read.
//   * by_keys = 0: 32 rows a wave, four waves share every block through a ring of four stages. by_keys = 1: four waves
//     take blocks in turn for the same 32 rows, each through memory of its own without a barrier, and are joined at the
//     end: for few rows over many keys, where the keys' bytes bound the call and not the matrix unit.
//   * A row that meets a number that is not finite is formed again by itself over its own keys: what lies in keys it
//     does not see (0 x infinity in the matrix product) never reaches it.
#include "attn_device.hpp"
#include "masked_kernel.h"

namespace zdraw {
namespace msk {

constexpr int KB = 32;                // keys per block
constexpr int kRow = D * 2;           // bytes of a row
constexpr int kBlock = KB * kRow;     // bytes of a K (or V) block
constexpr int kStages = 4;
constexpr int kLds = kStages * 2 * kBlock;
constexpr float kTau = 8.0f; // a row's reference point moves when a score (log2) lies this far above it: P <= 2^8 fits IEEE half

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
typedef const __attribute__((address_space(3))) bf16x8* lds_frag_t;
typedef __attribute__((address_space(3))) s16x4* lds_s16x4_t;
typedef const __attribute__((address_space(4))) unsigned* const_u32_t;

__device__ __forceinline__ float lane_f(float x, int src) { return __uint_as_float(__builtin_amdgcn_readlane((int)__float_as_uint(x), src)); }

// 1 KB of one operand, four rows of 256 bytes, to LDS: lane i's 16 bytes land at lds + 16 i.
__device__ __forceinline__ void rows_to_lds(const char* base, unsigned lane_off, unsigned lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 0\n\tglobal_load_lds_dwordx4 %1, %2" : : "s"(lds), "v"(lane_off), "s"(base) : "memory", "m0");
}

template <int N>
__device__ __forceinline__ void wait_loads() {
    asm volatile("s_waitcnt vmcnt(%0)" : : "n"(N) : "memory");
}

struct RowPos {
    int seq, tok, g;
};

// The keys a row sees, in its span's own numbering, and where it stands among them.
struct Range {
    int lo, hi, pos;
    bool live; // false: the row belongs to no sequence and is not written
};

__device__ __forceinline__ RowPos row_pos(const MaskArgs& a, const MaskJob& job, int seq, int r) {
    RowPos p;
    const int t = r / a.group;
    p.g = r - t * a.group;
    if (job.pooled) {
        p.seq = t / a.q_tokens;
        p.tok = t - p.seq * a.q_tokens;
    } else {
        p.seq = seq;
        p.tok = t;
    }
    return p;
}

__device__ __forceinline__ Range row_range(const MaskArgs& a, int kind, const KeySpan& sp, const RowPos& p) {
    Range r;
    r.lo = 0;
    r.live = true;
    if (kind == kRangeDocs) {
        int qs = 0, qe = a.q_tokens, ks = 0, ke = sp.keys, pre = 0, doc = 0;
        if (a.q_starts) {
            const unsigned* const qb = a.q_starts + (int64_t)p.seq * (a.documents + 1);
            const unsigned* const kb = a.k_starts + (int64_t)p.seq * (a.documents + 1);
            int d = 0, top = a.documents; // the last border at or below the row
            while (top - d > 1) {
                const int mid = (d + top) >> 1;
                if (qb[mid] <= (unsigned)p.tok) d = mid;
                else top = mid;
            }
            const unsigned s0 = qb[d], s1 = qb[d + 1];
            r.live = s0 <= (unsigned)p.tok && (unsigned)p.tok < s1;
            qs = r.live ? (int)s0 : 0;
            qe = (int)min(s1, (unsigned)a.q_tokens);
            ks = (int)min(kb[d], (unsigned)sp.keys);
            ke = max((int)min(kb[d + 1], (unsigned)sp.keys), ks);
            doc = d;
        }
        if (a.prefix) pre = (int)min(a.prefix[(int64_t)p.seq * max(a.documents, 1) + doc], (unsigned)(ke - ks));
        const int nk = ke - ks;
        const int at = p.tok - qs + nk - (qe - qs); // the last query stands on the last key
        int n = a.causal ? max(min(at + 1, nk), pre) : nk;
        n = r.live ? max(n, 0) : 0;
        r.lo = ks;
        r.hi = ks + n;
        r.pos = ks + at;
    } else {
        const int n = a.lens ? (int)min(a.lens[p.seq], (unsigned)a.own_keys) : 0;
        const int ql = a.q_lens ? (int)min(a.q_lens[p.seq], (unsigned)a.q_tokens) : a.q_tokens;
        r.live = p.tok < ql;
        const int at = p.tok + n - ql;
        if (kind == kRangePrefix) {
            r.hi = sp.keys;
            r.pos = sp.keys + at;
        } else {
            r.hi = a.causal ? max(min(at + 1, n), 0) : n;
            r.pos = at;
        }
        if (!r.live) r.hi = 0;
    }
    return r;
}

__device__ __forceinline__ int wave_min(int x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) x = min(x, __shfl_xor(x, o));
    return __builtin_amdgcn_readfirstlane(x);
}
__device__ __forceinline__ int wave_max(int x) {
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) x = max(x, __shfl_xor(x, o));
    return __builtin_amdgcn_readfirstlane(x);
}

// Address of key row j of a sequence and head; what is passed is uniform over the wave.
struct SpanBase {
    const char* k;
    const char* v;
    const_u32_t table; // this sequence's pages, or null
};
__device__ __forceinline__ SpanBase span_base(const KeySpan& sp, int seq, int kvh) {
    SpanBase b;
    b.k = sp.k + (int64_t)kvh * sp.k_hs;
    b.v = sp.v + (int64_t)kvh * sp.v_hs;
    b.table = nullptr;
    if (sp.table) {
        b.table = (const_u32_t)(sp.table + (int64_t)seq * sp.table_ld);
    } else {
        b.k += (int64_t)seq * sp.k_ss;
        b.v += (int64_t)seq * sp.v_ss;
    }
    return b;
}
__device__ __forceinline__ void row_at(const KeySpan& sp, const SpanBase& b, int j, const char*& k, const char*& v) {
    int64_t page = 0;
    int row = j;
    if (sp.table) {
        page = (int64_t)min(b.table[j >> sp.page_shift], (unsigned)(sp.pages - 1));
        row = j & sp.page_mask;
        k = b.k + page * sp.k_ss + (int64_t)row * sp.k_ts;
        v = b.v + page * sp.v_ss + (int64_t)row * sp.v_ts;
    } else {
        k = b.k + (int64_t)row * sp.k_ts;
        v = b.v + (int64_t)row * sp.v_ts;
    }
}

// Lane offsets of a four-row load: row lane / 16 of the four, chunk by the swizzle of LDS row 4 n + lane / 16.
struct LoadLane {
    unsigned q;          // lane / 16
    unsigned kc[4], vc;  // byte offset of the chunk in its row
    unsigned k_ts, v_ts;
};

// Loads rows j .. j + 3 of K and V (n = the first one's place in the block / 4); rows past `last` repeat it.
template <bool K, bool V>
__device__ __forceinline__ void load_rows(const KeySpan& sp, const SpanBase& b, const LoadLane& ln, int j, int last, int n, unsigned k_lds, unsigned v_lds) {
    const char *kp, *vp;
    row_at(sp, b, min(j, last), kp, vp);
    unsigned q = ln.q;
    if (j + 3 > last) q = min(q, (unsigned)max(last - j, 0));
    if (K) rows_to_lds(kp, q * ln.k_ts + ln.kc[n & 3], k_lds + (unsigned)n * 1024u);
    if (V) rows_to_lds(vp, q * ln.v_ts + ln.vc, v_lds + (unsigned)n * 1024u);
}

// What a lane keeps of its row across the key blocks. O^T: lane row l32, dims 32 b + 8 i + 4 h + j in o[b][4 i + j].
struct RowState {
    f32x16 o[4];
    float m, l; // reference point (log2), this lane's half of the denominator
};

template <bool F16>
__device__ __forceinline__ f32x16 mfma(const bf16x8& x, const bf16x8& y, const f32x16& c) {
    if constexpr (F16) return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, x), __builtin_bit_cast(f16x8, y), c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_32x32x16_bf16(x, y, c, 0, 0, 0);
}

template <bool F16>
__device__ __forceinline__ bf16x8 round8(const f32x16& p, int at) {
    f32x8 x;
#pragma unroll
    for (int i = 0; i < 8; i++) x[i] = p[at + i];
    if constexpr (F16) return __builtin_bit_cast(bf16x8, __builtin_convertvector(x, f16x8));
    else return __builtin_convertvector(x, bf16x8);
}

// A score of one key, log2, from the product q.k (cap and bias; the plain scale is applied by the caller's fma).
__device__ __forceinline__ float fancy_score(const MaskArgs& a, float dot, float slope, float dist) {
    float y;
    if (a.cap_in != 0.0f) {
        // cap tanh(s / cap): tanh x = 1 - 2 / (e^2x + 1) is 1 and -1 at the infinities and NaN at NaN; near 0 it is off by 2^-24 of the cap
        y = a.cap_out * (1.0f - 2.0f * __builtin_amdgcn_rcpf(__builtin_amdgcn_exp2f(dot * a.cap_in) + 1.0f));
    } else {
        y = dot * a.scale_log2;
    }
    return y - slope * fabsf(dist);
}

// Scores of a block -> P (16 bits), with the row's reference point, denominator and O kept up. `whole`: every row of the
// wave sees the whole block.
template <bool F16, bool FANCY>
__device__ __forceinline__ void softmax_block(const MaskArgs& a, f32x16& s, int j0, int h, const Range& r, float slope, bool whole, RowState& st, bf16x8 (&p)[2]) {
    float c = a.scale_log2;
    if constexpr (FANCY) {
        const float d0 = (float)(r.pos - j0 - 4 * h);
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = fancy_score(a, s[i], slope, d0 - (float)(8 * (i >> 2) + (i & 3)));
        c = 1.0f;
    }
    if (!whole) {
        const unsigned n = (unsigned)(r.hi - r.lo);
        const unsigned first = (unsigned)(j0 + 4 * h - r.lo);
#pragma unroll
        for (int i = 0; i < 16; i++) s[i] = first + (unsigned)(8 * (i >> 2) + (i & 3)) < n ? s[i] : -INFINITY;
    }
    float top = fmaxf(s[0], s[1]);
#pragma unroll
    for (int i = 2; i < 16; i += 2) top = fmaxf(top, fmaxf(s[i], s[i + 1]));
    top = pair_max(top) * c;
    const bool move = top > st.m + kTau; // (from -infinity: any score)
    if (__builtin_amdgcn_ballot_w64(move) != 0) {
        const float m = move ? top : st.m;
        const float f = move ? __builtin_amdgcn_exp2f(st.m - m) : 1.0f;
        st.m = m;
        st.l *= f;
#pragma unroll
        for (int b = 0; b < 4; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) st.o[b][i] *= f;
    }
    const float ref = st.m == -INFINITY ? 0.0f : st.m;
    float sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; i++) {
        s[i] = __builtin_amdgcn_exp2f(__builtin_fmaf(s[i], c, -ref));
        sum += s[i];
    }
    st.l += sum;
    p[0] = round8<F16>(s, 0);
    p[1] = round8<F16>(s, 8);
}

struct FragLane {
    unsigned k[8]; // byte offset of this lane's K fragment, dims 16 s + 8 h .. + 7 of key l32
    unsigned v[4]; // of its V patch: dims 32 b .. + 31, key 4 h + (lane & 15) / 4 (and 8, 16, 24 further)
};

__device__ __forceinline__ bf16x8 k_frag(unsigned k_lds, const FragLane& fl, int t) { return *(lds_frag_t)(k_lds + fl.k[t]); }
__device__ __forceinline__ s16x8 v_frag(unsigned v_lds, const FragLane& fl, int kb, int b) {
    const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(v_lds + fl.v[b] + (unsigned)(16 * kb * kRow)));
    const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t)(v_lds + fl.v[b] + (unsigned)((16 * kb + 8) * kRow)));
    return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
}

// One row by itself, all lanes of a wave: reference point, denominator and dims 2 lane, 2 lane + 1. Only the keys it sees
// are read. Slow; for rows whose tile met numbers that are not finite.
template <bool F16, bool FANCY>
__device__ void row_alone(const MaskArgs& a, const KeySpan& sp, const SpanBase& base, const char* q, int lo, int hi, int pos, float slope, int lane, float& m,
                          float& l, float& o0, float& o1) {
    auto pair = [](const char* p, float& x, float& y) __attribute__((always_inline)) {
        const unsigned w = *reinterpret_cast<const unsigned*>(p);
        if constexpr (F16) {
            typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
            const f16x2 t = __builtin_bit_cast(f16x2, w);
            x = (float)t[0];
            y = (float)t[1];
        } else {
            x = __uint_as_float(w << 16);
            y = __uint_as_float(w & 0xffff0000u);
        }
    };
    float q0, q1;
    pair(q + 4 * lane, q0, q1);
#pragma clang loop unroll(disable)
    for (int j = lo; j < hi; j++) {
        const char *kp, *vp;
        row_at(sp, base, j, kp, vp);
        float k0, k1, v0, v1;
        pair(kp + 4 * lane, k0, k1);
        pair(vp + 4 * lane, v0, v1);
        float s = q0 * k0 + q1 * k1;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) s += __shfl_xor(s, o);
        if constexpr (FANCY) s = fancy_score(a, s, slope, (float)(pos - j));
        else s *= a.scale_log2;
        if (!(s <= m)) { // (a NaN moves the reference to NaN, and stays)
            const float f = m == -INFINITY ? 0.0f : __builtin_amdgcn_exp2f(m - s);
            m = s;
            l *= f;
            o0 *= f;
            o1 *= f;
        }
        const float p = __builtin_amdgcn_exp2f(s - (m == -INFINITY ? 0.0f : m));
        l += p;
        o0 = __builtin_fmaf(p, v0, o0);
        o1 = __builtin_fmaf(p, v1, o1);
    }
}

template <bool F16>
__device__ __forceinline__ unsigned round2(float x, float y) {
    typedef float f32x2 __attribute__((ext_vector_type(2)));
    const f32x2 t = {x, y};
    if constexpr (F16) {
        typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned, __builtin_convertvector(t, f16x2));
    } else {
        typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
        return __builtin_bit_cast(unsigned, __builtin_convertvector(t, bf16x2));
    }
}

template <bool F16, bool FANCY>
__global__ void __launch_bounds__(256, 2) attn_masked_kernel(const MaskArgs a) {
    extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
    __shared__ int s_lo[2][4], s_hi[2][4];
    __shared__ float s_ml[4][KB][2];
    __shared__ unsigned s_bad;

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l32 = lane & 31;
    const int h = lane >> 5;
    const unsigned lds0 = __builtin_amdgcn_readfirstlane(lds_address(smem));

    // ---- which rows, which keys
    const int which = (int)blockIdx.x >= a.job[0].workgroups ? 1 : 0;
    const MaskJob& job = a.job[which];
    int item;
    {
        // consecutive items (tiles and shares of one head) on one XCD, whose L2 then holds the head's keys
        const int w = (int)blockIdx.x - (which ? a.job[0].workgroups : 0);
        const int xcd = w & 7, idx = w >> 3, per = job.workgroups >> 3, rem = job.workgroups & 7;
        item = idx + xcd * per + min(xcd, rem);
    }
    const int split = item % job.splits;
    const int rest = item / job.splits;
    const int tile = job.row_tiles - 1 - rest % job.row_tiles; // the last rows see the most keys: first
    const int sk = rest / job.row_tiles;
    const int kvh = sk % a.kv_heads;
    const int seq = sk / a.kv_heads;
    const bool by_keys = job.by_keys != 0;
    const int tile_rows = by_keys ? kMaskRowsByKeys : kMaskRowsByWave;
    const int row0 = tile * tile_rows + (by_keys ? 0 : 32 * wave);
    const int row = min(row0 + l32, job.rows - 1); // rows past the end work on the last one and are not written
    const RowPos rp = row_pos(a, job, seq, row);
    const int head = kvh * a.group + rp.g;
    const float slope = (FANCY && a.slopes) ? a.slopes[head] * 1.4426950408889634f : 0.0f;

    const char* const qrow = a.q + (int64_t)rp.seq * a.q_ss + (int64_t)rp.tok * a.q_ts + (int64_t)head * a.q_hs;
    bf16x8 qf[8];
#pragma unroll
    for (int s = 0; s < 8; s++) qf[s] = *reinterpret_cast<const bf16x8*>(qrow + 32 * s + 16 * h);

    FragLane fl;
#pragma unroll
    for (int s = 0; s < 8; s++) fl.k[s] = (unsigned)(l32 * kRow + ((2 * s + h) ^ (l32 & 15)) * 16);
    {
        const int tr = (lane & 15) >> 2;
#pragma unroll
        for (int b = 0; b < 4; b++) fl.v[b] = (unsigned)((4 * h + tr) * kRow + ((b ^ tr) * 32 + 16 * ((lane >> 4) & 1) + 4 * (lane & 3)) * 2);
    }
    LoadLane ln;
    ln.q = (unsigned)lane >> 4;
#pragma unroll
    for (int n = 0; n < 4; n++) ln.kc[n] = (((unsigned)lane & 15u) ^ (4u * n + ln.q)) * 16u;
    ln.vc = (((unsigned)lane & 15u) ^ (ln.q << 2)) * 16u;

    RowState st;
    st.m = -INFINITY;
    st.l = 0.f;
#pragma unroll
    for (int b = 0; b < 4; b++)
#pragma unroll
        for (int i = 0; i < 16; i++) st.o[b][i] = 0.f;
    bool live = true;
    int first[2] = {0, 0}, end[2] = {0, 0}; // the keys of each span that this workgroup walks
    Range range[2];

#pragma unroll
    for (int i = 0; i < 2; i++) {
        range[i] = Range{0, 0, 0, true};
        if (i >= job.spans) break;
        const KeySpan& sp = job.span[i];
        const Range r = row_range(a, job.kind[i], sp, rp);
        range[i] = r;
        live = r.live;
        const bool some = r.hi > r.lo;
        const int own_lo = wave_min(some ? r.lo : 0x7fffffff), own_hi = wave_max(some ? r.hi : 0);
        const int all_lo = wave_max(r.lo), all_hi = wave_min(r.hi); // what every row of the wave sees
        int lo = own_lo, hi = own_hi;
        if (!by_keys) {
            if (lane == 0) {
                s_lo[i][wave] = lo;
                s_hi[i][wave] = hi;
            }
            __syncthreads();
            lo = min(min(s_lo[i][0], s_lo[i][1]), min(s_lo[i][2], s_lo[i][3]));
            hi = max(max(s_hi[i][0], s_hi[i][1]), max(s_hi[i][2], s_hi[i][3]));
            lo = __builtin_amdgcn_readfirstlane(lo);
            hi = __builtin_amdgcn_readfirstlane(hi);
        }
        if (hi <= lo) continue; // no row sees a key of this span
        int nb = (hi - lo + KB - 1) / KB;
        if (job.splits > 1) {
            const int per = (nb + job.splits - 1) / job.splits;
            lo += split * per * KB;
            nb = max(min(per, nb - split * per), 0);
        }
        hi = min(hi, lo + nb * KB);
        if (nb == 0) continue;
        first[i] = lo;
        end[i] = hi;
        const int last = hi - 1;
        const SpanBase base = span_base(sp, seq, kvh);
        ln.k_ts = (unsigned)sp.k_ts;
        ln.v_ts = (unsigned)sp.v_ts;

        if (!by_keys) {
            auto fetch = [&](int b) __attribute__((always_inline)) {
                const unsigned at = lds0 + (unsigned)(b & (kStages - 1)) * (2u * kBlock);
                load_rows<true, true>(sp, base, ln, lo + b * KB + 8 * wave, last, 2 * wave, at, at + kBlock);
                load_rows<true, true>(sp, base, ln, lo + b * KB + 8 * wave + 4, last, 2 * wave + 1, at, at + kBlock);
            };
            fetch(0);
            fetch(1);
            fetch(2);
#pragma clang loop unroll(disable)
            for (int b = 0; b < nb; b++) {
                asm volatile("s_waitcnt vmcnt(8) lgkmcnt(0)\n\ts_barrier" : : : "memory");
                fetch(b + 3);
                const int j0 = lo + b * KB;
                if (j0 >= own_hi || j0 + KB <= own_lo) continue; // no row of this wave sees the block
                const unsigned kl = lds0 + (unsigned)(b & (kStages - 1)) * (2u * kBlock), vl = kl + kBlock;
                f32x16 s;
#pragma unroll
                for (int j = 0; j < 16; j++) s[j] = 0.f;
#pragma unroll
                for (int t = 0; t < 8; t++) s = mfma<F16>(k_frag(kl, fl, t), qf[t], s);
                bf16x8 p[2];
                softmax_block<F16, FANCY>(a, s, j0, h, r, slope, j0 >= all_lo && j0 + KB <= all_hi, st, p);
#pragma unroll
                for (int kb = 0; kb < 2; kb++)
#pragma unroll
                    for (int d = 0; d < 4; d++) st.o[d] = mfma<F16>(__builtin_bit_cast(bf16x8, v_frag(vl, fl, kb, d)), p[kb], st.o[d]);
            }
            asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");
        } else {
            const unsigned kl = lds0 + (unsigned)wave * (2u * kBlock), vl = kl + kBlock;
            if (wave < nb) {
#pragma unroll
                for (int n = 0; n < 8; n++) load_rows<true, false>(sp, base, ln, lo + wave * KB + 4 * n, last, n, kl, vl);
#pragma unroll
                for (int n = 0; n < 8; n++) load_rows<false, true>(sp, base, ln, lo + wave * KB + 4 * n, last, n, kl, vl);
            }
#pragma clang loop unroll(disable)
            for (int b = wave; b < nb; b += 4) {
                const bool more = b + 4 < nb;
                const int j0 = lo + b * KB;
                wait_loads<8>(); // K has arrived, V may be on its way
                bf16x8 kf[8];
#pragma unroll
                for (int t = 0; t < 8; t++) kf[t] = k_frag(kl, fl, t);
                asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
                if (more) {
#pragma unroll
                    for (int n = 0; n < 8; n++) load_rows<true, false>(sp, base, ln, j0 + 4 * KB + 4 * n, last, n, kl, vl);
                }
                f32x16 s;
#pragma unroll
                for (int j = 0; j < 16; j++) s[j] = 0.f;
#pragma unroll
                for (int t = 0; t < 8; t++) s = mfma<F16>(kf[t], qf[t], s);
                bf16x8 p[2];
                softmax_block<F16, FANCY>(a, s, j0, h, r, slope, j0 >= all_lo && j0 + KB <= all_hi, st, p);
                if (more) wait_loads<8>();
                else wait_loads<0>();
                s16x8 vf[2][4];
#pragma unroll
                for (int kb = 0; kb < 2; kb++)
#pragma unroll
                    for (int d = 0; d < 4; d++) vf[kb][d] = v_frag(vl, fl, kb, d);
                asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
                if (more) {
#pragma unroll
                    for (int n = 0; n < 8; n++) load_rows<false, true>(sp, base, ln, j0 + 4 * KB + 4 * n, last, n, kl, vl);
                }
#pragma unroll
                for (int kb = 0; kb < 2; kb++)
#pragma unroll
                    for (int d = 0; d < 4; d++) st.o[d] = mfma<F16>(__builtin_bit_cast(bf16x8, vf[kb][d]), p[kb], st.o[d]);
            }
        }
    }
    st.l = pair_sum(st.l);

    // ---- the rows leave: through LDS, so that they are stored as whole rows
    const bool here = live && row0 + l32 < job.rows;
    float* const part_o = a.part_o + (job.part_base + ((int64_t)(sk * job.row_tiles + tile) * job.splits + split) * tile_rows) * D;
    float* const part_ml = a.part_ml + (job.part_base + ((int64_t)(sk * job.row_tiles + tile) * job.splits + split) * tile_rows) * 2;
    unsigned bad = 0; // rows of this wave's 32 (by_keys: of the workgroup's) to be formed again

    if (!by_keys) {
        float z = 0.f;
#pragma unroll
        for (int b = 0; b < 4; b++)
#pragma unroll
            for (int i = 0; i < 16; i++) z = __builtin_fmaf(st.o[b][i], 0.0f, z);
        z = __builtin_fmaf(st.l, 0.0f, z);
        z = pair_sum(z);
        bad = (unsigned)__builtin_amdgcn_ballot_w64(here && !(z == 0.0f));
        if (a.direct) {
            const float inv = st.l > 0.f ? 1.0f / st.l : 0.f;
            unsigned char* const mine = smem + wave * (32 * kRow); // (the ring is idle; 16-byte chunks swizzled by row)
#pragma unroll
            for (int b = 0; b < 4; b++)
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const u32x2 w = {round2<F16>(st.o[b][4 * i] * inv, st.o[b][4 * i + 1] * inv), round2<F16>(st.o[b][4 * i + 2] * inv, st.o[b][4 * i + 3] * inv)};
                    *reinterpret_cast<u32x2*>(mine + l32 * kRow + (((4 * b + i) ^ (l32 & 15)) * 16) + 8 * h) = w;
                }
            asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");
            const unsigned good = (unsigned)__builtin_amdgcn_ballot_w64(here) & ~bad;
#pragma unroll
            for (int n = 0; n < 8; n++) {
                const int rr = 4 * n + (lane >> 4);
                const u32x4 w = *reinterpret_cast<const u32x4*>(mine + rr * kRow + (((lane & 15) ^ (rr & 15)) * 16));
                if ((good >> rr) & 1u) {
                    const RowPos p = row_pos(a, job, seq, row0 + rr);
                    char* const out = a.o + (int64_t)p.seq * a.o_ss + (int64_t)p.tok * a.o_ts + (int64_t)(kvh * a.group + p.g) * a.o_hs;
                    *reinterpret_cast<u32x4*>(out + 16 * (lane & 15)) = w;
                }
            }
        } else {
            const int at = 32 * wave + l32;
            if (here && st.l != 0.f) {
#pragma unroll
                for (int b = 0; b < 4; b++)
#pragma unroll
                    for (int i = 0; i < 4; i++)
                        *reinterpret_cast<f32x4*>(part_o + (int64_t)at * D + 32 * b + 8 * i + 4 * h) =
                            f32x4{st.o[b][4 * i], st.o[b][4 * i + 1], st.o[b][4 * i + 2], st.o[b][4 * i + 3]};
            }
            if (here && h == 0) {
                part_ml[2 * at] = st.m;
                part_ml[2 * at + 1] = st.l;
            }
        }
    } else {
        // the four waves' shares of the same rows, joined in their order
        if (tid == 0) s_bad = 0;
        if (h == 0) {
            s_ml[wave][l32][0] = st.m;
            s_ml[wave][l32][1] = st.l;
        }
        unsigned char* const mine = smem + wave * (2 * kBlock); // 32 x 512 bytes, 16-byte chunks swizzled by row
#pragma unroll
        for (int b = 0; b < 4; b++)
#pragma unroll
            for (int i = 0; i < 4; i++)
                *reinterpret_cast<f32x4*>(mine + l32 * (2 * kRow) + (((8 * b + 2 * i + h) ^ l32) * 16)) =
                    f32x4{st.o[b][4 * i], st.o[b][4 * i + 1], st.o[b][4 * i + 2], st.o[b][4 * i + 3]};
        __syncthreads();
        const int rr = tid >> 3, c8 = tid & 7; // eight threads a row, 16 dims each
        float m = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; w++) m = fmaxf(m, s_ml[w][rr][0]);
        float l = 0.f;
        f32x4 o[4];
#pragma unroll
        for (int i = 0; i < 4; i++) o[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int w = 0; w < 4; w++) {
            const float mw = s_ml[w][rr][0], lw = s_ml[w][rr][1];
            if (lw == 0.f) continue; // (a share without keys)
            const float f = __builtin_amdgcn_exp2f(mw - m);
            l += f * lw;
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const f32x4 x = *reinterpret_cast<const f32x4*>(smem + w * (2 * kBlock) + rr * (2 * kRow) + (((4 * c8 + i) ^ rr) * 16));
#pragma unroll
                for (int j = 0; j < 4; j++) o[i][j] = __builtin_fmaf(f, x[j], o[i][j]);
            }
        }
        float z = l * 0.0f;
#pragma unroll
        for (int i = 0; i < 4; i++)
#pragma unroll
            for (int j = 0; j < 4; j++) z = __builtin_fmaf(o[i][j], 0.0f, z);
#pragma unroll
        for (int x = 1; x < 8; x <<= 1) z += __shfl_xor(z, x);
        const unsigned alive = (unsigned)__builtin_amdgcn_ballot_w64(here);
        const bool mine_live = (alive >> rr) & 1u;
        const bool again = mine_live && !(z == 0.f);
        if (again && c8 == 0) atomicOr(&s_bad, 1u << rr);
        if (mine_live && !again) {
            if (a.direct) {
                const float inv = l > 0.f ? 1.0f / l : 0.f;
                const RowPos p = row_pos(a, job, seq, row0 + rr);
                char* const out = a.o + (int64_t)p.seq * a.o_ss + (int64_t)p.tok * a.o_ts + (int64_t)(kvh * a.group + p.g) * a.o_hs + 32 * c8;
                u32x4 w[2];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    w[i >> 1][2 * (i & 1)] = round2<F16>(o[i][0] * inv, o[i][1] * inv);
                    w[i >> 1][2 * (i & 1) + 1] = round2<F16>(o[i][2] * inv, o[i][3] * inv);
                }
                *reinterpret_cast<u32x4*>(out) = w[0];
                *reinterpret_cast<u32x4*>(out + 16) = w[1];
            } else {
#pragma unroll
                for (int i = 0; i < 4; i++) *reinterpret_cast<f32x4*>(part_o + (int64_t)rr * D + 16 * c8 + 4 * i) = o[i];
                if (c8 == 0) {
                    part_ml[2 * rr] = m;
                    part_ml[2 * rr + 1] = l;
                }
            }
        }
        __syncthreads();
        bad = s_bad;
        bad &= 0x11111111u << wave; // every wave forms a quarter of them
    }

    // ---- rows that met a number that is not finite
    bad = __builtin_amdgcn_readfirstlane(bad);
#pragma clang loop unroll(disable)
    while (bad != 0) {
        const int x = __builtin_ctz(bad);
        bad &= bad - 1;
        const RowPos p = row_pos(a, job, seq, row0 + x);
        const char* const q = a.q + (int64_t)p.seq * a.q_ss + (int64_t)p.tok * a.q_ts + (int64_t)(kvh * a.group + p.g) * a.q_hs;
        float m = -INFINITY, l = 0.f, o0 = 0.f, o1 = 0.f;
        const float sl = lane_f(slope, x);
#pragma unroll
        for (int i = 0; i < 2; i++) {
            if (i >= job.spans) break;
            const int lo = max(__builtin_amdgcn_readlane(range[i].lo, x), first[i]), hi = min(__builtin_amdgcn_readlane(range[i].hi, x), end[i]);
            row_alone<F16, FANCY>(a, job.span[i], span_base(job.span[i], seq, kvh), q, lo, hi, __builtin_amdgcn_readlane(range[i].pos, x), sl, lane, m, l, o0, o1);
        }
        if (a.direct) {
            const float inv = l == 0.f ? 0.f : 1.0f / l;
            char* const out = a.o + (int64_t)p.seq * a.o_ss + (int64_t)p.tok * a.o_ts + (int64_t)(kvh * a.group + p.g) * a.o_hs;
            *reinterpret_cast<unsigned*>(out + 4 * lane) = round2<F16>(o0 * inv, o1 * inv);
        } else {
            const int at = (by_keys ? 0 : 32 * wave) + x;
            part_o[(int64_t)at * D + 2 * lane] = o0;
            part_o[(int64_t)at * D + 2 * lane + 1] = o1;
            if (lane == 0) {
                part_ml[2 * at] = m;
                part_ml[2 * at + 1] = l;
            }
        }
    }
}

// The shares of each row's keys, joined in their order: half a wave a row.
template <bool F16>
__global__ void __launch_bounds__(256) attn_masked_merge_kernel(const MaskArgs a, int rows) {
    const int r = (int)blockIdx.x * 8 + ((int)threadIdx.x >> 5); // (sequence, key head, row of the sequence)
    const int c = (int)threadIdx.x & 31;
    if (r >= rows) return;
    const int per = a.q_tokens * a.group;
    const int sk = r / per;
    const int rr = r - sk * per;
    const int kvh = sk % a.kv_heads, seq = sk / a.kv_heads;
    const RowPos p{seq, rr / a.group, rr % a.group};
    if (!row_range(a, a.job[0].kind[0], a.job[0].span[0], p).live) return;
    float m = -INFINITY, l = 0.f;
    f32x4 o = f32x4{0.f, 0.f, 0.f, 0.f};
    for (int n = 0; n < a.jobs; n++) {
        const MaskJob& job = a.job[n];
        const int tr = job.by_keys ? kMaskRowsByKeys : kMaskRowsByWave;
        const int row = job.pooled ? seq * per + rr : rr;
        const int at_sk = job.pooled ? kvh : sk;
        const int tile = row / tr;
        const int64_t at = job.part_base + (int64_t)(at_sk * job.row_tiles + tile) * job.splits * tr + (row - tile * tr);
#pragma clang loop unroll_count(4)
        for (int s = 0; s < job.splits; s++) {
            const int64_t i = at + (int64_t)s * tr;
            const float ms = a.part_ml[2 * i], ls = a.part_ml[2 * i + 1];
            if (ls == 0.f) continue;
            const f32x4 x = *reinterpret_cast<const f32x4*>(a.part_o + i * D + 4 * c);
            const float top = fmaxf(m, ms); // (a NaN is in l and o by then)
            const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top), g = __builtin_amdgcn_exp2f(ms - top);
            l = l * f + ls * g;
#pragma unroll
            for (int j = 0; j < 4; j++) o[j] = o[j] * f + x[j] * g;
            m = top;
        }
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    char* const out = a.o + (int64_t)seq * a.o_ss + (int64_t)p.tok * a.o_ts + (int64_t)(kvh * a.group + p.g) * a.o_hs;
    *reinterpret_cast<u32x2*>(out + 8 * c) = u32x2{round2<F16>(o[0] * inv, o[1] * inv), round2<F16>(o[2] * inv, o[3] * inv)};
}

} // namespace msk

hipError_t masked_setup() {
    const void* const fns[4] = {reinterpret_cast<const void*>(&msk::attn_masked_kernel<false, false>), reinterpret_cast<const void*>(&msk::attn_masked_kernel<false, true>),
                                reinterpret_cast<const void*>(&msk::attn_masked_kernel<true, false>), reinterpret_cast<const void*>(&msk::attn_masked_kernel<true, true>)};
    for (const void* f : fns) {
        hipError_t e = hipFuncSetAttribute(f, hipFuncAttributeMaxDynamicSharedMemorySize, msk::kLds);
        if (e != hipSuccess) return e;
    }
    return hipSuccess;
}

hipError_t launch_masked(const MaskArgs& a, hipStream_t stream) {
    int wgs = 0;
    for (int i = 0; i < a.jobs; i++) wgs += a.job[i].workgroups;
    const bool fancy = a.cap_in != 0.0f || a.slopes != nullptr;
    const dim3 grid((unsigned)wgs), block(256);
    if (a.f16) {
        if (fancy) msk::attn_masked_kernel<true, true><<<grid, block, msk::kLds, stream>>>(a);
        else msk::attn_masked_kernel<true, false><<<grid, block, msk::kLds, stream>>>(a);
    } else {
        if (fancy) msk::attn_masked_kernel<false, true><<<grid, block, msk::kLds, stream>>>(a);
        else msk::attn_masked_kernel<false, false><<<grid, block, msk::kLds, stream>>>(a);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || a.direct) return e;
    const MaskJob& last = a.job[a.jobs - 1]; // tiled by sequence
    const int rows = last.seqs * a.kv_heads * last.rows;
    const dim3 mgrid((unsigned)((rows + 7) / 8));
    if (a.f16) msk::attn_masked_merge_kernel<true><<<mgrid, block, 0, stream>>>(a, rows);
    else msk::attn_masked_merge_kernel<false><<<mgrid, block, 0, stream>>>(a, rows);
    return hipGetLastError();
}

} // namespace zdraw
