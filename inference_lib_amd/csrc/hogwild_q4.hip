// Paged caches in 4 bits for gfx950 (MI355X, CDNA4, wave64): the append that quantises, the read that gives the values back, and
// the attention that reads the codes.
//
// A value is offset + scale * code, code in 0 .. 15, with a scale and an offset (fp16) for every token, kv head and group of 64
// channels: 9 bits per 2 channels against 32 in 16 bits.  Eight consecutive tokens (an octet) of a kv head lie together, 9 D / 2 bytes:
//
//   codes    4 D bytes.  Of a key octet: [8 tokens][D / 8 words]; word w of a token holds channels c .. c + 7,
//            c = 64 (r / 2) + 16 (w / (D / 32)) + 8 (r % 2), r = w % (D / 32).  Of a value octet: [D words], word c the octet's eight
//            tokens of channel c.  In a word the lower four nibbles are elements 0, 2, 4, 6 and the upper four 1, 3, 5, 7.
//   params   [D / 64 groups][8 scales, 8 offsets]
//
// Both orders are those in which the matrix instructions want them: a lane's share of a K operand (8 channels of one token per step
// of 32, both steps of a group in the same two groups of 16 channels) is D / 32 consecutive words of a key row, its share of a V^T
// operand (8 tokens of one channel) is one word, and a mask of a word gives two neighbouring elements in the halves of a register.
// The block (page) size is a multiple of 8, so an octet never spans two of them.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "hogwild_kernels.h"
#include "hogwild_device.h"

namespace hw {

// Values beyond, and infinities, are stored as this: offset + 15 scale then stays within fp16 however the two are rounded (by up to 16
// and 15 * 4), so that a cache holds finite values only.  65504, the largest fp16, over a group from 0 on would give 15 * 4368 = 65520.
constexpr float Q4_LIMIT = 65024.f;

template <int D>
struct Q4 {
    static constexpr int OCT = 9 * D / 2;        // bytes of an octet
    static constexpr int PAR = 4 * D;            // where its scales and offsets begin
    static constexpr int NG = D / 64;            // groups
    static constexpr int KROW = D / 2;           // bytes of a key's codes
    static constexpr int WPQ = D / 32;           // words of a key row that one lane multiplies
    static constexpr int NOC = D / 16;           // value words (channels) of a lane = 16-wide blocks of the output
};

// The nibbles of a word in pairs (elements 2i, 2i + 1), still in place: a code in bits 0..3 of each half or in bits 4..7.
constexpr u32 Q4_LO = 0x000F000Fu, Q4_HI = 0x00F000F0u, Q4_MAGIC = 0x64006400u;   // magic: 1024 in both halves, whose last bit counts 1

__device__ __forceinline__ u32 h2_bits(f16x2 x) { return __builtin_bit_cast(u32, x); }
__device__ __forceinline__ f16x2 h2_of(u32 x) { return __builtin_bit_cast(f16x2, x); }
__device__ __forceinline__ float h_lo(u32 x) { return (float)h2_of(x)[0]; }
__device__ __forceinline__ float h_hi(u32 x) { return (float)h2_of(x)[1]; }
__device__ __forceinline__ u32x4 load16(unsigned long long p) { return __builtin_nontemporal_load(reinterpret_cast<const HW_GLOBAL u32x4*>(p)); }

// ------------------------------------------------------------------------------------------------
// append and read
// ------------------------------------------------------------------------------------------------
// Reductions over the eight lanes of a token (lane % 8), by data-parallel-primitive moves.
__device__ __forceinline__ float oct_min(float v) {
    v = fminf(v, __int_as_float(row_dpp<0xB1>(__float_as_int(v))));
    v = fminf(v, __int_as_float(row_dpp<0x4E>(__float_as_int(v))));
    return fminf(v, __int_as_float(row_dpp<0x141>(__float_as_int(v))));
}
__device__ __forceinline__ float oct_max(float v) {
    v = fmaxf(v, __int_as_float(row_dpp<0xB1>(__float_as_int(v))));
    v = fmaxf(v, __int_as_float(row_dpp<0x4E>(__float_as_int(v))));
    return fmaxf(v, __int_as_float(row_dpp<0x141>(__float_as_int(v))));
}

// nibble position of element i (0..7) of a word
__device__ __forceinline__ constexpr int q4_shift(int i) { return 4 * ((i >> 1) + ((i & 1) << 2)); }

// Transposes the 8 x 8 nibbles that the lanes with one lane % 8 hold (lane / 8 = row i, one word each, its element j in nibble
// position j of the plain order 0..7): afterwards lane row i holds element i of rows 0..7.  Three rounds of exchanges with the lane
// 8, 16 and 32 away.
__device__ __forceinline__ u32 q4_transpose(u32 w, int lane) {
#pragma unroll
    for (int k = 0; k < 3; ++k) {
        const u32 mask = k == 0 ? 0x0F0F0F0Fu : k == 1 ? 0x00FF00FFu : 0x0000FFFFu;
        const int sh = 4 << k;
        const u32 other = (u32)__shfl_xor((int)w, 8 << k, 64);
        w = (lane >> (3 + k)) & 1 ? ((other >> sh) & mask) | (w & ~mask) : (w & mask) | ((other & mask) << sh);
    }
    return w;
}
// plain nibble order <-> the cache's (even elements below, odd ones above)
__device__ __forceinline__ u32 q4_spread(u32 w) {       // element i at q4_shift(i)
    u32 r = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) r |= ((w >> (4 * i)) & 15u) << q4_shift(i);
    return r;
}
__device__ __forceinline__ u32 q4_gather(u32 w) {
    u32 r = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) r |= ((w >> q4_shift(i)) & 15u) << (4 * i);
    return r;
}

// Where the octet `o` of sequence b lies, in octets from the cache's start; -1: nowhere (outside the table or the cache).
__device__ __forceinline__ long long q4_octet(const CopyBlocksArgs& a, int b, int h, int o) {
    const int per = a.block_size >> 3;
    const int bi = o / per;
    if (bi >= a.max_blocks) return -1;
    const int blk = a.block_table[(size_t)b * a.max_blocks + bi];
    if (blk < 0 || blk >= a.num_blocks) return -1;
    return ((long long)blk * a.Hkv + h) * per + (o - bi * per);
}

// One wave = one octet x one group of 64 channels of one (sequence, kv head), of the keys or of the values: lane = (token of the
// octet, eight channels).  The lane's channels are one word of a key row as they are; for the values the words are transposed over
// the lanes of the eight tokens.  Tokens of the octet that are not being appended keep their codes: the only writer of an octet is
// one wave, and what it does not replace it reads first (a decode step's append reads and writes 9 D / 2 bytes a head besides
// the token's own 2 D).  grid = (octets * groups * 2 / 4 waves, kv head, sequence).
template <class DT, int D, bool VEC>
__global__ __launch_bounds__(256) void append_q4_kernel(const CopyBlocksArgs a, int octets) {
    typedef typename Elem<DT>::store_t store_t;
    typedef Q4<D> G;
    const int lane = threadIdx.x & 63;
    const int item = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6));
    const int h = blockIdx.y, b = blockIdx.z;
    const int oi = item / (2 * G::NG), part = item - oi * (2 * G::NG);
    const bool keys = part < G::NG;
    const int g = keys ? part : part - G::NG;
    if (oi >= octets) return;
    const int first = a.seq_lengths[b];
    const int o = (first >> 3) + oi;                     // (floor: of a negative position the part from 0 on is appended, as by copy_to_blocks)
    const int i = lane >> 3, c = lane & 7;
    const int t = o * 8 + i - first;                     // new token of this lane
    const bool mine = t >= 0 && t < a.S_new;
    if (o < 0 || o * 8 >= first + a.S_new) return;       // uniform
    const long long at = q4_octet(a, b, h, o);
    if (at < 0) return;                                  // uniform
    char* oct = reinterpret_cast<char*>(keys ? a.kcache : a.vcache) + at * G::OCT;

    float x[8];
    {
        const store_t* src = reinterpret_cast<const store_t*>(keys ? a.key_states : a.value_states) +
                             ((long long)b * (keys ? a.ks_b : a.vs_b) + (long long)h * (keys ? a.ks_h : a.vs_h) +
                              (long long)(mine ? t : 0) * (keys ? a.ks_s : a.vs_s) + 64 * g + 8 * c);
        if constexpr (VEC) {
            constexpr int CH = Chunk<DT>::CH;
#pragma unroll
            for (int k = 0; k < 8 / CH; ++k) {
                float y[CH];
                Chunk<DT>::unpack(*reinterpret_cast<const u32x4*>(src + k * CH), y);
#pragma unroll
                for (int e = 0; e < CH; ++e) x[k * CH + e] = y[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[e] = Elem<DT>::to_float(src[e]);
        }
    }
    float lo = Q4_LIMIT, hi = -Q4_LIMIT;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        x[e] = x[e] != x[e] ? 0.f : fminf(fmaxf(x[e], -Q4_LIMIT), Q4_LIMIT);
        lo = fminf(lo, x[e]);
        hi = fmaxf(hi, x[e]);
    }
    lo = oct_min(lo);
    hi = oct_max(hi);
    const _Float16 mh = (_Float16)lo;
    const float m = (float)mh;
    const _Float16 sh = (_Float16)fmaxf((hi - m) / 15.f, 0.f);
    const float s = (float)sh;
    u32 w = 0;                                           // plain nibble order
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float code = s > 0.f ? fminf(fmaxf(__builtin_rintf((x[e] - m) / s), 0.f), 15.f) : 0.f;
        w |= (u32)code << (4 * e);
    }
    const u32 tokens = 0xffu & (u32)(((1 << min(max(first + a.S_new - o * 8, 0), 8)) - 1) & ~((1 << min(max(first - o * 8, 0), 8)) - 1));   // the octet's new tokens
    if (keys) {
        // channels 64 g + 8 c .. + 7: quarter c / 2, word (quarter) * WPQ + 2 g + c % 2
        if (mine) *reinterpret_cast<u32*>(oct + i * G::KROW + ((c >> 1) * G::WPQ + 2 * g + (c & 1)) * 4) = q4_spread(w);
    } else {
        w = q4_transpose(w, lane);                       // now: channel 64 g + 8 c + i, its eight tokens
        u32* dst = reinterpret_cast<u32*>(oct) + 64 * g + 8 * c + i;
        if (tokens != 0xffu) {
            u32 keep = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) keep |= (tokens >> e) & 1 ? 0u : 15u << (4 * e);
            w = (q4_gather(*dst) & keep) | (w & ~keep);
        }
        *dst = q4_spread(w);
    }
    if (mine && c == 0) {
        _Float16* par = reinterpret_cast<_Float16*>(oct + G::PAR + 32 * g) + i;
        par[0] = sh;
        par[8] = mh;
    }
}

// The values of positions first[b] .. first[b] + n - 1 as [B, Hkv, n, D]; positions outside the table or the cache give zeros.  The
// waves and lanes of append_q4_kernel, the other way round.
template <class DT, int D>
__global__ __launch_bounds__(256) void read_q4_kernel(const CopyBlocksArgs a, int octets) {
    typedef typename Elem<DT>::store_t store_t;
    typedef Q4<D> G;
    const int lane = threadIdx.x & 63;
    const int item = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6));
    const int h = blockIdx.y, b = blockIdx.z;
    const int oi = item / (2 * G::NG), part = item - oi * (2 * G::NG);
    const bool keys = part < G::NG;
    const int g = keys ? part : part - G::NG;
    if (oi >= octets) return;
    const int first = a.seq_lengths[b];
    const int i = lane >> 3, c = lane & 7;
    const int o = (first >> 3) + oi;                     // (floor, also of negative positions)
    const int t = oi * 8 + i - (first & 7);
    if (t < 0 || t >= a.S_new) return;
    const long long at = o < 0 ? -1 : q4_octet(a, b, h, o);
    const size_t row = ((size_t)b * a.Hkv + h) * a.S_new + t;
    store_t* dst = reinterpret_cast<store_t*>(const_cast<void*>(keys ? a.key_states : a.value_states)) + row * D + 64 * g + 8 * c;
    constexpr int CH = Chunk<DT>::CH;
    float y[8 / CH][CH];
#pragma unroll
    for (int e = 0; e < 8; ++e) y[e / CH][e % CH] = 0.f;
    if (at >= 0) {
        const char* oct = reinterpret_cast<const char*>(keys ? a.kcache : a.vcache) + at * G::OCT;
        const _Float16* par = reinterpret_cast<const _Float16*>(oct + G::PAR + 32 * g) + i;
        const float s = (float)par[0], m = (float)par[8];
        if (keys) {
            const u32 w = *reinterpret_cast<const u32*>(oct + i * G::KROW + ((c >> 1) * G::WPQ + 2 * g + (c & 1)) * 4);
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e / CH][e % CH] = __builtin_fmaf((float)((w >> q4_shift(e)) & 15u), s, m);
        } else {
            const u32* src = reinterpret_cast<const u32*>(oct) + 64 * g + 8 * c;
            const int sh = 4 * ((i >> 1) + ((i & 1) << 2));
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e / CH][e % CH] = __builtin_fmaf((float)((src[e] >> sh) & 15u), s, m);
        }
    }
#pragma unroll
    for (int k = 0; k < 8 / CH; ++k) *reinterpret_cast<u32x4*>(dst + k * CH) = Chunk<DT>::pack(y[k]);
}

// ------------------------------------------------------------------------------------------------
// attention
// ------------------------------------------------------------------------------------------------
// The bytes of one 32-token tile (four octets) that a lane holds: of the keys the rows of two tokens, one from each 16-token block of
// the product K Q^T (block b, row m of it: token 8 (m / 4) + 4 b + m % 4, so that lane quarter q finds the logits of octet q in its
// accumulators), the parameters of octet q's keys, and of the values octet q of D / 16 neighbouring channels and their parameters.
template <int D>
struct Q4Tile {
    typedef Q4<D> G;
    u32 k[2][G::WPQ];
    u32x4 ks[G::NG], km[G::NG];      // scales and offsets of the octet's eight keys
    u32 v[G::NOC];
    u32x4 vs, vm;
};

template <int W>
__device__ __forceinline__ void load_words(u32 (&dst)[W], unsigned long long p) {
    if constexpr (W == 2) {
        const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const HW_GLOBAL u32x2*>(p));
        dst[0] = x.x;
        dst[1] = x.y;
    } else {
#pragma unroll
        for (int j = 0; j < W / 4; ++j) {
            const u32x4 x = load16(p + 16 * j);
#pragma unroll
            for (int d = 0; d < 4; ++d) dst[4 * j + d] = x[d];
        }
    }
}

// Four registers of element pairs (0,1) (2,3) (4,5) (6,7) from a word, exactly the codes.
__device__ __forceinline__ u32x4 q4_codes(u32 w) {
    const f16x2 m1024 = {(_Float16)-1024.f, (_Float16)-1024.f}, inv = {(_Float16)0.0625f, (_Float16)0.0625f}, m64 = {(_Float16)-64.f, (_Float16)-64.f};
    const u32 w8 = w >> 8;
    u32x4 r;
    r[0] = h2_bits(h2_of((w & Q4_LO) | Q4_MAGIC) + m1024);
    r[1] = h2_bits(__builtin_elementwise_fma(h2_of((w & Q4_HI) | Q4_MAGIC), inv, m64));
    r[2] = h2_bits(h2_of((w8 & Q4_LO) | Q4_MAGIC) + m1024);
    r[3] = h2_bits(__builtin_elementwise_fma(h2_of((w8 & Q4_HI) | Q4_MAGIC), inv, m64));
    return r;
}

// The queries of a lane's row as B operands, and what the logits need of them: the products run on the bare codes, which fp16 holds
// exactly, against the queries times a power of two of their row's own (so bf16 queries lose nothing to fp16's range):
//   scale * q . k = sum_g s_g (sum_{e in g} q_e c_e) + m_g (sum_{e in g} q_e)
template <int D, int RB>
struct Q4Queries {
    u32x4 b[RB][D / 32];
    float sum[RB][Q4<D>::NG];        // sum of the group's queries, times the row's power of two
    float sc[RB];                    // scale * log2(e) over the power of two
};

template <class DT, int D, int RB>
__device__ __forceinline__ void q4_queries(Q4Queries<D, RB>& qq, int rb, unsigned long long row, int q, float sc) {
    typedef Q4<D> G;
    float x[G::WPQ][8];
    float top = 0.f;
#pragma unroll
    for (int r = 0; r < G::WPQ; ++r) {
        Chunk<DT>::unpack(*reinterpret_cast<const HW_GLOBAL u32x4*>(row + (64 * (r >> 1) + 16 * q + 8 * (r & 1)) * 2), x[r]);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf(x[r][e]));
    }
    top = quarter_max(top);
    // 2^f brings the largest of the row into [2^13, 2^14)
    const int f = min(max(14 - __builtin_amdgcn_frexp_expf(top), -90), 90);
    const float up = __builtin_ldexpf(1.f, f);
#pragma unroll
    for (int g = 0; g < G::NG; ++g) {
        float t = 0.f;
#pragma unroll
        for (int r = 2 * g; r < 2 * g + 2; ++r)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                x[r][e] *= up;
                t += x[r][e];
            }
        qq.sum[rb][g] = quarter_sum(t);
    }
#pragma unroll
    for (int r = 0; r < G::WPQ; ++r)
#pragma unroll
        for (int d = 0; d < 4; ++d) qq.b[rb][r][d] = Elem<F16>::pack2(x[r][2 * d], x[r][2 * d + 1]);
    qq.sc[rb] = sc * __builtin_ldexpf(1.f, -f);
}

constexpr float Q4_BELOW = 7.f, Q4_ABOVE = 15.f;   // weights are 2^7 where the reference is taken and stay below 2^15

// One tile against the rows of the workgroup.  MASKED: some row does not see all of it, or some of its tokens nobody sees (their bytes
// may be anything: the parameters of such values are cleared, their logits replaced).
template <int D, int RB, bool MASKED>
__device__ __forceinline__ void q4_compute(const Q4Tile<D>& t, const Q4Queries<D, RB>& qq, const int (&lim)[RB], int maxlim,
                                           WaveState<RB, Q4<D>::NOC>& st, int t0, int q) {
    typedef Q4<D> G;
    float p[RB][8];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
#pragma unroll
        for (int g = 0; g < G::NG; ++g) {
            const u32x4 a0 = q4_codes(t.k[b][2 * g]), a1 = q4_codes(t.k[b][2 * g + 1]);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                f32x4 acc = {0.f, 0.f, 0.f, 0.f};
                acc = Elem<F16>::mfma(a0, qq.b[rb][2 * g], acc);
                acc = Elem<F16>::mfma(a1, qq.b[rb][2 * g + 1], acc);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const u32 s2 = t.ks[g][2 * b + (r >> 1)], m2 = t.km[g][2 * b + (r >> 1)];
                    const float s = r & 1 ? h_hi(s2) : h_lo(s2), m = r & 1 ? h_hi(m2) : h_lo(m2);
                    float& x = p[rb][4 * b + r];
                    x = g == 0 ? m * qq.sum[rb][0] : __builtin_fmaf(m, qq.sum[rb][g], x);
                    x = __builtin_fmaf(s, acc[r], x);
                }
            }
        }
    }
    u32x4 pw[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        float top = NEG_BIG;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            p[rb][i] *= qq.sc[rb];
            if constexpr (MASKED) p[rb][i] = t0 + 8 * q + i < lim[rb] ? p[rb][i] : NEG_BIG;
            top = fmaxf(top, p[rb][i]);
        }
        // the reference moves only when a weight would leave the range that fp16 holds well
        if (__ballot(top > st.m[rb] + Q4_ABOVE) != 0 || st.fresh) {
            const float all = quarter_max(top);
            const float ref = all > st.m[rb] + Q4_ABOVE ? all - Q4_BELOW : st.m[rb];
            const float w = fast_exp2(st.m[rb] - ref);
            st.m[rb] = ref;
            st.l[rb] *= w;
#pragma unroll
            for (int c = 0; c < G::NOC; ++c) st.o[rb][c] *= w;
        }
        float l = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            float e = fast_exp2(p[rb][i] - st.m[rb]);
            if constexpr (MASKED) e = t0 + 8 * q + i < lim[rb] ? e : 0.f;      // (a row that has seen nothing yet: reference and logits are NEG_BIG)
            p[rb][i] = e;
            l += e;
        }
        st.l[rb] += l;
#pragma unroll
        for (int d = 0; d < 4; ++d) pw[rb][d] = Elem<F16>::pack2(p[rb][2 * d], p[rb][2 * d + 1]);
    }
    st.fresh = false;
    u32x4 vs = t.vs, vm = t.vm;
    if constexpr (MASKED) {
        const int seen = maxlim - t0 - 8 * q;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const u32 keep = seen > 2 * d + 1 ? 0xffffffffu : seen > 2 * d ? 0xffffu : 0u;
            vs[d] &= keep;
            vm[d] &= keep;
        }
    }
#pragma unroll
    for (int c = 0; c < G::NOC; ++c) {
        u32x4 a = q4_codes(t.v[c]);
#pragma unroll
        for (int d = 0; d < 4; ++d) a[d] = h2_bits(__builtin_elementwise_fma(h2_of(a[d]), h2_of(vs[d]), h2_of(vm[d])));
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) st.o[rb][c] = Elem<F16>::mfma(a, pw[rb], st.o[rb][c]);
    }
}

// Rows of the partial sums, and of what a workgroup of four waves hands over: as in store_partials, with the output channel of
// accumulator c, row i being i * D / 16 + c.
template <int D, int RB>
__device__ __forceinline__ void q4_store(WaveState<RB, D / 16>& st, Exchange<RB * 16, D>& ex, int wv, int n, int q, int lane, HW_GLOBAL float* part_o,
                                         HW_GLOBAL float* part_ml, size_t part, int nrows) {
    constexpr int NOC = D / 16, NSLOT = RB * NOC, SPW = NSLOT / NWAVES;
    static_assert(NSLOT % NWAVES == 0 && (NOC % SPW == 0), "a wave's share lies within one row block");
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const float l = quarter_sum(st.l[rb]);
#pragma unroll
        for (int c = 0; c < NOC; ++c) ex.o[wv][rb * NOC + c][lane] = st.o[rb][c];
        if (q == 0) {
            ex.m[rb * 16 + n][wv] = st.m[rb];
            ex.l[rb * 16 + n][wv] = l;
        }
    }
    __syncthreads();
    const int s0 = wv * SPW, rb = s0 / NOC, c0 = s0 % NOC, row = rb * 16 + n;
    if (row >= nrows) return;
    const f32x4 m4 = *reinterpret_cast<const f32x4*>(&ex.m[row][0]);
    const f32x4 l4 = *reinterpret_cast<const f32x4*>(&ex.l[row][0]);
    const float mm = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
    float wgt[NWAVES], lsum = 0.f;
#pragma unroll
    for (int w2 = 0; w2 < NWAVES; ++w2) {
        wgt[w2] = fast_exp2(m4[w2] - mm);
        lsum = __builtin_fmaf(l4[w2], wgt[w2], lsum);
    }
    float run[4][SPW];
#pragma unroll
    for (int j = 0; j < SPW; ++j) {
        f32x4 acc = ex.o[0][s0 + j][lane] * wgt[0];
#pragma unroll
        for (int w2 = 1; w2 < NWAVES; ++w2) acc += ex.o[w2][s0 + j][lane] * wgt[w2];
#pragma unroll
        for (int i = 0; i < 4; ++i) run[i][j] = acc[i];
    }
    HW_GLOBAL float* dst = part_o + (part + row) * D;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < SPW; ++j) dst[(4 * q + i) * NOC + c0 + j] = run[i][j];
    if (q == 0 && c0 == 0) *reinterpret_cast<HW_GLOBAL f32x2*>(part_ml + (part + row) * 2) = f32x2{mm, lsum};
}

// A workgroup = one kv head x up to 16 RB query rows of one sequence x every nsplit-th stripe of its 32-token tiles (four waves, each
// takes every (4 nsplit)-th tile).  Nothing goes through LDS but the waves' partial sums: a tile is loaded straight into the
// operands' lanes, one tile ahead of the one being multiplied, its table entries one further.
template <class DT, int D, int RB, int MINW>
__global__ __launch_bounds__(NTHREADS, MINW) void paged_q4_kernel(const PagedHeader args) {
    typedef Q4<D> G;
    constexpr int ROWS = RB * 16;
    __shared__ __attribute__((aligned(16))) Exchange<ROWS, D> ex;
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, q = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    PagedHeaderBits hb;
    paged_header_request(hb);
    WaveState<RB, G::NOC> st;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        st.m[rb] = NEG_BIG;
        st.l[rb] = 0.f;
#pragma unroll
        for (int c = 0; c < G::NOC; ++c) st.o[rb][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    st.fresh = true;
    const PagedDevHeader ph = paged_header_wait(hb);

    int bid = blockIdx.x;
    if (ph.flags & PH_XCD_REMAP) bid = (bid & 7) * (ph.nwg >> 3) + (bid >> 3);
    const int hi = fast_div(bid, ph.magic_nsplit);
    const int hkv = fast_div(hi, ph.magic_nitems);
    const int item = hi - hkv * ph.nitems, split = bid - hi * ph.nsplit;
    const int GQ = ph.Hq / ph.Hkv, T = ph.LW * ph.LS;
    const int cap = ph.block_size * ph.max_blocks, per = ph.block_size >> 3;
    const size_t slot = (size_t)(hkv * ph.nsplit + split) * ph.R;
    if (ph.cu_q != nullptr && item == 0) {
        // query tokens in front of the first sequence's and behind the last one's: nothing is seen
        const int from = min(max(ph.cu_q[ph.W], 0), T) * GQ, front = min(max(ph.cu_q[0], 0), T) * GQ;
        for (int r = tid; r < front + (ph.R - from); r += NTHREADS) {
            const size_t row = slot + (r < front ? r : from + r - front);
            for (int e = 0; e < D; ++e) ph.part_o[row * D + e] = 0.f;
            *reinterpret_cast<HW_GLOBAL f32x2*>(ph.part_ml + row * 2) = f32x2{NEG_BIG, 0.f};
        }
    }
    const PagedItem it = paged_item<ROWS>(ph, item, lane, GQ);
    if (!it.found) return;                  // the grid is sized for the worst case; uniform over the workgroup
    const int r0 = it.qs * GQ + it.rg * ROWS, rend = it.qe * GQ;
    if (r0 >= rend) return;
    const int NW = ph.nsplit * NWAVES, gw = split * NWAVES + wv;
    const HW_GLOBAL int* btw = ph.block_table + (size_t)it.w * ph.max_blocks;
    const unsigned long long kbase = reinterpret_cast<unsigned long long>(ph.kcache), vbase = reinterpret_cast<unsigned long long>(ph.vcache);

    for (int f = 0; f < ph.F; ++f) {
        const int flen = ph.frag_len[ph.cu_q != nullptr ? f * ph.W + it.w : f];
        Q4Queries<D, RB> qq;
        int lim[RB], maxlim = 0, minlim = 0x7fffffff;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const int r = r0 + rb * 16 + n, rc = min(r, rend - 1);
            const int ws = fast_div(rc, ph.magic_gq), gq = rc - ws * GQ;
            const int w = fast_div(ws, ph.magic_ls), s = ws - w * ph.LS;
            const int loc = ph.loc[(size_t)f * T + ws];
            const size_t qrow = (((size_t)f * ph.LW + w) * ph.Hq + hkv * GQ + gq) * ph.LS + s;
            q4_queries<DT, D, RB>(qq, rb, reinterpret_cast<unsigned long long>(ph.q) + qrow * (D * 2), q, ph.sc);
            const int seen = max(0, min(min(flen, cap), loc < cap ? loc + 1 : cap));
            lim[rb] = seen;
            maxlim = max(maxlim, seen);
            minlim = min(minlim, seen);      // (rows that pad the block repeat the last one)
        }
        maxlim = __builtin_amdgcn_readfirstlane(row_max16(maxlim));
        minlim = __builtin_amdgcn_readfirstlane(row_min16(minlim));
        const int tiles = (maxlim + TILE - 1) / TILE;
        if (gw >= tiles) continue;          // (no barrier before the end)
        const int last = (maxlim - 1) >> 3;    // octets behind it are read as this one, and masked

        auto octet_of = [&](int t) { return min(t * 4 + q, last); };
        auto entry = [&](int t) { return btw[fast_div(octet_of(t), ph.magic_bs)]; };
        auto request = [&](Q4Tile<D>& tr, int t, int e) {
            const int o = octet_of(t);
            const int blk = min(max(e, 0), ph.num_blocks - 1);
            const int rid = (blk * ph.Hkv + hkv) * per + (o - fast_div(o, ph.magic_bs) * per);
            const int krid = __shfl(rid, (n >> 2) << 4, 64);
            const unsigned long long krow = kbase + (unsigned long long)(unsigned)krid * G::OCT + (n & 3) * G::KROW + q * (G::WPQ * 4);
            load_words(tr.k[0], krow);
            load_words(tr.k[1], krow + 4 * G::KROW);
            const unsigned long long kp = kbase + (unsigned long long)(unsigned)rid * G::OCT + G::PAR;
#pragma unroll
            for (int g = 0; g < G::NG; ++g) {
                tr.ks[g] = load16(kp + 32 * g);
                tr.km[g] = load16(kp + 32 * g + 16);
            }
            const unsigned long long vp = vbase + (unsigned long long)(unsigned)rid * G::OCT;
            load_words(tr.v, vp + n * (G::NOC * 4));
            const unsigned long long vpp = vp + G::PAR + ((n * G::NOC) >> 6) * 32;
            tr.vs = load16(vpp);
            tr.vm = load16(vpp + 16);
        };
        auto compute = [&](const Q4Tile<D>& tr, int t) {
            if ((t + 1) * TILE <= minlim) q4_compute<D, RB, false>(tr, qq, lim, maxlim, st, t * TILE, q);
            else q4_compute<D, RB, true>(tr, qq, lim, maxlim, st, t * TILE, q);
        };
        Q4Tile<D> ta, tb;
        int e0 = entry(gw), e1 = entry(gw + NW);
        request(ta, gw, e0);
        for (int t = gw; t < tiles; t += 2 * NW) {
            e0 = entry(t + 2 * NW);
            request(tb, t + NW, e1);
            compute(ta, t);
            if (t + NW >= tiles) break;
            e1 = entry(t + 3 * NW);
            request(ta, t + 2 * NW, e0);
            compute(tb, t + NW);
        }
    }
    q4_store<D, RB>(st, ex, wv, n, q, lane, ph.part_o, ph.part_ml, slot + r0, min(ROWS, rend - r0));
}

// ------------------------------------------------------------------------------------------------
// launchers
// ------------------------------------------------------------------------------------------------
template <class DT>
static hipError_t launch_q4_dt(const PagedHeader& ph, int E, int rb, hipStream_t stream) {
    const dim3 grid(ph.nwg), threads(NTHREADS);
    if (E == 64) {
        if (rb == 1) hipLaunchKernelGGL((paged_q4_kernel<DT, 64, 1, 3>), grid, threads, 0, stream, ph);
        else if (rb == 2) hipLaunchKernelGGL((paged_q4_kernel<DT, 64, 2, 2>), grid, threads, 0, stream, ph);
        else return hipErrorInvalidValue;
    } else if (E == 128) {
        if (rb == 1) hipLaunchKernelGGL((paged_q4_kernel<DT, 128, 1, 2>), grid, threads, 0, stream, ph);
        else if (rb == 2) hipLaunchKernelGGL((paged_q4_kernel<DT, 128, 2, 1>), grid, threads, 0, stream, ph);
        else return hipErrorInvalidValue;
    } else if (E == 256) {
        if (rb == 1) hipLaunchKernelGGL((paged_q4_kernel<DT, 256, 1, 1>), grid, threads, 0, stream, ph);
        else return hipErrorInvalidValue;
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_paged_q4(const PagedHeader& ph, int dtype, int E, int rb, hipStream_t stream) {
    return dtype == 1 ? launch_q4_dt<F16>(ph, E, rb, stream) : launch_q4_dt<BF16>(ph, E, rb, stream);
}

// The octets that S_new tokens from any position on may touch, and the grid that takes them.
static dim3 q4_grid(const CopyBlocksArgs& a, int D, int* octets) {
    *octets = (a.S_new + 14) / 8;
    return dim3((unsigned)(((long long)*octets * 2 * (D / 64) + 3) / 4), (unsigned)a.Hkv, (unsigned)a.B);
}

template <class DT>
static hipError_t launch_append_q4_dt(const CopyBlocksArgs& a, bool vec, hipStream_t stream) {
    int octets;
    const dim3 grid = q4_grid(a, a.E, &octets);
    auto go = [&](auto d) {
        constexpr int D = decltype(d)::value;
        if (vec) hipLaunchKernelGGL((append_q4_kernel<DT, D, true>), grid, dim3(256), 0, stream, a, octets);
        else hipLaunchKernelGGL((append_q4_kernel<DT, D, false>), grid, dim3(256), 0, stream, a, octets);
    };
    if (a.E == 64) go(std::integral_constant<int, 64>{});
    else if (a.E == 128) go(std::integral_constant<int, 128>{});
    else go(std::integral_constant<int, 256>{});
    return hipGetLastError();
}

hipError_t launch_append_q4(const CopyBlocksArgs& a, int dtype, hipStream_t stream) {
    const int sz = dtype == 0 ? 4 : 2;
    const bool vec = (a.ks_b * sz) % 16 == 0 && (a.ks_h * sz) % 16 == 0 && (a.ks_s * sz) % 16 == 0 && (a.vs_b * sz) % 16 == 0 &&
                     (a.vs_h * sz) % 16 == 0 && (a.vs_s * sz) % 16 == 0 &&
                     ((reinterpret_cast<uintptr_t>(a.key_states) | reinterpret_cast<uintptr_t>(a.value_states)) & 15u) == 0;
    switch (dtype) {
        case 0: return launch_append_q4_dt<F32>(a, vec, stream);
        case 1: return launch_append_q4_dt<F16>(a, vec, stream);
        default: return launch_append_q4_dt<BF16>(a, vec, stream);
    }
}

template <class DT>
static hipError_t launch_read_q4_dt(const CopyBlocksArgs& a, hipStream_t stream) {
    int octets;
    const dim3 grid = q4_grid(a, a.E, &octets);
    if (a.E == 64) hipLaunchKernelGGL((read_q4_kernel<DT, 64>), grid, dim3(256), 0, stream, a, octets);
    else if (a.E == 128) hipLaunchKernelGGL((read_q4_kernel<DT, 128>), grid, dim3(256), 0, stream, a, octets);
    else hipLaunchKernelGGL((read_q4_kernel<DT, 256>), grid, dim3(256), 0, stream, a, octets);
    return hipGetLastError();
}

hipError_t launch_read_q4(const CopyBlocksArgs& a, int dtype, hipStream_t stream) {
    switch (dtype) {
        case 0: return launch_read_q4_dt<F32>(a, stream);
        case 1: return launch_read_q4_dt<F16>(a, stream);
        default: return launch_read_q4_dt<BF16>(a, stream);
    }
}

}  // namespace hw
