// Paged caches in 4 bits for gfx950 (MI355X, CDNA4, wave64): the append that quantises, the read that gives the values back, and
// the attention that reads the codes (each kernel's measurements stand above it).
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
    static constexpr int UNIT = D == 64 ? 5 : D == 128 ? 6 : 7;   // an octet is 9 << UNIT bytes
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

// What the decoding of a tile keeps in registers throughout (as literals the masks cost an instruction more a pair: an instruction
// with three operands takes none), and a block of zeros for products to begin with.
struct Q4Consts {
    u32 lo, hi, magic, one;
    f32x4 zero;
    __device__ __forceinline__ explicit Q4Consts(int lane) : lo(Q4_LO), hi(Q4_HI), magic(Q4_MAGIC), one(lane < 16 ? 0x3c003c00u : 0u), zero{0.f, 0.f, 0.f, 0.f} {
        asm volatile("" : "+v"(lo), "+v"(hi), "+v"(one), "+s"(magic));
    }
};

// Four registers of element pairs (0,1) (2,3) (4,5) (6,7) from a word: exactly the codes.
__device__ __forceinline__ u32x4 q4_codes(u32 w, const Q4Consts& k) {
    const f16x2 m1024 = {(_Float16)-1024.f, (_Float16)-1024.f}, inv = {(_Float16)0.0625f, (_Float16)0.0625f}, m64 = {(_Float16)-64.f, (_Float16)-64.f};
    const u32 w8 = w >> 8;
    u32x4 r;
    r[0] = h2_bits(h2_of((w & k.lo) | k.magic) + m1024);
    r[1] = h2_bits(__builtin_elementwise_fma(h2_of((w & k.hi) | k.magic), inv, m64));
    r[2] = h2_bits(h2_of((w8 & k.lo) | k.magic) + m1024);
    r[3] = h2_bits(__builtin_elementwise_fma(h2_of((w8 & k.hi) | k.magic), inv, m64));
    return r;
}

// ------------------------------------------------------------------------------------------------
// append and read
// ------------------------------------------------------------------------------------------------
// Of values that are no NaN, as one instruction each (fmaxf has every operand quieted first).
__device__ __forceinline__ float max3_nn(float a, float b, float c) {
    float r;
    asm("v_max3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float min3_nn(float a, float b, float c) {
    float r;
    asm("v_min3_f32 %0, %1, %2, %3" : "=v"(r) : "v"(a), "v"(b), "v"(c));
    return r;
}
__device__ __forceinline__ float max8(const float (&x)[8]) {
    return max_nn(max3_nn(max3_nn(max3_nn(x[0], x[1], x[2]), x[3], x[4]), x[5], x[6]), x[7]);
}
__device__ __forceinline__ float min8(const float (&x)[8]) {
    return min3_nn(min3_nn(min3_nn(min3_nn(x[0], x[1], x[2]), x[3], x[4]), x[5], x[6]), x[7], x[7]);
}
// Over the eight lanes of a token (lane % 8), by data-parallel-primitive moves.
template <int CTRL>
__device__ __forceinline__ float lane_dpp(float v) { return __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(v), CTRL, 0xf, 0xf, true)); }
__device__ __forceinline__ float oct_min(float v) {
    v = min3_nn(v, v, lane_dpp<0xB1>(v));
    v = min3_nn(v, v, lane_dpp<0x4E>(v));
    return min3_nn(v, v, lane_dpp<0x141>(v));
}
__device__ __forceinline__ float oct_max(float v) {
    v = max_nn(v, lane_dpp<0xB1>(v));
    v = max_nn(v, lane_dpp<0x4E>(v));
    return max_nn(v, lane_dpp<0x141>(v));
}

// nibble position of element i (0..7) of a word
__device__ __forceinline__ constexpr int q4_shift(int i) { return 4 * ((i >> 1) + ((i & 1) << 2)); }

// Transposes the 8 x 8 nibbles of the lanes with one lane % 8 (lane row = lane / 8, one word each): afterwards lane row i holds element
// i of rows 0..7, row r as element r.  Three rounds: bit k of the lane row changes places with that of the element, which stand in a
// word's places in the order of q4_shift (bit 0 of the element is 16 bits, bit 1 is 4, bit 2 is 8).  A lane takes from its partner
// the nibbles that `from` names, moved by the distance one way or (by a rotation, as the others are not taken) the other.
struct Q4Transpose {
    u32 from[3], turn[3];
    __device__ __forceinline__ explicit Q4Transpose(int lane) {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const u32 low = k == 0 ? 0x0000FFFFu : k == 1 ? 0x0F0F0F0Fu : 0x00FF00FFu;
            const int sh = k == 0 ? 16 : 4 * k;
            const bool up = (lane >> (3 + k)) & 1;
            from[k] = up ? low : ~low;
            turn[k] = up ? sh : 32 - sh;
        }
    }
    __device__ __forceinline__ u32 operator()(u32 w) const {
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            const u32 other = k == 0 ? (u32)row_dpp<0x128>((int)w) : (u32)__shfl_xor((int)w, 8 << k, 64);     // (half a row of sixteen on)
            w = (__builtin_amdgcn_alignbit(other, other, turn[k]) & from[k]) | (w & ~from[k]);
        }
        return w;
    }
};

// x / y to the nearest, as the division gives it, from r = 1 / y to the nearest: the remainder of the first quotient is exact and what it
// adds is, but for less than 2^-22 of a last place, and quotients by numbers of 11 bits stay 2^-12 of a last place away from
// the middle between two.  (Eight divisions a lane were a third of the append's instructions.)
__device__ __forceinline__ float q4_divide(float x, float y, float r) {
    const float q = x * r;
    return __builtin_fmaf(__builtin_fmaf(-q, y, x), r, q);
}

// Where the octet `o` of sequence b lies, in octets from the cache's start, and whether it lies anywhere (in the table and the cache; if
// not: at the start).
__device__ __forceinline__ long long q4_octet(const CopyBlocksArgs& a, int b, int h, int o, bool& there) {
    const int per = a.block_size >> 3;
    const int bi = max(o, 0) / per;
    const int blk = a.block_table[(size_t)b * a.max_blocks + min(bi, a.max_blocks - 1)];
    there = o >= 0 && bi < a.max_blocks && blk >= 0 && blk < a.num_blocks;
    return there ? ((long long)blk * a.Hkv + h) * per + (o - bi * per) : 0;
}

// One wave = one octet x one group of 64 channels of one (sequence, kv head), of the keys and of the values: lane = (token of the
// octet, eight channels).  The lane's channels are one word of a key row as they are; for the values the words are transposed over
// the lanes of the eight tokens.  Tokens of the octet that are not being appended keep their codes: the only writer of an octet's group
// is one wave, and what it does not replace it reads first (a decode step's append reads and writes 9 D / 2 bytes a head besides
// the token's own 2 D).  Both tensors' rows and the table entry are requested together.  The rows are
// read once and stream past the caches: 4 x 2048 tokens of 8 kv heads, D = 128, bf16 (43 MB) 17.4 us with cached loads, 14.2 without
// (3.0 TB/s; the arithmetic alone, some 330 instructions a wave, is 8 us).  grid = (octets * groups / 4 waves, kv head,
// sequence).
template <class DT, int D, bool VEC>
__global__ __launch_bounds__(256) void append_q4_kernel(const CopyBlocksArgs a, int octets) {
    typedef typename Elem<DT>::store_t store_t;
    typedef Q4<D> G;
    constexpr int CH = Chunk<DT>::CH;
    const int lane = threadIdx.x & 63;
    const int item = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6));
    const int h = blockIdx.y, b = blockIdx.z;
    const int oi = item / G::NG, g = item % G::NG;
    if (oi >= octets) return;
    const int first = a.seq_lengths[b];
    const int o = (first >> 3) + oi;                     // (floor: of a negative position the part from 0 on is appended, as by copy_to_blocks)
    const int i = lane >> 3, c = lane & 7;
    const int t = o * 8 + i - first;                     // new token of this lane
    const bool mine = t >= 0 && t < a.S_new;
    if (o < 0 || o * 8 >= first + a.S_new) return;       // uniform

    float x[2][8];
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        const store_t* src = reinterpret_cast<const store_t*>(kv == 0 ? a.key_states : a.value_states) +
                             ((long long)b * (kv == 0 ? a.ks_b : a.vs_b) + (long long)h * (kv == 0 ? a.ks_h : a.vs_h) +
                              (long long)(mine ? t : 0) * (kv == 0 ? a.ks_s : a.vs_s) + 64 * g + 8 * c);
        if constexpr (VEC) {
#pragma unroll
            for (int k = 0; k < 8 / CH; ++k) {
                float y[CH];
                Chunk<DT>::unpack(__builtin_nontemporal_load(reinterpret_cast<const u32x4*>(src + k * CH)), y);
#pragma unroll
                for (int e = 0; e < CH; ++e) x[kv][k * CH + e] = y[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) x[kv][e] = Elem<DT>::to_float(src[e]);
        }
    }
    bool there;
    const long long at = q4_octet(a, b, h, o, there) * G::OCT;
    const u32 tokens = 0xffu & (u32)(((1 << min(max(first + a.S_new - o * 8, 0), 8)) - 1) & ~((1 << min(max(first - o * 8, 0), 8)) - 1));   // the octet's new tokens
    const Q4Transpose transpose(lane);
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        float lo = min8(x[kv]), hi = max8(x[kv]), zero = 0.f;
#pragma unroll
        for (int e = 0; e < 8; ++e) zero = __builtin_fmaf(x[kv][e], 0.f, zero);
        // (NaN and what is beyond the limit are rare, and three instructions an element)
        if (__ballot(!(zero == 0.f) || lo < -Q4_LIMIT || hi > Q4_LIMIT) != 0) {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float y = x[kv][e];
                x[kv][e] = y != y ? 0.f : __builtin_amdgcn_fmed3f(y, -Q4_LIMIT, Q4_LIMIT);
            }
            lo = min8(x[kv]);
            hi = max8(x[kv]);
        }
        lo = oct_min(lo);
        hi = oct_max(hi);
        const _Float16 mh = (_Float16)lo;
        const float m = (float)mh;
        const _Float16 sh = (_Float16)fmaxf(q4_divide(hi - m, 15.f, 1.f / 15.f), 0.f);
        const float s = (float)sh, r = 1.f / (s > 0.f ? s : 1.f);
        // (codes as the last bits of 2^23 + code; the sum of the words that the 2^23 come to is taken off at the end)
        u32 w = 0, bias = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float code = __builtin_amdgcn_fmed3f(q4_divide(x[kv][e] - m, s, r), 0.f, 15.f) + 0x1p23f;
            w += __float_as_uint(code) << q4_shift(e);
            bias += 0x4B000000u << q4_shift(e);
        }
        w = s > 0.f ? w - bias : 0u;
        char* oct = reinterpret_cast<char*>(kv == 0 ? a.kcache : a.vcache) + at;
        if (kv == 0) {
            // channels 64 g + 8 c .. + 7: quarter c / 2, word (quarter) * WPQ + 2 g + c % 2
            if (there && mine) *reinterpret_cast<u32*>(oct + i * G::KROW + ((c >> 1) * G::WPQ + 2 * g + (c & 1)) * 4) = w;
        } else {
            w = transpose(w);                            // now: channel 64 g + 8 c + i, its eight tokens
            u32* dst = reinterpret_cast<u32*>(oct) + 64 * g + 8 * c + i;
            if (there && tokens != 0xffu) {
                u32 keep = 0;
#pragma unroll
                for (int e = 0; e < 8; ++e) keep |= (tokens >> e) & 1 ? 0u : 15u << q4_shift(e);
                w = (*dst & keep) | (w & ~keep);
            }
            if (there) *dst = w;
        }
        if (there && mine && c == 0) {
            _Float16* par = reinterpret_cast<_Float16*>(oct + G::PAR + 32 * g) + i;
            par[0] = sh;
            par[8] = mh;
        }
    }
}

// The values of positions first[b] .. first[b] + n - 1 as [B, Hkv, n, D]; positions outside the table or the cache give zeros.  The
// waves and lanes of append_q4_kernel, the other way round.  Bound by its writes: 4 x 2048 tokens of 8 kv heads, D = 128, to fp32 16.5 us
// (76 MB, 4.6 TB/s; stores that stream past the caches 21 us).
template <class DT, int D>
__global__ __launch_bounds__(256) void read_q4_kernel(const CopyBlocksArgs a, int octets) {
    typedef typename Elem<DT>::store_t store_t;
    typedef Q4<D> G;
    constexpr int CH = Chunk<DT>::CH;
    const int lane = threadIdx.x & 63;
    const int item = __builtin_amdgcn_readfirstlane((int)blockIdx.x * 4 + (int)(threadIdx.x >> 6));
    const int h = blockIdx.y, b = blockIdx.z;
    const int oi = item / G::NG, g = item % G::NG;
    if (oi >= octets) return;
    const int first = a.seq_lengths[b];
    const int i = lane >> 3, c = lane & 7;
    const int o = (first >> 3) + oi;                     // (floor, also of negative positions)
    const int t = oi * 8 + i - (first & 7);
    bool there;
    const long long at = q4_octet(a, b, h, o, there) * G::OCT;
    const char* koct = reinterpret_cast<const char*>(a.kcache) + at;
    const char* voct = reinterpret_cast<const char*>(a.vcache) + at;
    const u32 kw = *reinterpret_cast<const u32*>(koct + i * G::KROW + ((c >> 1) * G::WPQ + 2 * g + (c & 1)) * 4);
    const u32 vw = *reinterpret_cast<const u32*>(voct + (64 * g + 8 * c + i) * 4);
    const _Float16* kpar = reinterpret_cast<const _Float16*>(koct + G::PAR + 32 * g) + i;
    const _Float16* vpar = reinterpret_cast<const _Float16*>(voct + G::PAR + 32 * g) + i;
    const float ks = (float)kpar[0], km = (float)kpar[8], vs = (float)vpar[0], vm = (float)vpar[8];
    const Q4Transpose transpose(lane);
    const u32 words[2] = {kw, transpose(vw)};            // (of the values: token i, channels 64 g + 8 c .. + 7)
    const size_t row = ((size_t)b * a.Hkv + h) * a.S_new + t;
    if (t < 0 || t >= a.S_new) return;
#pragma unroll
    for (int kv = 0; kv < 2; ++kv) {
        const float sc = there ? (kv == 0 ? ks : vs) : 0.f, m = there ? (kv == 0 ? km : vm) : 0.f;
        const u32 even = words[kv] & 0x0F0F0F0Fu, odd = (words[kv] >> 4) & 0x0F0F0F0Fu;   // bytes: elements 0 4 1 5 and 2 6 3 7
        float y[8 / CH][CH];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int n = q4_shift(e) / 4;
            y[e / CH][e % CH] = __builtin_fmaf((float)(((n & 1 ? odd : even) >> (8 * (n >> 1))) & 0xffu), sc, m);
        }
        store_t* dst = reinterpret_cast<store_t*>(const_cast<void*>(kv == 0 ? a.key_states : a.value_states)) + row * D + 64 * g + 8 * c;
#pragma unroll
        for (int k = 0; k < 8 / CH; ++k) *reinterpret_cast<u32x4*>(dst + k * CH) = Chunk<DT>::pack(y[k]);
    }
}

// ------------------------------------------------------------------------------------------------
// attention
// ------------------------------------------------------------------------------------------------
// What a lane holds of one 32-token tile (four octets) in flight.  Of the keys the rows of two tokens, one from each 16-token block of
// the product K Q^T (block b, row m of it: token 8 (m / 4) + 4 b + m % 4, so that lane quarter q finds the logits of octet q in its
// accumulators); of the values octet q of D / 16 neighbouring channels; and its share of the parameters: the sixteen lanes of quarter
// q hold those of octet q between them (at D = 64 the keys' and the values' in one word a lane).  They go through the wave's own
// piece of LDS when the tile is multiplied, where every lane reads those it needs: loaded by every lane for itself they took 24 registers
// a tile instead of 2, and with them the second tile in flight.
template <int D>
struct Q4Tile {
    typedef Q4<D> G;
    static constexpr int NP = D <= 128 ? 1 : 2;          // parameter words of a lane: keys, and values (D > 64)
    u32 k[2][G::WPQ];
    u32 v[G::NOC];
    u32 kp[NP], vp[NP];
};
template <int D>
struct Q4Params {                                        // a wave's parameters in LDS
    static constexpr int OCTET = D == 64 ? 64 : Q4<D>::NG * 32;          // bytes between octets
    static constexpr int VALUES = D == 64 ? 32 : 4 * Q4<D>::NG * 32;     // where those of the values begin
    static constexpr int BYTES = 256 * Q4<D>::NG;
};

template <int W>
__device__ __forceinline__ void load_words(u32 (&dst)[W], unsigned long long p) {
    if constexpr (W == 1) {
        dst[0] = *reinterpret_cast<const HW_GLOBAL u32*>(p);
    } else if constexpr (W == 2) {
        const u32x2 x = *reinterpret_cast<const HW_GLOBAL u32x2*>(p);
        dst[0] = x.x;
        dst[1] = x.y;
    } else {
#pragma unroll
        for (int j = 0; j < W / 4; ++j) {
            const u32x4 x = *reinterpret_cast<const HW_GLOBAL u32x4*>(p + 16 * j);
#pragma unroll
            for (int d = 0; d < 4; ++d) dst[4 * j + d] = x[d];
        }
    }
}

// The first lane of every sixteen for all of them; and each lane's value one lane down.
__device__ __forceinline__ unsigned q4_first(unsigned v) { return (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x150, 0xf, 0xf, true); }
__device__ __forceinline__ unsigned q4_next(unsigned v) { return (unsigned)__builtin_amdgcn_mov_dpp((int)v, 0x12F, 0xf, 0xf, true); }

// The element pairs of a word in 5 instructions instead of the 9 of q4_codes: 2^-24 times the codes, the second and the fourth pair 16
// times that.  Bits 0..7 of a half are a subnormal number, which the matrix instructions take as it is.
__device__ __forceinline__ u32x4 q4_tiny(u32 w, const Q4Consts& k) {
    const u32 w8 = w >> 8;
    return u32x4{w & k.lo, w & k.hi, w8 & k.lo, w8 & k.hi};
}

// The logits.  The products run on the bare codes, which fp16 holds exactly, against the queries times a power of two of their row's own
// (so bf16 queries lose nothing to fp16's range); scales and offsets of the groups g join in fp32:
//   q . k = sum_g s_g (sum_{e in g} q_e c_e) + m_g (sum_{e in g} q_e)
// The second part and minus the reference of the exponentials (seed) are one product more for 16 tokens, of the offsets and a one with the
// sums of the queries and the seed, each as two fp16 numbers: by fp32 instructions it took 16 a tile and row block instead of 2.  What
// comes out counts in the units of the products; `sc` takes it to base 2.
//
// Sums of a wave over its tiles:
template <int RB, int NOC>
struct Q4State {
    f32x4 o[RB][NOC];
    float m[RB], l[RB];              // reference (base-2 units, NEG_BIG: none yet), this lane's part of the sum of the weights
    u32 seed[RB];                    // minus the reference in the products' units: two fp16 numbers, their sum is what it stands for
    float above[RB], unit[RB];       // in them, too: the logit (less the reference) beyond which that moves, and 1 in base 2
};

// More than 128 channels and rows of 16 together (QLDS): the operands lie in LDS, made ready by one wave for each 16 rows and read by
// the four for every tile, instead of in 32 registers of every wave, which then are too few for two waves on a SIMD.
template <int D>
struct Q4Block {                     // of 16 rows
    u32x4 b[D / 32];                 // (against q4_tiny: the second and fourth pair over 16)
    u32 sum;                         // lane quarter g: the sum of group g's queries in the units of the products, as two fp16 numbers
    float sc;                        // scale * log2(e) over those units
};
template <int D, int RB, bool QLDS>
struct Q4Queries {
    u32x4 b[QLDS ? 1 : RB][QLDS ? 1 : D / 32];
    u32x2 row[RB];                   // Q4Block's sum and sc (as two arrays the optimizer put them into memory)
    __device__ __forceinline__ u32 sum(int rb) const { return row[rb].x; }
    __device__ __forceinline__ float sc(int rb) const { return __uint_as_float(row[rb].y); }
};

// A number as the sum of two fp16 ones, 2^-22 of itself exact, the second times `up` (beyond what fp16 counts in: 2^-25 / up).
__device__ __forceinline__ u32 q4_pair(float x, float up) {
    const u32 hi = Elem<F16>::pack2(x, 0.f);
    return hi | Elem<F16>::pack2(0.f, (x - h_lo(hi)) * up);
}
// The sum of a row's queries is small in the products' units (2^-11 or so where its largest counts for much): its second half is kept
// this much larger and meets offsets that much smaller.
constexpr float Q4_LOW = 256.f;
// Logits stay within D 2^14 65024 2^-24 <= 16 256 of the products' units, and 2^7 is 448 of them at most (q4_queries): what lies beyond
// fp16's range are references of fragments with much larger queries.  44 000 units are more than 2^600 there, so either way one side's
// weights are nothing.
__device__ __forceinline__ u32 q4_seed(float x) { return q4_pair(fminf(fmaxf(x, -6.0e4f), 6.0e4f), 1.f); }

template <class DT, int D>
__device__ __forceinline__ void q4_queries(Q4Block<D>& qq, const u32x4 (&raw)[D / 32], float sc, int q) {
    typedef Q4<D> G;
    float x[G::WPQ][8];
    float top = 0.f;
#pragma unroll
    for (int r = 0; r < G::WPQ; ++r) {
        Chunk<DT>::unpack(raw[r], x[r]);
#pragma unroll
        for (int e = 0; e < 8; ++e) top = fmaxf(top, __builtin_fabsf(x[r][e]));
    }
    top = quarter_max(top);
    // 2^f brings the largest of the row into [2^13, 2^14), or less where a logit of 1 in base 2 would come to more than 64 units
    const int f = min(max(min(14 - __builtin_amdgcn_frexp_expf(top), 29 + __builtin_amdgcn_frexp_expf(sc)), -113), 90);
    const float up = __builtin_ldexpf(1.f, f);
    const float up16 = up * 0.0625f;
#pragma unroll
    for (int r = 0; r < G::WPQ; ++r)
#pragma unroll
        for (int d = 0; d < 4; ++d) qq.b[r][d] = Elem<F16>::pack2(x[r][2 * d] * (d & 1 ? up16 : up), x[r][2 * d + 1] * (d & 1 ? up16 : up));
    // their sums, as products with a key of ones: every row of the result holds them
    const u32x4 ones = {0x3c003c00u, 0x4c004c00u, 0x3c003c00u, 0x4c004c00u};     // 1, and 16 for the pairs over 16
    float sum = 0.f;
#pragma unroll
    for (int g = 0; g < G::NG; ++g) {
        f32x4 t = Elem<F16>::mfma(ones, qq.b[2 * g], f32x4{0.f, 0.f, 0.f, 0.f});
        t = Elem<F16>::mfma(ones, qq.b[2 * g + 1], t);
        sum = q == g ? t[0] * 0x1p-24f : sum;
    }
    qq.sum = q4_pair(sum, Q4_LOW);
    qq.sc = fmaxf(__builtin_ldexpf(sc, 24 - f), 1e-36f);      // (its inverse has to be finite; such logits are 0)
}

typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ f32x4 mfma_f16_k16(u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
}

constexpr float Q4_BELOW = 7.f, Q4_ABOVE = 15.f;   // weights are 2^7 where the reference is taken and stay below 2^15

// One tile against the rows of the workgroup.  `partial` (uniform): some row does not see all of it, or some of its tokens nobody sees
// (their bytes may be anything: the parameters of such values are cleared, their logits replaced).  SPLIT (fp16 results): the weights as the sum of
// two fp16 numbers, 2^-22 of themselves exact; with one the result is 1.5 times as far from the exact one as its own rounding makes it.
template <int D, int RB, bool SPLIT, bool QLDS>
__device__ __forceinline__ void q4_compute(bool partial, const Q4Tile<D>& t, char* par, const Q4Queries<D, RB, QLDS>& qq, const u32x4* q_lds, const int (&lim)[RB], int maxlim,
                                           Q4State<RB, Q4<D>::NOC>& st, const Q4Consts& cs, int t0, int n, int q, int lane) {
    typedef Q4<D> G;
    typedef Q4Params<D> P;
    // (the wave's own piece of LDS: its operations complete in order, so no barrier)
    if constexpr (Q4Tile<D>::NP == 1) {
        *reinterpret_cast<u32*>(par + lane * 4) = t.kp[0];
        if constexpr (D > 64) *reinterpret_cast<u32*>(par + P::VALUES + lane * 4) = t.vp[0];
    } else {
        *reinterpret_cast<u32x2*>(par + lane * 8) = u32x2{t.kp[0], t.kp[1]};
        *reinterpret_cast<u32x2*>(par + P::VALUES + lane * 8) = u32x2{t.vp[0], t.vp[1]};
    }
    asm volatile("" ::: "memory");
    __builtin_amdgcn_wave_barrier();
    const char* kpar = par + q * P::OCTET;
    f32x4 acc[G::NG][2][RB];
#pragma unroll
    for (int g = 0; g < G::NG; ++g)
#pragma unroll
        for (int b = 0; b < 2; ++b) {
            const u32x4 a0 = q4_tiny(t.k[b][2 * g], cs), a1 = q4_tiny(t.k[b][2 * g + 1], cs);
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const u32x4 b0 = QLDS ? q_lds[(rb * G::WPQ + 2 * g) * 64 + lane] : qq.b[QLDS ? 0 : rb][QLDS ? 0 : 2 * g];
                const u32x4 b1 = QLDS ? q_lds[(rb * G::WPQ + 2 * g + 1) * 64 + lane] : qq.b[QLDS ? 0 : rb][QLDS ? 0 : 2 * g + 1];
                acc[g][b][rb] = Elem<F16>::mfma(a0, b0, cs.zero);
                acc[g][b][rb] = Elem<F16>::mfma(a1, b1, acc[g][b][rb]);
            }
        }
    // the offsets' part: lane quarter g multiplies those of group g (others by zero) with both halves of the sum of its queries
    const char* mpar = par + (n >> 2) * P::OCTET + (q < G::NG ? q : 0) * 32 + 16 + (n & 3) * 2;
    f32x4 off[2][RB];
#pragma unroll
    for (int b = 0; b < 2; ++b) {
        const _Float16 m = *reinterpret_cast<const _Float16*>(mpar + 8 * b);
        const u32 mo = h2_bits(f16x2{m, m} * f16x2{(_Float16)1.f, (_Float16)(1.f / Q4_LOW)});
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) off[b][rb] = mfma_f16_k16(u32x2{mo, cs.one}, u32x2{qq.sum(rb), st.seed[rb]}, cs.zero);
    }
    float p[RB][8];
#pragma unroll
    for (int g = 0; g < G::NG; ++g) {
        const u32x4 ks = *reinterpret_cast<const u32x4*>(kpar + 32 * g);
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float s = i & 1 ? h_hi(ks[i >> 1]) : h_lo(ks[i >> 1]);
                p[rb][i] = __builtin_fmaf(s, acc[g][i >> 2][rb][i & 3], g == 0 ? off[i >> 2][rb][i & 3] : p[rb][i]);
            }
    }
    const char* vpar = par + P::VALUES + q * P::OCTET + ((n * G::NOC) >> 6) * 32;
    u32x4 vs = *reinterpret_cast<const u32x4*>(vpar), vm = *reinterpret_cast<const u32x4*>(vpar + 16);
    if (partial) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb)
#pragma unroll
            for (int i = 0; i < 8; ++i) p[rb][i] = t0 + 8 * q + i < lim[rb] ? p[rb][i] : -__builtin_inff();
        const int seen = maxlim - t0 - 8 * q;
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            const u32 keep = seen > 2 * d + 1 ? 0xffffffffu : seen > 2 * d ? 0xffffu : 0u;
            vs[d] &= keep;
            vm[d] &= keep;
        }
    }
    // the reference moves only when a weight would leave the range that fp16 holds well
    float top[RB];
    bool beyond = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        top[rb] = max8(p[rb]);
        beyond |= top[rb] > st.above[rb];
    }
    if (__ballot(beyond) != 0) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const float all = quarter_max(top[rb]);
            const bool have = st.m[rb] > NEG_BIG, move = all > st.above[rb];      // (of one row alike in all of its lanes)
            const float was = h_lo(st.seed[rb]) + h_hi(st.seed[rb]);
            const u32 moved = q4_seed(was - (all - Q4_BELOW * st.unit[rb])), seed = move ? moved : st.seed[rb];
            const float is = h_lo(seed) + h_hi(seed), up = was - is;
            const float shrink = fast_exp2(-up * qq.sc(rb)), w = have ? shrink : 1.f;
            const float m = -is * qq.sc(rb), above = Q4_ABOVE * st.unit[rb];
            st.m[rb] = move ? m : st.m[rb];
            st.seed[rb] = seed;
            st.above[rb] = move | have ? above : -3.0e38f;
            st.l[rb] *= w;
#pragma unroll
            for (int c = 0; c < G::NOC; ++c) st.o[rb][c] *= w;
#pragma unroll
            for (int i = 0; i < 8; ++i) p[rb][i] -= up;
        }
    }
    u32x4 pw[RB], pl[SPLIT ? RB : 1];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[rb][i] = fast_exp2(p[rb][i] * qq.sc(rb));
        st.l[rb] += ((p[rb][0] + p[rb][1]) + (p[rb][2] + p[rb][3])) + ((p[rb][4] + p[rb][5]) + (p[rb][6] + p[rb][7]));
#pragma unroll
        for (int d = 0; d < 4; ++d) {
            pw[rb][d] = Elem<F16>::pack2(p[rb][2 * d], p[rb][2 * d + 1]);
            if constexpr (SPLIT) pl[rb][d] = Elem<F16>::pack2(p[rb][2 * d] - h_lo(pw[rb][d]), p[rb][2 * d + 1] - h_hi(pw[rb][d]));
        }
    }
#pragma unroll
    for (int c = 0; c < G::NOC; ++c) {
        u32x4 a = q4_codes(t.v[c], cs);
#pragma unroll
        for (int d = 0; d < 4; ++d) a[d] = h2_bits(__builtin_elementwise_fma(h2_of(a[d]), h2_of(vs[d]), h2_of(vm[d])));
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            st.o[rb][c] = Elem<F16>::mfma(a, pw[rb], st.o[rb][c]);
            if constexpr (SPLIT) st.o[rb][c] = Elem<F16>::mfma(a, pl[rb], st.o[rb][c]);
        }
    }
}

// Where the results go that need no merge.
struct Q4Out {
    HW_GLOBAL char* out;
    HW_GLOBAL float* lse;
};
// Row r (query token * GQ + head in group) of a kv head, in rows of the result.
__device__ __forceinline__ size_t q4_out_row(const PagedDevHeader& ph, int r, int hkv) {
    const int GQ = ph.Hq / ph.Hkv, ws = fast_div(r, ph.magic_gq), w = fast_div(ws, ph.magic_ls);
    return ((size_t)w * ph.Hq + hkv * GQ + (r - ws * GQ)) * ph.LS + (ws - w * ph.LS);
}

// Rows of the partial sums (or of the result, PH_DIRECT), from what the four waves hand over: accumulator c, row i holds output channel
// i * D / 16 + c.  A wave takes whole rows, four at a time, sixteen lanes to a row and D / 16 neighbouring channels to a lane, so that what it
// writes are whole lines (by accumulators as they come a store is 64 pieces of 8 or 16 bytes: 0.5 to 4 % of a call).  In LDS a quarter's
// lanes change places so that those sixteen meet no bank twice.  What is left of the end is that the 8 MB of 512 workgroups of 32 rows have to
// reach memory: 2.9 us of a launch without any tiles, whose whole is 8.1 (empty launch 2.2, tables and first tile 1.4, queries 1.4).
template <class DT, int D, int RB>
__device__ __forceinline__ void q4_store(Q4State<RB, D / 16>& st, Exchange<RB * 16, D>& ex, int wv, int n, int q, int lane, const PagedDevHeader& ph,
                                         size_t part, int nrows, const Q4Out& out, int r0, int hkv) {
    constexpr int NOC = D / 16, NSLOT = RB * NOC;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const float l = quarter_sum(st.l[rb]);
#pragma unroll
        for (int c = 0; c < NOC; ++c) ex.o[wv][rb * NOC + c][q * 16 + (n ^ (4 * q))] = st.o[rb][c];
        if (q == 0) {
            ex.m[rb * 16 + n][wv] = st.m[rb];
            ex.l[rb * 16 + n][wv] = l;
        }
    }
    __syncthreads();
    const int i = lane & 3, from = (lane >> 2) & 3, nn = wv * 4 + (lane >> 4);
    const int e = (4 * from + i) * NOC;          // the lane's first channel
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const int row = rb * 16 + nn;
        if (row >= nrows) return;
        const f32x4 m4 = *reinterpret_cast<const f32x4*>(&ex.m[row][0]);
        const f32x4 l4 = *reinterpret_cast<const f32x4*>(&ex.l[row][0]);
        const float mm = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
        const float* src = reinterpret_cast<const float*>(&ex.o[0][rb * NOC][from * 16 + (nn ^ (4 * from))]) + i;
        float lsum = 0.f, run[NOC];
#pragma unroll
        for (int c = 0; c < NOC; ++c) run[c] = 0.f;
#pragma unroll
        for (int w2 = 0; w2 < NWAVES; ++w2) {
            const float wgt = fast_exp2(m4[w2] - mm);
            lsum = __builtin_fmaf(l4[w2], wgt, lsum);
#pragma unroll
            for (int c = 0; c < NOC; ++c) run[c] = __builtin_fmaf(src[(w2 * NSLOT + c) * 256], wgt, run[c]);
        }
        if (ph.flags & PH_DIRECT) {              // (the sums are all there are)
            const float inv = lsum > 0.f ? 1.f / lsum : 0.f;
            const size_t orow = q4_out_row(ph, r0 + row, hkv);
            HW_GLOBAL u32x2* dst = reinterpret_cast<HW_GLOBAL u32x2*>(out.out + (orow * D + e) * 2);
#pragma unroll
            for (int c = 0; c < NOC; c += 4)
                dst[c / 4] = u32x2{Elem<DT>::pack2(run[c] * inv, run[c + 1] * inv), Elem<DT>::pack2(run[c + 2] * inv, run[c + 3] * inv)};
            if (out.lse != nullptr && e == 0) out.lse[orow] = lsum > 0.f ? (mm + __builtin_amdgcn_logf(lsum)) * 0.69314718055994530942f : -__builtin_inff();
        } else {
            HW_GLOBAL f32x4* dst = reinterpret_cast<HW_GLOBAL f32x4*>(ph.part_o + (part + row) * D + e);
#pragma unroll
            for (int c = 0; c < NOC; c += 4) dst[c / 4] = f32x4{run[c], run[c + 1], run[c + 2], run[c + 3]};
            if (e == 0) *reinterpret_cast<HW_GLOBAL f32x2*>(ph.part_ml + (part + row) * 2) = f32x2{mm, lsum};
        }
    }
}

// A workgroup = one kv head x up to 16 RB query rows of one sequence x every nsplit-th stripe of its 32-token tiles (four waves, each
// takes every (4 nsplit)-th tile).  A tile is loaded straight into the operands' lanes, one ahead of the one being multiplied; the
// first ones are requested as soon as the rows' bounds are known, and the queries are made ready behind them.
//
// What bounds it: with few rows the stream of the codes, 5.5 to 6 TB/s from some thousand tokens on, and about 5 us before and behind it;
// with 32 rows the vector arithmetic (65 % of the issue slots over a prompt chunk, 80 % while both waves of a SIMD are there; the
// matrix units 30 %): of some 310 slots a tile 104 are for the values' codes, 40 for the keys', 74 for the softmax of each row block, 64
// of those for exponentials.  Measured (MI355X, us a layer with the merge, GB/s of what has to be read and TFLOP/s):
//   4 x 12 528 tokens, one query each, 40/8 heads, D = 128, bf16        18.1   3200
//   296 to 10 543 tokens, 16/8 heads, D = 256, bf16                     16.4   2480
//   2052 to 11 111 tokens, four queries each, 64/8, D = 128, f16        18.7   1710   191
//   1 / 8 / 32 / 64 packed queries on 12 528 each, 40/8, bf16           56     1060   480
//   1024 queries on 5120, 40/8, bf16                                    135           715
// One tile ahead is enough: two, or the loop arranged so that nothing waits for the tile in flight at its head, changed nothing (the other
// wave of the SIMD, or the other SIMDs at D = 256, cover it).  Loads that stay in the caches beat streaming ones everywhere, by up to
// 12 % (the halves of a line are requested apart, and the row groups of a sequence read the same tiles).  128-row workgroups that decode
// into LDS for their waves were built: half a barrier's wait a step, 456 against 325 us on the prompt chunk, 134 against 125 packed.  64
// rows a wave, one wave a SIMD: nothing runs beside the softmax then, 362 against 272 and 168 against 113.
template <class DT, int D, int RB, int MINW>
__global__ __launch_bounds__(NTHREADS, MINW) void paged_q4_kernel(const PagedHeader args, const Q4Out out) {
    typedef Q4<D> G;
    constexpr int ROWS = RB * 16;
    constexpr bool SPLIT = std::is_same<DT, F16>::value;
    constexpr bool QLDS = RB * D > 128;
    constexpr int QB = QLDS ? 1 : RB;       // row blocks whose queries a wave makes ready
    __shared__ __attribute__((aligned(16))) u32x4 q_lds[QLDS ? RB * G::WPQ * 64 : 1];
    __shared__ u32 q_sums[QLDS ? RB : 1][64];
    __shared__ u32 q_sc[QLDS ? RB : 1][16];
    __shared__ __attribute__((aligned(16))) Exchange<ROWS, D> ex;
    __shared__ __attribute__((aligned(16))) char par_lds[NWAVES][Q4Params<D>::BYTES];
    const int tid = threadIdx.x, lane = tid & 63, n = lane & 15, q = lane >> 4;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    PagedHeaderBits hb;
    paged_header_request(hb);
    const Q4Consts cs(lane);
    Q4State<RB, G::NOC> st;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        st.m[rb] = NEG_BIG;
        st.l[rb] = 0.f;
#pragma unroll
        for (int c = 0; c < G::NOC; ++c) st.o[rb][c] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const PagedDevHeader ph = paged_header_wait(hb);

    int bid = blockIdx.x;
    if (ph.flags & PH_XCD_REMAP) bid = (bid & 7) * (ph.nwg >> 3) + (bid >> 3);
    const int hi = fast_div(bid, ph.magic_nsplit);
    const int hkv = fast_div(hi, ph.magic_nitems);
    int item = hi - hkv * ph.nitems, split = bid - hi * ph.nsplit;
    int ns = ph.nsplit;                     // workgroups that share the sequence's tiles
    const int wg_slot = item * ns + split;
    const bool shared = (ph.flags & PH_SHARED) != 0;
    const int GQ = ph.Hq / ph.Hkv, T = ph.LW * ph.LS;
    const int cap = ph.block_size * ph.max_blocks, per = ph.block_size >> 3;
    const size_t slot = (size_t)(hkv * ph.nsplit + split) * ph.R;
    // Query tokens in front of the first sequence's and behind the last one's (a batch padded to a fixed size): nothing is seen.  All
    // workgroups of a kv head and split share them, in pieces of 16 bytes; one for all of them took 50 us for 900 tokens of 40 heads.
    const int cu_first = ph.cu_q != nullptr ? ph.cu_q[0] : 0, cu_last = ph.cu_q != nullptr ? ph.cu_q[ph.W] : T;
    auto fill_unseen = [&](int place_in_head) {
        const bool direct = (ph.flags & PH_DIRECT) != 0;
        const int front = min(max(cu_first, 0), T) * GQ, from = min(max(cu_last, 0), T) * GQ;
        const int rows = front + (ph.R - from), pieces = direct ? D / 8 : D / 4;
        for (int x = place_in_head * NTHREADS + tid; x < rows * pieces; x += ph.nitems * NTHREADS) {
            const int r = direct ? x / (D / 8) : x / (D / 4), c = x - r * pieces, row = r < front ? r : from + r - front;
            if (direct) {
                const size_t orow = q4_out_row(ph, row, hkv);
                reinterpret_cast<HW_GLOBAL u32x4*>(out.out + orow * (D * 2))[c] = u32x4{0u, 0u, 0u, 0u};
                if (out.lse != nullptr && c == 0) out.lse[orow] = -__builtin_inff();
            } else {
                reinterpret_cast<HW_GLOBAL f32x4*>(ph.part_o + (slot + row) * D)[c] = f32x4{0.f, 0.f, 0.f, 0.f};
                if (c == 0) *reinterpret_cast<HW_GLOBAL f32x2*>(ph.part_ml + (slot + row) * 2) = f32x2{NEG_BIG, 0.f};
            }
        }
    };
    const int last_octet = (cap >> 3) - 1;
    // what of an octet this lane loads
    const unsigned long long kbase = reinterpret_cast<unsigned long long>(ph.kcache), vbase = reinterpret_cast<unsigned long long>(ph.vcache);
    const unsigned long long klane = kbase + (n & 3) * G::KROW + q * (G::WPQ * 4), vlane = vbase + n * (G::NOC * 4);
    const unsigned long long kplane = D == 64 ? (n < 8 ? kbase : vbase) + G::PAR + (n & 7) * 4 : kbase + G::PAR + n * (4 * Q4Tile<D>::NP);
    const unsigned long long vplane = vbase + G::PAR + n * (4 * Q4Tile<D>::NP);
    int seq = 0, r0 = 0, rend = 0;          // sequence; first row (token * GQ + head in group), end of the sequence's rows
    int NW = 0, gw = 0;                     // waves that share the tiles of this (kv head, row group); this one
    const HW_GLOBAL int* btw = nullptr;
    auto uniform = [](int x) { return __builtin_amdgcn_readfirstlane(x); };
    auto take = [&](int w, int row_group, int qs, int qe) {
        seq = uniform(w);
        r0 = uniform(qs * GQ + row_group * ROWS);
        rend = uniform(qe * GQ);
        NW = ns * NWAVES;
        gw = split * NWAVES + wv;
        btw = ph.block_table + (size_t)seq * ph.max_blocks;
    };
    // A tile's octets are worked out for sixteen tiles of the wave at once, lane n of quarter q for octet q of the n-th, and handed
    // out from there (q4_first, q4_next): table entry, division and products by lane and tile were a sixth of a tile's instructions.
    auto octet_of = [&](int t) { return min(t * 4 + q, last_octet); };
    auto entry = [&](int t) { return btw[fast_div(octet_of(t), ph.magic_bs)]; };
    // where it starts in the caches, in D / 2 bytes (what the table says is clamped into them; there are less than 2^28 octets)
    auto place = [&](int t, int e) {
        const int o = octet_of(t);
        return 9u * (unsigned)((min(max(e, 0), ph.num_blocks - 1) * ph.Hkv + hkv) * per + (o - fast_div(o, ph.magic_bs) * per));
    };
    // one batch of independent loads: the table entries of the first tiles, the rows' bounds and queries
    int e = 0, flen = 0, loc[RB];
    u32x4 raw[QB][G::WPQ];
    auto fetch = [&](int f) {
        e = entry(gw + n * NW);
        flen = ph.frag_len[ph.cu_q != nullptr ? f * ph.W + seq : f];
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) loc[rb] = ph.loc[(size_t)f * T + fast_div(min(r0 + rb * 16 + n, rend - 1), ph.magic_gq)];
#pragma unroll
        for (int i = 0; i < QB; ++i) {
            const int rb = QLDS ? min(wv, RB - 1) : i;
            const int rc = min(r0 + rb * 16 + n, rend - 1), ws = fast_div(rc, ph.magic_gq), gq = rc - ws * GQ;
            const int w = fast_div(ws, ph.magic_ls), s = ws - w * ph.LS;
            const HW_GLOBAL char* row = ph.q + ((((size_t)f * ph.LW + w) * ph.Hq + hkv * GQ + gq) * ph.LS + s) * (D * 2);
#pragma unroll
            for (int r = 0; r < G::WPQ; ++r) raw[i][r] = *reinterpret_cast<const HW_GLOBAL u32x4*>(row + (64 * (r >> 1) + 16 * q + 8 * (r & 1)) * 2);
        }
    };
    {
        const PagedItem it = paged_item<ROWS>(ph, item, lane, GQ);
        if (it.found) take(it.w, it.rg, it.qs, it.qe);
        if (!it.found || r0 >= rend) {      // the grid is sized for the worst case; uniform over the workgroup
            if (ph.cu_q != nullptr) fill_unseen(item);
            return;
        }
    }
    int loc0 = 0, len0 = 0, first_slot = 0;
    if (shared) {
        loc0 = ph.loc[min(lane, ph.W - 1) * ph.LS];
        len0 = ph.frag_len[0];
    }
    // (what is requested holds for equal sequences: only where the share turns out another is it requested again)
    for (bool again = shared;; again = false) {
        fetch(0);
        if (!again) break;
        const PagedShare sh = paged_share(ph, item, split, lane, loc0, len0);
        if (!sh.found) return;              // uniform over the workgroup
        first_slot = sh.slot0;
        if (sh.w == item && sh.split == split && sh.ns == ns) break;
        item = uniform(sh.w);
        split = uniform(sh.split);
        ns = uniform(sh.ns);
        take(item, 0, item * ph.LS, item * ph.LS + ph.LS);
    }

    for (int f = 0; f < ph.F; ++f) {
        if (f > 0) fetch(f);
        int lim[RB], maxlim = 0, minlim = 0x7fffffff;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            lim[rb] = max(0, min(min(flen, cap), loc[rb] < cap ? loc[rb] + 1 : cap));
            maxlim = max(maxlim, lim[rb]);
            minlim = min(minlim, lim[rb]);       // (rows that pad the block repeat the last one)
        }
        maxlim = __builtin_amdgcn_readfirstlane(row_max16(maxlim));
        minlim = __builtin_amdgcn_readfirstlane(row_min16(minlim));
        const int tiles = (maxlim + TILE - 1) / TILE;
        if (!QLDS && gw >= tiles) continue;      // (no barrier before the end)
        int ahead = entry(gw + (16 + n) * NW);       // of the sixteen tiles after these
        unsigned at = place(gw + n * NW, e);
        const unsigned idle = uniform(at);           // a tile that does not exist: this octet again, four times
        at = gw + n * NW < tiles ? at : idle;
        auto request = [&](Q4Tile<D>& tr) {
            const unsigned rid = q4_first(at), krid = __shfl(rid, (n >> 2) << 4, 64);
            at = q4_next(at);
            const unsigned long long krow = klane + ((unsigned long long)krid << G::UNIT), oct = (unsigned long long)rid << G::UNIT;
            load_words(tr.k[0], krow);
            load_words(tr.k[1], krow + 4 * G::KROW);
            load_words(tr.kp, kplane + oct);
            if constexpr (D > 64) load_words(tr.vp, vplane + oct);
            load_words(tr.v, vlane + oct);
        };
        Q4Tile<D> tr[2];
        request(tr[0]);
        Q4Queries<D, RB, QLDS> qq;
        if constexpr (QLDS) {
            lds_barrier();                       // the fragment before is done with them
            if (wv < RB) {
                Q4Block<D> blk;
                q4_queries<DT, D>(blk, raw[0], ph.sc, q);
#pragma unroll
                for (int r = 0; r < G::WPQ; ++r) q_lds[(wv * G::WPQ + r) * 64 + lane] = blk.b[r];
                q_sums[wv][lane] = blk.sum;
                if (q == 0) q_sc[wv][n] = __builtin_bit_cast(u32, blk.sc);
            }
            lds_barrier();
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                qq.row[rb] = u32x2{q_sums[rb][lane], q_sc[rb][n]};
            }
        } else {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                Q4Block<D> blk;
                q4_queries<DT, D>(blk, raw[QLDS ? 0 : rb], ph.sc, q);
#pragma unroll
                for (int r = 0; r < G::WPQ; ++r) qq.b[QLDS ? 0 : rb][QLDS ? 0 : r] = blk.b[r];
                qq.row[rb] = u32x2{blk.sum, __builtin_bit_cast(u32, blk.sc)};
            }
        }
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            // (a fragment's products have units of their own; the reference goes on)
            st.unit[rb] = 1.f / qq.sc(rb);
            st.seed[rb] = st.m[rb] == NEG_BIG ? 0u : q4_seed(-st.m[rb] * st.unit[rb]);
            st.above[rb] = st.m[rb] == NEG_BIG ? -3.0e38f : Q4_ABOVE * st.unit[rb];
        }
        for (int t = gw, i = 1; gw < tiles;) {
#pragma unroll
            for (int u = 0; u < 2; ++u, ++i) {
                if (u == 1 && (i & 15) == 0) {
                    const int tn = t + (1 + n) * NW;
                    at = place(tn, ahead);
                    at = tn < tiles ? at : idle;
                    ahead = entry(tn + 16 * NW);
                }
                request(tr[u ^ 1]);
                q4_compute<D, RB, SPLIT, QLDS>((t + 1) * TILE > minlim, tr[u], par_lds[wv], qq, q_lds, lim, maxlim, st, cs, t * TILE, n, q, lane);
                t += NW;
                if (t >= tiles) goto tiles_done;
            }
        }
    tiles_done:;
    }
    q4_store<DT, D, RB>(st, ex, wv, n, q, lane, ph, shared ? (size_t)(hkv * ph.nitems * ph.nsplit + wg_slot) * (ph.LS * GQ) : slot + r0,
                        min(ROWS, rend - r0), out, r0, hkv);
    if (ph.cu_q != nullptr) fill_unseen(item);
    // where the merge finds the rows' partial sums
    if (shared && split == 0 && tid < rend - r0) {
        HW_GLOBAL int* row_tab = reinterpret_cast<HW_GLOBAL int*>(ph.part_ml + (size_t)ph.Hkv * ph.nsplit * ph.R * 2) + ((size_t)hkv * ph.R + r0) * 2;
        row_tab[2 * tid] = first_slot | (ns << 16);
        row_tab[2 * tid + 1] = tid;
    }
}

// ------------------------------------------------------------------------------------------------
// launchers
// ------------------------------------------------------------------------------------------------
template <class DT>
static hipError_t launch_q4_dt(const PagedHeader& ph, const Q4Out& out, int E, int rb, hipStream_t stream) {
    const dim3 grid(ph.nwg), threads(NTHREADS);
    if (E == 64) {
        if (rb == 1) hipLaunchKernelGGL((paged_q4_kernel<DT, 64, 1, 3>), grid, threads, 0, stream, ph, out);
        else if (rb == 2) hipLaunchKernelGGL((paged_q4_kernel<DT, 64, 2, 2>), grid, threads, 0, stream, ph, out);
        else return hipErrorInvalidValue;
    } else if (E == 128) {
        if (rb == 1) hipLaunchKernelGGL((paged_q4_kernel<DT, 128, 1, 2>), grid, threads, 0, stream, ph, out);
        else if (rb == 2) hipLaunchKernelGGL((paged_q4_kernel<DT, 128, 2, 2>), grid, threads, 0, stream, ph, out);
        else return hipErrorInvalidValue;
    } else if (E == 256) {
        if (rb == 1) hipLaunchKernelGGL((paged_q4_kernel<DT, 256, 1, 1>), grid, threads, 0, stream, ph, out);
        else return hipErrorInvalidValue;
    } else {
        return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

hipError_t launch_paged_q4(const PagedHeader& ph, void* out, float* lse, int dtype, int E, int rb, hipStream_t stream) {
    const Q4Out o = {(HW_GLOBAL char*)out, (HW_GLOBAL float*)lse};
    return dtype == 1 ? launch_q4_dt<F16>(ph, o, E, rb, stream) : launch_q4_dt<BF16>(ph, o, E, rb, stream);
}

// The octets that S_new tokens from any position on may touch, and the grid that takes them.
static dim3 q4_grid(const CopyBlocksArgs& a, int D, int* octets) {
    *octets = (a.S_new + 14) / 8;
    return dim3((unsigned)(((long long)*octets * (D / 64) + 3) / 4), (unsigned)a.Hkv, (unsigned)a.B);
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
