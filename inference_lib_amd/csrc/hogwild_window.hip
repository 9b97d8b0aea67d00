// Attention over paged caches with a sliding window and sinks, for gfx950 (MI355X, CDNA4, wave64).
//
//   o_r = sum_j p_j v_j,  p = softmax over { j <= l_r : l_r - j < window or j < sinks } of scale * q_r . k_j
//
// for the query rows r (a token and a head of the group that shares a kv head) at positions l_r of one sequence, whose keys and values
// lie in pages.  A workgroup owns one kv head and up to 16 or 32 rows of one sequence.  Its keys are two stretches of the sequence: the
// sinks, and the union of the rows' windows.  Both are cut into tiles of 32 tokens at multiples of 32, numbered through (tile_at), and
// tile k goes to wave k mod (4 * nsplit) of the workgroups that share the rows.
//
// Bound by what is loaded: 16 sequences that see 4096 tokens of 40/8 heads of 128 channels take 46 us a layer, 269 MB at 5.8 TB/s.  Smaller steps
// show the chain in front of the loads (positions, table entries, first tiles: 3 us) and the merge, 8 us together: 5 ragged sequences that see up to
// 1088 tokens of 256 channels, 36 MB, 15 us a layer; 4 sequences of 4 tokens that see 2048, 34 MB, 15.5 (a quarter of a pass over four layers,
// merges included); the least kernel 4.3 (one workgroup a group, no merge: one sequence that sees 64 tokens of 64 channels).
// Two row blocks share what is loaded, which pays where the tiles are many (see window_plan).
//
// Sequences with more rows (prompt chunks) go through window_wide_kernel: row groups of 256, whose waves share every tile through LDS.
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "hogwild_kernels.h"
#include "hogwild_device.h"

namespace hw {

// The logit of a token that a row does not see: its weight is 0 whatever the scale (a finite one times the least scales is next to 0).
constexpr float UNSEEN = -__builtin_inff();

// The bounds of a lane's rows: row n of row block rb sees the tokens below snk[rb], and from lo[rb] to lim[rb] - 1.
template <int RB>
struct Band {
    int lo[RB], lim[RB], snk[RB];
    __device__ __forceinline__ bool sees(int rb, int tok) const { return tok < snk[rb] || (tok >= lo[rb] && tok < lim[rb]); }
};

// Infinite and NaN values.  A row's weight of a token that it does not see is 0, which times an infinite value would be NaN.  Tiles that some
// row does not see all of are therefore looked over -- also where all rows see the same of them: a token that nobody sees has the values of one
// that is seen (issue_tile) -- and where one holds such values the products take 0 in their place, and every row that sees one gets it by
// itself: with ones in the place of the values and of the weights that are seen, a product is more than 0 where a row sees a value of the kind.  NaN counts as both infinities, whose sum it is.  (With rows at one position, single tokens, looking costs nothing that
// shows; zeros in the place of the values that they do not see, without a look: two layers of 16 sequences 92.7 -> 93.5 us, of drafts 62.2 -> 63.4.)
template <class DT>
struct Wild {
    static constexpr bool WIDE = Elem<DT>::size == 4;
    static constexpr u32 EXP = WIDE ? 0x7f800000u : std::is_same<DT, F16>::value ? 0x7c00u : 0x7f80u;
    static constexpr u32 ONE = WIDE ? 0x3f800000u : std::is_same<DT, F16>::value ? 0x3c00u : 0x3f80u;
    static constexpr u32 SIGN = WIDE ? 0x80000000u : 0x8000u;
    static constexpr u32 LOW = EXP & (0u - EXP);                // the exponent's lowest bit
    static constexpr u32 TWO = WIDE ? 1u : 0x10001u;
    // not 0 under the signs: an element's exponent is all ones
    static __device__ __forceinline__ u32 signs(u32 x) { return (x & EXP * TWO) + LOW * TWO; }
    static constexpr u32 SIGNS = SIGN * TWO;
    // element by element: `clean` the finite ones, `pos` and `neg` ones where they are infinite in that direction or NaN
    static __device__ __forceinline__ void split(u32 x, u32& clean, u32& pos, u32& neg) {
        clean = pos = neg = 0;
#pragma unroll
        for (int h = 0; h < (WIDE ? 1 : 2); ++h) {
            const u32 e = WIDE ? x : (x >> (16 * h)) & 0xffffu;
            const bool wild = (e & EXP) == EXP, nan = wild && (e & (SIGN - 1) & ~EXP) != 0;
            clean |= wild ? 0u : e << (16 * h);
            pos |= wild && (nan || (e & SIGN) == 0) ? ONE << (16 * h) : 0u;
            neg |= wild && (nan || (e & SIGN) != 0) ? ONE << (16 * h) : 0u;
        }
    }
    // the ones of a lane's eight tokens that row block rb of the band sees, as MFMA operands (16-bit types)
    template <int RB>
    static __device__ __forceinline__ u32x4 seen(const Band<RB>& band, int rb, int t0, int q) {
        u32x4 r;
#pragma unroll
        for (int d = 0; d < 4; ++d)
            r[d] = (band.sees(rb, t0 + slot_token(q, 2 * d)) ? ONE : 0u) | (band.sees(rb, t0 + slot_token(q, 2 * d + 1)) ? ONE << 16 : 0u);
        return r;
    }
    static __device__ __forceinline__ f32x4 add(f32x4 o, f32x4 pos, f32x4 neg) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            o[i] += pos[i] > 0.f ? __builtin_inff() : 0.f;
            o[i] -= neg[i] > 0.f ? __builtin_inff() : 0.f;
        }
        return o;
    }
};

// One 32-token tile against all rows of the wave: K in the staging slot, V in registers (see compute_tile, whose layouts these are).
// edge: not every row sees all of its tokens.
template <class DT, int D, int RB>
__device__ __forceinline__ void band_tile(const TileRegs<DT, D, D>& t, const u32x4* qreg, const Band<RB>& band, WaveState<RB, D / 16>& st, int t0, int n, int q,
                                          float sc, const char* kstage, bool edge) {
    typedef Geo<DT, D, D> G;
    constexpr float LAZY_LOG2 = 8.0f;     // how far a row's maximum may exceed the reference of its exponentials before that follows
    float s[RB][8], mxl[RB];
    {
        f32x4 sacc[RB][2];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb) {
            u32x4 kop[G::KJ];
#pragma unroll
            for (int j = 0; j < G::KJ; ++j) kop[j] = *reinterpret_cast<const u32x4*>(kstage + kstage_offset<G>(tb * 16 + n, 4 * j + q));
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < G::KJ; ++j) {
                    if constexpr (G::SZ == 2) acc = Elem<DT>::mfma(kop[j], qreg[rb * G::KJ + j], acc);
                    else {
#pragma unroll
                        for (int c = 0; c < 4; ++c)
                            acc = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(kop[j][c]), __uint_as_float(qreg[rb * G::KJ + j][c]), acc, 0, 0, 0);
                    }
                }
                sacc[rb][tb] = acc;
            }
        }
        bool need = false;
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            float mx = NEG_BIG;
#pragma unroll
            for (int idx = 0; idx < 8; ++idx) {
                s[rb][idx] = band.sees(rb, t0 + slot_token(q, idx)) ? sacc[rb][idx >> 2][idx & 3] : UNSEEN;
                mx = fmaxf(mx, s[rb][idx]);
            }
            mxl[rb] = mx;
            need = need || ((mx < -1.0e29f ? NEG_BIG : mx * sc) > st.m[rb] + LAZY_LOG2);
        }
        if (__builtin_amdgcn_ballot_w64(need) != 0) {
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                const float mx = quarter_max(mxl[rb]);
                const float mxs = mx < -1.0e29f ? NEG_BIG : mx * sc;
                const float mnew = mxs > st.m[rb] + LAZY_LOG2 ? mxs : st.m[rb];
                const float alpha = fast_exp2(st.m[rb] - mnew);
                st.m[rb] = mnew;
                st.l[rb] *= alpha;
                if (!st.fresh) {
#pragma unroll
                    for (int c = 0; c < G::NOC; ++c) st.o[rb][c] *= alpha;
                }
            }
        }
        st.fresh = false;
    }
    float p[RB][8];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const float mref = st.m[rb] < -1.0e29f ? 0.f : st.m[rb];      // (a row that has seen nothing yet: its slots give 0)
        float psum;
#pragma unroll
        for (int idx = 0; idx < 8; ++idx) {
            p[rb][idx] = fast_exp2(__builtin_fmaf(s[rb][idx], sc, -mref));
            psum = idx == 0 ? p[rb][0] : psum + p[rb][idx];
        }
        st.l[rb] += psum;
    }

    bool wild = false;
    if (edge) {                                                       // uniform over the wave
        u32 any = 0;
#pragma unroll
        for (int idx = 0; idx < 8; ++idx)
#pragma unroll
            for (int d = 0; d < G::VW; ++d) any |= Wild<DT>::signs(t.v[idx][d]);
        wild = __builtin_amdgcn_ballot_w64((any & Wild<DT>::SIGNS) != 0) != 0;
    }
    auto products = [&](auto wild_tag) {
        constexpr bool WILD = decltype(wild_tag)::value;
        if constexpr (G::SZ == 2) {
            u32x4 pp[RB], seen[RB];
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                pp[rb] = u32x4{Elem<DT>::pack2(p[rb][0], p[rb][1]), Elem<DT>::pack2(p[rb][2], p[rb][3]), Elem<DT>::pack2(p[rb][4], p[rb][5]),
                               Elem<DT>::pack2(p[rb][6], p[rb][7])};
                if constexpr (WILD) seen[rb] = Wild<DT>::seen(band, rb, t0, q);
            }
#pragma unroll
            for (int c = 0; c < G::NOC; ++c) {
                const int d = c / 2;                                  // dword d of a V row: the lane's elements for accumulators 2d and 2d + 1
                const u32 pick = c % 2 == 0 ? 0x05040100u : 0x07060302u;
                u32x4 v;
                v.x = __builtin_amdgcn_perm(t.v[1][d], t.v[0][d], pick);
                v.y = __builtin_amdgcn_perm(t.v[3][d], t.v[2][d], pick);
                v.z = __builtin_amdgcn_perm(t.v[5][d], t.v[4][d], pick);
                v.w = __builtin_amdgcn_perm(t.v[7][d], t.v[6][d], pick);
                if constexpr (WILD) {
                    u32x4 pos, neg;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        u32 a, b, e;
                        Wild<DT>::split(v[i], a, b, e);
                        v[i] = a;
                        pos[i] = b;
                        neg[i] = e;
                    }
                    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) st.o[rb][c] = Wild<DT>::add(st.o[rb][c], Elem<DT>::mfma(pos, seen[rb], z), Elem<DT>::mfma(neg, seen[rb], z));
                }
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) st.o[rb][c] = Elem<DT>::mfma(v, pp[rb], st.o[rb][c]);
            }
        } else {
#pragma unroll
            for (int c = 0; c < G::NOC; ++c)
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) {
                    [[maybe_unused]] f32x4 pos = {0.f, 0.f, 0.f, 0.f}, neg = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int idx = 0; idx < 8; ++idx) {
                        u32 v = t.v[idx][c];
                        if constexpr (WILD) {
                            const float seen = band.sees(rb, t0 + slot_token(q, idx)) ? 1.0f : 0.f;
                            u32 a, b, e;
                            Wild<DT>::split(v, a, b, e);
                            v = a;
                            pos = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(b), seen, pos, 0, 0, 0);
                            neg = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(e), seen, neg, 0, 0, 0);
                        }
                        st.o[rb][c] = __builtin_amdgcn_mfma_f32_16x16x4f32(__uint_as_float(v), p[rb][idx], st.o[rb][c], 0, 0, 0);
                    }
                    if constexpr (WILD) st.o[rb][c] = Wild<DT>::add(st.o[rb][c], pos, neg);
                }
        }
    };
    if (wild) products(std::true_type{});
    else products(std::false_type{});
}

// Which rows a work item stands for.  Packed queries: the row groups of `rows` rows are numbered through the sequences in order; an item behind
// the last of them is `spare`, of which there is one at least (the grid is sized for more row groups than there can be).
struct WindowItem {
    int w, rg, qs, qe;       // sequence, row group in it, its query tokens
    bool found;
    int spare, spares;       // not found: the how manieth of how many
    int first, end;          // and the query tokens that belong to sequences
};
__device__ __forceinline__ WindowItem window_item(const PagedDevHeader& ph, int rows, int item, int lane, int GQ) {
    WindowItem it = {0, 0, 0, 0, false, 0, 1, 0, 0};
    const int T = ph.LW * ph.LS;
    if (ph.cu_q == nullptr) {
        it.w = fast_div(item, ph.magic_nrg);
        it.rg = item - it.w * ph.nrg;
        it.qs = it.w * ph.LS;
        it.qe = it.qs + ph.LS;
        it.found = true;
        return it;
    }
    auto bound = [&](int x) { return min(max(x, 0), T); };      // a malformed array must not lead outside the buffers
    int base = 0;
    for (int c = 0; c < ph.W && !it.found; c += 64) {
        const int idx = c + lane;
        const int a0 = bound(ph.cu_q[min(idx, ph.W)]), a1 = bound(ph.cu_q[min(idx + 1, ph.W)]);
        const int cnt = idx < ph.W ? (max(a1 - a0, 0) * GQ + rows - 1) / rows : 0;
        const int inc = wave_scan_inclusive(cnt);
        const int total = __builtin_amdgcn_readlane(inc, 63);
        if (item < base + total) {
            const int l0 = __builtin_ctzll(__ballot(base + inc > item));
            it.w = c + l0;
            it.rg = item - base - __builtin_amdgcn_readlane(inc - cnt, l0);
            it.qs = __builtin_amdgcn_readlane(a0, l0);
            it.qe = __builtin_amdgcn_readlane(a1, l0);
            it.found = true;
        }
        base += total;
    }
    if (!it.found) {
        it.spare = item - base;
        it.spares = ph.nitems - base;
        it.first = bound(ph.cu_q[0]);
        it.end = bound(ph.cu_q[ph.W]);
    }
    return it;
}

// SMALL: the K cache is reached through one buffer descriptor (see make_cache_view).
template <class DT, int D, int RB, bool SMALL>
__global__ __launch_bounds__(NTHREADS, 1) void window_kernel(const WindowHeader args) {
    typedef Geo<DT, D, D> G;
    typedef typename Elem<DT>::store_t store_t;
    constexpr int ROWS = RB * 16;
    typedef hw::Exchange<ROWS, D> Ex;
    constexpr int SBYTES = NWAVES * G::KSTAGE;
    __shared__ __attribute__((aligned(16))) char q_lds[ROWS * G::QSTR];
    union Slot0 {
        char k[SBYTES];
        Ex ex;
    };
    __shared__ __attribute__((aligned(16))) Slot0 slot0;
    __shared__ __attribute__((aligned(16))) char slot1[SBYTES];

    const int tid = threadIdx.x;
    const int lane = tid & 63;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int n = lane & 15;
    const int q = lane >> 4;
    char* const kslots[2] = {slot0.k + wv * G::KSTAGE, slot1 + wv * G::KSTAGE};

    PagedHeaderBits hb;
    paged_header_request(hb);
    // K transfer i of a wave covers tile rows i * RPL .. i * RPL + RPL - 1; the bank swizzle is applied on the global side
    constexpr int RPL = 64 / G::CPR;
    const int lrow = lane / G::CPR, lslot = lane % G::CPR;
    auto k_chunk = [&](int i) -> unsigned {
        const int row = i * RPL + lrow;
        const int key = G::CPR >= 16 ? (row & 15) : ((row >> 1) & (G::CPR - 1));
        return (unsigned)((lslot ^ key) << 4);
    };
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
    const bool direct = (ph.flags & PH_DIRECT) != 0;
    [[maybe_unused]] CacheView all;              // the whole K cache
    if constexpr (SMALL) all = make_cache_view(ph, G::KROW);

    // logical workgroup id = ((kv head * nitems) + item) * nsplit + split; consecutive ids share an XCD
    int bid = blockIdx.x;
    if (ph.flags & PH_XCD_REMAP) bid = (bid & 7) * (ph.nwg >> 3) + (bid >> 3);
    const int hi = bid / ph.nsplit, split = bid - hi * ph.nsplit;
    const int hkv = hi / ph.nitems, item = hi - hkv * ph.nitems;
    const int GQ = ph.Hq / ph.Hkv;
    const int T = ph.LW * ph.LS;
    const int cap = ph.block_size * ph.max_blocks;

    const WindowItem it = window_item(ph, ROWS, item, lane, GQ);
    if (!it.found) {                        // uniform over the workgroup: zeros for query tokens that belong to no sequence
        const int before = it.first, rest = before + T - it.end;
        for (int i = it.spare; i < rest; i += it.spares) {
            const int t = i < before ? i : it.end + i - before;
            for (int x = tid; x < GQ * D; x += NTHREADS) {
                const int g = x / D, e = x - g * D;
                if (direct) {
                    const size_t orow = (size_t)t * ph.Hq + hkv * GQ + g;
                    reinterpret_cast<store_t*>(args.out)[orow * D + e] = Elem<DT>::from_float(0.f);
                    if (e == 0 && args.lse != nullptr) args.lse[orow] = -__builtin_inff();
                } else {
                    const size_t prow = (size_t)(hkv * ph.nsplit + split) * ph.R + (size_t)t * GQ + g;
                    ph.part_o[prow * D + e] = 0.f;
                    if (e == 0) *reinterpret_cast<HW_GLOBAL f32x2*>(ph.part_ml + prow * 2) = f32x2{NEG_BIG, 0.f};
                }
            }
        }
        return;
    }
    const int r0 = it.qs * GQ + it.rg * ROWS;    // first row (global numbering: token * GQ + head in group)
    const int rend = it.qe * GQ;
    if (r0 >= rend) return;                      // uniform over the workgroup
    const HW_GLOBAL int* btw = ph.block_table + (size_t)it.w * ph.max_blocks;

    DevHeader a;                                 // what QueryRotation / map_row need, in the [LW, Hq, LS] layout
    a.q = ph.q;
    a.loc = ph.loc;
    a.cos = nullptr;
    a.sin = nullptr;
    a.rq = nullptr;
    a.part_o = ph.part_o;
    a.part_ml = ph.part_ml;
    a.len_dev = nullptr;
    a.F = 1; a.W = ph.LW; a.Hq = ph.Hq; a.Hkv = ph.Hkv; a.S = ph.LS; a.R = rend;
    a.nrg = 1; a.wgs_per_head = ph.nsplit; a.nwg = ph.nwg;
    a.slot_stride = ph.nsplit; a.flags = KH_PREROTATED; a.sc = ph.sc;
    a.magic_gq = ph.magic_gq; a.magic_s = ph.magic_ls; a.magic_nrg = 0; a.magic_wg = 0;

    QueryRotation<DT, D, ROWS, G::QSTR, true> qrot;
    qrot.load(a, 0, hkv, r0, GQ, tid);
    const int NW = ph.nsplit * NWAVES, gw = split * NWAVES + wv;

    // The bounds of the rows (lane l: row l % ROWS; behind the last row, that row again), and of the workgroup: tokens [0, sink_end)
    // and [low, high).
    const int at = ph.loc[fast_div(min(r0 + (lane & (ROWS - 1)), rend - 1), ph.magic_gq)];
    const int lim1 = max(0, at < cap ? at + 1 : cap);
    const int lo1 = max(0, at < 0 ? 0 : at - args.window + 1);
    const int snk1 = min(args.sinks, lim1);
    Band<RB> band;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        band.lo[rb] = RB == 1 ? lo1 : __shfl(lo1, rb * 16 + n, 64);
        band.lim[rb] = RB == 1 ? lim1 : __shfl(lim1, rb * 16 + n, 64);
        band.snk[rb] = RB == 1 ? snk1 : __shfl(snk1, rb * 16 + n, 64);
    }
    const bool any = lo1 < lim1;                 // the row's window holds something
    const int high = wave_max(any ? lim1 : 0);
    const int low = -wave_max(any ? -lo1 : -0x7fffffff);
    const int sink_end = wave_max(snk1);
    const int all_from = wave_max(lo1), all_to = -wave_max(-lim1);                     // what every row's window holds
    const int sink_tiles = (sink_end + TILE - 1) / TILE;
    const int first = high > 0 ? max(low / TILE, sink_tiles) : 0;                    // first tile of the window
    const int tiles = sink_tiles + (high > 0 ? max((high + TILE - 1) / TILE - first, 0) : 0);
    auto tile_at = [&](int k) { return k < sink_tiles ? k : k - sink_tiles + first; };

    // block-table entry of the token this lane stands for in tile t
    auto bt_load = [&](int t) -> int {
        const int tok = min(t * TILE + (lane & 31), cap - 1);
        return btw[fast_div(tok, ph.magic_bs)];
    };
    auto edge = [&](int t) { return !(t * TILE >= all_from && t * TILE + TILE <= all_to); };
    // The loads of tile t, given its table entries: the same number of instructions whether or not the tile exists.  Tokens that no row
    // sees are replaced by one of the tile that some row does (there is one in every tile that exists), so that no byte of the cache
    // that is not seen is read; what a tile that does not exist reads is not used.
    auto issue_tile = [&](TileRegs<DT, D, D>& tr, char* kslot, int btv, int t) {
        const int t0 = t * TILE;
        const int tok_raw = t0 + (lane & 31);
        const int tok = min(tok_raw, cap - 1);
        const int bi = fast_div(tok, ph.magic_bs);
        const int blk = min(max(btv, 0), ph.num_blocks - 1);
        int rid = (blk * ph.Hkv + hkv) * ph.block_size + (tok - bi * ph.block_size);
        const int last = t0 + TILE > low && high > 0 ? high : sink_end;
        const int jstar = min(max(last - 1 - t0, 0), TILE - 1);
        const int rstar = __builtin_amdgcn_readlane(rid, jstar);
        rid = tok_raw < sink_end || (tok_raw >= low && tok_raw < high) ? rid : rstar;
        asm volatile("" ::: "memory");   // the transfers keep their place between the reads of the slot (see load_tile)
#pragma unroll
        for (int i = 0; i < G::KL; ++i) {
            const int r = __shfl(rid, i * RPL + lrow, 64);
            if constexpr (SMALL) {
                cache_transfer<HW_KV_AUX>(all, kslot + i * 1024, (unsigned)r * G::KROW + k_chunk(i));
            } else {
                const HW_GLOBAL char* src = ph.kcache + (unsigned long long)(unsigned)r * G::KROW + k_chunk(i);
                __builtin_amdgcn_global_load_lds(src, HW_LDS_PTR(kslot + i * 1024), 16, 0, HW_KV_AUX);
            }
        }
        asm volatile("" ::: "memory");
#pragma unroll
        for (int idx = 0; idx < 8; ++idx) {
            const int r = __shfl(rid, slot_token(q, idx), 64);
            const HW_GLOBAL char* src = ph.vcache + (unsigned long long)(unsigned)r * G::VROW + n * (G::VLD * 4);
#pragma unroll
            for (int hh = 0; hh < G::NVL; ++hh) {
                if constexpr (G::VLD == 4) {
                    const u32x4 x = __builtin_nontemporal_load(reinterpret_cast<const HW_GLOBAL u32x4*>(src + hh * 256));
                    tr.v[idx][hh * 4 + 0] = x.x;
                    tr.v[idx][hh * 4 + 1] = x.y;
                    tr.v[idx][hh * 4 + 2] = x.z;
                    tr.v[idx][hh * 4 + 3] = x.w;
                } else {
                    const u32x2 x = __builtin_nontemporal_load(reinterpret_cast<const HW_GLOBAL u32x2*>(src));
                    tr.v[idx][0] = x.x;
                    tr.v[idx][1] = x.y;
                }
            }
        }
    };

    int bt_a = bt_load(tile_at(gw)), bt_b = bt_load(tile_at(gw + NW));
    TileRegs<DT, D, D> tr[2];
    issue_tile(tr[0], kslots[0], bt_a, tile_at(gw));
    qrot.finish(a, q_lds, 0, hkv, r0, GQ, false, tid);
    lds_barrier();
    u32x4 qreg[RB * G::KJ];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb)
#pragma unroll
        for (int j = 0; j < G::KJ; ++j)
            qreg[rb * G::KJ + j] = *reinterpret_cast<const u32x4*>(q_lds + (rb * 16 + n) * G::QSTR + (4 * j + q) * 16);

    // Two tiles in flight per wave: request the table entries two tiles ahead, then the next tile, then compute the current one.  The last one or
    // two tiles are outside of the loop, where nothing is requested any more (this kernel alone, traced: 4 tokens of 4 sequences that see 2048
    // 15.0 -> 14.2 us, 5 ragged ones at 256 channels 14.2 -> 13.3; a third tile in flight instead: 5 % more than without).
    int k = gw;
    for (; k + 2 * NW < tiles; k += 2 * NW) {
        {
            const int bt_n = bt_load(tile_at(k + 2 * NW));
            issue_tile(tr[1], kslots[1], bt_b, tile_at(k + NW));
            wait_k_landed<G, 1>();
            band_tile<DT, D, RB>(tr[0], qreg, band, st, tile_at(k) * TILE, n, q, ph.sc, kslots[0], edge(tile_at(k)));
            bt_a = bt_n;
        }
        {
            const int bt_n = bt_load(tile_at(k + 3 * NW));
            issue_tile(tr[0], kslots[0], bt_a, tile_at(k + 2 * NW));
            wait_k_landed<G, 1>();
            band_tile<DT, D, RB>(tr[1], qreg, band, st, tile_at(k + NW) * TILE, n, q, ph.sc, kslots[1], edge(tile_at(k + NW)));
            bt_b = bt_n;
        }
    }
    if (k < tiles) {
        const bool two = k + NW < tiles;                             // (uniform over the wave)
        if (two) {
            issue_tile(tr[1], kslots[1], bt_b, tile_at(k + NW));
            wait_k_landed<G, 1>();
        } else wait_k_landed<G, 0>();
        band_tile<DT, D, RB>(tr[0], qreg, band, st, tile_at(k) * TILE, n, q, ph.sc, kslots[0], edge(tile_at(k)));
        if (two) {
            wait_k_landed<G, 0>();
            band_tile<DT, D, RB>(tr[1], qreg, band, st, tile_at(k + NW) * TILE, n, q, ph.sc, kslots[1], edge(tile_at(k + NW)));
        }
    }

    size_t orow[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) orow[rb] = map_row(a, min(r0 + rb * 16 + n, rend - 1), hkv, GQ).qrow;
    store_partials<DT, D, RB, true>(st, slot0.ex, wv, n, q, tid,
                                    direct ? reinterpret_cast<HW_GLOBAL float*>(reinterpret_cast<unsigned long long>(args.out)) : ph.part_o,
                                    direct ? reinterpret_cast<HW_GLOBAL float*>(reinterpret_cast<unsigned long long>(args.lse)) : ph.part_ml,
                                    (size_t)(hkv * ph.nsplit + split) * ph.R + r0, min(ROWS, rend - r0), direct, orow);
}

// ---- many rows -------------------------------------------------------------------------------------------------------------------
//
// Row groups of `rows` rows of one sequence (a last one of fewer), numbered through the sequences, `all` of them for every kv head.  The n
// workgroups of a head take q = all / n whole groups each, every n-th one (so that a prompt among sequences that decode falls to many: 60 of
// those and 512 tokens 261 -> 251 us, the prompt in front 230), and share the rest of them out.  Many of them (more than a third of n) evenly, in
// the order of the rows: workgroup i takes the stretch [i rest / n, (i + 1) rest / n), and a part of a group is that part of its tiles.  Few
// of them have workgroups to themselves, as many as their tiles and rows ask for (1, 8, 32 and 64 tokens behind 4096 at 40/8 heads: 48 -> 37 us),
// since a second opening in a workgroup costs as much as eleven tiles.  A workgroup that sees a whole group writes its result; parts leave partial
// sums in the workgroup's two slots (its first group's, and its last one's), which window_merge_kernel adds up.
//
// What bounds it (128 channels, 256 CUs at 2.0 GHz): a step of two tiles takes 2.2 us with 256 rows (0.95 PFLOP/s), 1.8 with 160, 1.2 with 64
// and fewer (the loads: 27 GB/s a CU).  Matrix products, exponentials with the rest of the softmax, and LDS reads are a microsecond each of
// the 2.2; leaving any one out saves a tenth, taking the logits a tile ahead 1 %.  Around the steps 6 us before the first one (row positions,
// table entries, tiles: a chain of loads), 1 to 3 of results or partial sums, 4 to 7 of the merge.  1024 tokens on 5120 that see 2048, 40/8 heads: 66 us
// a layer, 0.65 PFLOP/s.

constexpr int VMCNT_0 = 0x0f70;          // s_waitcnt: no vector memory operation outstanding, the other counters as they are

struct Deal {
    int all, whole, rest;                // row groups of a kv head; whole ones of a workgroup; what is shared out
    bool apart;                          // the latter have workgroups to themselves
    // the first 64 sequences, one a lane: their query tokens, row groups, and the groups up to and with them
    int qs, qe, count, upto;
    int first, parts;                    // apart: lane g, the workgroups of the g-th of the groups shared out
};
typedef int i32x4 __attribute__((ext_vector_type(4)));
__device__ __forceinline__ HW_GLOBAL i32x4* cuts_of(const WindowHeader& args, int hkv) {
    return reinterpret_cast<HW_GLOBAL i32x4*>(reinterpret_cast<unsigned long long>(args.cuts)) + (size_t)hkv * (args.most_cuts + 1);
}
__device__ __forceinline__ int bounded(int x, int T) { return min(max(x, 0), T); }        // a malformed array must not lead outside the buffers
__device__ __forceinline__ Deal window_deal(const WindowHeader& args, const PagedDevHeader& ph, int n, int lane, int GQ) {
    Deal d = {0, 0, 0, false, 0, 0, 0, 0, 0, 0};
    const int rows = args.rows, T = ph.LW * ph.LS;
    if (ph.cu_q == nullptr) d.all = ph.W * ph.nrg;
    else {
        for (int c = 0; c < ph.W; c += 64) {
            const int idx = c + lane;
            const int a0 = bounded(ph.cu_q[min(idx, ph.W)], T), a1 = bounded(ph.cu_q[min(idx + 1, ph.W)], T);
            const int cnt = idx < ph.W ? (max(a1 - a0, 0) * GQ + rows - 1) / rows : 0;
            const int inc = wave_scan_inclusive(cnt);
            if (c == 0) {
                d.qs = a0;
                d.qe = a1;
                d.count = cnt;
                d.upto = inc;
            }
            d.all += __builtin_amdgcn_readlane(inc, 63);
        }
    }
    d.whole = d.all / n;
    d.rest = d.all - d.whole * n;
    // (almost a group each: whole ones to as many workgroups take about as long, and nothing is left to merge)
    if (d.rest * 8 > n * 7) {
        ++d.whole;
        d.rest = 0;
    }
    if (d.rest == 0 || d.rest * 3 > n || d.rest > 64) return d;
    d.apart = true;
    int cost = 1;                                        // lane g: what the g-th of them costs
    if (ph.cu_q == nullptr || ph.W <= 64) {
        const int g = d.whole * n + min(lane, d.rest - 1);
        int qs, qe, rg;
        if (ph.cu_q == nullptr) {
            const int w = fast_div(g, ph.magic_nrg);
            qs = w * ph.LS;
            qe = qs + ph.LS;
            rg = g - w * ph.nrg;
        } else {
            int w = 0;                                   // the first sequence with more groups up to and with it
#pragma unroll
            for (int step = 32; step > 0; step >>= 1) w += __shfl(d.upto, w + step - 1, 64) <= g ? step : 0;
            qs = __shfl(d.qs, w, 64);
            qe = __shfl(d.qe, w, 64);
            rg = g - __shfl(d.upto - d.count, w, 64);
        }
        const int here = min((qe - qs) * GQ - rg * rows, rows);
        // the tiles that its last row sees, about, in fifths of a microsecond a step of two: with up to four row blocks as long as it needs to come
        // in, with four to a SIMD eleven; and an opening
        const int at = min(ph.loc[min(max(qs + (rg * rows + here - 1) / GQ, 0), T - 1)], ph.block_size * ph.max_blocks - 1);
        const int seen = at < 0 ? 0 : at < args.window ? at : args.window + min(args.sinks, at - args.window);
        cost = (seen / TILE + 11) * max(6, 3 + (here + 63) / 64 * 2);
    }
    // The least time t in which they are done with n workgroups, ceil(cost / t) for each: between the sum over n and over n - rest, where they
    // are enough in any case (n - rest is 2/3 n and more; the thousandth is for the roundings).
    const float mine = lane < d.rest ? (float)cost : 0.f;
    auto parts_in = [&](float t) { return (int)__builtin_ceilf(mine * __builtin_amdgcn_rcpf(t)); };
    const float sum = (float)__builtin_amdgcn_readlane(wave_scan_inclusive(lane < d.rest ? cost : 0), 63);
    float no = sum * __builtin_amdgcn_rcpf((float)n), yes = sum * __builtin_amdgcn_rcpf((float)(n - d.rest)) * 1.001f;
#pragma unroll 1
    for (int i = 0; i < 6; ++i) {
        const float t = 0.5f * (no + yes);
        if (__builtin_amdgcn_readlane(wave_scan_inclusive(parts_in(t)), 63) <= n) yes = t;
        else no = t;
    }
    d.parts = parts_in(yes);
    d.first = wave_scan_inclusive(d.parts) - d.parts;
    return d;
}
// Row group g < all: sequence, number in it, query tokens.
struct WindowGroup {
    int w, rg, qs, qe;
};
__device__ __forceinline__ WindowGroup window_group(const PagedDevHeader& ph, const Deal& d, int rows, int g, int lane, int GQ) {
    WindowGroup r;
    if (ph.cu_q != nullptr && ph.W <= 64) {
        r.w = __builtin_ctzll(__ballot(d.upto > g));
        r.rg = g - __builtin_amdgcn_readlane(d.upto - d.count, r.w);
        r.qs = __builtin_amdgcn_readlane(d.qs, r.w);
        r.qe = __builtin_amdgcn_readlane(d.qe, r.w);
    } else {
        const WindowItem it = window_item(ph, rows, g, lane, GQ);
        r.w = it.w;
        r.rg = it.rg;
        r.qs = it.qs;
        r.qe = it.qe;
    }
    return r;
}

// One 32-token tile, K and V images in LDS, against the wave's RB * 16 rows.  MASKED: some row may not see all of it.
template <class DT, int D, int RB, bool MASKED>
__device__ __forceinline__ void band_tile_lds(const u32x4* qreg, const Band<RB>& band, WaveState<RB, D / 16>& st, int t0, int n, int q, float sc,
                                              const char* kstage, const char* vimg, const unsigned* voff, bool edge) {
    typedef Geo<DT, D, D> G;
    constexpr float LAZY_LOG2 = 8.0f;
    f32x4 sacc[RB][2];
    {
        u32x4 kop[2][G::KJ];
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int j = 0; j < G::KJ; ++j) kop[tb][j] = *reinterpret_cast<const u32x4*>(kstage + kstage_offset<G>(tb * 16 + n, 4 * j + q));
#pragma unroll
        for (int tb = 0; tb < 2; ++tb)
#pragma unroll
            for (int rb = 0; rb < RB; ++rb) {
                f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int j = 0; j < G::KJ; ++j) acc = Elem<DT>::mfma(kop[tb][j], qreg[rb * G::KJ + j], acc);
                sacc[rb][tb] = acc;
            }
    }
    // the V^T operands, requested here: LDS answers while the exponentials are taken
    u32x4 vops[G::NOC];
#pragma unroll
    for (int c = 0; c < G::NOC; ++c) {
        const char* vp = vimg + voff[c];
        const u32x2 a0 = lds_read_tr16(vp), a1 = lds_read_tr16(vp + 16 * G::VROW);
        vops[c] = u32x4{a0.x, a0.y, a1.x, a1.y};     // tokens slot_token(q, 0..7) of element 16c + n
    }
    __builtin_amdgcn_sched_barrier(0);
    float s[RB][8], mxl[RB];
    bool need = false;
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        float mx = NEG_BIG;
        // (counted from the lane's first token: one subtraction and two comparisons a logit)
        const int base = t0 + slot_token(q, 0);
        [[maybe_unused]] const unsigned from = MASKED ? band.lo[rb] - base : 0, len = MASKED ? max(band.lim[rb] - band.lo[rb], 0) : 0;
        [[maybe_unused]] const int sink = MASKED ? band.snk[rb] - base : 0;
#pragma unroll
        for (int idx = 0; idx < 8; ++idx) {
            s[rb][idx] = sacc[rb][idx >> 2][idx & 3];
            if constexpr (MASKED) s[rb][idx] = (unsigned)slot_token(0, idx) - from < len || slot_token(0, idx) < sink ? s[rb][idx] : UNSEEN;
            mx = fmaxf(mx, s[rb][idx]);
        }
        mxl[rb] = mx;
        const float mine = MASKED ? (mx < -1.0e29f ? NEG_BIG : mx * sc) : mx * sc;
        need = need || (mine > st.m[rb] + LAZY_LOG2);
    }
    if (__builtin_amdgcn_ballot_w64(need) != 0) {
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) {
            const float mx = quarter_max(mxl[rb]);
            const float mxs = MASKED ? (mx < -1.0e29f ? NEG_BIG : mx * sc) : mx * sc;
            const float mnew = mxs > st.m[rb] + LAZY_LOG2 ? mxs : st.m[rb];
            const float alpha = fast_exp2(st.m[rb] - mnew);
            st.m[rb] = mnew;
            st.l[rb] *= alpha;
            if (!st.fresh) {
#pragma unroll
                for (int c = 0; c < G::NOC; ++c) st.o[rb][c] *= alpha;
            }
        }
    }
    st.fresh = false;
    u32x4 pp[RB];
#pragma unroll
    for (int rb = 0; rb < RB; ++rb) {
        const float mref = MASKED ? (st.m[rb] < -1.0e29f ? 0.f : st.m[rb]) : st.m[rb];
        float p[8], psum;
#pragma unroll
        for (int idx = 0; idx < 8; ++idx) {
            p[idx] = fast_exp2(__builtin_fmaf(s[rb][idx], sc, -mref));
            psum = idx == 0 ? p[0] : psum + p[idx];
        }
        st.l[rb] += psum;
        pp[rb] = u32x4{Elem<DT>::pack2(p[0], p[1]), Elem<DT>::pack2(p[2], p[3]), Elem<DT>::pack2(p[4], p[5]), Elem<DT>::pack2(p[6], p[7])};
    }
    if constexpr (MASKED) {
        if (edge) {                                                   // uniform over the wave
            // (nothing times them all: NaN where one is infinite or NaN; the matrix unit has time for it here, 32 registers looked at have not)
            f32x4 any[2] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
#pragma unroll
            for (int c = 0; c < G::NOC; ++c) any[c & 1] = Elem<DT>::mfma(vops[c], u32x4{0, 0, 0, 0}, any[c & 1]);
            const float sum = (any[0][0] + any[0][1] + any[0][2] + any[0][3]) + (any[1][0] + any[1][1] + any[1][2] + any[1][3]);
            if (__builtin_amdgcn_ballot_w64(sum != 0.f) != 0) {
                u32x4 seen[RB];
#pragma unroll
                for (int rb = 0; rb < RB; ++rb) seen[rb] = Wild<DT>::seen(band, rb, t0, q);
#pragma unroll
                for (int c = 0; c < G::NOC; ++c) {
                    u32x4 pos, neg;
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        u32 x, y, z;
                        Wild<DT>::split(vops[c][i], x, y, z);
                        vops[c][i] = x;
                        pos[i] = y;
                        neg[i] = z;
                    }
                    const f32x4 z = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int rb = 0; rb < RB; ++rb) st.o[rb][c] = Wild<DT>::add(st.o[rb][c], Elem<DT>::mfma(pos, seen[rb], z), Elem<DT>::mfma(neg, seen[rb], z));
                }
            }
        }
    }
#pragma unroll
    for (int c = 0; c < G::NOC; ++c)
#pragma unroll
        for (int rb = 0; rb < RB; ++rb) st.o[rb][c] = Elem<DT>::mfma(vops[c], pp[rb], st.o[rb][c]);
}

// NW waves of up to 32 rows each, two 16-row blocks NW blocks apart, which all take every tile of the group.  A tile comes into LDS once per workgroup, into a ring of NS slots in steps
// of TS tiles with one barrier each: a wave waits for its own transfers of the step, all waves meet, the step is complete, and the slots of
// the step before are free for the request behind the barrier.  The sequence's table entries come the same way: every wave brings those of
// the 32 tokens of the tiles of a step into a small ring of its own, one transfer a step, DP steps before it forms the addresses.  (A window
// may lie anywhere in a table of any length.)
template <class DT, int D, int NS, int NW, int TS>
__global__ __launch_bounds__(NW * 64, 1) void window_wide_kernel(const WindowHeader args) {
    typedef Geo<DT, D, D> G;
    typedef typename Elem<DT>::store_t store_t;
    constexpr int NT = NW * 64, ROWS = NW * 32;  // (rows of a group, at most)
    constexpr int NSTEP = NS / TS, DP = NSTEP - 1;
    constexpr int KBYTES = G::KSTAGE, VBYTES = TILE * G::VROW, SLOT = KBYTES + VBYTES;
    constexpr int TPW = SLOT / 1024 / NW;        // 1 KB transfers of a wave per tile
    constexpr int TPS = TS * TPW;
    constexpr int RPL = 64 / G::CPR;
    constexpr int ER = 2 * DP + 1;               // steps of table entries in a wave's ring
    static_assert(G::SZ == 2 && KBYTES == VBYTES && TPW >= 1 && NS % TS == 0 && DP >= 1 && (TS == 1 || TS == 2), "16-bit types");
    constexpr int OSTR = D + 4;                  // floats of a row on its way out
    static_assert(NW * 16 * OSTR * 4 <= NS * SLOT, "16 rows of every wave fit into the ring");
    __shared__ int entries[NW][ER][64];
    __shared__ __attribute__((aligned(16))) char ring[NS * SLOT];

    const int tid = threadIdx.x;
    const int wv = __builtin_amdgcn_readfirstlane(tid >> 6);

    PagedHeaderBits hb;
    paged_header_request(hb);
    // this wave's transfers of a tile: with an even number of them the same rows of both images (one look-up serves both), otherwise the first
    // half of the waves brings K, the second half V
    constexpr bool BOTH = TPW % 2 == 0;
    constexpr int NI = BOTH ? 2 : 1, NP = TPW / NI;
    static_assert((KBYTES / 1024) % NP == 0 && NW * NP * NI * 1024 == SLOT, "the waves' pieces tile both images");
    const bool k_wave = BOTH || wv < NW / 2;
    const int piece0 = (BOTH ? wv : (k_wave ? wv : wv - NW / 2)) * NP;
    unsigned my_image[NI];
    my_image[0] = lds_address(ring) + (k_wave ? 0 : KBYTES) + piece0 * 1024;
    if constexpr (BOTH) my_image[1] = my_image[0] + KBYTES;
    const unsigned my_entries = __builtin_amdgcn_readfirstlane(lds_address(entries) + wv * ER * 256);
    const PagedDevHeader ph = paged_header_wait(hb);

    int bid = blockIdx.x;                        // kv head * nsplit + workgroup of the head; consecutive ids share an XCD
    if (ph.flags & PH_XCD_REMAP) bid = (bid & 7) * (ph.nwg >> 3) + (bid >> 3);
    const int N = ph.nsplit;
    const int hkv = bid / N, me = bid - hkv * N;
    const int GQ = ph.Hq / ph.Hkv;
    const int T = ph.LW * ph.LS;
    const int cap = ph.block_size * ph.max_blocks;
    const int rows = args.rows;
    const Deal deal = window_deal(args, ph, N, tid & 63, GQ);
    unsigned long long image[NI];
    image[0] = reinterpret_cast<unsigned long long>(k_wave ? ph.kcache : ph.vcache);
    if constexpr (BOTH) image[1] = reinterpret_cast<unsigned long long>(ph.vcache);

    DevHeader a;                                 // what map_row needs, in the [LW, Hq, LS] layout
    a.Hq = ph.Hq; a.S = ph.LS;
    a.magic_gq = ph.magic_gq; a.magic_s = ph.magic_ls;

    int begin = me * deal.rest, end = begin + deal.rest, den = N;                     // the stretch, in den-ths of a group
    int part0 = begin / N, parts = deal.rest > 0 ? (end + N - 1) / N - part0 : 0;     // its groups
    if (deal.apart) {
        const unsigned long long owner = __ballot((tid & 63) < deal.rest && me >= deal.first && me < deal.first + deal.parts);
        parts = owner != 0 ? 1 : 0;
        part0 = owner != 0 ? __builtin_ctzll(owner) : 0;
        den = max(__builtin_amdgcn_readlane(deal.parts, part0), 1);
        begin = part0 * den + me - __builtin_amdgcn_readlane(deal.first, part0);
        end = begin + 1;
    }
    // word for window_merge_kernel: how many groups are shared out and how
    HW_GLOBAL i32x4* const cuts = cuts_of(args, hkv);
    if (N > 1 && me == 0 && tid == 0) cuts[0] = i32x4{deal.rest, deal.apart ? 1 : 0, 0, 0};
    for (int item = 0; item < deal.whole + parts; ++item) {
        const bool whole_one = item < deal.whole;
        const int cut = part0 + item - deal.whole;               // a part: of this one of the groups that are shared out
        const int g = whole_one ? item * N + me : N * deal.whole + cut;
        if (g >= deal.all) break;                                 // (the last workgroups, where almost a group each was left)
        const int from = whole_one ? 0 : max(begin - cut * den, 0), to = whole_one ? den : min(end - cut * den, den);
        const WindowGroup it = window_group(ph, deal, rows, g, tid & 63, GQ);
        const int r0 = it.qs * GQ + it.rg * rows, rend = min(it.qe * GQ, r0 + rows);
        const bool whole = from == 0 && to == den;
        if (!whole_one && from == 0 && tid == 0 && cut < args.most_cuts)        // which workgroups have it, and its rows
            cuts[cut + 1] = i32x4{me, deal.apart ? me + den - 1 : ((cut + 1) * N - 1) / deal.rest, r0, rend};
        const size_t pbase = ((size_t)hkv * 2 * N + 2 * me + (cut == part0 ? 0 : 1)) * ROWS;
        const HW_GLOBAL int* btw = ph.block_table + (size_t)it.w * ph.max_blocks;

        auto run = [&](auto rbx) {
            constexpr int RBX = decltype(rbx)::value;
            const int w0 = r0 + wv * 16;                 // the wave's first row; row block rb begins at w0 + rb * BLOCK
            constexpr int BLOCK = NW * 16;
            // (the lane as the compiler cannot see through it: what follows from it is formed here, per group, and does not stay in
            // registers through the tile loops of the other form, which have none to spare)
            int lane = tid & 63;
            asm volatile("" : "+v"(lane));
            const int n = lane & 15, q = lane >> 4;
            // the rows' positions (behind the last row, that row again): lane l rows l, 64 + l, ... of the group, and one of the wave's
            int at[ROWS / 64];
#pragma unroll
            for (int i = 0; i < ROWS / 64; ++i) at[i] = ph.loc[fast_div(min(r0 + 64 * i + lane, rend - 1), ph.magic_gq)];
            const int at_own = ph.loc[fast_div(min(w0 + n + (RBX == 1 ? 0 : (q & 1) * BLOCK), rend - 1), ph.magic_gq)];
            u32x4 qreg[RBX * G::KJ];
#pragma unroll
            for (int rb = 0; rb < RBX; ++rb) {
                const HW_GLOBAL char* qp = ph.q + map_row(a, min(w0 + rb * BLOCK + n, rend - 1), hkv, GQ).qrow * G::KROW;
#pragma unroll
                for (int j = 0; j < G::KJ; ++j) qreg[rb * G::KJ + j] = *reinterpret_cast<const HW_GLOBAL u32x4*>(qp + (4 * j + q) * 16);
            }
            const int lrow = lane / G::CPR, lslot = lane % G::CPR;
            unsigned chunk[NI][NP];                      // byte offset of the lane's 16 bytes in its row, by image and piece
            int trow[NP];                                // the tile row it belongs to
#pragma unroll
            for (int j = 0; j < NP; ++j) {
                const int row = (piece0 + j) * RPL + lrow;
                const int key = G::CPR >= 16 ? (row & 15) : ((row >> 1) & (G::CPR - 1));
                const unsigned kchunk = (unsigned)((lslot ^ key) << 4), vchunk = (unsigned)((lslot ^ (2 * vimg_segment_key<G::VROW>(row))) << 4);
                trow[j] = row;
                chunk[0][j] = k_wave ? kchunk : vchunk;
                if constexpr (BOTH) chunk[1][j] = vchunk;
            }
            unsigned voff[G::NOC];
            vtr_lane_offsets<G::VROW>(voff, lane);
            auto lim_of = [&](int x) { return max(0, x < cap ? x + 1 : cap); };
            auto lo_of = [&](int x) { return min(max(0, x < 0 ? 0 : x - args.window + 1), cap); };       // (so that it can be rounded up to tiles)
            int top = 0, bottom = -0x7fffffff, most = 0, above = 0, least = -0x7fffffff;
#pragma unroll
            for (int i = 0; i < ROWS / 64; ++i) {
                const int lim = lim_of(at[i]), lo = lo_of(at[i]);
                const bool any = lo < lim;               // the row's window holds something
                top = max(top, any ? lim : 0);
                bottom = max(bottom, any ? -lo : -0x7fffffff);
                most = max(most, lim);
                above = max(above, lo);
                least = max(least, -lim);
            }
            const int high = wave_max(top), low = -wave_max(bottom);                   // the windows of the group lie in [low, high)
            const int sink_end = min(args.sinks, wave_max(most));
            const int all_from = wave_max(above), all_to = -wave_max(least);           // what every row's window holds
            // the same of the wave's own rows
            const int own_high = wave_max(lo_of(at_own) < lim_of(at_own) ? lim_of(at_own) : 0), own_low = -wave_max(lo_of(at_own) < lim_of(at_own) ? -lo_of(at_own) : -0x7fffffff);
            const int own_from = wave_max(lo_of(at_own)), own_to = -wave_max(-lim_of(at_own)), own_sinks = min(args.sinks, wave_max(lim_of(at_own)));
            Band<RBX> band;
#pragma unroll
            for (int rb = 0; rb < RBX; ++rb) {
                const int x = RBX == 1 ? at_own : __shfl(at_own, rb * 16 + n, 64);
                band.lim[rb] = lim_of(x);
                band.lo[rb] = lo_of(x);
                band.snk[rb] = min(args.sinks, band.lim[rb]);
            }
            // Tiles: of the sinks, then of the windows; of them every row sees those numbered full0 .. full1 - 1 completely, which are taken last.
            const int sink_tiles = (sink_end + TILE - 1) / TILE;
            const int first = high > 0 ? max(low / TILE, sink_tiles) : 0, tiles = sink_tiles + (high > 0 ? max((high + TILE - 1) / TILE - first, 0) : 0);
            const int jump = first - sink_tiles;
            const int full0 = min(max((all_from + TILE - 1) / TILE - jump, sink_tiles), tiles), full1 = min(max(all_to / TILE - jump, full0), tiles);
            const int part = tiles - (full1 - full0);
            auto tile_at = [&](int k) {
                const int x = k + (k >= full0 ? full1 - full0 : 0) - (k >= part ? tiles - full0 : 0);
                return x + (x >= sink_tiles ? jump : 0);
            };
            // (a tile that is not seen completely takes half as long again as another)
            const int weight = 2 * tiles + part;
            auto tile_of = [&](int x) { return x <= 3 * part ? x / 3 : part + (x - 3 * part) / 2; };
            const int k0 = tile_of(weight * from / den), k1 = tile_of(weight * to / den);

            WaveState<RBX, G::NOC> st;
#pragma unroll
            for (int rb = 0; rb < RBX; ++rb) {
                st.m[rb] = NEG_BIG;
                st.l[rb] = 0.f;
#pragma unroll
                for (int c = 0; c < G::NOC; ++c) st.o[rb][c] = f32x4{0.f, 0.f, 0.f, 0.f};
            }
            st.fresh = true;

            if (k0 < k1) {                                            // uniform over the workgroup
                // the table entries of step s: lanes 0..31 those of its first tile's tokens, 32..63 of its second's
                auto request_entries = [&](int s, int slot) {
                    const int t = tile_at(k0 + s * TS + (TS - 1) * (lane >> 5));
                    const int tok = min(t * TILE + (lane & 31), cap - 1);
                    lds_transfer_flat<true, true>(__builtin_amdgcn_readfirstlane(my_entries + slot * 256), reinterpret_cast<unsigned long long>(btw + fast_div(tok, ph.magic_bs)));
                };
                // Source addresses of this wave's transfers of step s.  Tokens that no row sees are replaced by one of the tile that some row
                // sees; what a tile that does not exist reads is not used.  (Without branches: they would cut the tile loops into pieces.)
                auto addresses = [&](unsigned long long* src, int s, int slot) {
                    const int* ent = &entries[wv][slot][0];
#pragma unroll
                    for (int pp = 0; pp < TS; ++pp) {
                        const int t0 = tile_at(k0 + s * TS + pp) * TILE;
                        const bool windows = t0 + TILE > low && high > 0;             // (uniform)
                        const int lowest = windows ? low : sink_end - 1, highest = windows ? high - 1 : sink_end - 1;
#pragma unroll
                        for (int j = 0; j < NP; ++j) {
                            const int raw = t0 + trow[j];
                            const int moved = min(max(min(max(raw, lowest), highest) - t0, 0), TILE - 1);
                            const int tr = raw < sink_end ? trow[j] : moved;
                            const int tok = min(t0 + tr, cap - 1);
                            const int bi = fast_div(tok, ph.magic_bs);
                            const int blk = min(max(ent[pp * 32 + tr], 0), ph.num_blocks - 1);
                            const int rid = (blk * ph.Hkv + hkv) * ph.block_size + (tok - bi * ph.block_size);
#pragma unroll
                            for (int im = 0; im < NI; ++im) src[(pp * NP + j) * NI + im] = image[im] + (unsigned long long)(unsigned)rid * G::KROW + chunk[im][j];
                        }
                    }
                };
                auto request = [&](int step_slot, const unsigned long long* src) {
#pragma unroll
                    for (int pp = 0; pp < TS; ++pp)
#pragma unroll
                        for (int j = 0; j < NP; ++j)
#pragma unroll
                            for (int im = 0; im < NI; ++im)
                                lds_transfer_flat<true>(__builtin_amdgcn_readfirstlane(my_image[im] + (step_slot * TS + pp) * SLOT + j * 1024), src[(pp * NP + j) * NI + im]);
                };
                // Step i requests the entries of step i + 2 DP + 1 and the tiles of step i + DP, in this order, and forms the addresses of
                // step i + DP + 1 from the entries that step i - DP requested.  Steps -DP .. -1 here.
#pragma unroll
                for (int i = 0; i <= DP; ++i) request_entries(i, i);
                // (queries and positions as well; stated so that the compiler sees it: it would place its own wait for the queries where they
                // are used, inside the tile loops, and there it would also wait for the tiles in flight)
                __builtin_amdgcn_s_waitcnt(VMCNT_0);
                asm volatile("" ::: "memory");
                unsigned long long src[TPS];
                __syncthreads();                                      // everybody is done with the ring (the group before)
#pragma unroll
                for (int i = 0; i < DP; ++i) {
                    addresses(src, i, i);
                    request_entries(i + DP + 1, i + DP + 1);
                    request(i, src);
                }
                addresses(src, DP, DP);
                int sl = 0, es = 0, step = 0;                         // ring slots of this step's tiles and entries
                auto arrive = [&]() {
                    // this wave's transfers of the step have landed (loads complete in order; those of the DP - 1 steps since may be
                    // in flight), then every wave's; and every wave has left the step before, whose slots are free
                    asm volatile("s_waitcnt vmcnt(%0)\n\ts_barrier" ::"n"((DP - 1) * (TPS + 1)) : "memory");
                    request_entries(step + 2 * DP + 1, es);
                    request(sl == 0 ? NSTEP - 1 : sl - 1, src);
                    int es1 = es + DP + 1;
                    es1 = es1 >= ER ? es1 - ER : es1;
                    addresses(src, step + DP + 1, es1);
                };
                auto next = [&]() {
                    sl = sl + 1 == NSTEP ? 0 : sl + 1;
                    es = es + 1 == ER ? 0 : es + 1;
                    ++step;
                };
                // One instantiation of the arithmetic for tiles that some row may not see all of and one for the others, in loops of their
                // own (a step with both kinds, and a last one of one tile, are the first loop's).
                const bool live = w0 < rend;                          // (a wave without rows only takes part in the barriers)
                int k = k0;
                auto partly = [&]() {
                    arrive();
                    if (live) {
#pragma unroll 1
                        for (int pp = 0; pp < TS; ++pp) {
                            const int t0 = tile_at(k + pp) * TILE;
                            // (nothing of the tile is seen by the wave)
                            if (k + pp >= k1 || !(t0 < own_sinks || (t0 < own_high && t0 + TILE > own_low))) continue;
                            const char* slot = ring + (sl * TS + pp) * SLOT;
                            band_tile_lds<DT, D, RBX, true>(qreg, band, st, t0, n, q, ph.sc, slot, slot + KBYTES, voff,
                                                            !(t0 >= own_from && t0 + TILE <= own_to));
                        }
                    }
                    next();
                    k += TS;
                };
#pragma unroll 1
                while (k < k1 && k < part) partly();
                if (live) {
#pragma unroll 1
                    for (; k + TS <= k1; k += TS) {
                        arrive();
#pragma unroll 1
                        for (int pp = 0; pp < TS; ++pp) {
                            const char* slot = ring + (sl * TS + pp) * SLOT;
                            band_tile_lds<DT, D, RBX, false>(qreg, band, st, 0, n, q, ph.sc, slot, slot + KBYTES, voff, false);
                        }
                        next();
                    }
                    if (k < k1) {
                        arrive();
                        const char* slot = ring + sl * TS * SLOT;
                        band_tile_lds<DT, D, RBX, false>(qreg, band, st, 0, n, q, ph.sc, slot, slot + KBYTES, voff, false);
                    }
                } else {
#pragma unroll 1
                    for (; k < k1; k += TS) {
                        arrive();
                        next();
                    }
                }
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");      // the requests behind the last tile, before the ring is used again
            }

            // every wave stores its rows, staged through LDS so that they leave whole
            __syncthreads();
            float* stage = reinterpret_cast<float*>(ring) + wv * 16 * OSTR;
#pragma unroll
            for (int rb = 0; rb < RBX; ++rb) {
                const float lsum = quarter_sum(st.l[rb]);
                const float scale = !whole ? 1.0f : lsum > 0.f ? 1.0f / lsum : 0.f;
                const int row0 = w0 + rb * BLOCK;
                if (q == 0 && row0 + n < rend) {
                    if (!whole) *reinterpret_cast<HW_GLOBAL f32x2*>(ph.part_ml + (pbase + (row0 - r0) + n) * 2) = f32x2{st.m[rb], lsum};
                    else if (args.lse != nullptr)
                        args.lse[map_row(a, row0 + n, hkv, GQ).qrow] = lsum > 0.f ? (st.m[rb] + __builtin_amdgcn_logf(lsum)) * 0.69314718055994530942f : -__builtin_inff();
                }
#pragma unroll
                for (int c = 0; c < G::NOC; ++c) *reinterpret_cast<f32x4*>(stage + n * OSTR + 16 * c + 4 * q) = st.o[rb][c] * scale;
                const int nvalid = min(16, rend - row0);
#pragma unroll
                for (int ps = 0; ps < 16 * D / 256; ++ps) {
                    const int idx = ps * 256 + lane * 4;
                    const int rr = idx / D, e = idx % D;
                    if (rr < nvalid) {
                        const f32x4 x = *reinterpret_cast<const f32x4*>(stage + rr * OSTR + e);
                        if (whole)
                            *reinterpret_cast<u32x2*>(reinterpret_cast<store_t*>(args.out) + map_row(a, row0 + rr, hkv, GQ).qrow * D + e) =
                                u32x2{Elem<DT>::pack2(x[0], x[1]), Elem<DT>::pack2(x[2], x[3])};
                        else
                            *reinterpret_cast<HW_GLOBAL f32x4*>(ph.part_o + (pbase + (row0 - r0)) * D + idx) = x;
                    }
                }
            }
        };
        // (the waves of a workgroup may be in different ones: what they meet at are barriers, as many in both)
        if (r0 + wv * 16 + NW * 16 < rend) run(std::integral_constant<int, 2>{});
        else run(std::integral_constant<int, 1>{});
    }

    if (ph.cu_q != nullptr) {                    // zeros for query tokens that belong to no sequence
        const int before = bounded(ph.cu_q[0], T), after = bounded(ph.cu_q[ph.W], T), rest = before + T - after;
        for (int i = me; i < rest; i += N) {
            const size_t orow = (size_t)(i < before ? i : after + i - before) * ph.Hq + hkv * GQ;
            for (int x = tid; x < GQ * D; x += NT) reinterpret_cast<store_t*>(args.out)[orow * D + x] = 0;
            if (args.lse != nullptr)
                for (int x = tid; x < GQ; x += NT) args.lse[orow + x] = -__builtin_inff();
        }
    }
}

// The groups that lie across workgroups, as the attention kernel left word of them (cuts_of): a workgroup takes PER rows a thread, D / 4
// lanes a row, of one of them at a time; parts in their order.  A kv head's partial sums are read on the XCD that wrote them.
template <class DT, int D, int PER, int UN>
__global__ __launch_bounds__(256) void window_merge_kernel(const WindowHeader args) {
    typedef typename Elem<DT>::store_t store_t;
    constexpr int V4 = D / 4, RPB = 256 / V4, MOST = D == 256 ? WINDOW_ROWS_256 : WINDOW_ROWS;
    const int tid = threadIdx.x;
    PagedHeaderBits hb;
    paged_header_request(hb);
    const PagedDevHeader ph = paged_header_wait(hb);
    const int N = ph.nsplit, GQ = ph.Hq / ph.Hkv;
    const int homes = ph.flags & PH_XCD_REMAP && ph.Hkv % 8 == 0 ? 8 : 1, heads = ph.Hkv / homes;      // (kv heads of an XCD)
    const int blocks = (args.rows + RPB * PER - 1) / (RPB * PER);
    const int home = blockIdx.x % homes, step = gridDim.x / homes;
    const HW_GLOBAL i32x4* const cuts = cuts_of(args, 0);
    // (cuts first, then kv heads, then rows: where to begin does not depend on how many cuts there are)
    for (int x = blockIdx.x / homes; x < args.most_cuts * heads * blocks; x += step) {
        const int cut = x / (heads * blocks), hr = x - cut * heads * blocks;
        const int hkv = home * heads + hr / blocks, rblk = hr % blocks;
        const HW_GLOBAL i32x4* const mine = cuts + (size_t)hkv * (args.most_cuts + 1);
        const i32x4 all = mine[0], c = mine[cut + 1];
        const int rest = all.x;
        if (cut >= rest) return;
        const int first = c.x, last = c.y, r0 = c.z, rend = c.w;
        const int rr = rblk * RPB * PER + tid / V4, e = tid % V4 * 4;
        if (first == last || r0 + rr >= rend) continue;              // (one that saw the whole group has written the result)
        // (the slot of workgroup w: its first group's, or, for the one that begins the group in the middle of its stretch, the other)
        auto row_of = [&](int w, int k) { return ((size_t)hkv * 2 * N + 2 * w + (all.y != 0 || w * rest / N == cut ? 0 : 1)) * MOST + min(rr + k * RPB, rend - 1 - r0); };
        float m[PER], l[PER];
        f32x4 acc[PER];
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            m[i] = NEG_BIG;
            l[i] = 0.f;
            acc[i] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        for (int w = first; w <= last; w += UN) {
            f32x4 o[PER][UN];
            f32x2 ml[PER][UN];
#pragma unroll
            for (int i = 0; i < PER; ++i)
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    const size_t row = row_of(min(w + u, last), i);
                    o[i][u] = *reinterpret_cast<const HW_GLOBAL f32x4*>(ph.part_o + row * D + e);
                    ml[i][u] = *reinterpret_cast<const HW_GLOBAL f32x2*>(ph.part_ml + row * 2);
                    if (w + u > last) {
                        ml[i][u] = f32x2{NEG_BIG, 0.f};
                        o[i][u] = f32x4{0.f, 0.f, 0.f, 0.f};
                    }
                }
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                float mb = m[i];
#pragma unroll
                for (int u = 0; u < UN; ++u) mb = fmaxf(mb, ml[i][u].x);
                const float old = fast_exp2(m[i] - mb);
                acc[i] *= old;
                l[i] *= old;
#pragma unroll
                for (int u = 0; u < UN; ++u) {
                    const float x = fast_exp2(ml[i][u].x - mb);
                    acc[i] += o[i][u] * x;
                    l[i] += ml[i][u].y * x;
                }
                m[i] = mb;
            }
        }
        DevHeader a;
        a.Hq = ph.Hq; a.S = ph.LS;
        a.magic_gq = ph.magic_gq; a.magic_s = ph.magic_ls;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            if (r0 + rr + i * RPB >= rend) break;
            const float inv = l[i] > 0.f ? 1.0f / l[i] : 0.f;
            const size_t orow = map_row(a, r0 + rr + i * RPB, hkv, GQ).qrow;
            *reinterpret_cast<u32x2*>(reinterpret_cast<store_t*>(args.out) + orow * D + e) =
                u32x2{Elem<DT>::pack2(acc[i][0] * inv, acc[i][1] * inv), Elem<DT>::pack2(acc[i][2] * inv, acc[i][3] * inv)};
            if (args.lse != nullptr && e == 0) args.lse[orow] = l[i] > 0.f ? (m[i] + __builtin_amdgcn_logf(l[i])) * 0.69314718055994530942f : -__builtin_inff();
        }
    }
}

// ------------------------------------------------------------------------------------------------
// launchers
// ------------------------------------------------------------------------------------------------
template <class DT, int D, int NS, int NW, int TS>
static hipError_t launch_window_wide(const WindowHeader& wh, hipStream_t stream) {
    static_assert(NW * 32 == (D == 256 ? WINDOW_ROWS_256 : WINDOW_ROWS), "the planner's row groups");
    hipLaunchKernelGGL((window_wide_kernel<DT, D, NS, NW, TS>), dim3(wh.p.nwg), dim3(NW * 64), 0, stream, wh);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess || wh.p.nsplit == 1) return e;
    if (wh.most_cuts == 0 || (wh.p.cu_q == nullptr && wh.p.nitems % wh.p.nsplit == 0)) return e;
    constexpr int PER = 2, UN = 4, RPB = 1024 / D;
    const int all = wh.p.Hkv * wh.most_cuts * ((wh.rows + RPB * PER - 1) / (RPB * PER));
    hipLaunchKernelGGL((window_merge_kernel<DT, D, PER, UN>), dim3(all < 1024 ? all : 1024), dim3(256), 0, stream, wh);
    return hipGetLastError();
}

template <class DT, int D>
static hipError_t launch_window_d(const WindowHeader& wh, int rb, hipStream_t stream) {
    if constexpr (Elem<DT>::size == 2) {
        if (rb == WIDE_ROW_BLOCKS) {
            if constexpr (D == 256) return launch_window_wide<DT, D, 4, 4, 1>(wh, stream);
            else return launch_window_wide<DT, D, 6, 8, 2>(wh, stream);
        }
    }
    if constexpr (Elem<DT>::size == 2 && D <= 128) {
        if (rb == 2) {
            if (wh.p.flags & PH_SMALL) hipLaunchKernelGGL((window_kernel<DT, D, 2, true>), dim3(wh.p.nwg), dim3(NTHREADS), 0, stream, wh);
            else hipLaunchKernelGGL((window_kernel<DT, D, 2, false>), dim3(wh.p.nwg), dim3(NTHREADS), 0, stream, wh);
            return hipGetLastError();
        }
    }
    if (rb != 1) return hipErrorInvalidValue;
    if (wh.p.flags & PH_SMALL) hipLaunchKernelGGL((window_kernel<DT, D, 1, true>), dim3(wh.p.nwg), dim3(NTHREADS), 0, stream, wh);
    else hipLaunchKernelGGL((window_kernel<DT, D, 1, false>), dim3(wh.p.nwg), dim3(NTHREADS), 0, stream, wh);
    return hipGetLastError();
}

template <class DT>
static hipError_t launch_window_dt(const WindowHeader& wh, int D, int rb, hipStream_t stream) {
    if (D == 256) {
        if constexpr (Elem<DT>::size == 2) return launch_window_d<DT, 256>(wh, rb, stream);
        return hipErrorInvalidValue;
    }
    if (D == 128) return launch_window_d<DT, 128>(wh, rb, stream);
    if (D == 64) return launch_window_d<DT, 64>(wh, rb, stream);
    return hipErrorInvalidValue;
}

hipError_t launch_window_attention(const WindowHeader& wh, int dtype, int D, int rb, hipStream_t stream) {
    switch (dtype) {
        case 0: return launch_window_dt<F32>(wh, D, rb, stream);
        case 1: return launch_window_dt<F16>(wh, D, rb, stream);
        default: return launch_window_dt<BF16>(wh, D, rb, stream);
    }
}

}  // namespace hw
