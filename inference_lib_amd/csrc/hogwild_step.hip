// Serving steps around the paged caches, for gfx950 (MI355X, CDNA4, wave64):
//
//   packed_slots_kernel ..... a packed batch is laid out: where each sequence begins, every token's position and row of the caches
//   copy_to_slots_kernel .... keys and values of a packed batch go to their rows
//   verify_kernel ........... which drafts are accepted, and the token behind them
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "hogwild_kernels.h"
#include "hogwild_device.h"

namespace hw {

// ---- packed batches --------------------------------------------------------------------------------------------------------------

constexpr int SLOTS_THREADS = 256;

// Every workgroup adds up the numbers of new tokens for itself (W <= POOL_MAX_ROWS numbers, in LDS) and looks its tokens' sequences up there.
// Sums stop at `total`: min(a + b, total) of numbers up to total is associative and stays below 2^31.  Bound by latency: counts, scan, table,
// 2.4 us for 8 sequences of a token, 3.8 for 8192 rows of 32 sequences.
__global__ __launch_bounds__(SLOTS_THREADS) void packed_slots_kernel(const PackedBatchArgs a) {
    __shared__ int end[POOL_MAX_ROWS];       // tokens up to and with sequence w
    __shared__ int wave_end[SLOTS_THREADS / 64];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int per = (a.W + SLOTS_THREADS - 1) / SLOTS_THREADS;      // consecutive sequences of a thread
    int sum = 0;
    for (int i = 0; i < per; ++i) {
        const int w = tid * per + i;
        if (w < a.W) sum = min(sum + min(max(a.n_new[w], 0), a.total), a.total);
    }
    int inc = sum;
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const int v = __shfl_up(inc, d, 64);
        if (lane >= d) inc = min(inc + v, a.total);
    }
    if (lane == 63) wave_end[wv] = inc;
    int before = __shfl_up(inc, 1, 64);
    if (lane == 0) before = 0;
    __syncthreads();
    for (int i = 0; i < wv; ++i) before = min(before + wave_end[i], a.total);
    for (int i = 0; i < per; ++i) {
        const int w = tid * per + i;
        if (w < a.W) {
            before = min(before + min(max(a.n_new[w], 0), a.total), a.total);
            end[w] = before;
            if (blockIdx.x == 0) a.cu[w + 1] = before;
        }
    }
    if (blockIdx.x == 0 && tid == 0) a.cu[0] = 0;
    __syncthreads();
    const int cap = a.block_size * a.max_blocks;
    for (int i = blockIdx.x * SLOTS_THREADS + tid; i < a.total; i += gridDim.x * SLOTS_THREADS) {
        int lo = 0, hi = a.W;                // the first sequence that ends behind token i
        while (lo < hi) {
            const int mid = (lo + hi) >> 1;
            if (end[mid] > i) hi = mid;
            else lo = mid + 1;
        }
        int loc = -1, slot = -1;
        if (lo < a.W) {
            const long long at = (long long)a.positions[lo] + (i - (lo > 0 ? end[lo - 1] : 0));
            if (at >= 0 && at < cap) {
                const int j = (int)at / a.block_size;
                const int page = a.table[(size_t)lo * a.max_blocks + j];
                if (page >= 0 && page < a.num_blocks) {
                    loc = (int)at;
                    slot = page * a.block_size + ((int)at - j * a.block_size);
                }
            }
        }
        a.locations[i] = loc;
        a.slots[i] = slot;
    }
}

// One wave to a token: its row of the caches is found once, and its pieces of VEC bytes, keys then values, head by head, are dealt to the lanes,
// four of a lane in flight.  What is written streams past the caches, as attention reads it from there once in a step.  Bound by the
// writes: 8172 tokens of 8 heads of 128 channels in 16 bits, 67 MB read and written, 13 us (5.1 TB/s).
template <int VEC>
__global__ __launch_bounds__(256) void copy_to_slots_kernel(const CopySlotsArgs a, int sz, unsigned magic_k, unsigned magic_v) {
    typedef typename std::conditional<VEC == 16, u32x4, typename std::conditional<VEC == 4, u32, unsigned short>::type>::type piece_t;
    constexpr int UN = 4;
    const int lane = threadIdx.x & 63;
    const int t = __builtin_amdgcn_readfirstlane(blockIdx.x * 4 + (threadIdx.x >> 6));
    if (t >= a.total) return;
    const int slot = a.slots[t];
    if (slot < 0 || slot >= a.num_blocks * a.block_size) return;
    const int blk = slot / a.block_size, off = slot - blk * a.block_size;
    const int ck = a.E * sz / VEC, cv = a.Ev * sz / VEC, all_k = a.Hkv * ck, all = all_k + a.Hkv * cv;
    const char* const ks = reinterpret_cast<const char*>(a.key_states) + (long long)t * a.ks_t * sz;
    const char* const vs = reinterpret_cast<const char*>(a.value_states) + (long long)t * a.vs_t * sz;
    char* const kd = reinterpret_cast<char*>(a.kcache) + ((size_t)blk * a.Hkv * a.block_size + off) * a.E * sz;
    char* const vd = reinterpret_cast<char*>(a.vcache) + ((size_t)blk * a.Hkv * a.block_size + off) * a.Ev * sz;
    for (int x0 = lane; x0 < all; x0 += 64 * UN) {
        piece_t v[UN];
        char* dst[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) {
            const int x = min(x0 + 64 * u, all - 1);
            const bool is_k = x < all_k;
            const int y = is_k ? x : x - all_k, n = is_k ? ck : cv;
            const int h = n == 1 ? y : (int)__umulhi((unsigned)y, is_k ? magic_k : magic_v), c = y - h * n;
            v[u] = *reinterpret_cast<const piece_t*>((is_k ? ks + (long long)h * a.ks_h * sz : vs + (long long)h * a.vs_h * sz) + (size_t)c * VEC);
            dst[u] = (is_k ? kd : vd) + ((size_t)h * a.block_size * n + c) * VEC;
        }
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (x0 + 64 * u < all) __builtin_nontemporal_store(v[u], reinterpret_cast<piece_t*>(dst[u]));
    }
}

// ---- drafts ----------------------------------------------------------------------------------------------------------------------

// Probabilities are added up in chunks of VERIFY_CHUNK, by groups of 256 threads: 16 bytes in a row to a thread, two or four rows of the group to a
// chunk.  A thread's in their order, then the threads' of a row by a scan over the wave, then the waves and rows.  A chunk's sum and its
// running sum are the same additions wherever they are worked out, so a token is found where the sums say that it is, and it is the same in
// every call.  Bound by the two rows of probabilities that are read: 64 sequences, 128 000 in float32, 65.5 MB, 13.4 us (4.9 TB/s) and 6.4 for the
// draw, a chain of loads (sums, a chunk's probabilities) between scans.  One sequence of 32 000: 6.0 and 4.8 (half a microsecond more where
// the draw looks for the accepted drafts again).
constexpr int VERIFY_THREADS = 256, VERIFY_WAVES = VERIFY_THREADS / 64;
template <class DT>
struct Chunks {
    static constexpr int VEC = 16 / Elem<DT>::size, ROWS = VERIFY_CHUNK / (VERIFY_THREADS * VEC);
};

template <class DT>
__device__ __forceinline__ float prob_at(const void* base, long long i) {
    return Elem<DT>::to_float(reinterpret_cast<const typename Elem<DT>::store_t*>(base)[i]);
}
// What a probability counts in a sum: negative, infinite and NaN ones nothing.
__device__ __forceinline__ double weight_of(double x) { return x > 0.0 && x < __builtin_inf() ? x : 0.0; }

// Which drafts of sequence w are accepted, by every thread for itself: lane i of a wave looks at draft 64 c + i.
template <class DT, class TOK>
__device__ __forceinline__ VerifyRow verify_row(const VerifyArgs& a, int w, int lane) {
    VerifyRow r;
    r.n = a.n_drafts != nullptr ? min(max(a.n_drafts[w], 0), a.K) : a.K;
    r.accepted = r.n;
    r.draft = -1;
    const TOK* drafts = reinterpret_cast<const TOK*>(a.drafts) + (size_t)w * a.K;
    for (int c = 0; c < r.n; c += 64) {
        const int i = c + lane;
        const bool there = i < r.n;
        const long long x = there ? (long long)drafts[i] : -1;
        bool good = false;
        if (x >= 0 && x < a.V) {
            const float p = prob_at<DT>(a.target, w * a.tp_w + i * a.tp_k + x);
            const float q = a.draft_probs != nullptr ? prob_at<DT>(a.draft_probs, w * a.dp_w + i * a.dp_k + x) : 1.0f;
            good = (double)a.uniforms[(size_t)w * (a.K + 1) + i] * (double)q < (double)p;      // (exact: 24 bits times 24)
        }
        const unsigned long long bad = __ballot(there && !good);
        if (bad != 0) {
            const int l = __builtin_ctzll(bad);
            r.accepted = c + l;
            r.draft = __shfl(x, l, 64);
            break;
        }
    }
    return r;
}

// A thread's probabilities of chunk c; 0 behind the V-th.
template <class DT>
__device__ __forceinline__ void probs_at(const void* base, long long row, int V, int c, int t, float (&x)[Chunks<DT>::ROWS][Chunks<DT>::VEC]) {
    typedef typename Elem<DT>::store_t store_t;
    constexpr int VEC = Chunks<DT>::VEC, ROWS = Chunks<DT>::ROWS;
    const store_t* p = reinterpret_cast<const store_t*>(base) + row;
    const int i0 = c * VERIFY_CHUNK + t * VEC;
    if ((c + 1) * VERIFY_CHUNK <= V && (reinterpret_cast<uintptr_t>(p) & 15) == 0) {        // (uniform)
        u32x4 v[ROWS];
#pragma unroll
        for (int r = 0; r < ROWS; ++r) v[r] = __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p + i0 + r * VERIFY_THREADS * VEC));
#pragma unroll
        for (int r = 0; r < ROWS; ++r)
#pragma unroll
            for (int k = 0; k < VEC; ++k) {
                if constexpr (VEC == 4) x[r][k] = __uint_as_float(v[r][k]);
                else x[r][k] = Elem<DT>::to_float((store_t)(v[r][k / 2] >> (16 * (k & 1))));
            }
        return;
    }
#pragma unroll
    for (int r = 0; r < ROWS; ++r)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            const int i = i0 + r * VERIFY_THREADS * VEC + k;
            x[r][k] = i < V ? Elem<DT>::to_float(p[i]) : 0.f;
        }
}

// The weights of a thread's tokens of chunk c: what is left of the target's probabilities (left), and all of them.
template <class DT>
__device__ __forceinline__ void chunk_weights(const VerifyArgs& a, int w, const VerifyRow& r, int c, int t, double (&left)[Chunks<DT>::ROWS][Chunks<DT>::VEC],
                                              double (&all)[Chunks<DT>::ROWS][Chunks<DT>::VEC]) {
    constexpr int VEC = Chunks<DT>::VEC, ROWS = Chunks<DT>::ROWS;
    float p[ROWS][VEC], q[ROWS][VEC];
    const bool some = r.accepted < r.n;                  // a draft was not accepted
    probs_at<DT>(a.target, w * a.tp_w + r.accepted * a.tp_k, a.V, c, t, p);
    if (some && a.draft_probs != nullptr) probs_at<DT>(a.draft_probs, w * a.dp_w + r.accepted * a.dp_k, a.V, c, t, q);
    else {
#pragma unroll
        for (int i = 0; i < ROWS; ++i)
#pragma unroll
            for (int k = 0; k < VEC; ++k) q[i][k] = some && c * VERIFY_CHUNK + (i * VERIFY_THREADS + t) * VEC + k == r.draft ? 1.0f : 0.f;
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i)
#pragma unroll
        for (int k = 0; k < VEC; ++k) {
            all[i][k] = weight_of(p[i][k]);
            // (behind the V-th token p is 0, and so is what a negative probability of the draft's leaves)
            left[i][k] = some && c * VERIFY_CHUNK + (i * VERIFY_THREADS + t) * VEC + k < a.V ? weight_of((double)p[i][k] - (double)q[i][k]) : 0.0;
        }
}

// inclusive sum over the lanes of a wave (see wave_scan_inclusive; a lane that has nothing before it adds 0)
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_before(double v) {
    const unsigned long long x = __double_as_longlong(v);
    const u32 lo = __builtin_amdgcn_update_dpp(0, (u32)x, CTRL, ROWS, 0xf, false), hi = __builtin_amdgcn_update_dpp(0, (u32)(x >> 32), CTRL, ROWS, 0xf, false);
    return __longlong_as_double((unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_scan(double v) {
    v += dpp_before<0x111, 0xf>(v);
    v += dpp_before<0x112, 0xf>(v);
    v += dpp_before<0x114, 0xf>(v);
    v += dpp_before<0x118, 0xf>(v);
    v += dpp_before<0x142, 0xa>(v);
    v += dpp_before<0x143, 0xc>(v);
    return v;
}
__device__ __forceinline__ double lane_value(double v, int lane) {          // (lane: uniform)
    const unsigned long long x = __double_as_longlong(v);
    return __longlong_as_double((unsigned long long)(u32)__builtin_amdgcn_readlane((u32)(x >> 32), lane) << 32 | (u32)__builtin_amdgcn_readlane((u32)x, lane));
}

// Sums of the chunks (SUMS) and the token (DRAW).  In two launches the sums lie in `sums` and the accepted drafts in `rows`, the first with a
// workgroup to a chunk, the second with one to a sequence; in one, a workgroup of GROUPS groups of 256 threads does all of a sequence, with the sums in LDS.
template <class DT, class TOK, int GROUPS, bool SUMS, bool DRAW>
__global__ __launch_bounds__(VERIFY_THREADS * GROUPS) void verify_kernel(const VerifyArgs a) {
    constexpr bool BOTH = SUMS && DRAW;
    __shared__ double lds_sums[BOTH ? 2 * GROUPS : 1];
    constexpr int VEC = Chunks<DT>::VEC, ROWS = Chunks<DT>::ROWS;
    __shared__ double part[GROUPS][2][ROWS * VERIFY_WAVES];
    __shared__ int found[VERIFY_WAVES], last_one[VERIFY_WAVES];
    const int lane = threadIdx.x & 63, t = threadIdx.x % VERIFY_THREADS, grp = threadIdx.x / VERIFY_THREADS, wv = t >> 6;
    const int w = DRAW ? blockIdx.x : blockIdx.x / a.chunks;
    VerifyRow r;
    if constexpr (SUMS) r = verify_row<DT, TOK>(a, w, lane);
    else r = a.rows[w];
    if constexpr (!DRAW)
        if (threadIdx.x == 0 && blockIdx.x == w * a.chunks) a.rows[w] = r;
    double* const sums = BOTH ? lds_sums : a.sums + (size_t)w * a.chunks * 2;

    if constexpr (SUMS) {
        const int c_begin = DRAW ? 0 : blockIdx.x - w * a.chunks, c_end = DRAW ? a.chunks : c_begin + 1;
        for (int c0 = c_begin; c0 < c_end; c0 += GROUPS) {
            const int c = c0 + grp;                      // (behind the last: nothing there, nothing written)
            double left[ROWS][VEC], all[ROWS][VEC];
            chunk_weights<DT>(a, w, r, c, t, left, all);
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                double sl = 0.0, sa = 0.0;
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    sl += left[i][k];
                    sa += all[i][k];
                }
                sl = wave_scan(sl);
                sa = wave_scan(sa);
                if (lane == 63) {
                    part[grp][0][i * VERIFY_WAVES + wv] = sl;
                    part[grp][1][i * VERIFY_WAVES + wv] = sa;
                }
            }
            __syncthreads();
            if (t < 2 && c < c_end) {
                double s = part[grp][t][0];
                for (int i = 1; i < ROWS * VERIFY_WAVES; ++i) s += part[grp][t][i];
                sums[2 * c + t] = s;
            }
            __syncthreads();
        }
    }
    if constexpr (DRAW) {
        // The chunk in which the running sum passes u times the whole: lane = chunk, 64 at a time; every wave for itself.
        double total[2], mine64[2], run64[2];            // (of the first 64, which are all of them up to 262 144 tokens)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            mine64[k] = lane < a.chunks ? sums[2 * lane + k] : 0.0;
            run64[k] = wave_scan(mine64[k]);
            total[k] = lane_value(run64[k], 63);
        }
        for (int c0 = 64; c0 < a.chunks; c0 += 64) {
            const int c = c0 + lane;
#pragma unroll
            for (int k = 0; k < 2; ++k) total[k] += lane_value(wave_scan(c < a.chunks ? sums[2 * c + k] : 0.0), 63);
        }
        const int which = r.accepted < r.n && total[0] > 0.0 ? 0 : 1;
        const double aim = (double)a.uniforms[(size_t)w * (a.K + 1) + a.K] * total[which];
        int chunk = -1, holds = -1;                      // holds: the last chunk with a weight
        double base = 0.0, before = 0.0;
        for (int c0 = 0; c0 < a.chunks; c0 += 64) {
            const int c = c0 + lane;
            const double mine = c0 == 0 ? (which == 0 ? mine64[0] : mine64[1]) : c < a.chunks ? sums[2 * c + which] : 0.0;
            const double run = c0 == 0 ? (which == 0 ? run64[0] : run64[1]) : wave_scan(mine);
            const unsigned long long over = __ballot(mine > 0.0 && base + run > aim), some = __ballot(mine > 0.0);
            if (chunk < 0 && over != 0) {
                const int l = __builtin_ctzll(over);
                chunk = c0 + l;
                before = l > 0 ? base + lane_value(run, l - 1) : base;
            }
            if (some != 0) holds = c0 + 63 - __builtin_clzll(some);
            base += lane_value(run, 63);
        }
        const bool beyond = chunk < 0;                   // numbers from 1 on, or nothing has a weight
        if (beyond) chunk = holds;
        // the token in it; the last one with a weight where the sums' rounding leaves none over
        double x[ROWS][VEC], below[ROWS];                // weights; their sum in the row's threads of the wave before this one
        if (grp == 0 && chunk >= 0) {
            double left[ROWS][VEC], all[ROWS][VEC];
            chunk_weights<DT>(a, w, r, chunk, t, left, all);
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                double mine = 0.0;
#pragma unroll
                for (int k = 0; k < VEC; ++k) {
                    x[i][k] = which == 0 ? left[i][k] : all[i][k];
                    mine += x[i][k];
                }
                const double scan = wave_scan(mine), up = __shfl_up(scan, 1, 64);
                below[i] = lane > 0 ? up : 0.0;
                if (lane == 63) part[0][0][i * VERIFY_WAVES + wv] = scan;
            }
        }
        __syncthreads();
        int token = -1;
        if (grp == 0 && chunk >= 0) {
            int at = 0x7fffffff, last = -1;
            double at_wave = before;                     // the running sum where the wave's tokens of the row begin
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                for (int k = 0; k < VERIFY_WAVES; ++k) {
                    if (k == wv) {
                        double sum = at_wave + below[i];
#pragma unroll
                        for (int e = 0; e < VEC; ++e) {
                            sum += x[i][e];
                            const int tok = chunk * VERIFY_CHUNK + (i * VERIFY_THREADS + t) * VEC + e;
                            if (x[i][e] > 0.0) {
                                last = max(last, tok);
                                if (sum > aim && !beyond) at = min(at, tok);
                            }
                        }
                    }
                    at_wave += part[0][0][i * VERIFY_WAVES + k];
                }
            }
            at = -wave_max(-at);
            last = wave_max(last);
            if (lane == 0) {
                found[wv] = at;
                last_one[wv] = last;
            }
        }
        __syncthreads();
        if (chunk >= 0) {
            int at = found[0], last = last_one[0];
            for (int i = 1; i < VERIFY_WAVES; ++i) {
                at = min(at, found[i]);
                last = max(last, last_one[i]);
            }
            token = at != 0x7fffffff ? at : last;
        }
        const TOK* drafts = reinterpret_cast<const TOK*>(a.drafts) + (size_t)w * a.K;
        TOK* tokens = reinterpret_cast<TOK*>(a.tokens) + (size_t)w * (a.K + 1);
        for (int i = threadIdx.x; i <= a.K; i += VERIFY_THREADS * GROUPS) tokens[i] = i < r.accepted ? drafts[i] : (TOK)(i == r.accepted ? token : -1);
        if (threadIdx.x == 0) {
            a.accepted[w] = r.accepted;
            if (a.lengths != nullptr) {
                // (the drafts are the last of the step's tokens, behind one other at least)
                const long long brought = a.n_new != nullptr ? max(a.n_new[w], 0) : 1 + r.n, kept = min(brought, max(brought - r.n, 1ll) + r.accepted);
                a.lengths[w] = (int)min((long long)a.lengths[w], (long long)a.positions[w] + kept);
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------
// launchers
// ------------------------------------------------------------------------------------------------
hipError_t launch_packed_slots(const PackedBatchArgs& a, hipStream_t stream) {
    const int blocks = (a.total + SLOTS_THREADS - 1) / SLOTS_THREADS;
    hipLaunchKernelGGL(packed_slots_kernel, dim3(blocks < 1 ? 1 : blocks > 1024 ? 1024 : blocks), dim3(SLOTS_THREADS), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_copy_to_slots(const CopySlotsArgs& a, int dtype, hipStream_t stream) {
    const int sz = dtype == 0 ? 4 : 2;
    const bool vec16 = (a.E * sz) % 16 == 0 && (a.Ev * sz) % 16 == 0 && (a.ks_t * sz) % 16 == 0 && (a.ks_h * sz) % 16 == 0 && (a.vs_t * sz) % 16 == 0 &&
                       (a.vs_h * sz) % 16 == 0 &&
                       ((reinterpret_cast<uintptr_t>(a.key_states) | reinterpret_cast<uintptr_t>(a.value_states) | reinterpret_cast<uintptr_t>(a.kcache) |
                         reinterpret_cast<uintptr_t>(a.vcache)) & 15u) == 0;
    const int vec = vec16 ? 16 : sz;
    // y / n for y < 2^16 pieces of a token's keys, n < 2^16: exact with ceil(2^32 / n)
    auto magic = [&](int n) { return n > 1 ? (unsigned)(((1ull << 32) + n - 1) / n) : 0u; };
    const unsigned mk = magic(a.E * sz / vec), mv = magic(a.Ev * sz / vec);
    const dim3 grid(((unsigned)a.total + 3) / 4);
    if (vec == 16) hipLaunchKernelGGL((copy_to_slots_kernel<16>), grid, dim3(256), 0, stream, a, sz, mk, mv);
    else if (vec == 4) hipLaunchKernelGGL((copy_to_slots_kernel<4>), grid, dim3(256), 0, stream, a, sz, mk, mv);
    else hipLaunchKernelGGL((copy_to_slots_kernel<2>), grid, dim3(256), 0, stream, a, sz, mk, mv);
    return hipGetLastError();
}

template <class DT, class TOK>
static hipError_t launch_verify_dt(const VerifyArgs& a, hipStream_t stream) {
    if (a.sums == nullptr) {
        hipLaunchKernelGGL((verify_kernel<DT, TOK, VERIFY_GROUPS, true, true>), dim3(a.W), dim3(VERIFY_GROUPS * VERIFY_THREADS), 0, stream, a);
        return hipGetLastError();
    }
    hipLaunchKernelGGL((verify_kernel<DT, TOK, 1, true, false>), dim3((unsigned)a.W * a.chunks), dim3(VERIFY_THREADS), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((verify_kernel<DT, TOK, 1, false, true>), dim3(a.W), dim3(VERIFY_THREADS), 0, stream, a);
    return hipGetLastError();
}

hipError_t launch_verify(const VerifyArgs& a, int dtype, bool wide_tokens, hipStream_t stream) {
    auto go = [&](auto dt) {
        typedef decltype(dt) DT;
        return wide_tokens ? launch_verify_dt<DT, long long>(a, stream) : launch_verify_dt<DT, int>(a, stream);
    };
    switch (dtype) {
        case 0: return go(F32{});
        case 1: return go(F16{});
        default: return go(BF16{});
    }
}

}  // namespace hw
