// Serving steps around the paged caches, for gfx950 (MI355X, CDNA4, wave64):
//
//   packed_slots_kernel ..... a packed batch is laid out: where each sequence begins, every token's position and row of the caches
//   copy_to_slots_kernel .... keys and values of a packed batch go to their rows
//   verify_sums_kernel ...... which drafts are accepted, and the sums of the weights that the next token is drawn from
//   verify_draw_kernel ...... the token, by the running sum
#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "hogwild_kernels.h"
#include "hogwild_device.h"

namespace hw {

// ---- packed batches --------------------------------------------------------------------------------------------------------------

constexpr int SLOTS_THREADS = 256;

// Every workgroup adds up the numbers of new tokens for itself (W <= POOL_MAX_ROWS numbers, in LDS) and looks its tokens' sequences up there.
// Sums stop at `total`: min(a + b, total) of numbers up to total is associative and stays below 2^31.
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

// One piece of VEC bytes per thread and step: of the rows [token][keys, then values][head].
template <int VEC>
__global__ __launch_bounds__(256) void copy_to_slots_kernel(const CopySlotsArgs a, int sz) {
    const unsigned ck = a.E * sz / VEC, cv = a.Ev * sz / VEC, per = a.Hkv * (ck + cv);
    const size_t all = (size_t)a.total * per;
    const int rows = a.num_blocks * a.block_size;
    for (size_t x = (size_t)blockIdx.x * 256 + threadIdx.x; x < all; x += (size_t)gridDim.x * 256) {
        const size_t t = x / per;
        unsigned c = (unsigned)(x - t * per);
        const int slot = a.slots[t];
        if (slot < 0 || slot >= rows) continue;
        const int blk = slot / a.block_size, off = slot - blk * a.block_size;
        const bool is_k = c < a.Hkv * ck;
        if (!is_k) c -= a.Hkv * ck;
        const unsigned cr = is_k ? ck : cv, h = c / cr;
        c -= h * cr;
        const size_t dst_row = ((size_t)blk * a.Hkv + h) * a.block_size + off;
        const char* src = is_k ? reinterpret_cast<const char*>(a.key_states) + ((long long)t * a.ks_t + (long long)h * a.ks_h) * sz + (size_t)c * VEC
                               : reinterpret_cast<const char*>(a.value_states) + ((long long)t * a.vs_t + (long long)h * a.vs_h) * sz + (size_t)c * VEC;
        char* dst = is_k ? reinterpret_cast<char*>(a.kcache) + dst_row * a.E * sz + (size_t)c * VEC
                         : reinterpret_cast<char*>(a.vcache) + dst_row * a.Ev * sz + (size_t)c * VEC;
        if constexpr (VEC == 16) *reinterpret_cast<u32x4*>(dst) = *reinterpret_cast<const u32x4*>(src);
        else if constexpr (VEC == 4) *reinterpret_cast<u32*>(dst) = *reinterpret_cast<const u32*>(src);
        else *reinterpret_cast<unsigned short*>(dst) = *reinterpret_cast<const unsigned short*>(src);
    }
}

// ---- drafts ----------------------------------------------------------------------------------------------------------------------

constexpr int VERIFY_THREADS = 256;

template <class DT>
__device__ __forceinline__ float prob_at(const void* base, long long i) {
    return Elem<DT>::to_float(reinterpret_cast<const typename Elem<DT>::store_t*>(base)[i]);
}
// What a probability counts in a sum: negative, infinite and NaN ones nothing.
__device__ __forceinline__ double weight_of(double x) { return x > 0.0 && x < __builtin_inf() ? x : 0.0; }

struct VerifyRow {
    int n, accepted;
    long long draft;         // the first draft that is not accepted (accepted < n), a token or not
};
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

// Weight of token i: what is left of the target's probability (left), or all of it.
template <class DT>
__device__ __forceinline__ void weights_of(const VerifyArgs& a, int w, const VerifyRow& r, int i, double& left, double& all) {
    const double p = prob_at<DT>(a.target, w * a.tp_w + r.accepted * a.tp_k + i);
    all = weight_of(p);
    left = 0.0;
    if (r.accepted < r.n) {
        const double q = a.draft_probs != nullptr ? (double)prob_at<DT>(a.draft_probs, w * a.dp_w + r.accepted * a.dp_k + i) : (i == r.draft ? 1.0 : 0.0);
        left = weight_of(p - q);
    }
}

template <class DT, class TOK>
__global__ __launch_bounds__(VERIFY_THREADS) void verify_sums_kernel(const VerifyArgs a) {
    __shared__ double part[2][VERIFY_THREADS / 64];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int w = blockIdx.x / a.chunks, c = blockIdx.x - w * a.chunks;
    const VerifyRow r = verify_row<DT, TOK>(a, w, lane);
    double sl = 0.0, sa = 0.0;
    for (int i = c * VERIFY_CHUNK + tid; i < min((c + 1) * VERIFY_CHUNK, a.V); i += VERIFY_THREADS) {
        double left, all;
        weights_of<DT>(a, w, r, i, left, all);
        sl += left;
        sa += all;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        sl += __shfl_xor(sl, d, 64);
        sa += __shfl_xor(sa, d, 64);
    }
    if (lane == 0) {
        part[0][wv] = sl;
        part[1][wv] = sa;
    }
    __syncthreads();
    if (tid < 2) {
        double s = part[tid][0];
        for (int i = 1; i < VERIFY_THREADS / 64; ++i) s += part[tid][i];
        a.sums[((size_t)w * a.chunks + c) * 2 + tid] = s;
    }
}

// inclusive sum over the lanes of a wave
__device__ __forceinline__ double wave_scan(double v, int lane) {
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double x = __shfl_up(v, d, 64);
        if (lane >= d) v += x;
    }
    return v;
}

template <class DT, class TOK>
__global__ __launch_bounds__(VERIFY_THREADS) void verify_draw_kernel(const VerifyArgs a) {
    __shared__ double run_lds[VERIFY_THREADS / 64];
    __shared__ int found_lds[VERIFY_THREADS / 64], last_lds[VERIFY_THREADS / 64];
    const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
    const int w = blockIdx.x;
    const VerifyRow r = verify_row<DT, TOK>(a, w, lane);
    const double* sums = a.sums + (size_t)w * a.chunks * 2;
    // the chunk in which the running sum passes u times the whole (every wave for itself; sums in the order of the chunks)
    double total[2] = {0.0, 0.0};
    for (int c = 0; c < a.chunks; ++c) {
        total[0] += sums[2 * c];
        total[1] += sums[2 * c + 1];
    }
    const int which = r.accepted < r.n && total[0] > 0.0 ? 0 : 1;
    const double aim = (double)a.uniforms[(size_t)w * (a.K + 1) + a.K] * total[which];
    int chunk = -1, holds = -1;              // holds: the last chunk with a weight
    double base = 0.0, before = 0.0;
    for (int c = 0; c < a.chunks; ++c) {
        const double s = sums[2 * c + which];
        if (s > 0.0) {
            if (chunk < 0 && base + s > aim) {
                chunk = c;
                before = base;
            }
            holds = c;
        }
        base += s;
    }
    const bool beyond = chunk < 0;           // from 1 on, or nothing has a weight
    if (beyond) chunk = holds;
    int token = -1;
    if (chunk >= 0) {
        // within the chunk, 256 tokens at a time in their order; the last one with a weight where the sums' rounding leaves none over
        int last = -1;
        for (int i0 = chunk * VERIFY_CHUNK; i0 < min((chunk + 1) * VERIFY_CHUNK, a.V) && token < 0; i0 += VERIFY_THREADS) {
            const int i = i0 + tid;
            double left = 0.0, all = 0.0;
            if (i < a.V) weights_of<DT>(a, w, r, i, left, all);
            const double x = which == 0 ? left : all;
            double run = wave_scan(x, lane);
            if (lane == 63) run_lds[wv] = run;
            __syncthreads();
            double step = before;
            for (int k = 0; k < VERIFY_THREADS / 64; ++k) {
                if (k == wv) run += step;
                step += run_lds[k];
            }
            const unsigned long long over = __ballot(x > 0.0 && run > aim && !beyond), some = __ballot(x > 0.0);
            if (lane == 0) {
                found_lds[wv] = over != 0 ? i0 + wv * 64 + __builtin_ctzll(over) : -1;
                last_lds[wv] = some != 0 ? i0 + wv * 64 + 63 - __builtin_clzll(some) : -1;
            }
            __syncthreads();
            for (int k = 0; k < VERIFY_THREADS / 64; ++k) {
                if (token < 0) token = found_lds[k];
                last = max(last, last_lds[k]);
            }
            before = step;
            __syncthreads();
        }
        if (token < 0) token = last;
    }
    const TOK* drafts = reinterpret_cast<const TOK*>(a.drafts) + (size_t)w * a.K;
    TOK* tokens = reinterpret_cast<TOK*>(a.tokens) + (size_t)w * (a.K + 1);
    for (int i = tid; i <= a.K; i += VERIFY_THREADS) tokens[i] = i < r.accepted ? drafts[i] : (TOK)(i == r.accepted ? token : -1);
    if (tid == 0) {
        a.accepted[w] = r.accepted;
        if (a.lengths != nullptr) a.lengths[w] = (int)min((long long)a.lengths[w], (long long)a.positions[w] + 1 + r.accepted);
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
    const size_t all = (size_t)a.total * a.Hkv * ((size_t)(a.E + a.Ev) * sz / vec);
    size_t blocks = (all + 255) / 256;
    if (blocks > 8192) blocks = 8192;
    if (vec == 16) hipLaunchKernelGGL((copy_to_slots_kernel<16>), dim3((unsigned)blocks), dim3(256), 0, stream, a, sz);
    else if (vec == 4) hipLaunchKernelGGL((copy_to_slots_kernel<4>), dim3((unsigned)blocks), dim3(256), 0, stream, a, sz);
    else hipLaunchKernelGGL((copy_to_slots_kernel<2>), dim3((unsigned)blocks), dim3(256), 0, stream, a, sz);
    return hipGetLastError();
}

template <class DT, class TOK>
static hipError_t launch_verify_dt(const VerifyArgs& a, hipStream_t stream) {
    hipLaunchKernelGGL((verify_sums_kernel<DT, TOK>), dim3((unsigned)a.W * a.chunks), dim3(VERIFY_THREADS), 0, stream, a);
    const hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    hipLaunchKernelGGL((verify_draw_kernel<DT, TOK>), dim3(a.W), dim3(VERIFY_THREADS), 0, stream, a);
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
