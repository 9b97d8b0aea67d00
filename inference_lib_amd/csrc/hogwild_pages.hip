// The pages of paged caches, for gfx950 (MI355X): who holds them, and copies of them.
//
// A pool has num_blocks pages; row w of the block table names the pages of sequence w (entries outside 0 .. num_blocks - 1 name none),
// ref_counts[p] says how many rows name page p, 0 being a free page.  Everything lives in device memory and is worked out there, so
// that a step captured in a graph goes on allocating, forking and copying in its replays and nothing waits for the host.
//
//   fork_kernel ....... every row takes over its parent's pages (or gives its own back)
//   reserve_kernel .... pages for the tokens to come, copies of shared pages that are about to be written
//   compact_kernel .... which pages move where, so that those in use are the first ones
//   copy_pages_kernel . the pages themselves, of every tensor of the pool (layers, keys and values) in one launch
//   trim_kernel ....... pages that have left a sliding window are given back
//
// The first three are bound by latency: chains of a few dependent accesses to tables of some kilobytes.  One workgroup works out an
// allocation, because what one sequence gets depends on what the others took; its scans go over the free pages wave by wave.  The
// results depend on no order of execution: counts are integers, the i-th page wanted gets the i-th free one.

#include <hip/hip_runtime.h>
#include <stdint.h>

#include <type_traits>

#include "hogwild_kernels.h"
#include "hogwild_device.h"

namespace hw {

// Row w takes the pages with tokens of row parents[w] (all rows at once: the old rows are read before any is written), itself: the row
// stays as it is, no row of the table: it gives its pages back.  grid = chunks of `cols` columns; the chunk's old entries of all
// rows are held in LDS.
template <bool FREE>
__global__ __launch_bounds__(512) void fork_kernel(const PoolArgs a, const void* who, int cols) {
    extern __shared__ int lds[];
    int* const par = lds;
    int* const held = lds + a.W;
    int* const old = lds + 2 * a.W;
    const int tid = threadIdx.x, nt = blockDim.x;
    const int j0 = blockIdx.x * cols, nc = min(cols, a.max_blocks - j0);
    for (int w = tid; w < a.W; w += nt) {
        int p;
        if constexpr (FREE) p = reinterpret_cast<const unsigned char*>(who)[w] != 0 ? -1 : w;
        else p = reinterpret_cast<const int*>(who)[w];
        if (p < 0 || p >= a.W) p = -1;
        par[w] = p;
        const int len = p >= 0 ? max(a.lengths[p], 0) : 0;
        held[w] = (int)(((long long)len + a.block_size - 1) / a.block_size);
    }
    for (int x = tid; x < a.W * nc; x += nt) {
        const int w = x / nc, c = x - w * nc;
        old[x] = a.table[(size_t)w * a.max_blocks + j0 + c];
    }
    __syncthreads();
    for (int x = tid; x < a.W * nc; x += nt) {
        const int w = x / nc, c = x - w * nc, p = par[w];
        if (p == w) continue;
        const int was = old[x], is = p >= 0 && j0 + c < held[w] ? old[p * nc + c] : -1;
        if (was == is) continue;
        if (was >= 0 && was < a.num_blocks) atomicSub(a.refs + was, 1);
        if (is >= 0 && is < a.num_blocks) atomicAdd(a.refs + is, 1);
        a.table[(size_t)w * a.max_blocks + j0 + c] = is;
    }
    if (gridDim.x == 1) {                // (otherwise other workgroups still read them: fork_lengths_kernel)
        __syncthreads();                 // the pages' numbers make room for the lengths only when every wave has used them
        for (int w0 = 0; w0 < a.W; w0 += nt) {
            const int w = w0 + tid;
            if (w < a.W) held[w] = par[w] >= 0 ? a.lengths[par[w]] : 0;
        }
        __syncthreads();
        for (int w = tid; w < a.W; w += nt) a.lengths[w] = held[w];
    }
}

template <bool FREE>
__global__ __launch_bounds__(512) void fork_lengths_kernel(const PoolArgs a, const void* who) {
    extern __shared__ int lds[];
    for (int w = threadIdx.x; w < a.W; w += blockDim.x) {
        int p;
        if constexpr (FREE) p = reinterpret_cast<const unsigned char*>(who)[w] != 0 ? -1 : w;
        else p = reinterpret_cast<const int*>(who)[w];
        lds[w] = p < 0 || p >= a.W ? 0 : a.lengths[p];
    }
    __syncthreads();
    for (int w = threadIdx.x; w < a.W; w += blockDim.x) a.lengths[w] = lds[w];
}

constexpr int POOL_THREADS = 1024, POOL_WAVES = POOL_THREADS / 64;

// Exclusive prefix of one number per wave, by every thread for its wave; `total` over all waves.  Two barriers.
__device__ __forceinline__ int wave_base(int mine, int* lds, int wv, int lane, int& total) {
    __syncthreads();
    if (lane == 0) lds[wv] = mine;
    __syncthreads();
    const int v = lane < POOL_WAVES ? lds[lane] : 0;
    const int inc = wave_scan_inclusive(v);
    total = __builtin_amdgcn_readlane(inc, 63);
    return __builtin_amdgcn_readlane(inc - v, wv);
}

// Pages for n_new[w] more tokens of every sequence w: those that its row lacks from the page of its next token to that of its last
// one, and one in the place of each of them that other rows name as well.  Where the page of the next token holds tokens of the row already
// it is copied (the last of the rows that are about to write a page keeps it); the others hold none of its tokens (a length that was
// shortened), and neither do those behind the last new token, which the row gives up as far as others name them.  The pages that
// the rows want, row by row and in a row by position, get the free pages in ascending order; the first row whose wants go beyond the free
// pages gets none, and neither do the rows behind it that want any or keep a shared page.  positions[w] = where the new tokens go, or, for
// a row that gets nothing or asks for nothing, a position behind the table (which the appends leave out); taken[w] = how many, 0 for such a
// row.  From the first row on whose new tokens, those of all rows one behind the other, end behind `total` (a packed batch; negative: none), no
// row gets any.  Sixteen lanes to a row.
// Bound by latency: 6.1 us (with the copy launch behind it, in a graph) for 64 rows in a pool of 1024 pages, 43 of 131 072, whose counts it
// reads whole; that pages without tokens are looked for is 0.2 us of it, where a row names some 0.6.  What fits into a batch's rows: 1.4.
// A count is lowered at once where nothing depends on it any more; where a row wants a page only because others name its own, after
// all wants are served, by the pages that then stand in the list of the free ones.
__global__ __launch_bounds__(POOL_THREADS) void reserve_kernel(const PoolArgs a, const int* n_new, int total_rows, int* positions, int* taken, int* ws) {
    __shared__ int page[POOL_MAX_ROWS];      // the shared page that row w is about to write, or -1
    __shared__ int need[POOL_MAX_ROWS];      // pages wanted; then the wants of all rows up to this one
    __shared__ int behind[POOL_MAX_ROWS];    // pages behind the last new token that the row gives up
    __shared__ int scan[POOL_WAVES];
    __shared__ int copies, spare;            // spare: some row gives up pages that hold no tokens of it
    __shared__ int fits;                     // the rows before this one fit into the batch
    constexpr int RPT = POOL_MAX_ROWS / POOL_THREADS;      // consecutive rows of a thread, where rows are added up
    int* const list = ws + POOL_WS_HEADER;
    int* const pairs = list + a.num_blocks;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int l16 = tid & 15, g16 = tid >> 4, rows = POOL_THREADS / 16;
    const int cap = a.block_size * a.max_blocks;
    auto valid = [&](int p) { return p >= 0 && p < a.num_blocks; };
    auto sum16 = [](int v) {
#pragma unroll
        for (int d = 1; d < 16; d <<= 1) v += __shfl_xor(v, d, 64);
        return v;
    };
    if (tid == 0) {
        copies = spare = 0;
        fits = a.W;
    }
    __syncthreads();
    if (total_rows >= 0) {                   // (sums stop at total_rows + 1, below 2^29: associative, as those of packed_slots_kernel)
        const int most = total_rows + 1;
        auto add = [&](int sum, int w) { return w < a.W ? min(sum + min(max(n_new[w], 0), most), most) : sum; };
        int sum = 0;
#pragma unroll
        for (int i = 0; i < RPT; ++i) sum = add(sum, tid * RPT + i);
        int inc = sum;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int v = __shfl_up(inc, d, 64);
            if (lane >= d) inc = min(inc + v, most);
        }
        if (lane == 63) scan[wv] = inc;
        __syncthreads();
        int upto = __shfl_up(inc, 1, 64);
        if (lane == 0) upto = 0;
        for (int i = 0; i < wv; ++i) upto = min(upto + scan[i], most);
        for (int i = 0; i < RPT && upto < most; ++i) {
            upto = add(upto, tid * RPT + i);
            if (upto == most) atomicMin(&fits, tid * RPT + i);
        }
        __syncthreads();
    }
    const int in_batch = fits;
    struct Row {
        int len, nn, first, last;
        bool grows;
    };
    auto row_of = [&](int w) {
        Row r;
        r.len = a.lengths[w];
        r.nn = n_new[w];
        r.grows = r.nn > 0 && r.len >= 0 && (long long)r.len + r.nn <= cap && w < in_batch;
        r.first = r.grows ? r.len / a.block_size : 0;
        r.last = r.grows ? (r.len + r.nn - 1) / a.block_size : -1;
        return r;
    };
    for (int w = g16; w < a.W; w += rows) {
        const Row r = row_of(w);
        int miss = 0, p0 = -1, give = 0;
        if (r.grows) {
            const int* row = a.table + (size_t)w * a.max_blocks;
            const bool holds = r.len % a.block_size != 0;
            bool there = false;              // pages without tokens of the row, up to the entry behind the last one
            for (int j = r.first + l16; j <= min(r.last + 1, a.max_blocks - 1); j += 16) {
                const bool is = valid(row[j]);
                miss += j <= r.last && !is ? 1 : 0;
                there |= is && !(holds && j == r.first);
            }
            if (holds) {
                p0 = row[r.first];
                if (!valid(p0) || a.refs[p0] <= 1) p0 = -1;
            }
            if (((__ballot(there) >> (lane & 48)) & 0xffffu) != 0) {      // (rows that were filled ahead or shortened): which do others name?
                auto shared = [&](int j) { return valid(row[j]) && a.refs[row[j]] > 1; };
                int more = 0, run = 16;
                for (int j = r.first + l16; j <= r.last; j += 16) more += !(holds && j == r.first) && shared(j) ? 1 : 0;
                for (int j = r.last + 1 + l16; run == 16; j += 16) {
                    run = __builtin_ctz(~((unsigned)(__ballot(j < a.max_blocks && shared(j)) >> (lane & 48)) & 0xffffu));
                    give += run;
                }
                miss += more;
                if (more + give > 0) spare = 1;
            }
        }
        miss = sum16(miss);
        if (l16 == 0) {
            page[w] = p0;
            need[w] = miss;
            behind[w] = give;
        }
    }
    __syncthreads();
    const bool later = spare != 0;
    constexpr int COPY = 1 << 30;            // (needs are at most the columns of the table, below 2^30)
    for (int w = g16; w < a.W; w += rows) {
        const int p0 = page[w];
        if (p0 < 0) continue;
        int before = 0;
        for (int v = l16; v < w; v += 16) before += page[v] == p0 ? 1 : 0;
        before = sum16(before);
        if (l16 == 0 && before < a.refs[p0] - 1) need[w] = (need[w] + 1) | COPY;
    }
    __syncthreads();
    // wants of all rows up to each
    int total = 0;
    long long moves = 0;                     // bit i: the thread's row i copies (kept outside of `need`, which becomes the prefix)
    {
        int mine[RPT], sum = 0;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int w = tid * RPT + i;
            const int x = w < a.W ? need[w] : 0;
            sum += x & (COPY - 1);
            mine[i] = sum;
            if (x & COPY) moves |= 1ll << i;
        }
        const int inc = wave_scan_inclusive(sum);
        const int base = wave_base(__builtin_amdgcn_readlane(inc, 63), scan, wv, lane, total) + inc - sum;
#pragma unroll
        for (int i = 0; i < RPT; ++i) {
            const int w = tid * RPT + i;
            if (w < a.W) need[w] = (base + mine[i]) | ((moves >> i) & 1 ? COPY : 0);
        }
    }
    // the free pages: every wave a stretch of the counts, 64 at a time
    const int steps = (a.num_blocks + 64 * POOL_WAVES - 1) / (64 * POOL_WAVES);
    const int from = wv * steps * 64;
    int count = 0;
    for (int i = 0; i < steps; ++i) {
        const int p = from + i * 64 + lane;
        count += __popcll(__ballot(p < a.num_blocks && a.refs[min(p, a.num_blocks - 1)] == 0));
    }
    int n_free = 0;
    int at = wave_base(count, scan, wv, lane, n_free);
    const int listed = min(total, n_free);
    for (int i = 0; i < steps && at < listed; ++i) {
        const int p = from + i * 64 + lane;
        const bool is = p < a.num_blocks && a.refs[min(p, a.num_blocks - 1)] == 0;
        const unsigned long long bits = __ballot(is);
        const int rank = at + __popcll(bits & ((1ull << lane) - 1));
        if (is && rank < listed) list[rank] = p;
        at += __popcll(bits);
    }
    __syncthreads();
    struct Grant {
        int before, sofar;
        bool copy, granted;
    };
    auto grant_of = [&](int w, const Row& r) {
        Grant g;
        g.sofar = need[w] & (COPY - 1);
        g.before = w > 0 ? need[w - 1] & (COPY - 1) : 0;
        g.copy = (need[w] & COPY) != 0;
        g.granted = r.grows && ((g.sofar == g.before && page[w] < 0) || g.sofar <= n_free);
        return g;
    };
    auto finish = [&](int w, const Row& r, bool granted) {
        if (l16 == 0) {
            positions[w] = granted ? r.len : cap;
            if (taken != nullptr) taken[w] = granted ? r.nn : 0;
            if (granted) a.lengths[w] = r.len + r.nn;
        }
    };
    auto serve = [&](auto wait) {            // wait: counts are lowered behind it
        constexpr bool WAIT = decltype(wait)::value;
        for (int w = g16; w < a.W; w += rows) {
            const Row r = row_of(w);
            const Grant g = grant_of(w, r);
            if (g.granted) {
                int* row = a.table + (size_t)w * a.max_blocks;
                const bool holds = r.len % a.block_size != 0;
                int next = g.before;
                for (int j0 = r.first; j0 <= r.last && next < g.sofar; j0 += 16) {
                    const int j = j0 + l16;
                    const bool moved = g.copy && j == r.first;
                    const int old = row[min(j, r.last)];
                    bool want = moved || !valid(old);
                    if constexpr (WAIT) want = want || (!(holds && j == r.first) && a.refs[old] > 1);
                    want = want && j <= r.last;
                    const unsigned bits = (unsigned)(__ballot(want) >> (lane & 48)) & 0xffffu;
                    if (want) {
                        const int at = next + __popc(bits & ((1u << l16) - 1)), fresh = list[at];
                        row[j] = fresh;
                        a.refs[fresh] = 1;
                        if constexpr (WAIT) list[at] = valid(old) ? -2 - old : -1;
                        if (moved) {
                            if constexpr (!WAIT) atomicSub(a.refs + page[w], 1);
                            const int k = atomicAdd(&copies, 1);
                            pairs[2 * k] = page[w];
                            pairs[2 * k + 1] = fresh;
                        }
                    }
                    next += __popc(bits);
                }
            }
            if constexpr (!WAIT) finish(w, r, g.granted);
        }
    };
    if (!later) {
        serve(std::false_type{});
    } else {
        serve(std::true_type{});
        __syncthreads();
        for (int i = tid; i < listed; i += POOL_THREADS) {
            const int old = -2 - list[i];
            if (old >= 0) atomicSub(a.refs + old, 1);
        }
        for (int w = g16; w < a.W; w += rows) {
            const Row r = row_of(w);
            const bool granted = grant_of(w, r).granted;
            if (granted) {
                int* row = a.table + (size_t)w * a.max_blocks + r.last + 1;
                for (int j = l16; j < behind[w]; j += 16) {
                    atomicSub(a.refs + row[j], 1);
                    row[j] = -1;
                }
            }
            finish(w, r, granted);
        }
    }
    __syncthreads();
    if (tid == 0) ws[0] = copies;
}

// Pages in use (named by a row at least) behind as many places as there are such pages move to the places before that are not in use,
// both in ascending order: ws = {number of moves}, where to (by page, from the first such place on), the pairs.
__global__ __launch_bounds__(POOL_THREADS) void compact_kernel(const PoolArgs a, int* used, int* ws) {
    __shared__ int scan[POOL_WAVES];
    int* const to = ws + POOL_WS_HEADER;
    int* const pairs = to + a.num_blocks;
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int steps = (a.num_blocks + 64 * POOL_WAVES - 1) / (64 * POOL_WAVES);
    const int from = wv * steps * 64;
    auto in_use = [&](int p) { return p < a.num_blocks && a.refs[min(p, a.num_blocks - 1)] > 0; };
    int count = 0;
    for (int i = 0; i < steps; ++i) count += __popcll(__ballot(in_use(from + i * 64 + lane)));
    int n = 0;
    wave_base(count, scan, wv, lane, n);
    int movers = 0, places = 0;
    for (int i = 0; i < steps; ++i) {
        const int p = from + i * 64 + lane;
        const bool u = in_use(p);
        movers += __popcll(__ballot(u && p >= n));
        places += __popcll(__ballot(!u && p < n));
    }
    int moves = 0, same = 0;
    int m_at = wave_base(movers, scan, wv, lane, moves);
    int p_at = wave_base(places, scan, wv, lane, same);
    for (int i = 0; i < steps; ++i) {
        const int p = from + i * 64 + lane;
        const bool u = in_use(p), m = u && p >= n, f = !u && p < n;
        const unsigned long long mb = __ballot(m), fb = __ballot(f), below = (1ull << lane) - 1;
        if (m) pairs[2 * (m_at + __popcll(mb & below))] = p;
        if (f) pairs[2 * (p_at + __popcll(fb & below)) + 1] = p;
        if (!u && p >= n && p < a.num_blocks) to[p] = p;
        m_at += __popcll(mb);
        p_at += __popcll(fb);
    }
    __syncthreads();
    for (int r = tid; r < moves; r += POOL_THREADS) {
        const int s = pairs[2 * r], d = pairs[2 * r + 1];
        to[s] = d;
        a.refs[d] = a.refs[s];
        a.refs[s] = 0;
    }
    if (tid == 0) {
        ws[0] = moves;
        used[0] = n;
        ws[1] = n;
    }
}

// Copies of pages: grid.y = tensor, grid.x strides over (pair, 16 KB piece of a page), 16 bytes a lane and four loads of a thread in
// flight.  Bound by the writes, which stream past the caches (sources do not: a fork's copies all read one page): 47 copies of a page of
// 128 KB in each of 32 tensors (197 MB written) behind a fork and a reserve of 10 us, in all 57 us with cached stores, 51 without, 47 with
// 16 384 workgroups at most instead of 4096 (the copies 37, 5.4 TB/s); with sources read past the caches too 71.  (A launch that finds
// nothing to copy takes 4.4 us with 16 384, 2.4 with 4096.)  The pairs come in the
// arguments or, with their number, from device memory; a page that is written is neither read nor written by another pair.  With `to`, the block table's entries are renamed by the way (compaction).
template <class T>
__global__ __launch_bounds__(256) void copy_pages_kernel(const PageCopyArgs a) {
    constexpr int UN = 4;
    const int n = a.dev_pairs != nullptr ? a.dev_pairs_n[0] : a.n_pairs;
    if (a.to != nullptr && blockIdx.y == 0) {
        const int used = a.dev_pairs_n[1];
        for (size_t i = (size_t)blockIdx.x * 256 + threadIdx.x; i < a.table_entries; i += (size_t)gridDim.x * 256) {
            const int e = a.table[i];
            if (e >= used && e < a.num_blocks) a.table[i] = a.to[e];
        }
    }
    if (a.n_tensors == 0) return;
    char* const base = reinterpret_cast<char*>(a.ptr[blockIdx.y]);
    const unsigned per = a.bytes[blockIdx.y] / (unsigned)sizeof(T);              // items of a page
    const unsigned pieces = (per + 256 * UN - 1) / (256 * UN);
    const unsigned total = (unsigned)n * pieces;
    for (unsigned x = blockIdx.x; x < total; x += gridDim.x) {
        const unsigned k = x / pieces, i0 = (x - k * pieces) * (256 * UN) + threadIdx.x;
        const int s = a.dev_pairs != nullptr ? a.dev_pairs[2 * k] : a.pairs[2 * k], d = a.dev_pairs != nullptr ? a.dev_pairs[2 * k + 1] : a.pairs[2 * k + 1];
        const T* src = reinterpret_cast<const T*>(base + (size_t)s * a.bytes[blockIdx.y]);
        T* dst = reinterpret_cast<T*>(base + (size_t)d * a.bytes[blockIdx.y]);
        T v[UN];
#pragma unroll
        for (int u = 0; u < UN; ++u) v[u] = src[min(i0 + u * 256, per - 1)];
#pragma unroll
        for (int u = 0; u < UN; ++u)
            if (i0 + u * 256 < per) __builtin_nontemporal_store(v[u], dst + i0 + u * 256);
    }
}

// Tokens from position length on see, of the positions before it, those from length - window + 1 on and those below sinks: the pages in
// between are given back.  One workgroup per row; counts go down in any order.  Latency: 2.0 us for 4 rows, 4.9 for 256 rows of 784 entries.
__global__ __launch_bounds__(256) void trim_kernel(const PoolArgs a, int window, int sinks) {
    const int w = blockIdx.x;
    const int first = (int)min(((long long)sinks + a.block_size - 1) / a.block_size, (long long)a.max_blocks);
    const int last = (int)min(max((long long)a.lengths[w] - window + 1, 0ll) / a.block_size, (long long)a.max_blocks);
    int* const row = a.table + (size_t)w * a.max_blocks;
    for (int j = first + threadIdx.x; j < last; j += 256) {
        const int page = row[j];
        if (page < 0 || page >= a.num_blocks) continue;
        atomicSub(a.refs + page, 1);
        row[j] = -1;
    }
}

// ------------------------------------------------------------------------------------------------
// launchers
// ------------------------------------------------------------------------------------------------
hipError_t launch_trim(const PoolArgs& a, int window, int sinks, hipStream_t stream) {
    hipLaunchKernelGGL(trim_kernel, dim3(a.W), dim3(256), 0, stream, a, window, sinks);
    return hipGetLastError();
}

hipError_t launch_fork(const PoolArgs& a, const void* who, bool free_rows, hipStream_t stream) {
    int cols = 8192 / a.W;
    cols = cols < 1 ? 1 : cols > a.max_blocks ? a.max_blocks : cols;
    const int grid = (a.max_blocks + cols - 1) / cols;
    const size_t lds = ((size_t)a.W * cols + 2 * (size_t)a.W) * sizeof(int);
    if (free_rows) hipLaunchKernelGGL((fork_kernel<true>), dim3(grid), dim3(512), lds, stream, a, who, cols);
    else hipLaunchKernelGGL((fork_kernel<false>), dim3(grid), dim3(512), lds, stream, a, who, cols);
    hipError_t e = hipGetLastError();
    if (e != hipSuccess || grid == 1) return e;
    if (free_rows) hipLaunchKernelGGL((fork_lengths_kernel<true>), dim3(1), dim3(512), a.W * sizeof(int), stream, a, who);
    else hipLaunchKernelGGL((fork_lengths_kernel<false>), dim3(1), dim3(512), a.W * sizeof(int), stream, a, who);
    return hipGetLastError();
}

hipError_t launch_reserve(const PoolArgs& a, const int* n_new, int total, int* positions, int* taken, int* ws, hipStream_t stream) {
    hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(POOL_THREADS), 0, stream, a, n_new, total, positions, taken, ws);
    return hipGetLastError();
}

hipError_t launch_compact(const PoolArgs& a, int* used, int* ws, hipStream_t stream) {
    hipLaunchKernelGGL(compact_kernel, dim3(1), dim3(POOL_THREADS), 0, stream, a, used, ws);
    return hipGetLastError();
}

// most_pairs: what the number of pairs is at most (grids beyond what the pairs need leave at once)
hipError_t launch_copy_pages(const PageCopyArgs& a, int most_pairs, hipStream_t stream) {
    uintptr_t low = 0;
    unsigned most = 16;
    for (int t = 0; t < a.n_tensors; ++t) {
        low |= reinterpret_cast<uintptr_t>(a.ptr[t]) | a.bytes[t];
        if (a.bytes[t] > most) most = a.bytes[t];
    }
    const int item = (low & 15) == 0 ? 16 : (low & 3) == 0 ? 4 : 1;
    const unsigned long long pieces = ((unsigned long long)most / item + 1023) / 1024;
    unsigned long long gx = (unsigned long long)most_pairs * pieces;
    const unsigned gy = a.n_tensors > 0 ? (unsigned)a.n_tensors : 1;
    const unsigned long long room = 16384 / gy > 16 ? 16384 / gy : 16;
    if (a.to != nullptr && gx * 1024 < a.table_entries) gx = (a.table_entries + 1023) / 1024;
    if (gx > room) gx = room;
    if (gx < 1) gx = 1;
    const dim3 grid((unsigned)gx, gy);
    if (item == 16) hipLaunchKernelGGL((copy_pages_kernel<u32x4>), grid, dim3(256), 0, stream, a);
    else if (item == 4) hipLaunchKernelGGL((copy_pages_kernel<u32>), grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL((copy_pages_kernel<unsigned char>), grid, dim3(256), 0, stream, a);
    return hipGetLastError();
}

}  // namespace hw
