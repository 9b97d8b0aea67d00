// Fuzz of the 4-bit caches' validator and planner (inference_lib_amd/csrc/hogwild_plan.cpp), built with -fsanitize=address,undefined: what
// the kernels of hogwild_q4.hip rely on in every plan that is accepted.
// usage: q4_plan_fuzz <iterations> <seed>
#include <algorithm>
#include <cmath>
#include <cstdint>
#include <cstdio>
#include <cstdlib>
#include <random>
#include <vector>

#include "../../inference_lib_amd/csrc/hogwild_consts.h"
#include "../../inference_lib_amd/csrc/hogwild_plan.h"

using namespace hw::host;

static int failures = 0;
static long plans = 0, shares = 0, direct = 0;
#define CHECK(cond, ...)                                                   \
    do {                                                                   \
        if (!(cond)) {                                                     \
            if (failures++ < 20) { std::printf("FAIL %s:%d %s: ", __FILE__, __LINE__, #cond); std::printf(__VA_ARGS__); std::printf("\n"); } \
        }                                                                  \
    } while (0)

static void check_division(unsigned d, unsigned long long n_max, const char* what) {
    const unsigned m = magic_of((int)d);
    for (unsigned long long n = 0; n <= n_max; ++n) {
        const unsigned q = m ? (unsigned)((n * (unsigned long long)m) >> 32) : (unsigned)n;
        if (q != n / d) {
            CHECK(false, "%s: %llu / %u gives %u", what, n, d, q);
            return;
        }
    }
}

static void fuzz(std::mt19937_64& rng) {
    auto U = [&](long long lo, long long hi) { return (long long)(lo + rng() % (unsigned long long)(hi - lo + 1)); };
    alignas(16) static int32_t there[4];
    hw_paged_problem p{};
    p.dtype = U(0, 1) ? HW_BF16 : HW_F16;
    p.F = (int)U(1, U(0, 9) == 0 ? HW_MAX_FRAGMENTS + 1 : 4);
    p.Hkv = (int)(U(0, 3) == 0 ? U(1, 64) : 1 << U(0, 4));
    p.Hq = p.Hkv * (int)(U(0, 9) == 0 ? U(1, 4095) : U(1, 16));
    const int dims[3] = {64, 128, 256};
    p.E = p.Ev = dims[U(0, 2)];
    p.W = (int)(U(0, 3) == 0 ? U(1, 100000) : U(1, 80));
    p.S = (int)(U(0, 9) == 0 ? U(1, 4095) : U(1, 12));
    p.block_size = 8 * (int)(U(0, 3) == 0 ? U(1, 511) : 1 << U(0, 6));
    p.max_blocks = (int)(U(0, 1) ? U(1, (1 << 20) / p.block_size) : U(1, std::max(1, std::min(2000, (1 << 20) / p.block_size))));
    p.num_blocks = (int)U(1, 1 << U(0, 28));
    p.scale = 0.1f;
    p.splits = U(0, 3) == 0 ? (int)U(1, 80) : 0;
    p.row_blocks = (int)(U(0, 4) == 0 ? U(-1, 8) : 0);
    bool varlen = U(0, 1);
    if (U(0, 3) == 0) {               // a decode step or draft, mostly one whose workgroups are shared out by the lengths
        varlen = false;
        p.F = (int)U(1, 2);
        p.W = (int)U(1, 40);
        p.S = (int)U(1, 4);
        p.Hkv = 1 << U(0, 3);
        p.Hq = p.Hkv * (int)U(1, 5);
        p.E = p.Ev = U(0, 2) ? 256 : 128;
        p.num_blocks = 4096;
        p.splits = p.row_blocks = 0;
    }
    if (varlen) {
        p.cu_seqlens_q = there;       // only its presence matters here
        p.total_q = (int)U(0, U(0, 3) == 0 ? 200000 : 3000);
    }
    p.out = there; p.q = there; p.locations = there; p.fragment_lengths = there; p.key_cache = there; p.value_cache = there; p.block_table = there;
    switch (U(0, 12)) {               // something that is refused
        case 0: p.dtype = HW_F32; break;
        case 1: p.block_size += (int)U(1, 7); break;
        case 2: p.E = 96; break;
        case 3: p.Hq += p.Hkv > 1 ? 1 : 0; break;
        case 4: p.W = (int)U(-3, 0); break;
        case 5: p.max_blocks = (int)U(-3, 0); break;
        case 6: p.key_cache = (const char*)there + 4; break;
        default: break;
    }
    const int ok = paged_q4_validate(&p);
    const int cus = (int)(U(0, 3) == 0 ? U(1, 1024) : 256);
    hw_paged_plan plan;
    const int st = paged_q4_plan(&p, cus, &plan);
    if (ok == HW_OK) {
        // an octet's place is kept in 32 bits, in units of D / 2 bytes
        CHECK(9ull * ((unsigned long long)p.num_blocks * p.Hkv * (p.block_size / 8)) <= 0xffffffffull, "caches beyond what the kernel counts in");
        CHECK(p.E == p.Ev && p.block_size % 8 == 0 && p.dtype != HW_F32, "accepted");
    }
    if (st != HW_OK) {
        CHECK(st == HW_ERR_SHAPE, "status %d", st);
        return;
    }
    if (ok != HW_OK || p.E == 96) return;
    ++plans;
    const int gq = p.Hq / p.Hkv, D = p.E;
    const long long tokens = varlen ? p.total_q : (long long)p.W * p.S;
    CHECK(plan.rows == tokens * gq && plan.rows < (1 << 20), "rows");
    CHECK(plan.row_blocks == 1 || (plan.row_blocks == 2 && D <= 128), "row blocks %d at %d", plan.row_blocks, D);
    CHECK(plan.splits >= 1 && plan.splits <= 64 && (p.splits <= 0 || plan.splits == std::min(p.splits, 64)), "splits %d of %d", plan.splits, p.splits);
    CHECK((long long)plan.workgroups == (long long)p.Hkv * plan.row_groups * plan.splits && plan.workgroups < (1 << 20), "workgroups");
    // every row has its workgroup: of fixed lengths exactly, of packed ones for any lengths
    const int rpw = 16 * plan.row_blocks;
    if (!varlen) {
        const long long each = ((long long)p.S * gq + rpw - 1) / rpw;
        CHECK(plan.row_groups == p.W * each, "%d row groups, %d sequences of %lld", plan.row_groups, p.W, each);
    } else {
        for (int kind = 0; kind < 3; ++kind) {
            long long left = tokens, need = 0;
            for (int w = 0; w < p.W; ++w) {
                const long long n = w == p.W - 1 ? left : kind == 0 ? 0 : kind == 1 ? std::min<long long>(left, U(0, 3)) : std::min<long long>(left, U(0, 2 * tokens / p.W + 1));
                need += (n * gq + rpw - 1) / rpw;
                left -= n;
            }
            CHECK(need <= plan.row_groups, "%lld row groups of %d", need, plan.row_groups);
        }
    }
    // one workgroup writes the results where the table is short
    const long long tiles = ((long long)p.block_size * p.max_blocks + hw::TILE - 1) / hw::TILE;
    const int whole = D == 64 ? (plan.row_blocks == 1 ? 24 : 20) : D == 128 && plan.row_blocks == 1 ? 20 : 12;
    if (p.splits <= 0) {
        if (tiles <= whole) CHECK(plan.splits == 1, "%lld tiles in %d", tiles, plan.splits);
        CHECK(plan.splits <= std::max<long long>(1, (tiles + hw::NWAVES - 1) / hw::NWAVES), "%d splits of %lld tiles", plan.splits, tiles);
    }
    const size_t rows = plan.rows > 0 ? plan.rows : 1;
    CHECK(plan.workspace_bytes >= (size_t)p.Hkv * plan.splits * rows * ((size_t)D + 2) * sizeof(float), "workspace");
    if (plan.splits == 1) ++direct;
    if (plan.splits > 1 && paged_shared(&p, plan) && paged_q4_shares_save(&p, plan, cus) >= 0) {
        ++shares;
        // partial sums by workgroup, one row group a sequence, then two numbers a row for the merge; one lane a sequence
        CHECK(p.W <= 64 && plan.row_groups == p.W && p.S * gq <= rpw && plan.workgroups <= cus && plan.splits < (1 << 16), "shares of %d sequences", p.W);
        const size_t need = (size_t)p.Hkv * plan.row_groups * plan.splits * p.S * gq * ((size_t)D + 2) * sizeof(float) + (size_t)p.Hkv * plan.rows * 2 * sizeof(int);
        CHECK(paged_call_bytes(&p, plan) >= need, "workspace of shares");
        check_division((unsigned)(plan.rows / p.W), (unsigned long long)plan.rows, "row / rows of a sequence");
    }
    check_division((unsigned)plan.splits, (unsigned long long)plan.workgroups - 1, "workgroup / splits");
    check_division((unsigned)plan.row_groups, (unsigned long long)p.Hkv * plan.row_groups - 1, "(head, item) / items");
    if (!varlen) check_division((unsigned)(plan.row_groups / p.W), (unsigned long long)plan.row_groups - 1, "item / row groups of a sequence");
    check_division((unsigned)gq, (unsigned long long)tokens * gq + 31, "row / heads of a group");
    if (!varlen) check_division((unsigned)p.S, (unsigned long long)tokens + 31, "token / S");
    check_division((unsigned)(p.block_size / 8), (unsigned long long)(p.block_size / 8) * p.max_blocks - 1, "octet / octets of a block");
}

int main(int argc, char** argv) {
    const long iters = argc > 1 ? std::atol(argv[1]) : 2000;
    std::mt19937_64 rng(argc > 2 ? std::strtoull(argv[2], nullptr, 10) : 1);
    for (long i = 0; i < iters; ++i) fuzz(rng);
    std::printf("%ld iterations, %ld plans (%ld direct, %ld shared), %d failures\n", iters, plans, direct, shares, failures);
    CHECK(plans > iters / 4 && direct > iters / 40 && shares > iters / 40, "too few plans of a kind");
    return failures ? 1 : 0;
}
