// Decode attention of a batch whose sequences share the pages of a long prefix, over the paged bf16 cache.
//
// Attention over a set of keys is a maximum m, a sum l = sum e^(s - m) and a vector o = sum e^(s - m) v; two disjoint sets join by rescaling to the larger
// maximum.  So the prefix is computed once for all query rows of a K/V head, and each sequence adds its own keys:
//
//   attn_prefix   the batch's rows (sequences x drafted rows x query heads of the group) as tiles of 128, against the shared pages: the prefill kernel's
//                 scheme (S = Q K^T and O += P V as tcgen05.mma, one softmax thread per row, P and O in tensor memory, K and V pages by TMA), all rows see
//                 all keys.  The keys are shared out between CTAs until the GPU is full; every part leaves o, m and l.
//   attn_tail     per sequence and K/V head: the sequence's own keys (mma.sync, a warp has 16 keys of a page), then everything joined, divided, gated.
//
// A sequence shares the prefix if each of its rows sees all of it; another one (shorter, or empty) goes through its own table alone, in the second
// kernel.  The length of the prefix lies on the device, so that a captured step follows it; the host's bound only picks the parts.
//
// Nothing that a row does not see reaches it: K and V rows of the tiles' ends are masked and zeroed, and the last drafted keys, which some rows of a
// sequence see and others do not, are taken one by one (a probability of 0 times an infinity would not be 0).
// Roundings: scores, maxima, sums and O are 32-bit.  Probabilities enter P V as bf16, the type that the tensor cores take beside V: each is off by 2^-8 of itself at
// most, and the sums are of those that are not rounded.  On outputs of random values that is an error of 2.2e-3 in all, of which 1.7e-3 are the rounding of
// the outputs themselves; a second product with what is left of P would take it away, and the products bound the prefix already.
// What bounds it: the prefix, once read, by the tensor pipe and the exponentials from about 200 rows per K/V head on, else by its bytes; the tails by theirs.  61
// sequences x 2 rows behind 20000 keys of 128 values: 69 us with the tails; a tile of 64 keys takes 1600 clocks of two slots, nearly all of
// which the products take (a product of 64 columns with both operands in shared memory 71 clocks, of 128 with one in tensor memory 71).  32 behind 8192
// keys of 256 values 26, the tails beside the prefix; 128 behind 2048 keys of 64 values 20.
#include "attn_tile.cuh"
#include "hybrid.h"
#include "launch.h"
#include "tc_tile.cuh"

namespace llm {
namespace ash {
using namespace tc5;

constexpr int PAGE = 64, BQ = 128;
constexpr float RESCALE_STEP = 8.f;

// keys of the prefix, and whether sequence `b` takes part
LLM_DEVICE int prefix_of(const AttnSharedParams& p) { return p.splits > 0 ? max(0, min(*p.shared_len, p.max_pages * PAGE)) : 0; }
// tiles of the prefix in a part, and the parts that have any
LLM_DEVICE int tiles_per_part(int prefix, int splits) { return ((prefix + PAGE - 1) / PAGE + splits - 1) / splits; }
LLM_DEVICE int parts_of(int prefix, int splits) {
    const int per = tiles_per_part(prefix, splits);
    return per > 0 ? ((prefix + PAGE - 1) / PAGE + per - 1) / per : 0;
}
LLM_DEVICE bool shares(const AttnSharedParams& p, int b, int prefix) { return p.seq_lens[b] - (p.rows_per_seq - 1) >= prefix; }

// ------------------------------------------------------------------------------------------------
// prefix
// ------------------------------------------------------------------------------------------------
// Tiles of 64 keys (a page).  Each slot of 128 rows has two tiles of S in tensor memory (P in the first half of each), so that a product is always on its way while
// its softmax is at work: with one tile of 128 keys per slot a tile took 3550 clocks, of which the softmax waited 1500 (32 / 8 heads, 122 rows).
template <int D, int SLOTS>
struct Prefix {
    static constexpr int BK = 64, DA = D / 64, STAGES = D == 256 ? 2 : 4;     // keys of a tile, atoms of 64 values in a head, tiles of K and of V
    static constexpr int K_ATOM = BK * 128, TILE = DA * K_ATOM;
    static constexpr int OFF_K = SLOTS * DA * ATOM, OFF_V = OFF_K + STAGES * TILE, SMEM = OFF_V + STAGES * TILE + 1024;
    static constexpr int THREADS = SLOTS * 128 + 64;
    static constexpr uint32_t COL_O = SLOTS * 2 * BK;                         // behind the tiles of S: O per slot
    static constexpr uint32_t IDESC_S = instr_desc(BK), IDESC_O = instr_desc(D) | (1u << 16);       // bit 16: B is MN-major
    // Queries go on to tensor memory where that has room for them: a product for a tile's scores takes 41 clocks with them there, 71 with both operands in shared memory.
    static constexpr uint32_t COL_Q = COL_O + SLOTS * D;
    static constexpr bool Q_TMEM = COL_Q + SLOTS * D / 2 <= 512;
    static_assert(SMEM <= 225 * 1024 && COL_O + SLOTS * D <= 512, "a CTA's memories");
    static_assert(SLOTS * 128 * D * 4 <= OFF_V + STAGES * TILE, "results on their way out");
};
enum Bar { K_FULL = 0, K_EMPTY = 4, V_FULL = 8, V_EMPTY = 12, S_FULL = 16, P_FULL = 20, PV_DONE = 24, Q_FULL = 26, N_BARS };       // S_FULL, P_FULL: slot * 2 + tile of S

template <int D, int SLOTS>
__global__ void __launch_bounds__(Prefix<D, SLOTS>::THREADS, 1) attn_prefix_kernel(const __grid_constant__ CUtensorMap map_kv, const AttnSharedParams p, int* status) {
    using X = Prefix<D, SLOTS>;
    constexpr int BK = X::BK, DA = X::DA;
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t s_bars[N_BARS];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort[2];       // [1] stays 0 here (tc_common.cuh: restarts the wait clock when set)
    __shared__ int s_query[SLOTS * BQ];                    // where a row's query lies, in heads; -1: there is none
    pdl_wait();
    pdl_trigger();                   // the tails may begin: what they read was there before this kernel
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int kvh = blockIdx.y, split = blockIdx.z, G = p.n_heads / p.n_kv_heads;
    const int rows_all = p.n_seqs * p.rows_per_seq * G, row_first = blockIdx.x * (SLOTS * BQ);
    const bool both = SLOTS == 2 && row_first + BQ < rows_all;
    const int keys = prefix_of(p), tiles = (keys + BK - 1) / BK, per = tiles_per_part(keys, p.splits);
    const int tile0 = split * per, nt = min(tiles, tile0 + per) - tile0;
    const size_t part = ((size_t)kvh * rows_all + row_first) * p.splits + split;        // of the first row; the next one is `splits` further
    if (nt <= 0) return;                                   // uniform for the CTA, before any barrier or allocation; nobody reads this part
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bars = smem_u32(s_bars);
    auto bar = [&](int i) { return bars + i * 8; };
    if (tid == 0) {
        s_abort[0] = 0; s_abort[1] = 0;
        for (int i = 0; i < N_BARS; ++i) mbar_init(bar(i), i == Q_FULL ? (both ? 8 : 4) : i >= P_FULL && i < P_FULL + 4 ? 4 : 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    if (warp == SLOTS * 4 + 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    volatile int* abort_flag = s_abort;
    auto buffer = [](int slot, int j) { return slot * 2 + (j & 1); };         // tile of S
    auto phase = [](int j) { return (uint32_t)((j >> 1) & 1); };              // of its barriers

    if (warp < SLOTS * 4) {
        // ------------------------------ softmax: one thread per query row (== TMEM lane) ------------------------------
        const int slot = warp >> 2, row = tid & 127;
        if (slot == 0 || both) {
            const int m0 = row_first + slot * BQ;
            const uint32_t sQ = base + slot * DA * ATOM;
            s_query[slot * BQ + row] = m0 + row < rows_all ? (m0 + row) / G * p.n_heads + kvh * G + (m0 + row) % G : -1;
            asm volatile("bar.sync %0, 128;" ::"r"(1 + slot) : "memory");
#pragma unroll 8
            for (int idx = row; idx < BQ * (D / 8); idx += 128) {
                const int r = idx / (D / 8), u = idx % (D / 8), from = s_query[slot * BQ + r];
                // (a row that there is not: zeros, nothing is read)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(atom_addr(sQ + (u >> 3) * ATOM, r, u & 7)), "l"(p.q + (size_t)max(from, 0) * D + u * 8), "r"(from >= 0 ? 16 : 0) : "memory");
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
            const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16), t_o = t_lane + X::COL_O + slot * D;
            if constexpr (X::Q_TMEM) {
                asm volatile("bar.sync %0, 128;" ::"r"(1 + slot) : "memory");
#pragma unroll
                for (int a = 0; a < DA; ++a) {
                    uint32_t w[32];
#pragma unroll
                    for (int u = 0; u < 8; ++u)
                        asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(w[4 * u]), "=r"(w[4 * u + 1]), "=r"(w[4 * u + 2]), "=r"(w[4 * u + 3]) : "r"(atom_addr(sQ + a * ATOM, row, u)));
                    tmem_st32(t_lane + X::COL_Q + slot * (D / 2) + a * 32, w);
                }
                tmem_wait_st();
                tc_fence_before();
            } else {
                fence_proxy_async();
            }
            __syncwarp();
            mbar_arrive_if(bar(Q_FULL), lane == 0);

            const float sl2 = p.scale * LOG2E;
            float m = -INFINITY, l = 0.f;
            bool ok = true;
            for (int j = 0; j < nt; ++j) {
                const int buf = buffer(slot, j);
                const uint32_t t_s = t_lane + buf * BK;
                ok = mbar_wait_warp(bar(S_FULL + buf), phase(j), abort_flag);
                if (!ok) break;
                tc_fence_after();
                uint32_t s[BK / 32][32];
#pragma unroll
                for (int c = 0; c < BK / 32; ++c) tmem_ld32_issue(t_s + c * 32, s[c]);
#pragma unroll
                for (int c = 0; c < BK / 32; ++c) tmem_wait_ld(s[c]);
                const int hi = keys - (tile0 + j) * BK;    // keys of the tile that there are
                if (hi < BK) {
                    // the tile's end: no scores, and V rows of zeros (P is 0 there, whatever the page holds)
#pragma unroll
                    for (int c = 0; c < BK / 32; ++c)
#pragma unroll
                        for (int i = 0; i < 32; ++i) s[c][i] = c * 32 + i < hi ? s[c][i] : 0xff800000u;       // -inf
                    ok = mbar_wait_warp(bar(V_FULL + j % X::STAGES), j / X::STAGES & 1, abort_flag);
                    if (!ok) break;
                    const uint32_t v = base + X::OFF_V + j % X::STAGES * X::TILE;
                    for (int idx = row; idx < (BK - hi) * DA * 8; idx += 128) {
                        const int r = hi + idx / (DA * 8), u = idx % (DA * 8);
                        st_shared_v4(v + (u >> 3) * X::K_ATOM + r * 128 + ((u & 7) << 4), make_uint4(0, 0, 0, 0));
                    }
                    fence_proxy_async();
                }
                float mx4[BK / 32];
#pragma unroll
                for (int c = 0; c < BK / 32; ++c) {
                    mx4[c] = __uint_as_float(s[c][0]);
#pragma unroll
                    for (int i = 1; i < 32; ++i) mx4[c] = fmaxf(mx4[c], __uint_as_float(s[c][i]));
                }
                float mx = mx4[0];
#pragma unroll
                for (int c = 1; c < BK / 32; ++c) mx = fmaxf(mx, mx4[c]);
                const float top = mx * sl2;
                const bool raise = top > m + RESCALE_STEP;                // also the first keys, where m is -inf
                const float factor = raise ? ex2(m - top) : 1.f;
                if (raise) m = top;
                if (j > 0 && __any_sync(0xffffffffu, raise)) {
                    // this tile's S was issued in front of the last tile's P V: O has to be complete
                    ok = mbar_wait_warp(bar(PV_DONE + slot), (j - 1) & 1, abort_flag);
                    if (!ok) break;
                    tc_fence_after();
#pragma unroll
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t r[32];
                        tmem_ld_n<32>(t_o + c * 32, r);
#pragma unroll
                        for (int i = 0; i < 32; ++i) r[i] = __float_as_uint(__uint_as_float(r[i]) * factor);
                        tmem_st32(t_o + c * 32, r);
                    }
                }
                const float mb = m == -INFINITY ? 0.f : m;
                float sum[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < BK / 32; ++c) {
                    uint32_t w[16];
#pragma unroll
                    for (int i = 0; i < 32; i += 2) {
                        const float p0 = ex2(fmaf(__uint_as_float(s[c][i]), sl2, -mb)), p1 = ex2(fmaf(__uint_as_float(s[c][i + 1]), sl2, -mb));
                        sum[(i >> 1) & 1] += p0;
                        sum[2 + ((i >> 1) & 1)] += p1;
                        w[i >> 1] = pack_bf16(p0, p1);
                    }
                    tmem_st_n<16>(t_s + c * 16, w);
                }
                l = l * factor + ((sum[0] + sum[1]) + (sum[2] + sum[3]));
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                mbar_arrive_if(bar(P_FULL + buf), lane == 0);
            }
            // the last product is complete (the one before it first: a wait tells apart two neighbouring phases only)
            ok = ok && (nt < 2 || mbar_wait_warp(bar(PV_DONE + slot), (nt - 2) & 1, abort_flag)) && mbar_wait_warp(bar(PV_DONE + slot), (nt - 1) & 1, abort_flag);
            if (both) asm volatile("bar.sync 3, 256;" ::: "memory");            // both slots' products are done with Q, K and V
            if (ok) {
                // O through shared memory, so that a warp writes whole rows (a row per thread took 15000 clocks); 16-byte units XOR-swizzled
                tc_fence_after();
                const size_t at = part + (size_t)(slot * BQ + row) * p.splits;
                if (m0 + row < rows_all) *reinterpret_cast<float2*>(p.part_ml + at * 2) = make_float2(m, l);
                const uint32_t mine = base + (slot * BQ + (warp & 3) * 32) * (D * 4);
#pragma unroll
                for (int c = 0; c < D / 32; ++c) {
                    uint32_t r[32];
                    tmem_ld_n<32>(t_o + c * 32, r);
#pragma unroll
                    for (int u = 0; u < 8; ++u) st_shared_v4(mine + lane * (D * 4) + (((c * 8 + u) ^ (lane & 7)) << 4), make_uint4(r[4 * u], r[4 * u + 1], r[4 * u + 2], r[4 * u + 3]));
                }
                __syncwarp();
                constexpr int UNITS = D / 4;                // of a row
#pragma unroll 8
                for (int i = lane; i < 32 * UNITS; i += 32) {
                    const int r = i / UNITS, u = i % UNITS, row_of = (warp & 3) * 32 + r;
                    float4 v;
                    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(mine + r * (D * 4) + ((u ^ (r & 7)) << 4)));
                    if (m0 + row_of < rows_all) *(reinterpret_cast<float4*>(p.part_o + (part + (size_t)(slot * BQ + row_of) * p.splits) * D) + u) = v;
                }
            }
        }
    } else if (warp == SLOTS * 4) {
        // ------------------------------ K and V pages, 64 values at a time ------------------------------
        if (elect_one()) {
            bool ok = true;
            const int* table = p.block_table + (size_t)p.prefix_row * p.max_pages + tile0;
            auto load = [&](int j, int page, int kv, int full, int empty) {
                const int b = j % X::STAGES;
                ok = mbar_wait(bar(empty + b), (j / X::STAGES & 1) ^ 1, abort_flag);
                if (!ok) return;
                mbar_arrive_expect_tx(bar(full + b), X::TILE);
                const uint32_t dst = base + (kv ? X::OFF_V : X::OFF_K) + b * X::TILE;
                const int y = ((page * 2 + kv) * p.n_kv_heads + kvh) * PAGE;
#pragma unroll
                for (int a = 0; a < DA; ++a) tma_load_2d(dst + a * X::K_ATOM, &map_kv, a * 64, y, bar(full + b));
            };
            // K a tile ahead of V: its places become free before V's do
            int page = LLM_CHECK_INDEX(table[0], p.n_pages), next = LLM_CHECK_INDEX(nt > 1 ? table[1] : 0, p.n_pages);
            load(0, page, 0, K_FULL, K_EMPTY);
            for (int j = 0; j < nt && ok; ++j) {
                const int after = j + 2 < nt ? table[j + 2] : 0;
                if (j + 1 < nt) load(j + 1, next, 0, K_FULL, K_EMPTY);
                if (ok) load(j, page, 1, V_FULL, V_EMPTY);
                page = next;
                next = LLM_CHECK_INDEX(after, p.n_pages);
            }
        }
    } else if (elect_one()) {
        // ------------------------------ products ------------------------------
        const int slots = both ? 2 : 1;
        auto issue_s = [&](int slot, int j) {
            const uint64_t q = smem_desc_sw128(base + slot * DA * ATOM), k = smem_desc_sw128(base + X::OFF_K + j % X::STAGES * X::TILE);
#pragma unroll
            for (int ks = 0; ks < D / 16; ++ks) {           // (a descriptor counts 16 bytes)
                const uint64_t keys16 = k + (ks >> 2) * (X::K_ATOM / 16) + 2 * (ks & 3);
                if constexpr (X::Q_TMEM) mma_f16_ts(tmem + buffer(slot, j) * BK, tmem + X::COL_Q + slot * (D / 2) + ks * 8, keys16, X::IDESC_S, ks > 0 ? 1u : 0u);
                else mma_f16(tmem + buffer(slot, j) * BK, q + (ks >> 2) * (ATOM / 16) + 2 * (ks & 3), keys16, X::IDESC_S, ks > 0 ? 1u : 0u);
            }
            mma_commit(bar(S_FULL + buffer(slot, j)));
        };
        auto issue_o = [&](int slot, int j) {
            const uint64_t v = smem_desc_mn_sw128(base + X::OFF_V + j % X::STAGES * X::TILE, X::K_ATOM);
#pragma unroll
            for (int ks = 0; ks < BK / 16; ++ks)            // 16 keys: 8 TMEM columns of P, 16 rows of the V tile
                mma_f16_ts(tmem + X::COL_O + slot * D, tmem + buffer(slot, j) * BK + ks * 8, v + ks * (16 * 128 / 16), X::IDESC_O, j > 0 || ks > 0 ? 1u : 0u);
            mma_commit(bar(PV_DONE + slot));
        };
        auto scores = [&](int j) {                          // of a tile of keys, all slots
            if (!mbar_wait(bar(K_FULL + j % X::STAGES), j / X::STAGES & 1, abort_flag)) return false;
            tc_fence_after();
            return true;
        };
        bool ok = mbar_wait(bar(Q_FULL), 0, abort_flag);
        for (int j = 0; j < min(2, nt) && ok; ++j) {
            ok = scores(j);
            if (!ok) break;
            for (int slot = 0; slot < slots; ++slot) issue_s(slot, j);
            mma_commit(bar(K_EMPTY + j % X::STAGES));
        }
        for (int j = 0; j < nt && ok; ++j) {
            ok = mbar_wait(bar(V_FULL + j % X::STAGES), j / X::STAGES & 1, abort_flag);
            for (int slot = 0; slot < slots && ok; ++slot) {
                ok = mbar_wait(bar(P_FULL + buffer(slot, j)), phase(j), abort_flag);
                if (!ok) break;
                tc_fence_after();
                issue_o(slot, j);
            }
            if (ok) mma_commit(bar(V_EMPTY + j % X::STAGES));
            if (j + 2 >= nt) continue;
            // The scores of tile j + 2 take the columns that P of tile j lies in.  Products of two shapes have no promised order, so P V is waited for; the other
            // slot's, or the softmax of tile j + 1, is at work meanwhile
            ok = ok && scores(j + 2);
            for (int slot = 0; slot < slots && ok; ++slot) {
                ok = mbar_wait(bar(PV_DONE + slot), j & 1, abort_flag);
                if (!ok) break;
                tc_fence_after();
                issue_s(slot, j + 2);
            }
            if (ok) mma_commit(bar(K_EMPTY + (j + 2) % X::STAGES));
        }
    }
    tc_fence_before();
    __syncthreads();
    teardown(abort_flag, tid, status);
    if (warp == SLOTS * 4 + 1) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

// ------------------------------------------------------------------------------------------------
// tails
// ------------------------------------------------------------------------------------------------
constexpr int MAX_PARTS = 64;
template <int D>
struct Tail {
    static constexpr int STAGES = 2, SUB = 16 * D * 2, PER_WARP = STAGES * 2 * SUB;      // SUB: a warp's 16 keys of K or V
    static constexpr int ROW = D + 8;                       // of a merged row: eight rows of an accumulator start 32 bytes apart, no two in one bank
    static constexpr int MERGE = 5 * 16 * (ROW + 2) * 4 + 16 * MAX_PARTS * 4;         // four warps' results and that of the last drafted keys; weights of parts
    static constexpr int BYTES = 4 * PER_WARP > MERGE ? 4 * PER_WARP : MERGE;
};

// A row among the lanes of a warp: D / 32 values each, four (two) neighbours at a time
template <int D> LLM_DEVICE int column(int e) { return D == 64 ? (threadIdx.x & 31) * 2 + e : (e >> 2) * 128 + (threadIdx.x & 31) * 4 + (e & 3); }
template <int D> LLM_DEVICE void load_row(const float* x, float (&v)[D / 32]) {
    if constexpr (D == 64) {
        const float2 t = __ldcg(reinterpret_cast<const float2*>(x + column<D>(0)));
        v[0] = t.x; v[1] = t.y;
    } else {
#pragma unroll
        for (int e = 0; e < D / 32; e += 4) {
            const float4 t = __ldcg(reinterpret_cast<const float4*>(x + column<D>(e)));
            v[e] = t.x; v[e + 1] = t.y; v[e + 2] = t.z; v[e + 3] = t.w;
        }
    }
}
template <int D> LLM_DEVICE void load_row_shared(const float* x, float (&v)[D / 32]) {
    if constexpr (D == 64) {
        const float2 t = *reinterpret_cast<const float2*>(x + column<D>(0));
        v[0] = t.x; v[1] = t.y;
    } else {
#pragma unroll
        for (int e = 0; e < D / 32; e += 4) {
            const float4 t = *reinterpret_cast<const float4*>(x + column<D>(e));
            v[e] = t.x; v[e + 1] = t.y; v[e + 2] = t.z; v[e + 3] = t.w;
        }
    }
}
template <int D> LLM_DEVICE void store_row(float* x, const float (&v)[D / 32]) {
    if constexpr (D == 64) {
        *reinterpret_cast<float2*>(x + column<D>(0)) = make_float2(v[0], v[1]);
    } else {
#pragma unroll
        for (int e = 0; e < D / 32; e += 4) *reinterpret_cast<float4*>(x + column<D>(e)) = make_float4(v[e], v[e + 1], v[e + 2], v[e + 3]);
    }
}
// `n` <= MAX_PARTS sets of keys, whose results lie `step` rows apart, join two rows.  Maxima and sums of all sets first, a lane each, which gives every set its
// weight (kept in `w`); the values of many sets of both rows are on their way meanwhile (a row after the other, eight sets at a time, it was 17000 clocks for six rows of 18
// parts of 256).
template <int D> LLM_DEVICE void join_parts(float (&m)[2], float (&l)[2], float (&acc)[2][D / 32], const float* part_o, const float* part_ml, const size_t (&first)[2], int step, int n,
                                            float* const (&w)[2]) {
    constexpr int N = D / 32, DEEP = N == 2 ? 16 : 8;
    const int lane = threadIdx.x & 31;
    float2 ml[2][2];
    float v[2][DEEP][N];
#pragma unroll
    for (int r = 0; r < 2; ++r)
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const int s = k * 32 + lane;
            ml[r][k] = s < n ? __ldcg(reinterpret_cast<const float2*>(part_ml + (first[r] + (size_t)s * step) * 2)) : make_float2(-INFINITY, 0.f);
        }
    auto load = [&](int s0) {
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int k = 0; k < DEEP; ++k) load_row<D>(part_o + (first[r] + (size_t)min(s0 + k, n - 1) * step) * D, v[r][k]);
    };
    load(0);
#pragma unroll
    for (int r = 0; r < 2; ++r) {
        const float top = fmaxf(m[r], warp_max(fmaxf(ml[r][0].x, ml[r][1].x))), base = top == -INFINITY ? 0.f : top;
        float sum = 0.f;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            const float c = ex2(ml[r][k].x - base);
            sum += c * ml[r][k].y;
            w[r][k * 32 + lane] = c;
        }
        const float old = ex2(m[r] - base);
        l[r] = l[r] * old + warp_sum(sum);
        m[r] = top;
#pragma unroll
        for (int e = 0; e < N; ++e) acc[r][e] *= old;
    }
    __syncwarp();
    for (int s0 = 0; s0 < n; s0 += DEEP) {
        if (s0 > 0) load(s0);
#pragma unroll
        for (int r = 0; r < 2; ++r)
#pragma unroll
            for (int k = 0; k < DEEP; ++k) {
                const float c = w[r][s0 + k];               // (0 from n on)
#pragma unroll
                for (int e = 0; e < N; ++e) acc[r][e] += c * v[r][k][e];
            }
    }
    __syncwarp();
}

template <int D>
__global__ void __launch_bounds__(128, D == 64 ? 4 : D == 128 ? 3 : 1) attn_tail_kernel(const AttnSharedParams p) {
    extern __shared__ __align__(128) uint8_t smem[];
    using SM = Tail<D>;
    pdl_trigger();
    if (p.splits == 0) pdl_wait();                          // no prefix kernel in front: the rows come from the one before
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int kvh = blockIdx.x, split = blockIdx.y, seq = blockIdx.z;
    const int G = p.n_heads / p.n_kv_heads, R = p.rows_per_seq, rows = G * R;
    const int prefix = prefix_of(p), seq_len = max(0, min(p.seq_lens[seq], p.max_pages * PAGE));
    const bool joins = prefix > 0 && shares(p, seq, prefix);
    // keys [start, stop) are seen by every row, [stop, seq_len) by the later ones; row r sees keys < seq_len - (R - 1 - r)
    const int start = joins ? prefix : 0, stop = max(start, seq_len - (R - 1));
    const int page0 = start / PAGE, n_pages = (stop + PAGE - 1) / PAGE;
    const int per = (max(0, n_pages - page0) + (int)gridDim.y - 1) / (int)gridDim.y;
    const int pg0 = page0 + split * per, pg1 = stop > start ? min(n_pages, pg0 + per) : pg0;
    const int* btab = p.block_table + (size_t)seq * p.max_pages;
    const uint32_t wbase = smem_u32(smem) + warp * SM::PER_WARP;
    auto page_of = [&](int pg, int kv) {
        const size_t page = (size_t)LLM_CHECK_INDEX(btab[pg], p.n_pages);
        return p.kv + ((page * 2 + kv) * p.n_kv_heads + kvh) * (size_t)(PAGE * D);
    };
    auto query = [&](int i) { return p.q + ((size_t)(seq * R + i / G) * p.n_heads + kvh * G + i % G) * D; };

    auto issue = [&](int pg, int stage) {
        if (pg < pg1) {
            const __nv_bfloat16 *kp = page_of(pg, 0) + (size_t)warp * 16 * D, *vp = page_of(pg, 1) + (size_t)warp * 16 * D;
            const uint32_t kb = wbase + stage * 2 * SM::SUB, vb = kb + SM::SUB;
            constexpr int UPR = D / 8;                       // 16-byte units per row
#pragma unroll
            for (int t = 0; t < 16 * UPR / 32; ++t) {
                const int idx = t * 32 + lane, row = idx / UPR, unit = idx % UPR;
                cp_async16(tile_addr<D>(kb, row, unit), kp + row * D + unit * 8);
                cp_async16(tile_addr<D>(vb, row, unit), vp + row * D + unit * 8);
            }
        }
        cp_async_commit();
    };
#pragma unroll
    for (int s = 0; s < SM::STAGES - 1; ++s) issue(pg0 + s, s);

    // Q fragments: MMA row i <-> (row i / G of the sequence, head i % G of the group)
    uint32_t qa[D / 16][4];
    const int i0 = lane >> 2, i1 = i0 + 8;
    {
        const int cq = (lane & 3) * 2;
        const __nv_bfloat16 *q0 = i0 < rows ? query(i0) : nullptr, *q1 = i1 < rows ? query(i1) : nullptr;
#pragma unroll
        for (int ks = 0; ks < D / 16; ++ks) {
            const int d0 = ks * 16 + cq;
            qa[ks][0] = q0 ? *reinterpret_cast<const uint32_t*>(q0 + d0) : 0u;
            qa[ks][1] = q1 ? *reinterpret_cast<const uint32_t*>(q1 + d0) : 0u;
            qa[ks][2] = q0 ? *reinterpret_cast<const uint32_t*>(q0 + d0 + 8) : 0u;
            qa[ks][3] = q1 ? *reinterpret_cast<const uint32_t*>(q1 + d0 + 8) : 0u;
        }
    }
    float o[D / 8][4];
#pragma unroll
    for (int n = 0; n < D / 8; ++n)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[n][i] = 0.f;
    float m0 = -INFINITY, m1 = -INFINITY, l0 = 0.f, l1 = 0.f;
    const float sl2 = p.scale * LOG2E;

    for (int pg = pg0; pg < pg1; ++pg) {
        const int stage = (pg - pg0) % SM::STAGES;
        issue(pg + SM::STAGES - 1, (pg - pg0 + SM::STAGES - 1) % SM::STAGES);
        cp_async_wait<SM::STAGES - 1>();
        __syncwarp();
        const uint32_t kb = wbase + stage * 2 * SM::SUB, vb = kb + SM::SUB;
        const int first = pg * PAGE + warp * 16, lo = start - first, hi = stop - first;       // this warp's keys that count: [lo, hi) of 16
        if (lo > 0 || hi < 16) {
            constexpr int UPR = D / 8;
            for (int idx = lane; idx < 16 * UPR; idx += 32) {
                const int row = idx / UPR;
                if (row < lo || row >= hi) st_shared_v4(tile_addr<D>(vb, row, idx % UPR), make_uint4(0, 0, 0, 0));
            }
            __syncwarp();
        }
        float s[2][4];
        qk_16keys<D>(qa, kb, lane, s);
        float mx0 = -INFINITY, mx1 = -INFINITY;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int key = (lane & 3) * 2 + nb * 8 + e;
                const bool in = key >= lo && key < hi;
                s[nb][e] = in ? s[nb][e] * sl2 : -INFINITY;
                s[nb][2 + e] = in ? s[nb][2 + e] * sl2 : -INFINITY;
                mx0 = fmaxf(mx0, s[nb][e]);
                mx1 = fmaxf(mx1, s[nb][2 + e]);
            }
        }
        mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 1)); mx0 = fmaxf(mx0, __shfl_xor_sync(0xffffffffu, mx0, 2));
        mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 1)); mx1 = fmaxf(mx1, __shfl_xor_sync(0xffffffffu, mx1, 2));
        const float nm0 = fmaxf(m0, mx0), nm1 = fmaxf(m1, mx1);
        const float base0 = nm0 == -INFINITY ? 0.f : nm0, base1 = nm1 == -INFINITY ? 0.f : nm1;
        const float c0 = exp2f(m0 - base0), c1 = exp2f(m1 - base1);
        m0 = nm0; m1 = nm1;
        float ps0 = 0.f, ps1 = 0.f;
#pragma unroll
        for (int nb = 0; nb < 2; ++nb) {
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                s[nb][e] = exp2f(s[nb][e] - base0); ps0 += s[nb][e];
                s[nb][2 + e] = exp2f(s[nb][2 + e] - base1); ps1 += s[nb][2 + e];
            }
        }
        l0 = l0 * c0 + ps0; l1 = l1 * c1 + ps1;
#pragma unroll
        for (int n = 0; n < D / 8; ++n) { o[n][0] *= c0; o[n][1] *= c0; o[n][2] *= c1; o[n][3] *= c1; }
        uint32_t pa[4];
        pa[0] = pack_bf16(s[0][0], s[0][1]); pa[1] = pack_bf16(s[0][2], s[0][3]);
        pa[2] = pack_bf16(s[1][0], s[1][1]); pa[3] = pack_bf16(s[1][2], s[1][3]);
        pv_16keys<D>(pa, vb, lane, o);
        __syncwarp();
    }
    cp_async_wait<0>();
    l0 += __shfl_xor_sync(0xffffffffu, l0, 1); l0 += __shfl_xor_sync(0xffffffffu, l0, 2);
    l1 += __shfl_xor_sync(0xffffffffu, l1, 1); l1 += __shfl_xor_sync(0xffffffffu, l1, 2);
    __syncthreads();

    // ---- the four warps' results (disjoint keys) and those of the last drafted keys, in shared memory ----
    constexpr int VPL = D / 32, ROW = SM::ROW;
    const int sets = R > 1 ? 5 : 4;
    float* s_o = reinterpret_cast<float*>(smem);             // [5][16][ROW]
    float* s_ml = s_o + 5 * 16 * ROW;                        // [5][16][2]
    float* s_w = s_ml + 5 * 16 * 2;                          // [16][MAX_PARTS]
#pragma unroll
    for (int n = 0; n < D / 8; ++n) {
        const int col = n * 8 + (lane & 3) * 2;
        *reinterpret_cast<float2*>(&s_o[(warp * 16 + i0) * ROW + col]) = make_float2(o[n][0], o[n][1]);
        *reinterpret_cast<float2*>(&s_o[(warp * 16 + i1) * ROW + col]) = make_float2(o[n][2], o[n][3]);
    }
    if ((lane & 3) == 0) {
        s_ml[(warp * 16 + i0) * 2] = m0; s_ml[(warp * 16 + i0) * 2 + 1] = l0;
        s_ml[(warp * 16 + i1) * 2] = m1; s_ml[(warp * 16 + i1) * 2 + 1] = l1;
    }
    for (int i = warp; R > 1 && i < rows; i += 4) {          // a warp per row: keys stop .. seq_len - (R - 1 - r), one by one
        float m = -INFINITY, l = 0.f, acc[VPL], x[VPL];
#pragma unroll
        for (int e = 0; e < VPL; ++e) { acc[e] = 0.f; x[e] = 0.f; }
        const int end = seq_len - (R - 1 - i / G);
        if (split == 0 && stop < end) {
#pragma unroll
            for (int e = 0; e < VPL; ++e) x[e] = __bfloat162float(query(i)[column<D>(e)]);
            for (int key = stop; key < end; ++key) {
                const size_t at = (size_t)(key % PAGE) * D;
                const __nv_bfloat16 *k = page_of(key / PAGE, 0) + at, *v = page_of(key / PAGE, 1) + at;
                float kx[VPL], vx[VPL], d = 0.f;
#pragma unroll
                for (int e = 0; e < VPL; ++e) { kx[e] = __bfloat162float(k[column<D>(e)]); vx[e] = __bfloat162float(v[column<D>(e)]); }
#pragma unroll
                for (int e = 0; e < VPL; ++e) d += x[e] * kx[e];
                const float score = warp_sum(d) * sl2, top = fmaxf(m, score);
                if (top == -INFINITY && score == -INFINITY) continue;       // (a score that is no number goes on, and makes the row one that is none)
                const float c = exp2f(m - top), w = exp2f(score - top);
                m = top;
                l = l * c + w;
#pragma unroll
                for (int e = 0; e < VPL; ++e) acc[e] = acc[e] * c + w * vx[e];
            }
        }
        store_row<D>(&s_o[(4 * 16 + i) * ROW], acc);
        if (lane == 0) { s_ml[(4 * 16 + i) * 2] = m; s_ml[(4 * 16 + i) * 2 + 1] = l; }
    }
    __syncthreads();

    // the quotient and the gate
    struct Gate { __nv_bfloat16 x[VPL]; };
    auto gate_of = [&](int i) {                              // on its way while the parts are
        Gate g;
        const __nv_bfloat16* x = p.gate + (size_t)(seq * R + i / G) * p.gate_token + (size_t)(kvh * G + i % G) * p.gate_head;
#pragma unroll
        for (int e = 0; e < VPL; ++e) g.x[e] = p.gate ? x[column<D>(e)] : __nv_bfloat16();
        return g;
    };
    auto finish = [&](int i, float l, float (&acc)[VPL], const Gate& g) {
        const size_t token = (size_t)seq * R + i / G;
        const int head = kvh * G + i % G;
        const float inv = l == 0.f ? 0.f : 1.f / l;          // (a sum that is not a number makes the row one)
#pragma unroll
        for (int e = 0; e < VPL; ++e) {
            acc[e] = l == 0.f ? 0.f : acc[e] * inv;
            if (p.gate) acc[e] *= __fdividef(1.f, 1.f + __expf(-__bfloat162float(g.x[e])));
        }
        __nv_bfloat16* dst = p.out + (token * p.n_heads + head) * D;
#pragma unroll
        for (int e = 0; e < VPL; e += 2) *reinterpret_cast<uint32_t*>(dst + column<D>(e)) = pack_bf16(acc[e], acc[e + 1]);
    };
    const int S = (int)gridDim.y;
    const size_t mine = (((size_t)seq * p.n_kv_heads + kvh) * S + split) * 16;
    // rows i and i + 4 (the same one twice at the end): the prefix's parts join them
    auto prefix_parts = [&](int i, int i2, float (&m)[2], float (&l)[2], float (&acc)[2][VPL]) {
        const size_t first = ((size_t)kvh * p.n_seqs + seq) * rows;
        const size_t at[2] = {(first + i) * p.splits, (first + i2) * p.splits};
        float* const w[2] = {s_w + i * MAX_PARTS, s_w + i2 * MAX_PARTS};
        join_parts<D>(m, l, acc, p.part_o, p.part_ml, at, 1, parts_of(prefix, p.splits), w);
    };
    if (S == 1 && p.splits > 0) pdl_wait();                  // the prefix kernel's parts
    for (int i = warp; i < rows; i += 8) {
        const int i2 = i + 4 < rows ? i + 4 : i;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, acc[2][VPL] = {};
        Gate g[2] = {gate_of(i), gate_of(i2)};
        if (S == 1 && joins) prefix_parts(i, i2, m, l, acc);
#pragma unroll
        for (int r = 0; r < 2; ++r) {
            const int row = r ? i2 : i;
            if (r && i2 == i) break;
            float top = m[r];
            for (int w = 0; w < sets; ++w) top = fmaxf(top, s_ml[(w * 16 + row) * 2]);
            const float base = top == -INFINITY ? 0.f : top, old = ex2(m[r] - base);
            l[r] *= old;
#pragma unroll
            for (int e = 0; e < VPL; ++e) acc[r][e] *= old;
#pragma unroll 2
            for (int w = 0; w < sets; ++w) {
                const float wm = s_ml[(w * 16 + row) * 2], wl = s_ml[(w * 16 + row) * 2 + 1], c = ex2(wm - base);
                float v[VPL];
                load_row_shared<D>(&s_o[(w * 16 + row) * ROW], v);
                l[r] += c * wl;
#pragma unroll
                for (int e = 0; e < VPL; ++e) acc[r][e] += c * v[e];
            }
            if (S == 1) {
                finish(row, l[r], acc[r], g[r]);
            } else {
                store_row<D>(p.tail_o + (mine + row) * D, acc[r]);
                if (lane == 0) *reinterpret_cast<float2*>(p.tail_ml + (mine + row) * 2) = make_float2(top, l[r]);
            }
        }
    }
    if (S == 1) return;

    // ---- the last CTA of this (sequence, K/V head) joins the parts of its tail ----
    __shared__ int s_last;
    __syncthreads();
    if (threadIdx.x == 0) {
        unsigned t;      // releases this CTA's parts (every thread's, through the barrier) and acquires the others'
        asm volatile("atom.acq_rel.gpu.global.add.u32 %0, [%1], 1;" : "=r"(t) : "l"(&p.tickets[seq * p.n_kv_heads + kvh]) : "memory");
        s_last = t == (unsigned)S - 1;
        if (s_last) p.tickets[seq * p.n_kv_heads + kvh] = 0u;
    }
    __syncthreads();
    if (!s_last) return;
    if (p.splits > 0) pdl_wait();
    for (int i = warp; i < rows; i += 8) {
        const int i2 = i + 4 < rows ? i + 4 : i;
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f}, acc[2][VPL] = {};
        const size_t first = ((size_t)seq * p.n_kv_heads + kvh) * S * 16;
        const size_t at[2] = {first + i, first + i2};
        float* const w[2] = {s_w + i * MAX_PARTS, s_w + i2 * MAX_PARTS};
        join_parts<D>(m, l, acc, p.tail_o, p.tail_ml, at, 16, S, w);
        if (joins) prefix_parts(i, i2, m, l, acc);
        finish(i, l[0], acc[0], gate_of(i));
        if (i2 != i) finish(i2, l[1], acc[1], gate_of(i2));
    }
}

template <class K> static cudaError_t smem_for(K kernel, int bytes) { return cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes); }

template <int D, int SLOTS> static cudaError_t prefix(const AttnSharedParams& p, const CUtensorMap& map, int* status, cudaStream_t st) {
    using X = Prefix<D, SLOTS>;
    const cudaError_t e = smem_for(attn_prefix_kernel<D, SLOTS>, X::SMEM);
    if (e != cudaSuccess) return e;
    const int rows = p.n_seqs * p.rows_per_seq * (p.n_heads / p.n_kv_heads);
    return launch_pdl(attn_prefix_kernel<D, SLOTS>, dim3((rows + SLOTS * BQ - 1) / (SLOTS * BQ), p.n_kv_heads, p.splits), dim3(X::THREADS), X::SMEM, st, map, p, status);
}
template <int D> static cudaError_t tail(const AttnSharedParams& p, cudaStream_t st) {
    const cudaError_t e = smem_for(attn_tail_kernel<D>, Tail<D>::BYTES + 1024);
    if (e != cudaSuccess) return e;
    return launch_pdl(attn_tail_kernel<D>, dim3(p.n_kv_heads, p.tail_splits, p.n_seqs), dim3(128), Tail<D>::BYTES + 1024, st, p);
}

}  // namespace ash

// Parts of the keys: as many CTAs as fill the GPU once, two tiles (pages) of keys in each at least.
AttnSharedPlan attn_shared_plan(int n_seqs, int rows_per_seq, int n_heads, int n_kv_heads, int head_dim, int max_shared, int max_tail, int max_tickets) {
    AttnSharedPlan plan = {0, 1, 0, 0};
    const int G = n_heads / n_kv_heads;
    const long long rows = (long long)n_seqs * rows_per_seq * G;
    if (max_shared > 0 && rows > 0) {
        const int per_cta = head_dim == 256 || rows <= ash::BQ ? ash::BQ : 2 * ash::BQ, bk = ash::PAGE;
        const long long ctas = (rows + per_cta - 1) / per_cta * n_kv_heads, tiles = (max_shared + bk - 1) / bk;
        long long s = sm_count() / ctas;
        if (s > (tiles + 1) / 2) s = (tiles + 1) / 2;
        if (s > ash::MAX_PARTS) s = ash::MAX_PARTS;
        plan.splits = s < 1 ? 1 : (int)s;
    }
    const long long pairs = (long long)n_seqs * n_kv_heads, pages = (max_tail + ash::PAGE - 1) / ash::PAGE;
    long long t = pairs > 0 ? sm_count() * (head_dim == 256 ? 1 : head_dim == 128 ? 2 : 4) / pairs : 1;
    if (t > (pages + 1) / 2) t = (pages + 1) / 2;
    if (t > ash::MAX_PARTS) t = ash::MAX_PARTS;
    plan.tail_splits = t < 1 || pairs > max_tickets ? 1 : (int)t;
    plan.prefix_rows = rows * n_kv_heads * plan.splits;
    plan.tail_rows = plan.tail_splits > 1 ? pairs * plan.tail_splits * 16 : 0;
    return plan;
}

cudaError_t launch_attn_shared(const AttnSharedParams& p, int* status, cudaStream_t st) {
    if (p.n_seqs == 0) return cudaSuccess;
    if (p.n_heads % p.n_kv_heads || p.n_heads / p.n_kv_heads * p.rows_per_seq > 16) return cudaErrorInvalidValue;
    if (p.splits > 0) {
        // the cache as a matrix of head_dim columns: 64 rows per page, K or V, and head
        CUtensorMap map;
        const uint64_t rows = (uint64_t)p.n_pages * 2 * p.n_kv_heads * ash::PAGE;
        if (rows > INT32_MAX || !tc5::make_map(&map, p.kv, p.head_dim, rows, p.head_dim, ash::PAGE)) return cudaErrorInvalidValue;
        const bool two = (long long)p.n_seqs * p.rows_per_seq * (p.n_heads / p.n_kv_heads) > ash::BQ;
        cudaError_t e = cudaErrorInvalidValue;
        if (p.head_dim == 64) e = two ? ash::prefix<64, 2>(p, map, status, st) : ash::prefix<64, 1>(p, map, status, st);
        if (p.head_dim == 128) e = two ? ash::prefix<128, 2>(p, map, status, st) : ash::prefix<128, 1>(p, map, status, st);
        if (p.head_dim == 256) e = ash::prefix<256, 1>(p, map, status, st);
        if (e != cudaSuccess) return e;
    }
    if (p.head_dim == 64) return ash::tail<64>(p, st);
    if (p.head_dim == 128) return ash::tail<128>(p, st);
    if (p.head_dim == 256) return ash::tail<256>(p, st);
    return cudaErrorInvalidValue;
}

LLM_DEFINE_BOUNDS_STATUS_READER(bounds_status_attn_shared)

}  // namespace llm
