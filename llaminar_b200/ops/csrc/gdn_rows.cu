// The gated delta rule over several new rows of every sequence, one row after the other: the rows of a speculative verification, and prompts
// (short ones, and head sizes that the chunk-parallel kernels do not have).
//
//     y = silu(causal convolution of q | k | v)      q = y_q / |y_q| / sqrt(d),  k = y_k / |y_k|
//     a = exp(ssm_a softplus(alpha + dt_bias))       b = sigmoid(beta)
//     u = b (v - a S^T k)       S = a S + k u^T      o = S^T q       out = o / rms(o) * norm_w * silu(z)
//
// A CTA takes one value head of one sequence after the other; four neighbouring threads keep a column of the d x d state in registers, so that both products
// with the state are sums inside a thread (and two exchanges) and a row costs no barrier.  q, k and v of a block of four rows are convolved, normed and left in shared memory
// first; the next state, rows and gates are on their way meanwhile.
// What bounds it: few rows, the state's bytes (64 KB read per head at d = 128; written too unless the state is left alone); more rows, the chain of a row.  Prompts
// of 32 / 16 heads: one sequence of 16 rows 23 us, 32 of them 157 us.
//
// gdn_commit brings the state behind the accepted rows: a streaming pass, S = a S + k u^T for each of them, bound by the state's bytes in both
// directions (32 sequences x 48 heads: 200 MB in 35 us, 5.7 TB/s).
//
// (reference: the recurrence of src/v2/kernels/cuda/gdn/CUDAGatedDeltaNetKernels.cu and the verifier's state capture rows,
//  src/v2/models/qwen35/Qwen35Graph.cpp:886-887.)
#include <algorithm>

#include "hybrid.h"
#include "launch.h"
#include "pairs.cuh"
#include "tc_tile.cuh"

namespace llm {

constexpr int TB = 4;                                        // rows prepared together
constexpr int DRAFT_ROWS = 8;                                // most rows of a sequence that are drafts

struct GdnSeq {
    int first, rows;
    bool fresh;
    size_t slot;
};
LLM_DEVICE GdnSeq gdn_seq(const GdnParams& p, int b) {
    GdnSeq s;
    if (p.cu) {
        s.first = max(0, min(p.cu[b], p.n_rows));
        s.rows = max(0, min(p.cu[b + 1], p.n_rows) - s.first);
    } else {
        s.first = b * p.rows_per_seq;
        s.rows = p.rows_per_seq;
    }
    s.fresh = p.positions && s.rows > 0 && p.positions[s.first] == 0;
    s.slot = (size_t)LLM_CHECK_INDEX(p.slots[b], p.n_slots);
    return s;
}

// Four neighbouring threads have a column of the state, a quarter of its rows each.  What the next block of rows (or the next item's first one) needs is loaded
// while a block is at work, and the state of the next item too.  K4: four taps; another number of taps loads its rows when it needs them.
template <int D, bool KEEP, bool K4>
__global__ void __launch_bounds__(4 * D, 1) gdn_rows_kernel(const GdnParams p) {
    constexpr int THREADS = 4 * D, WARPS = THREADS / 32, EPL = D / 32, QUARTER = D / 4, ROW = D + 16;        // a quarter of a vector starts four banks behind the one before
    __shared__ __align__(16) float s_q[TB][ROW], s_k[TB][ROW];
    __shared__ float s_v[TB][D], s_o[TB][D], s_a[TB], s_b[TB];
    extern __shared__ __align__(16) float s_state[];         // two states [D][D], a quarter's 16-byte units XORed so that a column's four threads meet other banks
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int j = tid >> 2, part = tid & 3;                  // column of the state, quarter of its rows
    const int items = p.n_seqs * p.n_v, K = K4 ? 4 : p.K;
    pdl_wait();                                              // (no trigger: the windows behind it are shifted without waiting)
    auto seq_of = [&](int item) { return gdn_seq(p, min(item, items - 1) / p.n_v); };
    auto unit_of = [](int row, int u) { return u ^ (2 * (row / QUARTER)) % (D / 4); };       // 16-byte unit u of a row of the state

    auto fetch = [&](int item, const GdnSeq& q, int buffer) {
        if (item < items && q.rows > 0 && !q.fresh) {
            const float* from = p.rec + (q.slot * p.n_v + item % p.n_v) * (size_t)(D * D);
            float* to = s_state + buffer * D * D;
#pragma unroll 8
            for (int u = tid; u < D * D / 4; u += THREADS) {
                const int row = u / (D / 4);
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(to + row * D + unit_of(row, u % (D / 4)) * 4)), "l"(from + (size_t)u * 4) : "memory");
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };

    // this thread's channel: of q, k and v in the first three quarters of the threads
    const int kind = tid / D, i_ch = tid % D;
    auto channel = [&](int h) {
        const int kh = (h + p.v_head_offset) % p.n_k;
        return (kind == 0 ? kh : kind == 1 ? p.n_k + kh : 2 * p.n_k + h) * D + i_ch;
    };
    struct Block {                                           // of rows, as they were loaded
        float before[3], w[4];
        __nv_bfloat16 x[TB + 3], z[(TB + WARPS - 1) / WARPS][EPL], alpha, beta;
    };
    constexpr int MINE = (TB + WARPS - 1) / WARPS;           // rows of a block that a warp finishes
    auto load = [&](int item, const GdnSeq& q, int t0, Block& k) {
        const int h = item % p.n_v, last = q.rows - 1;
        if (q.rows == 0) return;
        if (K4 && kind < 3) {
            const int c = channel(h);
#pragma unroll
            for (int i = 0; i < TB + 3; ++i) k.x[i] = p.in[(size_t)(q.first + min(max(t0 + i - 3, 0), last)) * p.in_row + c];        // (behind the last row: that one)
#pragma unroll
            for (int i = 0; i < 4; ++i) k.w[i] = p.conv_w[(size_t)c * 4 + i];
            if (t0 == 0 && !q.fresh) {
                const float* x = p.conv + (q.slot * p.C + c) * (size_t)3;
#pragma unroll
                for (int i = 0; i < 3; ++i) k.before[i] = x[i];
            }
        }
        if (kind == 3 && i_ch < TB) {
            const __nv_bfloat16* ab = p.in + (size_t)(q.first + min(t0 + i_ch, last)) * p.in_row + p.ab_off;
            k.alpha = ab[h];
            k.beta = ab[p.n_v + h];
        }
#pragma unroll
        for (int r = 0; r < MINE; ++r) {
            const __nv_bfloat16* x = p.in + (size_t)(q.first + min(t0 + r * WARPS + warp, last)) * p.in_row + p.z_off + h * D;
#pragma unroll
            for (int e = 0; e < EPL; ++e)
                if (r * WARPS + warp < TB) k.z[r][e] = x[e * 32 + lane];
        }
    };

    int item = blockIdx.x, buffer = 0;
    GdnSeq q = seq_of(item), q1 = seq_of(item + gridDim.x);
    fetch(item, q, 0);
    Block now;
    load(item, q, 0, now);
    float gain[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) gain[e] = p.norm_w[e * 32 + lane];

    for (; item < items; item += gridDim.x, buffer ^= 1) {
        const int h = item % p.n_v, b = item / p.n_v, next = item + gridDim.x;
        const GdnSeq q2 = seq_of(next + gridDim.x);          // used by the item after this one
        fetch(next, q1, buffer ^ 1);
        if (q.rows == 0) {
            if (next < items) load(next, q1, 0, now);
            q = q1; q1 = q2;
            continue;
        }
        float* state = p.rec + ((q.slot * p.n_v + h) * D + part * QUARTER) * (size_t)D + j;
        f32x2 S[QUARTER / 2];
#pragma unroll 1
        for (int t0 = 0; t0 < q.rows; t0 += TB) {
            const int n = min(TB, q.rows - t0);
            // ---- convolution, SiLU, gates ----
            if (kind < 3) {
                float y[TB];
                if (K4) {
                    float x[TB + 3];
#pragma unroll
                    for (int i = 0; i < TB + 3; ++i) x[i] = i < 3 && t0 == 0 ? q.fresh ? 0.f : now.before[i % 3] : __bfloat162float(now.x[i]);
#pragma unroll
                    for (int i = 0; i < TB; ++i) y[i] = now.w[0] * x[i] + now.w[1] * x[i + 1] + now.w[2] * x[i + 2] + now.w[3] * x[i + 3];
                } else {
                    const int c = channel(h);
#pragma unroll
                    for (int r = 0; r < TB; ++r) y[r] = 0.f;
                    for (int i = 0; i < K; ++i) {
                        const float w = p.conv_w[(size_t)c * K + i];
#pragma unroll
                        for (int r = 0; r < TB; ++r) {
                            const int t = t0 + r + i - (K - 1);
                            y[r] += w * (t >= 0 ? __bfloat162float(p.in[(size_t)(q.first + min(t, q.rows - 1)) * p.in_row + c]) : q.fresh ? 0.f : p.conv[(q.slot * p.C + c) * (size_t)(K - 1) + (K - 1 + t)]);
                        }
                    }
                }
#pragma unroll
                for (int i = 0; i < TB; ++i) {
                    const float v = silu(y[i]);
                    if (kind == 2) s_v[i][i_ch] = v;
                    else (kind ? s_k : s_q)[i][i_ch + i_ch / QUARTER * 4] = v;
                }
            } else if (i_ch < n) {
                const float x = __bfloat162float(now.alpha) + p.dt_bias[h];
                s_a[i_ch] = expf(p.ssm_a[h] * (x > 20.f ? x : log1pf(expf(x))));
                s_b[i_ch] = 1.f / (1.f + expf(-__bfloat162float(now.beta)));
            }
            float z[MINE][EPL];
#pragma unroll
            for (int r = 0; r < MINE; ++r)
#pragma unroll
                for (int e = 0; e < EPL; ++e) z[r][e] = __bfloat162float(now.z[r][e]);
            // the next block is on its way from here on
            if (t0 + TB < q.rows) load(item, q, t0 + TB, now);
            else if (next < items) load(next, q1, 0, now);
            __syncthreads();
            // ---- norms, a warp per vector ----
            for (int i = warp; i < 2 * n; i += WARPS) {
                float* x = i < n ? s_q[i] : s_k[i - n];
                float ss = 0.f, v[EPL];
#pragma unroll
                for (int e = 0; e < EPL; ++e) {
                    const int k = e * 32 + lane;
                    v[e] = x[k + k / QUARTER * 4];
                    ss += v[e] * v[e];
                }
                const float r = rsqrtf(warp_sum(ss) + 1e-6f) * (i < n ? rsqrtf((float)D) : 1.f);
#pragma unroll
                for (int e = 0; e < EPL; ++e) {
                    const int k = e * 32 + lane;
                    x[k + k / QUARTER * 4] = v[e] * r;
                    if (KEEP && i >= n) p.keep_k[((size_t)(q.first + t0 + i - n) * p.n_v + h) * D + k] = v[e] * r;
                }
            }
            if (t0 == 0) asm volatile("cp.async.wait_group 1;" ::: "memory");     // this item's state; the next one's may still be on its way
            __syncthreads();
            if (t0 == 0) {
                const float* x = s_state + buffer * D * D + part * QUARTER * D + unit_of(part * QUARTER, j >> 2) * 4 + (j & 3);
#pragma unroll
                for (int i = 0; i < QUARTER / 2; ++i) S[i] = q.fresh ? pair(0.f, 0.f) : pair(x[2 * i * D], x[(2 * i + 1) * D]);
            }
            // ---- the rows ----
#pragma unroll 1
            for (int i = 0; i < n; ++i) {
                const float a = s_a[i];
                const float4 *k = reinterpret_cast<const float4*>(&s_k[i][part * (QUARTER + 4)]), *x = reinterpret_cast<const float4*>(&s_q[i][part * (QUARTER + 4)]);
                f32x2 d0 = pair(0.f, 0.f), d1 = d0, o0 = d0, o1 = d0;
#pragma unroll
                for (int e = 0; e < QUARTER / 4; ++e) {
                    const float4 f = k[e];
                    d0 = fma2(S[2 * e], pair(f.x, f.y), d0);
                    d1 = fma2(S[2 * e + 1], pair(f.z, f.w), d1);
                }
                const float2 e0 = both(d0), e1 = both(d1);
                float dot = (e0.x + e0.y) + (e1.x + e1.y);
                dot += __shfl_xor_sync(0xffffffffu, dot, 1);
                dot += __shfl_xor_sync(0xffffffffu, dot, 2);
                const float u = s_b[i] * (s_v[i][j] - a * dot);
#pragma unroll
                for (int e = 0; e < QUARTER / 4; ++e) {
                    const float4 f = k[e], g = x[e];
                    S[2 * e] = fma2(pair(f.x, f.y), pair(u, u), mul2(S[2 * e], pair(a, a)));
                    S[2 * e + 1] = fma2(pair(f.z, f.w), pair(u, u), mul2(S[2 * e + 1], pair(a, a)));
                    o0 = fma2(S[2 * e], pair(g.x, g.y), o0);
                    o1 = fma2(S[2 * e + 1], pair(g.z, g.w), o1);
                }
                const float2 f0 = both(o0), f1 = both(o1);
                float o = (f0.x + f0.y) + (f1.x + f1.y);
                o += __shfl_xor_sync(0xffffffffu, o, 1);
                o += __shfl_xor_sync(0xffffffffu, o, 2);
                if (part == 0) {
                    s_o[i][j] = o;
                    if (KEEP) {
                        const size_t at = (size_t)(q.first + t0 + i) * p.n_v + h;
                        p.keep_u[at * D + j] = u;
                        if (j == 0) p.keep_a[at] = a;
                    }
                }
            }
            __syncthreads();
            // ---- gated norm, a warp per row ----
#pragma unroll
            for (int r = 0; r < MINE; ++r) {
                const int i = r * WARPS + warp;
                if (i >= n) break;
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < EPL; ++e) ss += s_o[i][e * 32 + lane] * s_o[i][e * 32 + lane];
                const float f = rsqrtf(warp_sum(ss) / D + p.eps);
                __nv_bfloat16* dst = p.out + (size_t)(q.first + t0 + i) * p.out_row + h * D;
#pragma unroll
                for (int e = 0; e < EPL; ++e) dst[e * 32 + lane] = __float2bfloat16(s_o[i][e * 32 + lane] * f * gain[e] * silu(z[r][e]));
            }
        }
        if (KEEP) {                                          // a share of the convolution's inputs, for the commit
            const int c0 = (int)((long long)p.C * h / p.n_v), c1 = (int)((long long)p.C * (h + 1) / p.n_v);
            for (int i = tid; i < (c1 - c0) * q.rows; i += THREADS) {
                const int t = i / (c1 - c0), c = c0 + i % (c1 - c0);
                p.keep_x[((size_t)b * p.rows_per_seq + t) * p.C + c] = p.in[(size_t)(q.first + t) * p.in_row + c];
            }
        } else {
#pragma unroll
            for (int i = 0; i < QUARTER / 2; ++i) {
                const float2 x = both(S[i]);
                state[(size_t)(2 * i) * D] = x.x;
                state[(size_t)(2 * i + 1) * D] = x.y;
            }
        }
        q = q1; q1 = q2;
    }
}

// Drafted rows: at most TB of every sequence, in one block.  The states arrive by bulk copies, two at a time, an eighth each, 16 bytes further than the one before:
// the eight threads of two columns meet other banks.  (By 16-byte copies of all threads, 73 us at three rows of 32 x 48 heads, the loads in front of the
// barriers waited behind them.)  The state is left alone, so no row needs one of its own: with S in front of the first row, A_r the product of the decays up to row r
// and w_i = u_i decayed from row i to row r,
//     a S_r-1^T k_r = A_r S^T k_r + sum_{i<r} w_i (k_i.k_r)       o_r = A_r S^T q_r + sum_{i<=r} w_i (k_i.q_r)
// All products with S are one pass, and the chain of the rows is one of single numbers.  Two columns a thread, since what k and q take of shared memory's
// bandwidth is the longest phase.  (Row after row, the state in registers, 1700 clocks a row, 60 us; in one pass with a column a thread 51; now 46, 15 of them the
// states' bytes.)
template <int D, int TB, bool K4>
__global__ void __launch_bounds__(4 * D, D == 128 ? 1 : D == 64 ? 2 : 4) gdn_draft_kernel(const GdnParams p) {
    using namespace tc5;
    constexpr int THREADS = 4 * D, WARPS = THREADS / 32, EPL = D / 32, EIGHTH = D / 8, ROW = D + 32, STRIDE = EIGHTH * D + 4;
    __shared__ __align__(16) float s_q[TB][ROW], s_k[TB][ROW];
    __shared__ float s_v[TB][D], s_o[TB][D], s_a[TB], s_b[TB], s_kk[TB][TB], s_kq[TB][TB];
    __shared__ __align__(8) uint64_t s_bar[2];
    __shared__ int s_abort[2];                               // [1] stays 0 here (tc_common.cuh: restarts the wait clock when set)
    extern __shared__ __align__(16) float s_state[];         // two states of eight parts, STRIDE apart
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int j = tid >> 3, part = tid & 7, col = 2 * j + (part & 1);         // two columns, an eighth of their rows; the column whose sums end up here
    const int items = p.n_seqs * p.n_v, K = K4 ? 4 : p.K, n = p.rows_per_seq;
    const uint32_t bars = smem_u32(s_bar);
    volatile int* abort_flag = s_abort;
    if (tid == 0) {
        s_abort[0] = 0; s_abort[1] = 0;
        mbar_init(bars, 1);
        mbar_init(bars + 8, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    auto slot_of = [&](int item) { return (size_t)LLM_CHECK_INDEX(p.slots[item / p.n_v], p.n_slots); };
    auto fetch = [&](int item, size_t slot, int buffer) {    // by one thread
        const float* from = p.rec + (slot * p.n_v + item % p.n_v) * (size_t)(D * D);
        fence_proxy_async();                                 // what stood there has been read
        mbar_arrive_expect_tx(bars + buffer * 8, D * D * 4);
#pragma unroll
        for (int i = 0; i < 8; ++i) bulk_load(smem_u32(s_state + (buffer * 8 + i) * STRIDE), from + i * EIGHTH * D, EIGHTH * D * 4, bars + buffer * 8);
    };
    const int kind = tid / D, i_ch = tid % D;                // this thread's channel: of q, k and v in the first three quarters of the threads
    struct Rows {                                            // an item's, as they were loaded
        float before[3], w[4], ssm_a, dt;
        __nv_bfloat16 x[TB], z[EPL], alpha, beta;
    };
    auto channel = [&](int h) {
        const int kh = (h + p.v_head_offset) % p.n_k;
        return (kind == 0 ? kh : kind == 1 ? p.n_k + kh : 2 * p.n_k + h) * D + i_ch;
    };
    auto load = [&](int item, size_t slot, Rows& r) {
        const int h = item % p.n_v, first = item / p.n_v * n;
        if (kind < 3) {
            const int c = channel(h);
#pragma unroll
            for (int i = 0; i < TB; ++i) r.x[i] = p.in[(size_t)(first + min(i, n - 1)) * p.in_row + c];
            if (K4) {
                const float* window = p.conv + (slot * p.C + c) * (size_t)3;
#pragma unroll
                for (int i = 0; i < 4; ++i) r.w[i] = p.conv_w[(size_t)c * 4 + i];
#pragma unroll
                for (int i = 0; i < 3; ++i) r.before[i] = window[i];
            }
        } else if (i_ch < n) {
            const __nv_bfloat16* ab = p.in + (size_t)(first + i_ch) * p.in_row + p.ab_off;
            r.alpha = ab[h]; r.beta = ab[p.n_v + h];
            r.ssm_a = p.ssm_a[h]; r.dt = p.dt_bias[h];
        }
        if (warp < n) {
            const __nv_bfloat16* x = p.in + (size_t)(first + warp) * p.in_row + p.z_off + h * D;
#pragma unroll
            for (int e = 0; e < EPL; ++e) r.z[e] = x[e * 32 + lane];
        }
    };
    int item = blockIdx.x, buffer = 0;
    uint32_t phase = 0;                                      // of both barriers: it turns with every second item
    size_t slot = slot_of(item), slot1 = slot_of(min(item + (int)gridDim.x, items - 1));
    if (tid == THREADS - 1) fetch(item, slot, 0);             // (of the warps with the least to convolve)
    Rows now;
    load(item, slot, now);
    float gain[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) gain[e] = p.norm_w[e * 32 + lane];
    for (; item < items; item += gridDim.x) {
        const int h = item % p.n_v, b = item / p.n_v, first = b * n, next = item + gridDim.x;
        if (tid == THREADS - 1 && next < items) fetch(next, slot1, buffer ^ 1);          // (its place was read two barriers ago)
        const size_t slot2 = slot_of(min(next + (int)gridDim.x, items - 1));
        // ---- convolution, SiLU, gates ----
        if (kind < 3) {
            const int c = channel(h);
            float y[TB];
            if (K4) {
                float x[TB + 3];
#pragma unroll
                for (int i = 0; i < 3; ++i) x[i] = now.before[i];
#pragma unroll
                for (int i = 0; i < TB; ++i) x[i + 3] = __bfloat162float(now.x[i]);
#pragma unroll
                for (int i = 0; i < TB; ++i) y[i] = now.w[0] * x[i] + now.w[1] * x[i + 1] + now.w[2] * x[i + 2] + now.w[3] * x[i + 3];
            } else {
                const float* window = p.conv + (slot * p.C + c) * (size_t)(K - 1);
#pragma unroll
                for (int r = 0; r < TB; ++r) y[r] = 0.f;
                for (int i = 0; i < K; ++i) {
                    const float w = p.conv_w[(size_t)c * K + i];
#pragma unroll
                    for (int r = 0; r < TB; ++r) {
                        const int t = r + i - (K - 1);
                        y[r] += w * (t >= 0 ? __bfloat162float(p.in[(size_t)(first + min(t, n - 1)) * p.in_row + c]) : window[K - 1 + t]);
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                if (i >= n) break;
                const float v = silu(y[i]);
                if (kind == 2) s_v[i][i_ch] = v;
                else (kind ? s_k : s_q)[i][i_ch + i_ch / EIGHTH * 4] = v;
                // the convolution's inputs, for the commit: a channel of q and k by the first value head that reads it
                if (kind == 2 || (h < p.n_k && p.n_v >= p.n_k)) p.keep_x[((size_t)b * n + i) * p.C + c] = now.x[i];
            }
        } else {
            if (i_ch < n) {
                const float x = __bfloat162float(now.alpha) + now.dt;
                s_a[i_ch] = expf(now.ssm_a * (x > 20.f ? x : log1pf(expf(x))));
                s_b[i_ch] = 1.f / (1.f + expf(-__bfloat162float(now.beta)));
            }
            if (p.n_v < p.n_k) {                             // key heads that no value head reads: all of q and k, shared out
                const int all = 2 * p.n_k * D, c0 = (int)((long long)all * h / p.n_v), c1 = (int)((long long)all * (h + 1) / p.n_v);
                for (int c = c0 + i_ch; c < c1; c += D)
                    for (int i = 0; i < n; ++i) p.keep_x[((size_t)b * n + i) * p.C + c] = p.in[(size_t)(first + i) * p.in_row + c];
            }
        }
        float z[EPL];                                        // of the row that this warp finishes
#pragma unroll
        for (int e = 0; e < EPL; ++e) z[e] = __bfloat162float(now.z[e]);
        if (next < items) load(next, slot1, now);            // on their way from here on
        __syncthreads();
        // ---- norms, a warp per row ----
        if (warp < n) {
            float qs = 0.f, ks = 0.f, q[EPL], k[EPL];
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
                const int at = e * 32 + lane, to = at + at / EIGHTH * 4;
                q[e] = s_q[warp][to]; k[e] = s_k[warp][to];
                qs += q[e] * q[e]; ks += k[e] * k[e];
            }
            const float rq = rsqrtf(warp_sum(qs) + 1e-6f) * rsqrtf((float)D), rk = rsqrtf(warp_sum(ks) + 1e-6f);
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
                const int at = e * 32 + lane, to = at + at / EIGHTH * 4;
                s_q[warp][to] = q[e] * rq; s_k[warp][to] = k[e] * rk;
                p.keep_k[((size_t)(first + warp) * p.n_v + h) * D + at] = k[e] * rk;
            }
        }
        mbar_wait_warp(bars + buffer * 8, phase, abort_flag);
        f32x2 S[2][EIGHTH / 2];
        {
            const float* x = s_state + (buffer * 8 + part) * STRIDE + 2 * j;
#pragma unroll
            for (int i = 0; i < EIGHTH / 2; ++i) {
                const float2 even = *reinterpret_cast<const float2*>(x + 2 * i * D), odd = *reinterpret_cast<const float2*>(x + (2 * i + 1) * D);
                S[0][i] = pair(even.x, odd.x);
                S[1][i] = pair(even.y, odd.y);
            }
        }
        __syncthreads();
        if (abort_flag[0]) break;
        // ---- k.k and k.q of two rows, a warp per pair ----
        for (int x = warp; x < n * (n + 1) / 2; x += WARPS) {
            int r = 0;
#pragma unroll
            for (int e = 1; e < TB; ++e) r += x >= e * (e + 1) / 2;
            const int i = x - r * (r + 1) / 2;
            float kk = 0.f, kq = 0.f;
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
                const int at = e * 32 + lane, to = at + at / EIGHTH * 4;
                const float ki = s_k[i][to];
                kk += ki * s_k[r][to];
                kq += ki * s_q[r][to];
            }
            kk = warp_sum(kk);
            kq = warp_sum(kq);
            if (lane == 0) { s_kk[r][i] = kk; s_kq[r][i] = kq; }
        }
        // ---- S^T k and S^T q of all rows, with the state in front of them ----
        float dot[TB], o[TB];
#pragma unroll
        for (int r = 0; r < TB; ++r) {
            if (r >= n) break;
            const float4 *k4 = reinterpret_cast<const float4*>(&s_k[r][part * (EIGHTH + 4)]), *q4 = reinterpret_cast<const float4*>(&s_q[r][part * (EIGHTH + 4)]);
            f32x2 d[2] = {pair(0.f, 0.f), pair(0.f, 0.f)}, x[2] = {d[0], d[0]};
#pragma unroll
            for (int e = 0; e < EIGHTH / 4; ++e) {
                const float4 f = k4[e], g = q4[e];
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    d[c] = fma2(S[c][2 * e + 1], pair(f.z, f.w), fma2(S[c][2 * e], pair(f.x, f.y), d[c]));
                    x[c] = fma2(S[c][2 * e + 1], pair(g.z, g.w), fma2(S[c][2 * e], pair(g.x, g.y), x[c]));
                }
            }
            const float2 d0 = both(d[0]), d1 = both(d[1]), x0 = both(x[0]), x1 = both(x[1]);
            const bool odd = part & 1;
            const float ds[2] = {d0.x + d0.y, d1.x + d1.y}, xs[2] = {x0.x + x0.y, x1.x + x1.y};
            dot[r] = (odd ? ds[1] : ds[0]) + __shfl_xor_sync(0xffffffffu, odd ? ds[0] : ds[1], 1);
            o[r] = (odd ? xs[1] : xs[0]) + __shfl_xor_sync(0xffffffffu, odd ? xs[0] : xs[1], 1);
        }
#pragma unroll
        for (int off = 2; off < 8; off <<= 1)
#pragma unroll
            for (int r = 0; r < TB; ++r) {
                if (r >= n) break;
                dot[r] += __shfl_xor_sync(0xffffffffu, dot[r], off);
                o[r] += __shfl_xor_sync(0xffffffffu, o[r], off);
            }
        __syncthreads();
        // ---- the rows: their corrections, each decayed up to the row at hand, take the place of the states in between ----
        float w[TB], all = 1.f;
#pragma unroll
        for (int r = 0; r < TB; ++r) {
            if (r >= n) break;
            const float a = s_a[r];
            all *= a;
            float x = all * dot[r], y = all * o[r];
#pragma unroll
            for (int i = 0; i < r; ++i) {
                w[i] *= a;
                x = fmaf(w[i], s_kk[r][i], x);
                y = fmaf(w[i], s_kq[r][i], y);
            }
            w[r] = s_b[r] * (s_v[r][col] - x);
            if (part < 2) {
                s_o[r][col] = fmaf(w[r], s_kq[r][r], y);
                const size_t at = (size_t)(first + r) * p.n_v + h;
                p.keep_u[at * D + col] = w[r];
                if (col == 0) p.keep_a[at] = a;
            }
        }
        __syncthreads();
        // ---- gated norm, a warp per row ----
        if (warp < n) {
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < EPL; ++e) ss += s_o[warp][e * 32 + lane] * s_o[warp][e * 32 + lane];
            const float f = rsqrtf(warp_sum(ss) / D + p.eps);
            __nv_bfloat16* dst = p.out + (size_t)(first + warp) * p.out_row + h * D;
#pragma unroll
            for (int e = 0; e < EPL; ++e) dst[e * 32 + lane] = __float2bfloat16(s_o[warp][e * 32 + lane] * f * gain[e] * silu(z[e]));
        }
        slot = slot1; slot1 = slot2;
        phase ^= (uint32_t)buffer;
        buffer ^= 1;
    }
    __syncthreads();
    teardown(abort_flag, tid, p.status);
}

// One thread per channel of a sequence.  K - 1 values of [old window | rows], from the `n`th on; kept rows come from keep_x.
template <bool KEPT>
LLM_DEVICE void gdn_shift(const GdnParams& p, const GdnSeq& q, int b, int c, int n) {
    float* w = p.conv + (q.slot * p.C + c) * (size_t)(p.K - 1);
    for (int i = 0; i < p.K - 1; ++i) {                      // w[i] comes from place n + i >= i: not yet overwritten
        const int t = n + i - (p.K - 1);
        float x;
        if (t < 0) x = q.fresh ? 0.f : w[n + i];
        else if (KEPT) x = __bfloat162float(p.keep_x[((size_t)b * p.rows_per_seq + t) * p.C + c]);
        else x = __bfloat162float(p.in[(size_t)(q.first + t) * p.in_row + c]);
        w[i] = x;
    }
}

__global__ void __launch_bounds__(256) gdn_windows_kernel(const GdnParams p) {
    const int c = blockIdx.x * 256 + threadIdx.x, b = blockIdx.y;
    const GdnSeq q = gdn_seq(p, b);
    if (c < p.C && q.rows > 0) gdn_shift<false>(p, q, b, c, q.rows);
    pdl_wait();                                             // (the scan of the chunk form reads no windows and runs beside this)
}

// A block has half a state at d = 128, a whole one otherwise: 32 KB at most, so that an SM has four or more of them on their way.  The kept rows come in together.
template <int D> constexpr int COMMIT_PARTS = D == 128 ? 2 : 1;
template <int D>
__global__ void __launch_bounds__(256, 4) gdn_commit_kernel(const GdnParams p, const int* accepted) {
    constexpr int BLOCK = 16;                                // kept rows in shared memory at a time
    __shared__ __align__(16) float s_u[BLOCK][D], s_k[BLOCK][D];
    __shared__ float s_a[BLOCK];
    const int b = blockIdx.y, tid = threadIdx.x, R = p.rows_per_seq;
    pdl_wait();
    const int n = max(0, min(accepted[b], R));
    if (n == 0) return;
    const GdnSeq q = gdn_seq(p, b);
    constexpr int PARTS = COMMIT_PARTS<D>;
    if ((int)blockIdx.x >= p.n_v * PARTS) {                  // the convolution's windows
        const int c = ((int)blockIdx.x - p.n_v * PARTS) * 256 + tid;
        if (c < p.C) gdn_shift<true>(p, q, b, c, n);
        return;
    }
    const int h = blockIdx.x / PARTS;
    const size_t kept = (size_t)b * R * p.n_v + h;           // of the sequence's first kept row; the next one is n_v further
    constexpr int QUADS = D / 4, STEP = 256 / QUADS, PER = D / PARTS / STEP;       // a thread has PER rows i of four columns
    const int j4 = tid % QUADS, i0 = blockIdx.x % PARTS * (D / PARTS) + tid / QUADS;
    float4* state = reinterpret_cast<float4*>(p.rec + (q.slot * p.n_v + h) * (size_t)(D * D)) + i0 * QUADS + j4;
    f32x2 S[PER][2];
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const float4 x = __ldcs(state + e * STEP * QUADS);
        S[e][0] = pair(x.x, x.y);
        S[e][1] = pair(x.z, x.w);
    }
    for (int r0 = 0; r0 < n; r0 += BLOCK) {
        const int rows = min(BLOCK, n - r0);
        __syncthreads();
#pragma unroll 4
        for (int i = tid; i < rows * QUADS; i += 256) {
            const int r = i / QUADS, c = i % QUADS * 4;
            const size_t at = (kept + (size_t)(r0 + r) * p.n_v) * D + c;
            const float4 u = *reinterpret_cast<const float4*>(p.keep_u + at), k = *reinterpret_cast<const float4*>(p.keep_k + at);
            *reinterpret_cast<float4*>(&s_u[r][c]) = u;
            *reinterpret_cast<float4*>(&s_k[r][c]) = k;
        }
        if (tid < rows) s_a[tid] = p.keep_a[kept + (size_t)(r0 + tid) * p.n_v];
        __syncthreads();
#pragma unroll 1
        for (int r = 0; r < rows; ++r) {
            const float4 u = *reinterpret_cast<const float4*>(&s_u[r][j4 * 4]);
            const f32x2 a = pair(s_a[r], s_a[r]), u0 = pair(u.x, u.y), u1 = pair(u.z, u.w);
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const float k = s_k[r][i0 + e * STEP];
                S[e][0] = fma2(pair(k, k), u0, mul2(a, S[e][0]));
                S[e][1] = fma2(pair(k, k), u1, mul2(a, S[e][1]));
            }
        }
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) {
        const float2 x = both(S[e][0]), y = both(S[e][1]);
        state[e * STEP * QUADS] = make_float4(x.x, x.y, y.x, y.y);
    }
}

LLM_DEFINE_BOUNDS_STATUS_READER(bounds_status_gdn_rows)

template <int D> static cudaError_t rows_of(const GdnParams& p, cudaStream_t st) {
    constexpr int SMEM = 2 * D * D * 4;
    const long long items = (long long)p.n_v * p.n_seqs;
    if (items > INT32_MAX / 2) return cudaErrorInvalidValue;
    const unsigned ctas = (unsigned)std::min<long long>(items, sm_count() * (D == 128 ? 1 : D == 64 ? 2 : 4));        // as many as fit at once
    auto go = [&](auto kernel) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return e;
        return launch_pdl(kernel, dim3(ctas), dim3(4 * D), SMEM, st, p);
    };
    if (p.keep_u) return p.K == 4 ? go(gdn_rows_kernel<D, true, true>) : go(gdn_rows_kernel<D, true, false>);
    return p.K == 4 ? go(gdn_rows_kernel<D, false, true>) : go(gdn_rows_kernel<D, false, false>);
}
template <int D> static cudaError_t drafts_of(const GdnParams& p, cudaStream_t st) {
    constexpr int SMEM = 2 * (D * D + 4 * 8) * 4;
    const long long items = (long long)p.n_v * p.n_seqs;
    if (items > INT32_MAX / 2) return cudaErrorInvalidValue;
    const unsigned ctas = (unsigned)std::min<long long>(items, sm_count() * (D == 128 ? 1 : D == 64 ? 2 : 4));        // as many as fit at once
    auto go = [&](auto kernel) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return e;
        return launch_pdl(kernel, dim3(ctas), dim3(4 * D), SMEM, st, p);
    };
    constexpr int MOST = D == 32 ? 4 : DRAFT_ROWS;           // a warp finishes a row
    if (p.rows_per_seq > 4 && MOST > 4) return p.K == 4 ? go(gdn_draft_kernel<D, MOST, true>) : go(gdn_draft_kernel<D, MOST, false>);
    return p.K == 4 ? go(gdn_draft_kernel<D, 4, true>) : go(gdn_draft_kernel<D, 4, false>);
}
cudaError_t launch_gdn_rows(const GdnParams& p, cudaStream_t st) {
    if (p.n_seqs == 0 || p.n_rows == 0) return cudaSuccess;
    if (p.keep_u && p.rows_per_seq <= (p.d == 32 ? 4 : DRAFT_ROWS)) {
        switch (p.d) {
            case 32: return drafts_of<32>(p, st);
            case 64: return drafts_of<64>(p, st);
            case 128: return drafts_of<128>(p, st);
            default: return cudaErrorNotSupported;
        }
    }
    switch (p.d) {
        case 32: return rows_of<32>(p, st);
        case 64: return rows_of<64>(p, st);
        case 128: return rows_of<128>(p, st);
        default: return cudaErrorNotSupported;
    }
}
cudaError_t launch_gdn_windows(const GdnParams& p, cudaStream_t st) {
    if (p.n_seqs == 0 || p.n_rows == 0) return cudaSuccess;
    return launch_pdl(gdn_windows_kernel, dim3((p.C + 255) / 256, p.n_seqs), dim3(256), 0, st, p);
}
cudaError_t launch_gdn_commit(const GdnParams& p, const int* accepted, cudaStream_t st) {
    if (p.n_seqs == 0 || p.rows_per_seq == 0) return cudaSuccess;
    const dim3 grid(p.n_v * (p.d == 128 ? COMMIT_PARTS<128> : 1) + (p.C + 255) / 256, p.n_seqs);
    switch (p.d) {
        case 32: return launch_pdl(gdn_commit_kernel<32>, grid, dim3(256), 0, st, p, accepted);
        case 64: return launch_pdl(gdn_commit_kernel<64>, grid, dim3(256), 0, st, p, accepted);
        case 128: return launch_pdl(gdn_commit_kernel<128>, grid, dim3(256), 0, st, p, accepted);
        default: return cudaErrorNotSupported;
    }
}

}  // namespace llm
