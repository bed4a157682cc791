// The gated delta rule over several new rows of every sequence, one row after the other: the rows of a speculative verification, and prompts
// (short ones, and head sizes that the chunk-parallel kernels do not have).
//
//     y = silu(causal convolution of q | k | v)      q = y_q / |y_q| / sqrt(d),  k = y_k / |y_k|
//     a = exp(ssm_a softplus(alpha + dt_bias))       b = sigmoid(beta)
//     u = b (v - a S^T k)       S = a S + k u^T      o = S^T q       out = o / rms(o) * norm_w * silu(z)
//
// A CTA has one value head of one sequence; two neighbouring threads keep a column of the d x d state in registers, so that both products with the state are
// sums inside a thread (and one exchange) and a row costs no barrier.  q, k and v of a block of four rows are convolved, normed and left in shared memory
// first; the loads of the state, of the rows and of the gates are all on their way together.
// What bounds it: few rows, the state's bytes (64 KB read per head at d = 128; written too unless the state is left alone); more rows, the chain of a row.
//
// gdn_commit brings the state behind the accepted rows: a streaming pass, S = A S + sum_r k_r (u_r prod_{s > r} a_s)^T, bound by the
// state's bytes in both directions.
//
// (reference: the recurrence of src/v2/kernels/cuda/gdn/CUDAGatedDeltaNetKernels.cu and the verifier's state capture rows,
//  src/v2/models/qwen35/Qwen35Graph.cpp:886-887.)
#include "hybrid.h"
#include "pairs.cuh"

namespace llm {

constexpr int TB = 4;                                        // rows prepared together

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

// K4: four taps, a row loaded once per channel; another number of taps loads rows again.
template <int D, bool KEEP, bool K4>
__global__ void __launch_bounds__(2 * D, D == 128 ? 2 : 4) gdn_rows_kernel(const GdnParams p) {
    constexpr int WARPS = 2 * D / 32, EPL = D / 32, HALF = D / 2, ROW = D + 4;             // the second half of a vector starts four banks further
    constexpr int MINE = (TB + WARPS - 1) / WARPS;           // rows of a block that a warp finishes
    __shared__ __align__(16) float s_q[TB][ROW], s_k[TB][ROW];
    __shared__ float s_v[TB][D], s_o[TB][D], s_a[TB], s_b[TB];
    extern __shared__ __align__(16) float s_state[];         // [D][D]; the second half of the rows with its columns XORed by 16, so that a column's two threads meet other banks
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int j = tid >> 1, part = tid & 1;                  // column of the state, half of its rows
    const int items = p.n_seqs * p.n_v;
    // the state of an item, on its way while the item before it is at work
    auto fetch = [&](int item) {
        if (item < items) {
            const GdnSeq q = gdn_seq(p, item / p.n_v);
            if (q.rows > 0 && !q.fresh) {
                const float* from = p.rec + (q.slot * p.n_v + item % p.n_v) * (size_t)(D * D);
#pragma unroll 8
                for (int u = tid; u < D * D / 4; u += 2 * D) {
                    const int row = u / (D / 4), at = u % (D / 4) ^ (row >= HALF ? 4 : 0);
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(smem_u32(s_state + row * D + at * 4)), "l"(from + (size_t)u * 4) : "memory");
                }
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    fetch(blockIdx.x);
    float gain[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) gain[e] = p.norm_w[e * 32 + lane];

    for (int item = blockIdx.x; item < items; item += gridDim.x) {
        const int h = item % p.n_v, b = item / p.n_v;
        const GdnSeq q = gdn_seq(p, b);
        if (q.rows == 0) {
            fetch(item + gridDim.x);
            continue;
        }
        const int K = K4 ? 4 : p.K, kh = (h + p.v_head_offset) % p.n_k;
        const float* window = p.conv + q.slot * (size_t)p.C * (K - 1);
        float* state = p.rec + ((q.slot * p.n_v + h) * D + part * HALF) * (size_t)D + j;
        const float ssm_a = p.ssm_a[h], dt = p.dt_bias[h];
        // this thread's channel of q (first half of the threads) or k, and of v (first half)
        const int c_qk = tid < D ? kh * D + tid : (p.n_k + kh) * D + tid - D, c_v = 2 * p.n_k * D + h * D + tid;

        // channel c of n rows from t0: convolution and SiLU
        auto convolved = [&](int c, int t0, int n, float (&y)[TB]) {
            auto row = [&](int t) { return p.in[(size_t)(q.first + min(t, q.rows - 1)) * p.in_row + c]; };      // (behind the last row: that one)
            auto before = [&](int t) { return q.fresh ? 0.f : window[(size_t)c * (K - 1) + (K - 1 + t)]; };    // t < 0
            if (K4) {
                float x[TB + 3], w[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) w[i] = p.conv_w[(size_t)c * 4 + i];
                __nv_bfloat16 in[TB + 3];
#pragma unroll
                for (int i = 0; i < TB + 3; ++i) in[i] = row(max(t0 + i - 3, 0));
                if (t0 == 0) {
#pragma unroll
                    for (int i = 0; i < 3; ++i) x[i] = before(i - 3);
                } else {
#pragma unroll
                    for (int i = 0; i < 3; ++i) x[i] = __bfloat162float(in[i]);
                }
#pragma unroll
                for (int i = 3; i < TB + 3; ++i) x[i] = __bfloat162float(in[i]);
#pragma unroll
                for (int i = 0; i < TB; ++i) y[i] = w[0] * x[i] + w[1] * x[i + 1] + w[2] * x[i + 2] + w[3] * x[i + 3];
            } else {
#pragma unroll
                for (int i = 0; i < TB; ++i) y[i] = 0.f;
                for (int i = 0; i < K; ++i) {
                    const float w = p.conv_w[(size_t)c * K + i];
#pragma unroll
                    for (int r = 0; r < TB; ++r) {
                        const int t = t0 + r + i - (K - 1);
                        y[r] += w * (t >= 0 ? __bfloat162float(row(t)) : before(t));
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < TB; ++i) y[i] = silu(y[i]);
        };

        f32x2 S[HALF / 2];
        for (int t0 = 0; t0 < q.rows; t0 += TB) {
            const int n = min(TB, q.rows - t0);
            __nv_bfloat16 z[MINE][EPL];                          // of the rows that this warp finishes
#pragma unroll
            for (int r = 0; r < MINE; ++r) {
                const __nv_bfloat16* x = p.in + (size_t)(q.first + min(t0 + r * WARPS + warp, q.rows - 1)) * p.in_row + p.z_off + h * D;
#pragma unroll
                for (int e = 0; e < EPL; ++e) z[r][e] = x[e * 32 + lane];
            }
            float alpha = 0.f, beta = 0.f;
            if (tid < n) {
                const __nv_bfloat16* ab = p.in + (size_t)(q.first + t0 + tid) * p.in_row + p.ab_off;
                alpha = __bfloat162float(ab[h]);
                beta = __bfloat162float(ab[p.n_v + h]);
            }
            float y[TB], v[TB];
            convolved(c_qk, t0, n, y);
            if (tid < D) convolved(c_v, t0, n, v);
            float(*to)[ROW] = tid < D ? s_q : s_k;
            const int i_qk = tid & (D - 1), at = i_qk + (i_qk >= HALF ? 4 : 0);
#pragma unroll
            for (int i = 0; i < TB; ++i) {
                to[i][at] = y[i];
                if (tid < D) s_v[i][tid] = v[i];
            }
            if (tid < n) {
                const float x = alpha + dt;
                s_a[tid] = expf(ssm_a * (x > 20.f ? x : log1pf(expf(x))));
                s_b[tid] = 1.f / (1.f + expf(-beta));
            }
            __syncthreads();
            for (int i = warp; i < 2 * n; i += WARPS) {          // a warp norms one vector
                float* x = i < n ? s_q[i] : s_k[i - n];
                float ss = 0.f, e_v[EPL];
#pragma unroll
                for (int e = 0; e < EPL; ++e) {
                    const int k = e * 32 + lane;
                    e_v[e] = x[k + (k >= HALF ? 4 : 0)];
                    ss += e_v[e] * e_v[e];
                }
                const float r = rsqrtf(warp_sum(ss) + 1e-6f) * (i < n ? rsqrtf((float)D) : 1.f);
#pragma unroll
                for (int e = 0; e < EPL; ++e) {
                    const int k = e * 32 + lane;
                    x[k + (k >= HALF ? 4 : 0)] = e_v[e] * r;
                    if (KEEP && i >= n) p.keep_k[((size_t)(q.first + t0 + i - n) * p.n_v + h) * D + k] = e_v[e] * r;
                }
            }
            if (t0 == 0) {
                asm volatile("cp.async.wait_group 0;" ::: "memory");
                __syncthreads();
                const float* x = s_state + part * HALF * D + (j ^ (part << 4));
#pragma unroll
                for (int i = 0; i < HALF / 2; ++i) S[i] = q.fresh ? pair(0.f, 0.f) : pair(x[2 * i * D], x[(2 * i + 1) * D]);
            }
            __syncthreads();
            if (t0 == 0) fetch(item + gridDim.x);
#pragma unroll 1
            for (int i = 0; i < n; ++i) {
                const float a = s_a[i];
                const float4 *k = reinterpret_cast<const float4*>(&s_k[i][part * (HALF + 4)]), *x = reinterpret_cast<const float4*>(&s_q[i][part * (HALF + 4)]);
                f32x2 d0 = pair(0.f, 0.f), d1 = d0, o0 = d0, o1 = d0;
#pragma unroll
                for (int e = 0; e < HALF / 4; ++e) {
                    const float4 f = k[e];
                    d0 = fma2(S[2 * e], pair(f.x, f.y), d0);
                    d1 = fma2(S[2 * e + 1], pair(f.z, f.w), d1);
                }
                const float2 e0 = both(d0), e1 = both(d1);
                float dot = (e0.x + e0.y) + (e1.x + e1.y);
                dot += __shfl_xor_sync(0xffffffffu, dot, 1);
                const float u = s_b[i] * (s_v[i][j] - a * dot);
#pragma unroll
                for (int e = 0; e < HALF / 4; ++e) {
                    const float4 f = k[e], g = x[e];
                    S[2 * e] = fma2(pair(f.x, f.y), pair(u, u), mul2(S[2 * e], pair(a, a)));
                    S[2 * e + 1] = fma2(pair(f.z, f.w), pair(u, u), mul2(S[2 * e + 1], pair(a, a)));
                    o0 = fma2(S[2 * e], pair(g.x, g.y), o0);
                    o1 = fma2(S[2 * e + 1], pair(g.z, g.w), o1);
                }
                const float2 f0 = both(o0), f1 = both(o1);
                float o = (f0.x + f0.y) + (f1.x + f1.y);
                o += __shfl_xor_sync(0xffffffffu, o, 1);
                if (part == 0) {
                    s_o[i][j] = o;
                    if (KEEP) {
                        const size_t at_row = (size_t)(q.first + t0 + i) * p.n_v + h;
                        p.keep_u[at_row * D + j] = u;
                        if (j == 0) p.keep_a[at_row] = a;
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int r = 0; r < MINE; ++r) {                     // gated norm, a warp per row
                const int i = r * WARPS + warp;
                if (i >= n) break;
                float ss = 0.f;
#pragma unroll
                for (int e = 0; e < EPL; ++e) ss += s_o[i][e * 32 + lane] * s_o[i][e * 32 + lane];
                const float f = rsqrtf(warp_sum(ss) / D + p.eps);
                __nv_bfloat16* dst = p.out + (size_t)(q.first + t0 + i) * p.out_row + h * D;
#pragma unroll
                for (int e = 0; e < EPL; ++e) dst[e * 32 + lane] = __float2bfloat16(s_o[i][e * 32 + lane] * f * gain[e] * silu(__bfloat162float(z[r][e])));
            }
        }
        if (KEEP) {                                              // a share of the convolution's inputs, for the commit
            const int c0 = (int)((long long)p.C * h / p.n_v), c1 = (int)((long long)p.C * (h + 1) / p.n_v);
            for (int i = tid; i < (c1 - c0) * q.rows; i += 2 * D) {
                const int t = i / (c1 - c0), c = c0 + i % (c1 - c0);
                p.keep_x[((size_t)b * p.rows_per_seq + t) * p.C + c] = p.in[(size_t)(q.first + t) * p.in_row + c];
            }
        } else {
#pragma unroll
            for (int i = 0; i < HALF / 2; ++i) {
                const float2 x = both(S[i]);
                state[(size_t)(2 * i) * D] = x.x;
                state[(size_t)(2 * i + 1) * D] = x.y;
            }
        }
    }
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
    if (c >= p.C || q.rows == 0) return;
    gdn_shift<false>(p, q, b, c, q.rows);
}

template <int D>
__global__ void __launch_bounds__(256) gdn_commit_kernel(const GdnParams p, const int* accepted) {
    constexpr int BLOCK = 16;                                // kept rows in shared memory at a time
    __shared__ __align__(16) float s_u[BLOCK][D], s_k[BLOCK][D];
    const int b = blockIdx.y, tid = threadIdx.x, R = p.rows_per_seq;
    const int n = max(0, min(accepted[b], R));
    if (n == 0) return;
    const GdnSeq q = gdn_seq(p, b);
    if ((int)blockIdx.x >= p.n_v) {                          // the convolution's windows
        const int c = ((int)blockIdx.x - p.n_v) * 256 + tid;
        if (c < p.C) gdn_shift<true>(p, q, b, c, n);
        return;
    }
    const int h = blockIdx.x;
    const size_t kept = (size_t)b * R * p.n_v + h;           // of the sequence's first kept row; the next one is n_v further
    float4* state = reinterpret_cast<float4*>(p.rec + (q.slot * p.n_v + h) * (size_t)(D * D));
    constexpr int QUADS = D / 4, STEP = 256 / QUADS, PER = D / STEP;         // a thread has PER rows i of four columns
    const int j4 = tid % QUADS, i0 = tid / QUADS;
    float4 S[PER];
#pragma unroll
    for (int e = 0; e < PER; ++e) S[e] = state[(size_t)(i0 + e * STEP) * QUADS + j4];
    float all = 1.f;
    for (int r = 0; r < n; ++r) all *= p.keep_a[kept + (size_t)r * p.n_v];
#pragma unroll
    for (int e = 0; e < PER; ++e) { S[e].x *= all; S[e].y *= all; S[e].z *= all; S[e].w *= all; }
    float after = 1.f;                                       // decays behind row r
    for (int r1 = n; r1 > 0; r1 -= BLOCK) {
        const int r0 = max(0, r1 - BLOCK);
        __syncthreads();
        for (int r = r1 - 1; r >= r0; --r) {
            const size_t at = kept + (size_t)r * p.n_v;
            if (tid < D) { s_u[r - r0][tid] = after * p.keep_u[at * D + tid]; s_k[r - r0][tid] = p.keep_k[at * D + tid]; }
            after *= p.keep_a[at];
        }
        __syncthreads();
        for (int r = 0; r < r1 - r0; ++r) {
            const float4 u = *reinterpret_cast<const float4*>(&s_u[r][j4 * 4]);
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const float k = s_k[r][i0 + e * STEP];
                S[e].x += k * u.x; S[e].y += k * u.y; S[e].z += k * u.z; S[e].w += k * u.w;
            }
        }
    }
#pragma unroll
    for (int e = 0; e < PER; ++e) state[(size_t)(i0 + e * STEP) * QUADS + j4] = S[e];
}

LLM_DEFINE_BOUNDS_STATUS_READER(bounds_status_gdn_rows)

template <int D> static cudaError_t rows_of(const GdnParams& p, cudaStream_t st) {
    constexpr int SMEM = D * D * 4, CTAS = D == 128 ? 2 : 4;                  // CTAs of an SM
    const long long items = (long long)p.n_v * p.n_seqs;
    if (items > INT32_MAX / 2) return cudaErrorInvalidValue;
    auto go = [&](auto kernel) {
        const cudaError_t e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, SMEM);
        if (e != cudaSuccess) return e;
        kernel<<<(unsigned)(items < 148 * CTAS ? items : 148 * CTAS), 2 * D, SMEM, st>>>(p);
        return cudaGetLastError();
    };
    if (p.keep_u) return p.K == 4 ? go(gdn_rows_kernel<D, true, true>) : go(gdn_rows_kernel<D, true, false>);
    return p.K == 4 ? go(gdn_rows_kernel<D, false, true>) : go(gdn_rows_kernel<D, false, false>);
}
cudaError_t launch_gdn_rows(const GdnParams& p, cudaStream_t st) {
    if (p.n_seqs == 0 || p.n_rows == 0) return cudaSuccess;
    switch (p.d) {
        case 32: return rows_of<32>(p, st);
        case 64: return rows_of<64>(p, st);
        case 128: return rows_of<128>(p, st);
        default: return cudaErrorNotSupported;
    }
}
cudaError_t launch_gdn_windows(const GdnParams& p, cudaStream_t st) {
    if (p.n_seqs == 0 || p.n_rows == 0) return cudaSuccess;
    gdn_windows_kernel<<<dim3((p.C + 255) / 256, p.n_seqs), 256, 0, st>>>(p);
    return cudaGetLastError();
}
cudaError_t launch_gdn_commit(const GdnParams& p, const int* accepted, cudaStream_t st) {
    if (p.n_seqs == 0 || p.rows_per_seq == 0) return cudaSuccess;
    const dim3 grid(p.n_v + (p.C + 255) / 256, p.n_seqs);
    switch (p.d) {
        case 32: gdn_commit_kernel<32><<<grid, 256, 0, st>>>(p, accepted); break;
        case 64: gdn_commit_kernel<64><<<grid, 256, 0, st>>>(p, accepted); break;
        case 128: gdn_commit_kernel<128><<<grid, 256, 0, st>>>(p, accepted); break;
        default: return cudaErrorNotSupported;
    }
    return cudaGetLastError();
}

}  // namespace llm
