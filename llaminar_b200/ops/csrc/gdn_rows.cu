// The gated delta rule over several new rows of every sequence, one row after the other: the rows of a speculative verification, and prompts
// (short ones, and head sizes that the chunk-parallel kernels do not have).
//
//     y = silu(causal convolution of q | k | v)      q = y_q / |y_q| / sqrt(d),  k = y_k / |y_k|
//     a = exp(ssm_a softplus(alpha + dt_bias))       b = sigmoid(beta)
//     u = b (v - a S^T k)       S = a S + k u^T      o = S^T q       out = o / rms(o) * norm_w * silu(z)
//
// A CTA has one value head of one sequence; thread j keeps column j of the d x d state in registers, so that both products with the state are
// sums inside a thread and a row costs no barrier.  q and k of a block of rows are convolved, normed and left in shared memory first.
// What bounds it: few rows, the state's bytes (64 KB read per head at d = 128; written too unless the state is left alone); more rows, the
// 4 d operations of a column on the FP32 pipes, about 0.6 us a row.
//
// gdn_commit brings the state behind the accepted rows: a streaming pass, S = A S + sum_r k_r (u_r prod_{s > r} a_s)^T, bound by the
// state's bytes in both directions.
//
// (reference: the recurrence of src/v2/kernels/cuda/gdn/CUDAGatedDeltaNetKernels.cu and the verifier's state capture rows,
//  src/v2/models/qwen35/Qwen35Graph.cpp:886-887.)
#include "common.cuh"
#include "hybrid.h"

namespace llm {

constexpr int TB = 8;                                        // rows prepared together

// x of channel c, `t` rows behind the sequence's first row (t < 0: the window before it)
LLM_DEVICE float gdn_input(const GdnParams& p, int first, int t, int c, const float* window, bool fresh) {
    if (t >= 0) return __bfloat162float(p.in[(size_t)(first + t) * p.in_row + c]);
    return fresh ? 0.f : window[(size_t)c * (p.K - 1) + (p.K - 1 + t)];
}

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

template <int D, bool KEEP>
__global__ void __launch_bounds__(D) gdn_rows_kernel(const GdnParams p) {
    constexpr int WARPS = D / 32, EPL = D / 32;
    __shared__ __align__(16) float s_q[TB][D], s_k[TB][D], s_o[TB][D];
    __shared__ float s_a[TB], s_b[TB];
    const int h = blockIdx.x, b = blockIdx.y, j = threadIdx.x, lane = j & 31, warp = j >> 5;
    const GdnSeq q = gdn_seq(p, b);
    if (q.rows == 0) return;
    const int kh = (h + p.v_head_offset) % p.n_k;
    const int cq = kh * D + j, ck = p.n_k * D + kh * D + j, cv = 2 * p.n_k * D + h * D + j;
    const float* window = p.conv + q.slot * (size_t)p.C * (p.K - 1);
    float* state = p.rec + (q.slot * p.n_v + h) * (size_t)(D * D) + j;
    float S[D];
#pragma unroll
    for (int i = 0; i < D; ++i) S[i] = q.fresh ? 0.f : state[(size_t)i * D];
    const float ssm_a = p.ssm_a[h], dt = p.dt_bias[h];
    float gain[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) gain[e] = p.norm_w[e * 32 + lane];

    for (int t0 = 0; t0 < q.rows; t0 += TB) {
        const int n = min(TB, q.rows - t0);
        float v[TB];
#pragma unroll
        for (int i = 0; i < TB; ++i) {
            v[i] = 0.f;
            if (i >= n) continue;
            float yq = 0.f, yk = 0.f, yv = 0.f;
            for (int w = 0; w < p.K; ++w) {
                const int t = t0 + i + w - (p.K - 1);
                yq += p.conv_w[(size_t)cq * p.K + w] * gdn_input(p, q.first, t, cq, window, q.fresh);
                yk += p.conv_w[(size_t)ck * p.K + w] * gdn_input(p, q.first, t, ck, window, q.fresh);
                yv += p.conv_w[(size_t)cv * p.K + w] * gdn_input(p, q.first, t, cv, window, q.fresh);
            }
            s_q[i][j] = yq / (1.f + expf(-yq));
            s_k[i][j] = yk / (1.f + expf(-yk));
            v[i] = yv / (1.f + expf(-yv));
        }
        if (j < n) {
            const __nv_bfloat16* ab = p.in + (size_t)(q.first + t0 + j) * p.in_row + p.ab_off;
            const float x = __bfloat162float(ab[h]) + dt;
            s_a[j] = expf(ssm_a * (x > 20.f ? x : log1pf(expf(x))));
            s_b[j] = 1.f / (1.f + expf(-__bfloat162float(ab[p.n_v + h])));
        }
        __syncthreads();
        for (int i = warp; i < 2 * n; i += WARPS) {          // a warp norms one vector
            float* x = i < n ? s_q[i] : s_k[i - n];
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < EPL; ++e) ss += x[e * 32 + lane] * x[e * 32 + lane];
            const float r = 1.f / sqrtf(warp_sum(ss) + 1e-6f) * (i < n ? 1.f / sqrtf((float)D) : 1.f);
#pragma unroll
            for (int e = 0; e < EPL; ++e) x[e * 32 + lane] *= r;
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < TB; ++i) {
            if (i >= n) continue;
            const float a = s_a[i];
            float dot[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < D; e += 4) {
                const float4 k = *reinterpret_cast<const float4*>(&s_k[i][e]);
                dot[0] += S[e] * k.x; dot[1] += S[e + 1] * k.y; dot[2] += S[e + 2] * k.z; dot[3] += S[e + 3] * k.w;
            }
            const float u = s_b[i] * (v[i] - a * ((dot[0] + dot[1]) + (dot[2] + dot[3])));
            float o[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int e = 0; e < D; e += 4) {
                const float4 k = *reinterpret_cast<const float4*>(&s_k[i][e]), x = *reinterpret_cast<const float4*>(&s_q[i][e]);
                S[e] = a * S[e] + k.x * u; S[e + 1] = a * S[e + 1] + k.y * u; S[e + 2] = a * S[e + 2] + k.z * u; S[e + 3] = a * S[e + 3] + k.w * u;
                o[0] += S[e] * x.x; o[1] += S[e + 1] * x.y; o[2] += S[e + 2] * x.z; o[3] += S[e + 3] * x.w;
            }
            s_o[i][j] = (o[0] + o[1]) + (o[2] + o[3]);
            if (KEEP) {
                const size_t at = ((size_t)(q.first + t0 + i) * p.n_v + h);
                p.keep_u[at * D + j] = u;
                p.keep_k[at * D + j] = s_k[i][j];
                if (j == 0) p.keep_a[at] = a;
            }
        }
        __syncthreads();
        for (int i = warp; i < n; i += WARPS) {              // gated norm, a warp per row
            const size_t row = q.first + t0 + i;
            const __nv_bfloat16* z = p.in + row * p.in_row + p.z_off + h * D;
            float ss = 0.f;
#pragma unroll
            for (int e = 0; e < EPL; ++e) ss += s_o[i][e * 32 + lane] * s_o[i][e * 32 + lane];
            const float r = 1.f / sqrtf(warp_sum(ss) / D + p.eps);
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
                const float g = __bfloat162float(z[e * 32 + lane]);
                p.out[row * p.out_row + h * D + e * 32 + lane] = __float2bfloat16(s_o[i][e * 32 + lane] * r * gain[e] * (g / (1.f + expf(-g))));
            }
        }
        __syncthreads();
    }
    if (!KEEP) {
#pragma unroll
        for (int i = 0; i < D; ++i) state[(size_t)i * D] = S[i];
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
    if (p.keep_x) {
        for (int t = 0; t < q.rows; ++t) p.keep_x[((size_t)b * p.rows_per_seq + t) * p.C + c] = p.in[(size_t)(q.first + t) * p.in_row + c];
    } else {
        gdn_shift<false>(p, q, b, c, q.rows);
    }
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

template <int D> static void rows_of(const GdnParams& p, cudaStream_t st) {
    const dim3 grid(p.n_v, p.n_seqs);
    if (p.keep_u) gdn_rows_kernel<D, true><<<grid, D, 0, st>>>(p);
    else gdn_rows_kernel<D, false><<<grid, D, 0, st>>>(p);
}
cudaError_t launch_gdn_rows(const GdnParams& p, cudaStream_t st) {
    if (p.n_seqs == 0 || p.n_rows == 0) return cudaSuccess;
    switch (p.d) {
        case 32: rows_of<32>(p, st); break;
        case 64: rows_of<64>(p, st); break;
        case 128: rows_of<128>(p, st); break;
        default: return cudaErrorNotSupported;
    }
    return cudaGetLastError();
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
