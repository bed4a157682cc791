// Rows of a projection -> queries and entries of the paged cache, with the norm and the rotation of a part of every head on the way.
//
// A row is [query | gate] per head (gate optional, left where it is), keys, values.  Queries and keys are RMS-normed per head, then the first `rot` values of a head
// turn by position x frequency, pairs (i, i + rot / 2) or (2i, 2i + 1), and grow by a common factor (scaled rotations); the rest passes.  Keys and values go to
// their page as bf16, or as 8-bit numbers with one scale per 32 values (the layout and the scales of rope_kv).
//
// Angles are formed in 64 bits as turns, position x frequency / 2 pi, of which the whole turns are dropped before the sine: in 32 bits an angle at position 200000 is
// 2^-7 off.  A warp has a token (or a part of its heads: few tokens) and forms them once; a lane has D / 32 neighbouring values of a head, partners of the
// first kind come from the lane rot / 2 values away.  What bounds it: the bytes of the rows, read and written once (8190 rows of 24
// gated heads of 256 values: 207 MB in 44 us, 4.7 TB/s); below a few hundred rows the launch and a warp's chain (32 rows 4.4 us, 700 rows into 8-bit pages 7.0 us).
// (reference: src/v2/kernels/cuda/ops/CUDARoPEKernels.cu, ring append of src/v2/kernels/cuda/kvcache/CUDARingKVCache.cu.)
#include <cuda_fp16.h>

#include "hybrid.h"
#include "launch.h"
#include "pairs.cuh"

namespace llm {

constexpr int PAGE = 64, WARPS = 4;

// N bf16 values as they lie in memory (N = 2, 4, 8)
template <int N> struct Raw {
    uint32_t w[N / 2];
    LLM_DEVICE f32x2 two(int i) const { return pair(bf16_lo(w[i]), bf16_hi(w[i])); }
};
template <int N> LLM_DEVICE Raw<N> load_raw(const __nv_bfloat16* x, bool whole) {
    Raw<N> r;
    if (!whole) {
#pragma unroll
        for (int i = 0; i < N / 2; ++i) r.w[i] = __bfloat16_as_ushort(x[2 * i]) | (uint32_t)__bfloat16_as_ushort(x[2 * i + 1]) << 16;
    } else if (N == 8) {
        const uint4 v = *reinterpret_cast<const uint4*>(x);
        r.w[0] = v.x; r.w[1 % (N / 2)] = v.y; r.w[2 % (N / 2)] = v.z; r.w[3 % (N / 2)] = v.w;
    } else if (N == 4) {
        const uint2 v = *reinterpret_cast<const uint2*>(x);
        r.w[0] = v.x; r.w[1 % (N / 2)] = v.y;
    } else {
        r.w[0] = *reinterpret_cast<const uint32_t*>(x);
    }
    return r;
}
template <int N> LLM_DEVICE void store_raw(__nv_bfloat16* x, const Raw<N>& r) {            // aligned: the caches and the queries are dense
    if (N == 8) *reinterpret_cast<uint4*>(x) = make_uint4(r.w[0], r.w[1 % (N / 2)], r.w[2 % (N / 2)], r.w[3 % (N / 2)]);
    else if (N == 4) *reinterpret_cast<uint2*>(x) = make_uint2(r.w[0], r.w[1 % (N / 2)]);
    else *reinterpret_cast<uint32_t*>(x) = r.w[0];
}

// sums of B values over a warp, as reciprocal roots of their means.  Four go through the lanes together: each step halves what a lane carries
// on, so that four sums take 10 exchanges and one root instead of 20 and four.
template <int B> LLM_DEVICE void roots(float (&ss)[B], float scale, float eps) {
    const int lane = threadIdx.x & 31;
    if constexpr (B == 4) {
        const bool up = lane & 16, up2 = lane & 8;
        const float x0 = (up ? ss[2] : ss[0]) + __shfl_xor_sync(0xffffffffu, up ? ss[0] : ss[2], 16), x1 = (up ? ss[3] : ss[1]) + __shfl_xor_sync(0xffffffffu, up ? ss[1] : ss[3], 16);
        float z = (up2 ? x1 : x0) + __shfl_xor_sync(0xffffffffu, up2 ? x0 : x1, 8);
        z += __shfl_xor_sync(0xffffffffu, z, 4);
        z += __shfl_xor_sync(0xffffffffu, z, 2);
        z += __shfl_xor_sync(0xffffffffu, z, 1);
        const float r = rsqrtf(z * scale + eps);
#pragma unroll
        for (int j = 0; j < 4; ++j) ss[j] = __shfl_sync(0xffffffffu, r, (j >> 1) * 16 + (j & 1) * 8);
    } else {
#pragma unroll
        for (int j = 0; j < B; ++j) ss[j] = rsqrtf(warp_sum(ss[j]) * scale + eps);
    }
}

// One value becomes own * gain * cos +- partner * gain of the partner * sin, all times the head's reciprocal root: gains and angles are multiplied once per
// token, and the partners come as they were loaded, two values a word.  D / 32 values a lane, BATCH heads at a time, the next ones on their way.
// ODD: halves that end inside a lane's values.
template <int D, int BATCH, bool ODD>
__global__ void __launch_bounds__(32 * WARPS, ODD ? 1 : D == 256 ? 4 : 6) rope_part_kernel(const RopePartParams p) {
    constexpr int N = D / 32;
    __shared__ float2 s_angles[WARPS][D / 2];
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, item = blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (item >= p.n_tokens * p.parts) return;
    const int t = item / p.parts, part = item - t * p.parts;
    const int heads = p.n_heads + 2 * p.n_kv_heads, per = (heads + p.parts - 1) / p.parts;
    const int h0 = part * per, h1 = min(heads, h0 + per);
    if (h0 >= h1) return;
    const int pos = p.positions[t], half = p.rot / 2, i0 = lane * N;
    const __nv_bfloat16* row = p.rows + (size_t)t * p.row + i0;
    auto source = [&](int h) { return row + (size_t)(h < p.n_heads ? h * p.q_stride : p.n_heads * p.q_stride + (h - p.n_heads) * D); };
    Raw<N> next[BATCH];
#pragma unroll
    for (int j = 0; j < BATCH; ++j) next[j] = load_raw<N>(source(min(h0 + j, h1 - 1)), p.whole);
    float cs[N], sn[N];                                      // with the sign that the partner has
    uint32_t turns[N / 2];                                   // the words' values that turn, as a mask
    auto partner_of = [&](int i) { return i >= p.rot ? i : p.interleaved ? i ^ 1 : i < half ? i + half : i - half; };
    if (h0 < p.n_heads + p.n_kv_heads) {
#pragma unroll
        for (int k = 0; k < N / 2; ++k) {                    // a lane forms the angles of every 32nd pair
            const int i = k * 32 + lane;
            if (i >= half) break;
            const double x = (double)pos * p.freqs[i] * 0.15915494309189533577;       // in turns
            float s, c;
            sincospif(2.f * (float)(x - rint(x)), &s, &c);
            s_angles[threadIdx.x >> 5][i] = make_float2(c * p.magnitude, s * p.magnitude);
        }
        __syncwarp();
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int i = i0 + e;
            const bool first = p.interleaved ? !(e & 1) : i < half;
            const int index = p.interleaved ? i >> 1 : first ? i : i - half;
            cs[e] = 1.f; sn[e] = 0.f;
            if (e % 2 == 0) turns[e / 2] = 0;
            if (i >= p.rot) continue;
            turns[e / 2] |= e % 2 ? 0xffff0000u : 0xffffu;
            const float2 x = s_angles[threadIdx.x >> 5][index];
            cs[e] = x.x; sn[e] = first ? -x.y : x.y;
        }
    }
    uint8_t* page = nullptr;
    if (h1 > p.n_heads) {
        const int seq = LLM_CHECK_INDEX(p.seq_ids[t], p.n_seqs), slot = LLM_CHECK_INDEX(pos >> 6, p.max_pages);          // (a shift: -1 is no page, not the first one)
        page = p.kv + (size_t)LLM_CHECK_INDEX(p.block_table[(size_t)seq * p.max_pages + slot], p.n_pages) * p.page_bytes;
    }

    // heads [a, b) of one kind (0: queries, 1: keys, 2: values); the first batch is in `next`, the last one leaves what comes behind b there
    auto heads_of = [&](int a, int b, int kind) {
        const float* gain = kind == 0 ? p.q_norm : kind == 1 ? p.k_norm : nullptr;
        f32x2 own[N / 2], partner[N / 2];
        if (kind < 2) {
#pragma unroll
            for (int e = 0; e < N; e += 2) {
                own[e / 2] = pair(cs[e] * (gain ? gain[i0 + e] : 1.f), cs[e + 1] * (gain ? gain[i0 + e + 1] : 1.f));
                partner[e / 2] = pair(sn[e] * (gain ? gain[partner_of(i0 + e)] : 1.f), sn[e + 1] * (gain ? gain[partner_of(i0 + e + 1)] : 1.f));
            }
        }
        for (int b0 = a; b0 < b; b0 += BATCH) {
            Raw<N> raw[BATCH];
#pragma unroll
            for (int j = 0; j < BATCH; ++j) raw[j] = next[j];
            const int n0 = min(b0 + BATCH, b);               // kinds begin a batch of their own
            if (n0 < h1) {
#pragma unroll
                for (int j = 0; j < BATCH; ++j) next[j] = load_raw<N>(source(min(n0 + j, h1 - 1)), p.whole);
            }
            float r[BATCH];
            if (gain) {
#pragma unroll
                for (int j = 0; j < BATCH; ++j) {
                    f32x2 ss = pair(0.f, 0.f);
#pragma unroll
                    for (int e = 0; e < N / 2; ++e) ss = fma2(raw[j].two(e), raw[j].two(e), ss);
                    const float2 x = both(ss);
                    r[j] = x.x + x.y;
                }
                roots<BATCH>(r, 1.f / D, p.eps);
            }
#pragma unroll
            for (int j = 0; j < BATCH; ++j) {
                const int h = b0 + j;
                if (h >= b) break;
                f32x2 y[N / 2];
                if (kind < 2) {
                    Raw<N> x;
                    if (p.interleaved) {
#pragma unroll
                        for (int e = 0; e < N / 2; ++e) x.w[e] = __byte_perm(raw[j].w[e], 0, 0x1032);
                    } else if (!ODD) {                       // a lane's partners are the neighbours of one another
                        const int lane_of = partner_of(i0) / N;
#pragma unroll
                        for (int e = 0; e < N / 2; ++e) x.w[e] = __shfl_sync(0xffffffffu, raw[j].w[e], lane_of);
                    } else {
#pragma unroll
                        for (int e = 0; e < N; ++e) {
                            const int from = partner_of(i0 + e);
                            uint32_t v = 0;
#pragma unroll
                            for (int k = 0; k < N / 2; ++k) {
                                const uint32_t w = __shfl_sync(0xffffffffu, raw[j].w[k], from / N);
                                if (from % N / 2 == k) v = w;
                            }
                            v = from & 1 ? v >> 16 : v & 0xffffu;
                            x.w[e / 2] = e & 1 ? x.w[e / 2] | v << 16 : v;
                        }
                    }
#pragma unroll
                    for (int e = 0; e < N / 2; ++e) {
                        x.w[e] &= turns[e];                  // what passes meets no partner (an infinity times 0 is not 0)
                        y[e] = fma2(x.two(e), partner[e], mul2(raw[j].two(e), own[e]));
                        if (gain) y[e] = mul2(y[e], pair(r[j], r[j]));
                    }
                    if (kind == 0 || !p.q8) {
#pragma unroll
                        for (int e = 0; e < N / 2; ++e) {
                            const float2 v = both(y[e]);
                            raw[j].w[e] = pack_bf16(v.x, v.y);
                        }
                    }
                } else if (p.q8) {
#pragma unroll
                    for (int e = 0; e < N / 2; ++e) y[e] = raw[j].two(e);
                }
                if (kind == 0) {
                    store_raw<N>(p.q_out + ((size_t)t * p.n_heads + h) * D + i0, raw[j]);
                    continue;
                }
                const size_t at = ((size_t)(kind - 1) * p.n_kv_heads + (h - p.n_heads - (kind - 1) * p.n_kv_heads)) * PAGE + (pos & (PAGE - 1));
                if (!p.q8) {
                    store_raw<N>(reinterpret_cast<__nv_bfloat16*>(page) + at * D + i0, raw[j]);
                    continue;
                }
                // 8-bit: largest magnitude of the 32 values / 127, rounded up to seven bits behind the point (no value clips; see rope_kv for why seven)
                float top = 0.f;
#pragma unroll
                for (int e = 0; e < N / 2; ++e) {
                    const float2 v = both(y[e]);
                    top = fmaxf(top, fmaxf(fabsf(v.x), fabsf(v.y)));
                }
#pragma unroll
                for (int o = 1; o < 32 / N; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
                const __half hs = __float2half_rn(__uint_as_float((__float_as_uint(top * (1.0f / 127.0f)) + 0xFFFFu) & 0xFFFF0000u));
                const float s = __half2float(hs), inv = s > 0.f ? 1.0f / s : 0.f;
                uint32_t w[2] = {0u, 0u};
#pragma unroll
                for (int e = 0; e < N; ++e) {
                    const float2 v = both(y[e / 2]);
                    w[e / 4] |= (uint32_t)(uint8_t)(int8_t)max(-127, min(127, __float2int_rn((e & 1 ? v.y : v.x) * inv))) << (8 * (e & 3));
                }
                uint8_t* d8 = page + at * D + i0;
                if (N == 8) *reinterpret_cast<uint2*>(d8) = make_uint2(w[0], w[1]);
                else if (N == 4) *reinterpret_cast<uint32_t*>(d8) = w[0];
                else *reinterpret_cast<unsigned short*>(d8) = (unsigned short)w[0];
                if ((lane & (32 / N - 1)) == 0) reinterpret_cast<__half*>(page + p.scale_off)[at * (D / 32) + i0 / 32] = hs;
            }
        }
    };
    const int q1 = min(h1, p.n_heads), k1 = min(h1, p.n_heads + p.n_kv_heads);
    if (h0 < q1) heads_of(h0, q1, 0);
    if (max(h0, q1) < k1) heads_of(max(h0, q1), k1, 1);
    if (max(h0, k1) < h1) heads_of(max(h0, k1), h1, 2);
}

cudaError_t launch_rope_part(const RopePartParams& args, cudaStream_t st) {
    RopePartParams p = args;
    if (p.n_tokens == 0) return cudaSuccess;
    const int heads = p.n_heads + 2 * p.n_kv_heads;
    // A warp takes all heads of a token where the tokens give every SM `per_sm` warps, else the heads are shared out; up to eight heads go one at a time.
    const int per_sm = p.head_dim == 256 ? 8 : 16;
    p.parts = 1;
    while ((long long)p.n_tokens * p.parts < sm_count() * per_sm && p.parts < heads) p.parts *= 2;
    if (p.parts > heads) p.parts = heads;
    const long long ctas = ((long long)p.n_tokens * p.parts + WARPS - 1) / WARPS;
    if (ctas > INT32_MAX) return cudaErrorInvalidValue;
    const bool few = (heads + p.parts - 1) / p.parts <= 8;
    const bool odd = !p.interleaved && p.rot / 2 % (p.head_dim / 32);
    auto go = [&](auto one, auto many, auto any) { return launch_pdl(odd ? any : few ? one : many, dim3((unsigned)ctas), dim3(32 * WARPS), 0, st, p); };
    if (p.head_dim == 64) return go(rope_part_kernel<64, 1, false>, rope_part_kernel<64, 4, false>, rope_part_kernel<64, 1, true>);
    if (p.head_dim == 128) return go(rope_part_kernel<128, 1, false>, rope_part_kernel<128, 4, false>, rope_part_kernel<128, 1, true>);
    if (p.head_dim == 256) return go(rope_part_kernel<256, 1, false>, rope_part_kernel<256, 4, false>, rope_part_kernel<256, 1, true>);
    return cudaErrorInvalidValue;
}

LLM_DEFINE_BOUNDS_STATUS_READER(bounds_status_rope_part)

}  // namespace llm
