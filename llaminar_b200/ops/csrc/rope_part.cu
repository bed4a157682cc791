// Rows of a projection -> queries and entries of the paged cache, with the norm and the rotation of a part of every head on the way.
//
// A row is [query | gate] per head (gate optional, left where it is), keys, values.  Queries and keys are RMS-normed per head, then the first `rot` values of a head
// turn by position x frequency, pairs (i, i + rot / 2) or (2i, 2i + 1), and grow by a common factor (scaled rotations); the rest passes.  Keys and values go to
// their page as bf16, or as 8-bit numbers with one scale per 32 values (the layout and the scales of rope_kv).
//
// Angles are formed in 64 bits as turns, position x frequency / 2 pi, of which the whole turns are dropped before the sine: in 32 bits an angle at position 200000 is
// 2^-7 off.  A warp has a token (or a part of its heads: few tokens) and forms them once; a lane has D / 32 neighbouring values of a head, partners of the
// first kind come from the lane rot / 2 values away.  What bounds it: the bytes of the rows, read and written once.
// (reference: src/v2/kernels/cuda/ops/CUDARoPEKernels.cu, ring append of src/v2/kernels/cuda/kvcache/CUDARingKVCache.cu.)
#include <cuda_fp16.h>

#include "common.cuh"
#include "hybrid.h"
#include "launch.h"

namespace llm {

constexpr int PAGE = 64, WARPS = 4;

// N bf16 values as they lie in memory (N = 2, 4, 8)
template <int N> struct Raw { uint32_t w[N / 2]; };
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
template <int N> LLM_DEVICE void store_raw(__nv_bfloat16* x, const float (&v)[N]) {        // aligned: the caches and the queries are dense
    uint32_t w[N / 2];
#pragma unroll
    for (int i = 0; i < N / 2; ++i) w[i] = pack_bf16(v[2 * i], v[2 * i + 1]);
    if (N == 8) *reinterpret_cast<uint4*>(x) = make_uint4(w[0], w[1 % (N / 2)], w[2 % (N / 2)], w[3 % (N / 2)]);
    else if (N == 4) *reinterpret_cast<uint2*>(x) = make_uint2(w[0], w[1 % (N / 2)]);
    else *reinterpret_cast<uint32_t*>(x) = w[0];
}

// D / 32 values a lane, BATCH heads at a time
template <int D, int BATCH>
__global__ void __launch_bounds__(32 * WARPS) rope_part_kernel(const RopePartParams p) {
    constexpr int N = D / 32;
    pdl_trigger();
    pdl_wait();
    const int lane = threadIdx.x & 31, item = blockIdx.x * WARPS + (threadIdx.x >> 5);
    if (item >= p.n_tokens * p.parts) return;
    const int t = item / p.parts, part = item - t * p.parts;
    const int heads = p.n_heads + 2 * p.n_kv_heads, per = (heads + p.parts - 1) / p.parts;
    const int h0 = part * per, h1 = min(heads, h0 + per);
    const int pos = p.positions[t], half = p.rot / 2, i0 = lane * N;
    const __nv_bfloat16* row = p.rows + (size_t)t * p.row + i0;
    auto source = [&](int h) { return row + (size_t)(h < p.n_heads ? h * p.q_stride : p.n_heads * p.q_stride + (h - p.n_heads) * D); };
    float cs[N], sn[N];
    if (h0 < p.n_heads + p.n_kv_heads) {
#pragma unroll
        for (int e = 0; e < N; ++e) {
            const int i = i0 + e, pair = p.interleaved ? i >> 1 : i < half ? i : i - half;
            cs[e] = 1.f; sn[e] = 0.f;
            if (i >= p.rot) continue;
            if (p.interleaved && (e & 1)) { cs[e] = cs[e - 1]; sn[e] = sn[e - 1]; continue; }
            const double turns = (double)pos * p.freqs[pair] * 0.15915494309189533577;
            float s, c;
            sincospif(2.f * (float)(turns - rint(turns)), &s, &c);
            cs[e] = c * p.magnitude; sn[e] = s * p.magnitude;
        }
    }
    uint8_t* page = nullptr;
    if (h1 > p.n_heads) {
        const int seq = LLM_CHECK_INDEX(p.seq_ids[t], p.n_seqs), slot = LLM_CHECK_INDEX(pos / PAGE, p.max_pages);
        page = p.kv + (size_t)LLM_CHECK_INDEX(p.block_table[(size_t)seq * p.max_pages + slot], p.n_pages) * p.page_bytes;
    }
    for (int b0 = h0; b0 < h1; b0 += BATCH) {
        Raw<N> raw[BATCH];
#pragma unroll
        for (int j = 0; j < BATCH; ++j) raw[j] = load_raw<N>(source(min(b0 + j, h1 - 1)), p.whole);
#pragma unroll
        for (int j = 0; j < BATCH; ++j) {
            const int h = b0 + j;
            if (h >= h1) break;
            const bool is_q = h < p.n_heads, is_k = !is_q && h < p.n_heads + p.n_kv_heads;
            float x[N];
#pragma unroll
            for (int e = 0; e < N; e += 2) { x[e] = bf16_lo(raw[j].w[e / 2]); x[e + 1] = bf16_hi(raw[j].w[e / 2]); }
            if (is_q || is_k) {
                const float* gain = is_q ? p.q_norm : p.k_norm;
                if (gain) {
                    float ss = 0.f;
#pragma unroll
                    for (int e = 0; e < N; ++e) ss += x[e] * x[e];
                    const float r = rsqrtf(warp_sum(ss) / D + p.eps);
#pragma unroll
                    for (int e = 0; e < N; ++e) x[e] *= r * gain[i0 + e];
                }
                float y[N];                                  // the partners
                if (p.interleaved) {
#pragma unroll
                    for (int e = 0; e < N; e += 2) { y[e] = -x[e + 1]; y[e + 1] = x[e]; }
                } else if (half % N == 0) {
                    const int from = i0 < half ? lane + half / N : lane - half / N;
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const float v = __shfl_sync(0xffffffffu, x[e], from & 31);
                        y[e] = i0 < half ? -v : v;
                    }
                } else {                                     // a part whose halves end inside a lane's values
#pragma unroll
                    for (int e = 0; e < N; ++e) {
                        const int i = i0 + e, from = i < half ? i + half : i - half;
                        y[e] = 0.f;
#pragma unroll
                        for (int k = 0; k < N; ++k) {
                            const float v = __shfl_sync(0xffffffffu, x[k], (from / N) & 31);
                            if (from % N == k) y[e] = i < half ? -v : v;
                        }
                    }
                }
#pragma unroll
                for (int e = 0; e < N; ++e)
                    if (i0 + e < p.rot) x[e] = x[e] * cs[e] + y[e] * sn[e];
            }
            if (is_q) {
                store_raw<N>(p.q_out + ((size_t)t * p.n_heads + h) * D + i0, x);
                continue;
            }
            const size_t at = ((size_t)(is_k ? 0 : 1) * p.n_kv_heads + (is_k ? h - p.n_heads : h - p.n_heads - p.n_kv_heads)) * PAGE + pos % PAGE;
            if (!p.q8) {
                store_raw<N>(reinterpret_cast<__nv_bfloat16*>(page) + at * D + i0, x);
                continue;
            }
            // 8-bit: largest magnitude of the 32 values / 127, rounded up to seven bits behind the point (no value clips; see rope_kv for why seven)
            float top = 0.f;
#pragma unroll
            for (int e = 0; e < N; ++e) top = fmaxf(top, fabsf(x[e]));
#pragma unroll
            for (int o = 1; o < 32 / N; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
            const __half hs = __float2half_rn(__uint_as_float((__float_as_uint(top * (1.0f / 127.0f)) + 0xFFFFu) & 0xFFFF0000u));
            const float s = __half2float(hs), inv = s > 0.f ? 1.0f / s : 0.f;
            uint32_t w[2] = {0u, 0u};
#pragma unroll
            for (int e = 0; e < N; ++e) w[e / 4] |= (uint32_t)(uint8_t)(int8_t)max(-127, min(127, __float2int_rn(x[e] * inv))) << (8 * (e & 3));
            uint8_t* d8 = page + at * D + i0;
            if (N == 8) *reinterpret_cast<uint2*>(d8) = make_uint2(w[0], w[1]);
            else if (N == 4) *reinterpret_cast<uint32_t*>(d8) = w[0];
            else *reinterpret_cast<unsigned short*>(d8) = (unsigned short)w[0];
            if ((lane & (32 / N - 1)) == 0) reinterpret_cast<__half*>(page + p.scale_off)[at * (D / 32) + i0 / 32] = hs;
        }
    }
}

cudaError_t launch_rope_part(const RopePartParams& args, cudaStream_t st) {
    RopePartParams p = args;
    if (p.n_tokens == 0) return cudaSuccess;
    const int heads = p.n_heads + 2 * p.n_kv_heads;
    // a warp takes all heads of a token where the tokens fill the GPU's warps, else the heads are shared out
    p.parts = 1;
    while ((long long)p.n_tokens * p.parts < 148 * 16 && p.parts < heads) p.parts *= 2;
    if (p.parts > heads) p.parts = heads;
    const long long ctas = ((long long)p.n_tokens * p.parts + WARPS - 1) / WARPS;
    if (ctas > INT32_MAX) return cudaErrorInvalidValue;
    const bool few = (heads + p.parts - 1) / p.parts < 4;
    auto go = [&](auto one, auto many) { return launch_pdl(few ? one : many, dim3((unsigned)ctas), dim3(32 * WARPS), 0, st, p); };
    if (p.head_dim == 64) return go(rope_part_kernel<64, 1>, rope_part_kernel<64, 4>);
    if (p.head_dim == 128) return go(rope_part_kernel<128, 1>, rope_part_kernel<128, 4>);
    if (p.head_dim == 256) return go(rope_part_kernel<256, 1>, rope_part_kernel<256, 4>);
    return cudaErrorInvalidValue;
}

LLM_DEFINE_BOUNDS_STATUS_READER(bounds_status_rope_part)

}  // namespace llm
