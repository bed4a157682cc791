// The gated delta rule over prompts, chunk-parallel on the 5th-generation tensor cores (d = 128).
//
// A sequence is cut into chunks of 64 rows.  With G_t the running sum of the log decays inside a chunk, M[t, i] = e^(G_t - G_i) for i <= t, and S the state
// in front of the chunk, the corrections of a chunk solve a triangular system, and everything else is matrix products:
//
//     (I + A) U = R       A[t, i] = b_t M[t, i] k_t.k_i  (i < t)      R_t = b_t (v_t - e^(G_t) S^T k_t)
//     o_t = e^(G_t) S^T q_t + sum_{i<=t} M[t, i] (q_t.k_i) u_i        S' = e^(G_C) S + sum_i e^(G_C - G_i) k_i u_i^T
//
// Every exponent is <= 0.  Two launches:
//
//   gdn_chunk_prep   per chunk and key head: convolutions, norms, gates, k.k and q.k (mma.sync), then per value head P[t, i] = M[t, i] q_t.k_i and the inverse
//                    T = (I + A)^-1: blocks of 16 rows on the diagonal by forward substitution (a thread per column), the others from them by products,
//                    T_ij = -T_ii sum_k A_ik T_kj, a warp per column of blocks.  All chunks at once.
//   gdn_chunk_scan   per sequence and value head, chunk after chunk:  S^T k, S^T q, U = T R, P U and the state's sum as tcgen05.mma with M = 128 value
//                    columns, the left operand (S, R, U) in tensor memory and T, P, K, Q in shared memory.  A thread has one value column: what it reads
//                    from an accumulator it scales, splits and writes back as the next product's operand without leaving its lane.
//
// Everything stays at 32-bit accuracy: each operand is split into two fp16 numbers (22 bits), which takes three products.  The range comes from
// powers of two: k, T and q, P are bounded by 1 in magnitude and have fixed factors (a row's update is a contraction, so no entry of T exceeds 1); S,
// R and U are scaled per value column, to 2^13 .. 2^14 at the largest.  (With q, P and the S and U that only the output sees as single fp16 numbers an output whose
// sum cancels was 2^-7 off behind the gated norm.)  G is summed in 64 bits: differences of sums near -100 would cost a 32-bit one 2^-17.
//
// What bounds it: the scan's chain along the state, 7450 clocks a chunk: the state as an operand 1290, S^T k 1070, R 1280, U 500, U as an operand 960, the
// state's sum 990, the state 530, and 200 for each of four signals (U before its products had all 64 columns: three groups of four at 41 clocks now).  Operands are in tensor memory since a product of 64 (128) columns takes 41 (71) clocks so and
// 71 (100) with both in shared memory.  8192 rows of 16 / 48 heads take 608 us (57 by the bytes), five sequences of 900 rows on average 188 (preparation
// 86, scan 102), 37 rows 30.5.
// Every mbarrier wait is bounded; on a timeout the kernel raises the status word and tears down.
//
// (reference: the chunk kernels of src/v2/kernels/cuda/gdn/CUDAGatedDeltaNetKernels.cu.)
#include <cuda_fp16.h>

#include "hybrid.h"
#include "launch.h"
#include "pairs.cuh"
#include "tc_tile.cuh"

namespace llm {
namespace gdc {
using namespace tc5;

constexpr int D = 128, C = 64;
// one chunk of a key head: K and Q as two fp16 numbers each, [2 halves of d][64 rows][128 bytes], swizzled as the products read them
constexpr int IMG = C * D * 2;                              // 16 KB
constexpr int OFF_KHI = 0, OFF_KLO = IMG, OFF_QHI = 2 * IMG, OFF_QLO = 3 * IMG, KEY_BYTES = 4 * IMG;
// one chunk of a value head: T and P likewise [64 rows][128 bytes], b v transposed [128 columns][64 rows] fp32, four vectors
constexpr int TRI = C * C * 2;                              // 8 KB
constexpr int OFF_THI = 0, OFF_PHI = 2 * TRI, OFF_PLO = 3 * TRI, OFF_V = 4 * TRI, VALS = C * D * 4, OFF_VEC = OFF_V + VALS, VEC_BYTES = 4 * C * 4, HEAD_BYTES = OFF_VEC + VEC_BYTES;
static_assert(KEY_BYTES % 1024 == 0 && HEAD_BYTES % 1024 == 0, "tiles start on swizzle atoms");
enum Vec { V_BE = 0, V_EG = C, V_EL = 2 * C, V_ALL = 3 * C };               // b e^G, e^G, e^(G_C - G), e^G_C
constexpr float SK = 4096.f, SQ = 16384.f;                  // factors of k, T and of q, P

LLM_DEVICE int rows_of(const GdnParams& p, int b, int& first) {
    first = max(0, min(p.cu[b], p.n_rows));
    return max(0, min(p.cu[b + 1], p.n_rows) - first);
}
// chunks of the sequences in front of sequence `b` (whole warp)
LLM_DEVICE int chunks_before(const GdnParams& p, int b) {
    int n = 0, first;
    for (int i = threadIdx.x & 31; i < b; i += 32) n += (rows_of(p, i, first) + C - 1) / C;
    return __reduce_add_sync(0xffffffffu, n);
}
// the sequence that chunk `u` of the batch belongs to, and that sequence's first chunk (whole warp); -1: none
LLM_DEVICE int sequence_of(const GdnParams& p, int u, int& at) {
    const int lane = threadIdx.x & 31;
    at = 0;
    for (int b0 = 0; b0 < p.n_seqs; b0 += 32) {
        int first;
        const int n = b0 + lane < p.n_seqs ? (rows_of(p, b0 + lane, first) + C - 1) / C : 0;
        int sum = n;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += x;
        }
        const unsigned m = __ballot_sync(0xffffffffu, at + sum > u);
        if (m) {
            const int l = __ffs(m) - 1;
            at += __shfl_sync(0xffffffffu, sum - n, l);
            return b0 + l;
        }
        at += __shfl_sync(0xffffffffu, sum, 31);
    }
    return -1;
}

struct Chunk {                                              // rows [row0, row0 + n) of a sequence that starts at `first`
    int first, row0, n, slot;
    bool fresh;
};

// four neighbours as they lie; the host says whether 8-byte loads may be used
LLM_DEVICE uint2 four(const __nv_bfloat16* x, bool aligned) {
    if (aligned) return *reinterpret_cast<const uint2*>(x);
    return make_uint2(__bfloat16_as_ushort(x[0]) | (uint32_t)__bfloat16_as_ushort(x[1]) << 16, __bfloat16_as_ushort(x[2]) | (uint32_t)__bfloat16_as_ushort(x[3]) << 16);
}
// sigmoid of a row's second gate
LLM_DEVICE float beta(const GdnParams& p, const Chunk& ch, int t, int h) { return 1.f / (1.f + expf(-__bfloat162float(p.in[(size_t)(ch.row0 + t) * p.in_row + p.ab_off + p.n_v + h]))); }
LLM_DEVICE f32x2 two_of(uint32_t w) { return pair(bf16_lo(w), bf16_hi(w)); }
// x / (1 + e^-x).  The exponential and the reciprocal are the approximate ones, a few 2^-23 off (and the exponent's own rounding, 2^-24 of it), far below the half
// step of the bf16 outputs, 2^-8.  gdn_rows.cu has the like from other instructions, so the two forms' last bits differ.
LLM_DEVICE f32x2 silu2(f32x2 x) {
    const float2 e = both(mul2(x, pair(-1.44269504f, -1.44269504f)));
    float2 r = both(add2(pair(ex2(e.x), ex2(e.y)), pair(1.f, 1.f)));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.x) : "f"(r.x));
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r.y) : "f"(r.y));
    return mul2(x, pair(r.x, r.y));
}

// Eight rows from t0 of the chunk and the three in front of them, channels c .. c + 3, as they lie.  They are loaded without a branch, from places inside of the
// sequence, so that all of them are on their way together, and before the work that they do not depend on; `conv_rows` puts zeros in the place of what
// lies behind the chunk's rows, and the window in that of what lies before the sequence's first one.
constexpr int ROWS = 8;
LLM_DEVICE const __nv_bfloat16* row_of(const GdnParams& p, const Chunk& ch, int t, int c) {
    return p.in + (size_t)min(max(ch.row0 + t, ch.first), ch.row0 + ch.n - 1) * p.in_row + c;
}
struct Rows {
    uint2 raw[ROWS + 3];
    float4 taps[4];                                         // of a channel
};
LLM_DEVICE void load_rows(const GdnParams& p, const Chunk& ch, int t0, int c, Rows& x) {
#pragma unroll
    for (int e = 0; e < 4; ++e) x.taps[e] = *reinterpret_cast<const float4*>(p.conv_w + (size_t)(c + e) * 4);
#pragma unroll
    for (int i = 0; i < ROWS + 3; ++i) x.raw[i] = four(row_of(p, ch, t0 + i - 3, c), true);
}
// Convolution and SiLU of those rows; zeros behind the chunk's.  FAST: four taps, all on their boundaries; otherwise the rows are loaded here, tap by tap.
template <bool FAST>
LLM_DEVICE void conv_rows(const GdnParams& p, const Chunk& ch, int t0, int c, const Rows& in, f32x2 (&y)[ROWS][2]) {
    const int K = FAST ? 4 : p.K;
    auto before = [&](f32x2 (&x)[2], int t) {               // r < 0: of the window
        const int r = ch.row0 + t - ch.first;
        if (r >= 0) return;
        x[0] = x[1] = pair(0.f, 0.f);
        if (ch.fresh) return;
        const float* w = p.conv + ((size_t)ch.slot * p.C + c) * (K - 1) + (K - 1 + r);
        x[0] = pair(w[0], w[K - 1]);
        x[1] = pair(w[2 * (K - 1)], w[3 * (K - 1)]);
    };
    const bool edge = ch.row0 + t0 - (K - 1) < ch.first;
    if (FAST) {
        f32x2 x[ROWS + 3][2];
#pragma unroll
        for (int i = 0; i < ROWS + 3; ++i) {
            const bool there = t0 + i - 3 < ch.n;
            x[i][0] = two_of(there ? in.raw[i].x : 0u);
            x[i][1] = two_of(there ? in.raw[i].y : 0u);
        }
        if (edge) {
#pragma unroll
            for (int i = 0; i < 3; ++i) before(x[i], t0 + i - 3);
        }
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const float4 a = in.taps[2 * e], b = in.taps[2 * e + 1];
            const f32x2 w0 = pair(a.x, b.x), w1 = pair(a.y, b.y), w2 = pair(a.z, b.z), w3 = pair(a.w, b.w);
#pragma unroll
            for (int i = 0; i < ROWS; ++i) y[i][e] = fma2(w3, x[i + 3][e], fma2(w2, x[i + 2][e], fma2(w1, x[i + 1][e], mul2(w0, x[i][e]))));
        }
    } else {
#pragma unroll
        for (int i = 0; i < ROWS; ++i) y[i][0] = y[i][1] = pair(0.f, 0.f);
        for (int w = 0; w < K; ++w) {
            const float* f = p.conv_w + (size_t)c * K + w;
            const f32x2 f0 = pair(f[0], f[K]), f1 = pair(f[2 * K], f[3 * K]);
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                const int t = t0 + i + w - (K - 1);
                const uint2 v = four(row_of(p, ch, t, c), false);
                f32x2 x[2] = {two_of(t < ch.n ? v.x : 0u), two_of(t < ch.n ? v.y : 0u)};
                if (edge) before(x, t);
                y[i][0] = fma2(f0, x[0], y[i][0]);
                y[i][1] = fma2(f1, x[1], y[i][1]);
            }
        }
    }
#pragma unroll
    for (int i = 0; i < ROWS; ++i) {
        const bool there = t0 + i < ch.n;
#pragma unroll
        for (int e = 0; e < 2; ++e) y[i][e] = there ? silu2(y[i][e]) : pair(0.f, 0.f);
    }
}
// Sums of eight numbers over the warp's lanes: a lane ends up with that of number lane / 4
LLM_DEVICE float sums8(float (&v)[8], int lane) {
#pragma unroll
    for (int n = 4; n; n >>= 1) {
        const bool up = lane & (4 * n);
#pragma unroll
        for (int i = 0; i < n; ++i) {
            const float mine = up ? v[i + n] : v[i], other = up ? v[i] : v[i + n];
            v[i] = mine + __shfl_xor_sync(0xffffffffu, other, 4 * n);
        }
    }
    v[0] += __shfl_xor_sync(0xffffffffu, v[0], 2);
    return v[0] + __shfl_xor_sync(0xffffffffu, v[0], 1);
}

LLM_DEVICE uint32_t pack_half(float a, float b) {
    const __half2 v = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t*>(&v);
}
LLM_DEVICE float2 unpack_half(uint32_t w) { return __half22float2(*reinterpret_cast<const __half2*>(&w)); }
// two numbers as fp16 and what that leaves of them as fp16
LLM_DEVICE void split2(float a, float b, uint32_t& hi, uint32_t& lo) {
    hi = pack_half(a, b);
    const float2 h = unpack_half(hi);
    lo = pack_half(a - h.x, b - h.y);
}

LLM_DEVICE void split2(f32x2 v, uint32_t& hi, uint32_t& lo) {
    const float2 x = both(v);
    hi = pack_half(x.x, x.y);
    const float2 h = unpack_half(hi), l = both(fma2(pair(h.x, h.y), pair(-1.f, -1.f), v));
    lo = pack_half(l.x, l.y);
}
LLM_DEVICE float top2(float t, f32x2 v) {
    const float2 x = both(v);
    return fmaxf(t, fmaxf(fabsf(x.x), fabsf(x.y)));
}

LLM_DEVICE void ldsm4(uint32_t addr, uint32_t (&r)[4]) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(addr));
}
LLM_DEVICE void mma16(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// byte of column c's values of rows 4 q .. 4 q + 3: neighbours both for a lane of every fourth column (who writes) and for a lane of each (who reads)
LLM_DEVICE int val_at(int c, int q) { return q * (D * 16) + (c & 3) * (D * 4) + (((c >> 2) ^ (2 * (c & 3))) << 4); }
// byte of 16-byte unit u (0 .. 15) of row t in an image of K or Q
LLM_DEVICE int img_at(int t, int u) { return (u >> 3) * (IMG / 2) + t * 128 + (((u ^ t) & 7) << 4); }

constexpr int PREP_HEADS = 3;                               // value heads whose triangular systems are solved at the same time
constexpr int PREP_A = 2 * C * C * 4, PREP_DIAG = PREP_A + PREP_HEADS * 2 * TRI;           // k.k and q.k, then the matrices A (as two fp16 numbers), all where the images were
constexpr int PREP_SMEM = PREP_DIAG + PREP_HEADS * C * 16 * 4;                              // and their diagonal blocks in fp32
static_assert(PREP_DIAG >= KEY_BYTES, "the images");
constexpr float SX = 1024.f;                                // factor of sum_k A_ik T_kj = -(I + A_ii) T_ij, at most 17
constexpr int PREP_THREADS = 256, BAD_HEADS = 64;           // (of a key head's value heads, those 64 apart share a place)

struct ChunkParams {
    GdnParams g;
    uint8_t* ws;                                            // [units][n_ks] chunks of key heads, then [units][n_v] of value heads
    int n_ks, u0, units, first;                             // key heads in use, first chunk of this pass, chunks of it, whether it is the first pass
    int* status;
    int in_aligned, out_aligned;
};
LLM_DEVICE uint8_t* key_chunk(const ChunkParams& p, int u, int ks) { return p.ws + ((size_t)u * p.n_ks + ks) * KEY_BYTES; }
LLM_DEVICE uint8_t* head_chunk(const ChunkParams& p, int u, int h) { return p.ws + (size_t)p.units * p.n_ks * KEY_BYTES + ((size_t)u * p.g.n_v + h) * HEAD_BYTES; }

template <bool FAST>
__global__ void __launch_bounds__(PREP_THREADS, 2) gdn_chunk_prep_kernel(const ChunkParams cp) {
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ __align__(16) float2 s_G[PREP_HEADS][C];          // a sum as a float and what that leaves of it
    __shared__ float s_b[PREP_HEADS][C];
    __shared__ int s_chunk[6], s_bad[1 + BAD_HEADS];        // first rows whose keys, and whose values of a head, are not finite
    const GdnParams& p = cp.g;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int ks = blockIdx.x, u = blockIdx.y;              // value heads ks, ks + n_k, ... read this key head
    if (cp.first) pdl_wait();
    if (tid <= BAD_HEADS) s_bad[tid] = C;
    if (warp == 0) {
        int at;
        const int b = sequence_of(p, cp.u0 + u, at);
        if (lane == 0) {
            s_chunk[0] = b;
            if (b >= 0) {
                int first;
                const int n = rows_of(p, b, first), row0 = first + (cp.u0 + u - at) * C;
                s_chunk[1] = first; s_chunk[2] = row0; s_chunk[3] = min(C, first + n - row0);
                if (row0 - (p.K - 1) < first) {             // the window is read here alone
                    s_chunk[4] = LLM_CHECK_INDEX(p.slots[b], p.n_slots);
                    s_chunk[5] = p.positions[first];
                }
            }
        }
    }
    __syncthreads();
    // From the second pass on this kernel starts beside the scan of the pass before, which reads other memory.  The next launch waits for this one alone, so its last block waits for
    // that scan.
    const bool waits = blockIdx.x == gridDim.x - 1 && blockIdx.y == gridDim.y - 1;
    if (s_chunk[0] < 0) {
        if (waits) pdl_wait();
        return;
    }
    const Chunk ch = {s_chunk[1], s_chunk[2], s_chunk[3], s_chunk[4], s_chunk[5] == 0};
    const int kh = (ks + p.v_head_offset) % p.n_k;
    const uint32_t sm = smem_u32(smem);

    // ---- q, k, then b v of the value heads, transposed: a warp has eight rows, a lane four channels.  One loop, so that its code is fetched once ----
    {
        const int parts = 2 + (p.n_v - ks + p.n_k - 1) / p.n_k;
        auto channel = [&](int part) { return (part < 2 ? part * p.n_k + kh : 2 * p.n_k + ks + (part - 2) * p.n_k) * D + lane * 4; };
        Rows in;
        if (FAST) load_rows(p, ch, warp * ROWS, channel(0), in);
#pragma unroll 1
        for (int part = 0; part < parts; ++part) {
            f32x2 y[ROWS][2];
            conv_rows<FAST>(p, ch, warp * ROWS, channel(part), in, y);
            if (FAST && part + 1 < parts) load_rows(p, ch, warp * ROWS, channel(part + 1), in);
            float mine;                                     // a row's factor, in lanes 4 row .. 4 row + 3
            if (part < 2) {
                float ss[ROWS];
#pragma unroll
                for (int i = 0; i < ROWS; ++i) {
                    const float2 q = both(fma2(y[i][0], y[i][0], mul2(y[i][1], y[i][1])));
                    ss[i] = q.x + q.y;
                }
                mine = rsqrtf(sums8(ss, lane) + 1e-6f) * (part ? SK : SQ * 0.08838834764831845f);        // 128^-1/2
            } else {
                const int t = warp * ROWS + (lane >> 2);
                mine = t < ch.n ? beta(p, ch, t, ks + (part - 2) * p.n_k) : 0.f;
            }
#pragma unroll
            for (int i = 0; i < ROWS; ++i) {
                const float r = __shfl_sync(0xffffffffu, mine, 4 * i);
                y[i][0] = mul2(y[i][0], pair(r, r));
                y[i][1] = mul2(y[i][1], pair(r, r));
            }
            // A product of the chunk has all of its rows, those that do not see a row times 0: a key or a value that is not finite would reach the rows in front of
            // it.  Zeros take its place; from its row on the head's outputs, and its state, are no numbers (the gates, below).
            if (part > 0) {
                f32x2 any = pair(0.f, 0.f);                 // not finite if one of them is not (or, looked at again, if products overflow)
#pragma unroll
                for (int i = 0; i < ROWS; ++i) any = fma2(y[i][0], y[i][1], any);
                const float2 f = both(any);
                if (__any_sync(0xffffffffu, (f.x + f.y) * 0.f != 0.f)) {
                    unsigned rows = 0;
#pragma unroll
                    for (int i = 0; i < ROWS; ++i) {
                        const float2 g = both(fma2(y[i][1], pair(0.f, 0.f), mul2(y[i][0], pair(0.f, 0.f))));
                        rows |= g.x + g.y != 0.f ? 1u << i : 0u;
                    }
                    rows = __reduce_or_sync(0xffffffffu, rows);
#pragma unroll
                    for (int i = 0; i < ROWS; ++i)
                        if (rows >> i & 1) y[i][0] = y[i][1] = pair(0.f, 0.f);
                    if (lane == 0 && rows) atomicMin(&s_bad[part == 1 ? 0 : 1 + (part - 2) % BAD_HEADS], warp * ROWS + __ffs(rows) - 1);
                }
            }
            if (part < 2) {
                uint8_t* img = key_chunk(cp, u, ks);
#pragma unroll
                for (int i = 0; i < ROWS; ++i) {
                    uint2 hi, lo;
                    split2(y[i][0], hi.x, lo.x);
                    split2(y[i][1], hi.y, lo.y);
                    const int at_hi = (part ? OFF_KHI : OFF_QHI) + img_at(warp * ROWS + i, lane >> 1) + (lane & 1) * 8, at_lo = at_hi + IMG;
                    *reinterpret_cast<uint2*>(smem + at_hi) = hi; *reinterpret_cast<uint2*>(img + at_hi) = hi;
                    *reinterpret_cast<uint2*>(smem + at_lo) = lo; *reinterpret_cast<uint2*>(img + at_lo) = lo;
                }
            } else {
                uint8_t* dst = head_chunk(cp, u, ks + (part - 2) * p.n_k) + OFF_V;
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    float2 x[4][2];
#pragma unroll
                    for (int i = 0; i < 4; ++i) { x[i][0] = both(y[4 * q + i][0]); x[i][1] = both(y[4 * q + i][1]); }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        *reinterpret_cast<float4*>(dst + val_at(lane * 4 + 2 * e, 2 * warp + q)) = make_float4(x[0][e].x, x[1][e].x, x[2][e].x, x[3][e].x);
                        *reinterpret_cast<float4*>(dst + val_at(lane * 4 + 2 * e + 1, 2 * warp + q)) = make_float4(x[0][e].y, x[1][e].y, x[2][e].y, x[3][e].y);
                    }
                }
            }
        }
    }
    __syncthreads();

    // ---- k.k (warps 0 - 3) and q.k (warps 4 - 7, from the other end: as much for each quarter of the SM), 16 rows a warp, up to the diagonal ----
    {
        const bool kk = warp < 4;
        const int w = kk ? warp : 7 - warp, mat = lane >> 3, r8 = lane & 7;
        float acc[8][4];
#pragma unroll
        for (int n = 0; n < 8; ++n)
#pragma unroll
            for (int e = 0; e < 4; ++e) acc[n][e] = 0.f;
#pragma unroll 2
        for (int s = 0; s < 8; ++s) {
            uint32_t ah[4], al[4];
            const int a_at = img_at(16 * w + (lane & 15), 2 * s + (lane >> 4));
            ldsm4(sm + (kk ? OFF_KHI : OFF_QHI) + a_at, ah);
            ldsm4(sm + (kk ? OFF_KLO : OFF_QLO) + a_at, al);
#pragma unroll
            for (int n = 0; n < 4; ++n) {
                if (n > w) break;
                uint32_t bh[4], bl[4];
                const int b_at = img_at(16 * n + (mat >> 1) * 8 + r8, 2 * s + (mat & 1));
                ldsm4(sm + OFF_KHI + b_at, bh);
                ldsm4(sm + OFF_KLO + b_at, bl);
                mma16(acc[2 * n], ah, bh[0], bh[1]);
                mma16(acc[2 * n + 1], ah, bh[2], bh[3]);
                mma16(acc[2 * n], al, bh[0], bh[1]);
                mma16(acc[2 * n + 1], al, bh[2], bh[3]);
                mma16(acc[2 * n], ah, bl[0], bl[1]);
                mma16(acc[2 * n + 1], ah, bl[2], bl[3]);
            }
        }
        __syncthreads();                                    // the images have been read: the products take their place
        float* dst = reinterpret_cast<float*>(smem) + (kk ? 0 : C * C);
        const float f = kk ? 1.f / (SK * SK) : 1.f / SK;    // q.k keeps its factor SQ
#pragma unroll
        for (int n = 0; n < 8; ++n) {
            if (n > 2 * w + 1) break;
            const int t = 16 * w + (lane >> 2), i = 8 * n + (lane & 3) * 2;
            *reinterpret_cast<float2*>(dst + t * C + i) = make_float2(acc[n][0] * f, acc[n][1] * f);
            *reinterpret_cast<float2*>(dst + (t + 8) * C + i) = make_float2(acc[n][2] * f, acc[n][3] * f);
        }
    }
    const float* s_kk = reinterpret_cast<const float*>(smem);
    const float* s_qk = s_kk + C * C;

    for (int h0 = ks, place = 0; h0 < p.n_v; h0 += PREP_HEADS * p.n_k, place += PREP_HEADS) {
        const int nh = min(PREP_HEADS, (p.n_v - h0 + p.n_k - 1) / p.n_k);
        __syncthreads();
        // ---- gates: a warp per head, two rows a lane ----
        if (warp < nh) {
            const int h = h0 + warp * p.n_k;
            const float a = p.ssm_a[h], dt = p.dt_bias[h];
            float g[2], b[2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const int t = 2 * lane + e;
                g[e] = b[e] = 0.f;
                if (t < ch.n) {
                    const __nv_bfloat16* ab = p.in + (size_t)(ch.row0 + t) * p.in_row + p.ab_off;
                    const float x = __bfloat162float(ab[h]) + dt;
                    // -10000 is a decay of 0, and differences of sums that hold some of them stay numbers (of two infinities they would not)
                    const float log_decay = a * (x > 20.f ? x : log1pf(expf(x)));
                    g[e] = log_decay < -10000.f ? -10000.f : log_decay;
                    b[e] = beta(p, ch, t, h);
                }
            }
            int bad = min(s_bad[0], s_bad[1 + (place + warp) % BAD_HEADS]);
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const unsigned m = __ballot_sync(0xffffffffu, g[e] * b[e] != g[e] * b[e]);
                if (m) bad = min(bad, 2 * (__ffs(m) - 1) + e);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e)
                if (2 * lane + e >= bad) g[e] = b[e] = 0.f;
            // sums in units of ln 2, as exp2 takes them
            const double l0 = (double)g[0] * 1.4426950408889634, l1 = (double)g[1] * 1.4426950408889634;
            double sum = l0 + l1;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const double x = __shfl_up_sync(0xffffffffu, sum, o);
                if (lane >= o) sum += x;
            }
            const double G1 = sum, G0 = sum - l1, all = __shfl_sync(0xffffffffu, sum, 31);
            const float f0 = (float)G0, f1 = (float)G1;
            s_G[warp][2 * lane] = make_float2(f0, (float)(G0 - f0)); s_G[warp][2 * lane + 1] = make_float2(f1, (float)(G1 - f1));
            s_b[warp][2 * lane] = b[0]; s_b[warp][2 * lane + 1] = b[1];
            float2* vec = reinterpret_cast<float2*>(head_chunk(cp, u, h) + OFF_VEC);
            const float e0 = ex2((float)G0), e1 = ex2((float)G1), ea = bad < C ? __int_as_float(0x7fffffff) : ex2((float)all);
            vec[V_BE / 2 + lane] = make_float2(b[0] * e0, b[1] * e1);
            vec[V_EG / 2 + lane] = make_float2(2 * lane >= bad ? __int_as_float(0x7fffffff) : e0, 2 * lane + 1 >= bad ? __int_as_float(0x7fffffff) : e1);
            vec[V_EL / 2 + lane] = make_float2(ex2((float)(all - G0)), ex2((float)(all - G1)));
            vec[V_ALL / 2 + lane] = make_float2(ea, ea);
        }
        __syncthreads();
        // ---- A and P, up to the diagonal's blocks.  16 rows and 2, 4, 6, 8 units of eight columns for each block of rows ----
#pragma unroll 1
        for (int item = tid; item < nh * 320; item += PREP_THREADS) {
            const int hi = item / 320, k = item % 320, tb = (k >= 32) + (k >= 96) + (k >= 192), off = k - 16 * tb * (tb + 1), half = off >> 1;
            const int row = tb == 0 ? half : tb == 1 ? half >> 1 : tb == 2 ? (half * 43) >> 7 : half >> 2;       // off / (2 tb + 2), off < 128
            const int t = 16 * tb + row, unit = off - 2 * (tb + 1) * row;
            uint8_t* dst = head_chunk(cp, u, h0 + hi * p.n_k);
            uint8_t* A = smem + PREP_A + hi * 2 * TRI;
            const float2 Gt = s_G[hi][t];
            const float b = s_b[hi][t];
            float a8[8], p8[8], G4[4][4], kk[8], qk[8];
#pragma unroll
            for (int e = 0; e < 4; ++e) *reinterpret_cast<float4*>(G4[e]) = *reinterpret_cast<const float4*>(&s_G[hi][unit * 8 + 2 * e]);
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                *reinterpret_cast<float4*>(kk + e) = *reinterpret_cast<const float4*>(s_kk + t * C + unit * 8 + e);
                *reinterpret_cast<float4*>(qk + e) = *reinterpret_cast<const float4*>(s_qk + t * C + unit * 8 + e);
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int i = unit * 8 + e;
                const float m = ex2((Gt.x - G4[e >> 1][2 * (e & 1)]) + (Gt.y - G4[e >> 1][2 * (e & 1) + 1]));
                p8[e] = i <= t ? m * qk[e] : 0.f;
                a8[e] = i < t ? b * m * kk[e] : 0.f;
            }
            if (unit >> 1 == tb) {
                float* diag = reinterpret_cast<float*>(smem + PREP_DIAG) + hi * C * 16 + t * 16 + (unit & 1) * 8;
                *reinterpret_cast<float4*>(diag) = make_float4(a8[0], a8[1], a8[2], a8[3]);
                *reinterpret_cast<float4*>(diag + 4) = make_float4(a8[4], a8[5], a8[6], a8[7]);
            }
            uint4 ph, pl, ah, al;
#pragma unroll
            for (int e = 0; e < 8; ++e) a8[e] *= SK;
            split2(a8[0], a8[1], ah.x, al.x); split2(a8[2], a8[3], ah.y, al.y); split2(a8[4], a8[5], ah.z, al.z); split2(a8[6], a8[7], ah.w, al.w);
            split2(p8[0], p8[1], ph.x, pl.x); split2(p8[2], p8[3], ph.y, pl.y); split2(p8[4], p8[5], ph.z, pl.z); split2(p8[6], p8[7], ph.w, pl.w);
            const int at = t * 128 + (((unit ^ t) & 7) << 4);
            *reinterpret_cast<uint4*>(A + at) = ah;
            *reinterpret_cast<uint4*>(A + TRI + at) = al;
            *reinterpret_cast<uint4*>(dst + OFF_PHI + at) = ph;
            *reinterpret_cast<uint4*>(dst + OFF_PLO + at) = pl;
        }
        // zeros of P above them: 16 rows and 6, 4, 2 units
#pragma unroll 1
        for (int item = tid; item < nh * 192; item += PREP_THREADS) {
            const int hi = item / 192, k = item % 192, tb = (k >= 96) + (k >= 160);
            const int row = tb == 0 ? k / 6 : tb == 1 ? (k - 96) >> 2 : (k - 160) >> 1;
            const int t = 16 * tb + row, unit = 2 * (tb + 1) + (tb == 0 ? k - 6 * row : tb == 1 ? (k - 96) & 3 : (k - 160) & 1);
            uint8_t* at = head_chunk(cp, u, h0 + hi * p.n_k) + t * 128 + (((unit ^ t) & 7) << 4);
            *reinterpret_cast<uint4*>(at + OFF_PHI) = make_uint4(0, 0, 0, 0);
            *reinterpret_cast<uint4*>(at + OFF_PLO) = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
        // ---- the diagonal's blocks of T, in the place of A's: a thread per column ----
        if (tid < nh * C) {
            const int hi = tid / C, j = tid % C, at = j & 15;
            const float* diag = reinterpret_cast<const float*>(smem + PREP_DIAG) + hi * C * 16 + (j & ~15) * 16;
            float x[16];
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float sum = i == at ? 1.f : 0.f;
#pragma unroll
                for (int m = 0; m < i; m += 4) {
                    const float4 a = *reinterpret_cast<const float4*>(diag + i * 16 + m);       // zeros from column i on
                    sum -= a.x * x[m];
                    if (m + 1 < i) sum -= a.y * x[m + 1];
                    if (m + 2 < i) sum -= a.z * x[m + 2];
                    if (m + 3 < i) sum -= a.w * x[m + 3];
                }
                x[i] = sum;
            }
            uint8_t* T = smem + PREP_A + hi * 2 * TRI + (j & 7) * 2;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float f = x[i] * SK;
                const __half h = __float2half_rn(f), l = __float2half_rn(f - __half2float(h));
                const int t = (j & ~15) + i, row = t * 128 + (((j >> 3) ^ (t & 7)) << 4);
                *reinterpret_cast<__half*>(T + row) = h;
                *reinterpret_cast<__half*>(T + TRI + row) = l;
            }
        }
        __syncthreads();
        // ---- the other blocks, T_ij transposed at (j, i): a left operand of the next product as it comes out ----
#pragma unroll 1
        for (int item = warp; item < nh * 3; item += PREP_THREADS / 32) {
            const int hi = item % nh, j = item / nh, mat = lane >> 3, r8 = lane & 7;
            const uint32_t A = sm + PREP_A + hi * 2 * TRI;
            // 16 x 16 block (bi, bj) as the right operand of a product with its transpose
            auto right = [&](int bi, int bj, uint32_t (&h)[4], uint32_t (&l)[4]) {
                const int row = 16 * bi + (mat >> 1) * 8 + r8;
                const uint32_t at = A + row * 128 + (((2 * bj + (mat & 1)) ^ (row & 7)) << 4);
                ldsm4(at, h);
                ldsm4(at + TRI, l);
            };
            auto product = [&](float (&acc)[2][4], const uint32_t (&ah)[4], const uint32_t (&al)[4], const uint32_t (&bh)[4], const uint32_t (&bl)[4]) {
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    mma16(acc[n], ah, bh[2 * n], bh[2 * n + 1]);
                    mma16(acc[n], al, bh[2 * n], bh[2 * n + 1]);
                    mma16(acc[n], ah, bl[2 * n], bl[2 * n + 1]);
                }
            };
            auto left = [&](const float (&acc)[2][4], float f, uint32_t (&h)[4], uint32_t (&l)[4]) {
#pragma unroll
                for (int e = 0; e < 4; ++e) split2(acc[e >> 1][2 * (e & 1)] * f, acc[e >> 1][2 * (e & 1) + 1] * f, h[e], l[e]);
            };
            uint32_t th[4][4], tl[4][4];                    // T_kj transposed, k = j, j + 1, ... (from place 0 on)
            {
                const int row = 16 * j + (mat >> 1) * 8 + r8;
                const uint32_t at = A + row * 128 + (((2 * j + (mat & 1)) ^ (row & 7)) << 4);
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(th[0][0]), "=r"(th[0][1]), "=r"(th[0][2]), "=r"(th[0][3]) : "r"(at));
                asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(tl[0][0]), "=r"(tl[0][1]), "=r"(tl[0][2]), "=r"(tl[0][3]) : "r"(at + TRI));
            }
#pragma unroll
            for (int step = 1; step < 4; ++step) {
                const int i = j + step;
                if (i > 3) break;
                float acc[2][4] = {};
                uint32_t bh[4], bl[4], xh[4], xl[4];
#pragma unroll
                for (int k = 0; k < step; ++k) {
                    right(i, j + k, bh, bl);
                    product(acc, th[k], tl[k], bh, bl);
                }
                left(acc, SX / (SK * SK), xh, xl);
                float out[2][4] = {};
                right(i, i, bh, bl);
                product(out, xh, xl, bh, bl);
                left(out, -1.f / SX, th[step], tl[step]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {               // rows lane / 4 (+ 8), columns of the 8-value unit e / 2
                    const int row = 16 * j + (lane >> 2) + (e & 1) * 8;
                    uint8_t* at = smem + PREP_A + hi * 2 * TRI + row * 128 + (((2 * i + (e >> 1)) ^ (row & 7)) << 4) + (lane & 3) * 4;
                    *reinterpret_cast<uint32_t*>(at) = th[step][e];
                    *reinterpret_cast<uint32_t*>(at + TRI) = tl[step][e];
                }
            }
        }
        __syncthreads();
        pdl_trigger();                                      // the scan's blocks may come up
        // ---- T as the scan reads it: the blocks below the diagonal back from their transposes, in the place of A's ----
#pragma unroll 1
        for (int item = warp; item < nh * 12; item += PREP_THREADS / 32) {
            const int part = item % (nh * 2), pr = item / (nh * 2);        // head and half of the number; block (i, j)
            const int i = pr == 0 ? 1 : pr < 3 ? 2 : 3, j = pr - i * (i - 1) / 2, mat = lane >> 3, r8 = lane & 7;
            uint8_t* T = smem + PREP_A + part * TRI;
            uint32_t x[4];
            const uint32_t from = smem_u32(T) + (16 * j + 8 * (mat & 1) + r8) * 128 + (((2 * i + (mat >> 1)) ^ r8) << 4);
            asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(x[0]), "=r"(x[1]), "=r"(x[2]), "=r"(x[3]) : "r"(from));
#pragma unroll
            for (int m = 0; m < 4; ++m) {
                const int t = 16 * i + 8 * (m >> 1) + (lane >> 2);
                *reinterpret_cast<uint32_t*>(T + t * 128 + (((2 * j + (m & 1)) ^ (t & 7)) << 4) + (lane & 3) * 4) = x[m];
            }
            __syncwarp();                                   // all lanes have the transpose: zeros above the diagonal
            const int above = 16 * j + (lane & 15);
            *reinterpret_cast<uint4*>(T + above * 128 + (((2 * i + (lane >> 4)) ^ (above & 7)) << 4)) = make_uint4(0, 0, 0, 0);
        }
        __syncthreads();
#pragma unroll 4
        for (int item = tid; item < nh * 2 * (TRI / 16); item += PREP_THREADS) {
            const int hi = item / (2 * TRI / 16), at = item % (2 * TRI / 16) * 16;
            *reinterpret_cast<uint4*>(head_chunk(cp, u, h0 + hi * p.n_k) + OFF_THI + at) = *reinterpret_cast<const uint4*>(smem + PREP_A + hi * 2 * TRI + at);
        }
    }
    if (waits) pdl_wait();
}

// ------------------------------------------------------------------------------------------------
// scan
// ------------------------------------------------------------------------------------------------
// Warps 0-3 and 4-7 are the two math groups: a thread has a value column (== TMEM lane), the groups share out a row's columns.  Warps 8-11 write the output,
// warp 12 copies, warp 13 allocates tensor memory and issues the products.
constexpr int THREADS = 512;
constexpr int REGS_MATH = 176, REGS_OUT = 104, REGS_REST = 56, REGS_LAUNCH = 128;
static_assert(2 * REGS_MATH + REGS_OUT + REGS_REST <= 4 * REGS_LAUNCH, "a warpgroup would wait for registers that nobody gives back");
// shared memory: K, T and the vectors in two stages; V, Q and P, which are free again while their chunk is still at work, once; the output's rows
constexpr int ST_T = 2 * IMG, ST_VEC = ST_T + 2 * TRI, STAGE_BYTES = ST_VEC + VEC_BYTES;
constexpr int SM_V = 2 * STAGE_BYTES, SM_Q = SM_V + VALS, SM_P = SM_Q + 2 * IMG, SM_O = SM_P + 2 * TRI, SCAN_SMEM = SM_O + C * D * 4 + 1024;
static_assert(STAGE_BYTES % 1024 == 0 && SM_Q % 1024 == 0 && SM_P % 1024 == 0, "tiles start on swizzle atoms");
static_assert(SCAN_SMEM <= 227 * 1024, "shared memory of a CTA");
// tensor memory columns; the state's sum takes the columns of the state operand, U those of S^T k, U' those of R
constexpr uint32_t T_SHI = 0, T_SLO = 64, T_DS = 0, T_KS = 128, T_QS = 192, T_PU = 256, T_RHI = 320, T_RLO = 352, T_UHI = 384, T_ULO = 416;
__host__ __device__ constexpr uint32_t idesc(int n) { return (1u << 4) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(128 >> 4) << 24); }     // fp16 x fp16 -> fp32, M = 128

enum Bar { IN_FULL = 0, IN_EMPTY = 2, V_FULL = 4, V_EMPTY, Q_FULL, Q_EMPTY, P_FULL, P_EMPTY, S_RDY, KS_DONE = S_RDY + 2, R_RDY, U_DONE, U_RDY, UO_RDY, DS_DONE, O_DONE, O_FREE, N_BARS };

// the power of two that brings `top` into [2^13, 2^14), and its inverse
LLM_DEVICE void scale_for(float top, float& s, float& inv) {
    const int e = (int)(__float_as_uint(top) >> 23);        // 0 .. 255: top >= 0
    const int b = min(253, 267 - e);
    s = __uint_as_float((uint32_t)b << 23);
    inv = __uint_as_float((uint32_t)(254 - b) << 23);
}
LLM_DEVICE void tmem_ld16_issue(uint32_t taddr, uint32_t (&r)[16]) {       // readable behind the next wait, and `keep`
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]) : "r"(taddr));
}
template <int N> LLM_DEVICE void keep(uint32_t (&r)[N]) {
#pragma unroll
    for (int i = 0; i < N; ++i) asm volatile("" : "+r"(r[i]));
}
LLM_DEVICE f32x2 pair_of(uint32_t a, uint32_t b) { return pair(__uint_as_float(a), __uint_as_float(b)); }
LLM_DEVICE void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
LLM_DEVICE float4 lds4(uint32_t a) {
    float4 v;
    asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(a));
    return v;
}

__global__ void __launch_bounds__(THREADS, 1) gdn_chunk_scan_kernel(const ChunkParams cp) {
    extern __shared__ uint8_t smem_raw[];
    __shared__ __align__(8) uint64_t s_bars[N_BARS];
    __shared__ uint32_t s_tmem;
    __shared__ int s_abort[2];                              // [1] stays 0 here (tc_common.cuh: restarts the wait clock when set)
    __shared__ int s_first[3];
    __shared__ float s_top[3][2][D];                        // largest magnitudes of a column, per math group
    __shared__ float s_inv[2][2][D];                        // inverse scales of S and U, by parity of the chunk
    const GdnParams& p = cp.g;
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int h = blockIdx.x, b = blockIdx.y;
    if (warp == 0) {
        const int before = chunks_before(p, b);
        if (lane == 0) s_first[0] = before;
    }
    __syncthreads();
    int first;
    const int n_rows = rows_of(p, b, first), u_first = s_first[0];
    const int c0 = max(0, cp.u0 - u_first), c1 = min((n_rows + C - 1) / C, cp.u0 + cp.units - u_first);
    if (c0 >= c1) return;                                   // uniform for the CTA, before any barrier or allocation
    const int nc = c1 - c0, u_ws = u_first + c0 - cp.u0;    // chunks of this pass, the first one's place in the workspace
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;
    const uint32_t bars = smem_u32(s_bars);
    auto bar = [&](int i) { return bars + i * 8; };
    if (tid == 0) {
        s_abort[0] = 0; s_abort[1] = 0;
        for (int i = 0; i < N_BARS; ++i) {
            int n = 1;
            if (i == IN_EMPTY || i == IN_EMPTY + 1) n = 1 + 8 + 4;                   // the products, the math and the output warps
            if (i == S_RDY || i == S_RDY + 1 || i == R_RDY || i == U_RDY || i == UO_RDY || i == V_EMPTY) n = 8;
            if (i == O_FREE) n = 4;
            mbar_init(bar(i), n);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_proxy_async();
    }
    if (warp == 13) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(&s_tmem)), "r"(512) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_wait();                                             // for this pass' chunks, and the scan before it
    pdl_trigger();                                          // what comes next writes nothing that is read here
    const uint32_t tmem = s_tmem;
    volatile int* abort_flag = s_abort;
    auto stage = [&](int c) { return base + (c & 1) * STAGE_BYTES; };
    auto phase = [](int c) { return (uint32_t)((c >> 1) & 1); };               // of a stage's barriers

    if (warp < 8) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(REGS_MATH));
        const int w = warp >> 2, col = tid & 127;
        const uint32_t t_lane = tmem + ((uint32_t)((warp & 3) * 32) << 16);
        const bool fresh = c0 == 0 && p.positions[first] == 0;
        const int slot = LLM_CHECK_INDEX(p.slots[b], p.n_slots);
        float* state = p.rec + ((size_t)slot * p.n_v + h) * (D * D) + (size_t)w * 64 * D + col;
        f32x2 S[32];
#pragma unroll
        for (int i = 0; i < 32; ++i) S[i] = fresh ? pair(0.f, 0.f) : pair(state[(size_t)(2 * i) * D], state[(size_t)(2 * i + 1) * D]);
        // largest magnitude of the column over both groups
        auto column_top = [&](int which, float mine) {
            s_top[which][w][col] = mine;
            tc_fence_before();
            bar_sync(1, 256);
            tc_fence_after();
            return fmaxf(mine, s_top[which][w ^ 1][col]);
        };
        float top_s = 0.f;                                  // of the state
#pragma unroll
        for (int i = 0; i < 32; ++i) top_s = top2(top_s, S[i]);
        bool ok = true;                                     // after a wait that gave up all go on, without further waits, since they meet at barriers
        for (int c = 0; c < nc; ++c) {
            const uint32_t vec = stage(c) + ST_VEC, vals = base + SM_V + val_at(col, 0);
            float s, inv;
            // ---- the state as an operand ----
            {
                scale_for(column_top(0, top_s), s, inv);
                if (w == 0) s_inv[c & 1][0][col] = inv;
#pragma unroll
                for (int half = 0; half < 2; ++half) {       // S^T k begins with the first half
                    uint32_t hi[16], lo[16];
#pragma unroll
                    for (int i = 0; i < 16; ++i) split2(mul2(S[16 * half + i], pair(s, s)), hi[i], lo[i]);
                    tmem_st_n<16>(t_lane + T_SHI + w * 32 + half * 16, hi);
                    tmem_st_n<16>(t_lane + T_SLO + w * 32 + half * 16, lo);
                    tmem_wait_st();
                    tc_fence_before();
                    __syncwarp();
                    mbar_arrive_if(bar(S_RDY + half), lane == 0);
                }
            }
            // ---- R = b v - b e^G S^T k ----
            ok = ok && mbar_wait_warp(bar(IN_FULL + (c & 1)), phase(c), abort_flag) && mbar_wait_warp(bar(V_FULL), c & 1, abort_flag);
            {
                float4 v[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) v[q] = lds4(vals + (8 * w + q) * (D * 16));
                ok = ok && mbar_wait_warp(bar(KS_DONE), c & 1, abort_flag);
                tc_fence_after();
                uint32_t x[32];
                tmem_ld_n<32>(t_lane + T_KS + w * 32, x);
                const float f = -inv * (1.f / SK);
                const f32x2 f2 = pair(f, f);
                f32x2 r[16];
                float top = 0.f;
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    const float4 be = lds4(vec + (V_BE + 32 * w + 4 * q) * 4);
                    r[2 * q] = fma2(mul2(pair(be.x, be.y), f2), pair_of(x[4 * q], x[4 * q + 1]), pair(v[q].x, v[q].y));
                    r[2 * q + 1] = fma2(mul2(pair(be.z, be.w), f2), pair_of(x[4 * q + 2], x[4 * q + 3]), pair(v[q].z, v[q].w));
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) top = top2(top, r[i]);
                scale_for(column_top(1, top), s, inv);
                uint32_t hi[16], lo[16];
#pragma unroll
                for (int i = 0; i < 16; ++i) split2(mul2(r[i], pair(s, s)), hi[i], lo[i]);
                tmem_st_n<16>(t_lane + T_RHI + w * 16, hi);
                tmem_st_n<16>(t_lane + T_RLO + w * 16, lo);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                mbar_arrive_if(bar(R_RDY), lane == 0);
                mbar_arrive_if(bar(V_EMPTY), lane == 0);
            }
            // ---- U = T R; U e^(G_C - G) for the state ----
            float4 el[8];
#pragma unroll
            for (int q = 0; q < 8; ++q) el[q] = lds4(vec + (V_EL + 32 * w + 4 * q) * 4);
            const float decay = lds4(vec + V_ALL * 4).x;
            ok = ok && mbar_wait_warp(bar(U_DONE), c & 1, abort_flag);
            tc_fence_after();
            {
                uint32_t x[32], hi[16], lo[16];
                tmem_ld_n<32>(t_lane + T_KS + w * 32, x);
                const float f = inv * (1.f / SK);
                float top = 0.f;
#pragma unroll
                for (int i = 0; i < 32; i += 2) top = top2(top, pair_of(x[i], x[i + 1]));
                scale_for(column_top(2, top), s, inv);       // of the accumulator as it is: its own factor f goes into the inverse
                inv *= f;
                f32x2 a[16];
#pragma unroll
                for (int q = 0; q < 8; ++q) {
                    a[2 * q] = mul2(pair_of(x[4 * q], x[4 * q + 1]), pair(s, s));
                    a[2 * q + 1] = mul2(pair_of(x[4 * q + 2], x[4 * q + 3]), pair(s, s));
                    split2(mul2(a[2 * q], pair(el[q].x, el[q].y)), hi[2 * q], lo[2 * q]);
                    split2(mul2(a[2 * q + 1], pair(el[q].z, el[q].w)), hi[2 * q + 1], lo[2 * q + 1]);
                }
                tmem_st_n<16>(t_lane + T_RHI + w * 16, hi);
                tmem_st_n<16>(t_lane + T_RLO + w * 16, lo);
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                mbar_arrive_if(bar(U_RDY), lane == 0);
                // the state's sum is on its way: U for the output
#pragma unroll
                for (int i = 0; i < 16; ++i) split2(a[i], hi[i], lo[i]);
                tmem_st_n<16>(t_lane + T_UHI + w * 16, hi);
                tmem_st_n<16>(t_lane + T_ULO + w * 16, lo);
                if (w == 0) s_inv[c & 1][1][col] = inv;
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                mbar_arrive_if(bar(UO_RDY), lane == 0);
                mbar_arrive_if(bar(IN_EMPTY + (c & 1)), lane == 0);
            }
            // ---- S = e^G_C S + sum ----
            ok = ok && mbar_wait_warp(bar(DS_DONE), c & 1, abort_flag);
            tc_fence_after();
            const float f = inv * (1.f / SK);
            top_s = 0.f;
#pragma unroll
            for (int half = 0; half < 2; ++half) {
                uint32_t x[32];
                tmem_ld_n<32>(t_lane + T_DS + w * 64 + half * 32, x);
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    S[half * 16 + i] = fma2(pair(f, f), pair_of(x[2 * i], x[2 * i + 1]), mul2(pair(decay, decay), S[half * 16 + i]));
                    top_s = top2(top_s, S[half * 16 + i]);
                }
            }
        }
        if (ok) {
#pragma unroll
            for (int i = 0; i < 32; ++i) {
                const float2 x = both(S[i]);
                state[(size_t)(2 * i) * D] = x.x;
                state[(size_t)(2 * i + 1) * D] = x.y;
            }
        }
    } else if (warp < 12) {
        // ------------------------------ output: o, gated norm ------------------------------
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_OUT));
        const int ow = warp - 8, col = tid & 127;
        const uint32_t t_lane = tmem + ((uint32_t)(ow * 32) << 16);
        const f32x2 gain0 = pair(p.norm_w[lane * 4], p.norm_w[lane * 4 + 1]), gain1 = pair(p.norm_w[lane * 4 + 2], p.norm_w[lane * 4 + 3]);
        const bool in_aligned = cp.in_aligned, out_aligned = cp.out_aligned;
        bool ok = true;
        for (int c = 0; c < nc; ++c) {
            const int row0 = first + (c0 + c) * C, n = min(C, first + n_rows - row0);
            uint2 z[C / 4];                                 // the rows' gates, on their way while the chunk is at work
#pragma unroll
            for (int i = 0; i < C / 4; ++i) {
                const __nv_bfloat16* x = p.in + (size_t)(row0 + min(i * 4 + ow, n - 1)) * p.in_row + p.z_off + h * D + lane * 4;
                z[i] = four(x, in_aligned);
            }
            ok = ok && mbar_wait_warp(bar(O_DONE), c & 1, abort_flag);
            tc_fence_after();
            bar_sync(2, 128);                               // the last chunk's rows have been read
            const uint32_t vec = stage(c) + ST_VEC, rows = base + SM_O;
            const float fs = s_inv[c & 1][0][col] * (1.f / SQ), fu = s_inv[c & 1][1][col] * (1.f / SQ);
#pragma unroll
            for (int part = 0; part < 4; ++part) {
                uint32_t a[16], e[16];
                tmem_ld16_issue(t_lane + T_QS + part * 16, a);
                tmem_ld_n<16>(t_lane + T_PU + part * 16, e);
                keep(a);
#pragma unroll
                for (int q = 0; q < 4; ++q) {
                    const float4 eg = lds4(vec + (V_EG + part * 16 + q * 4) * 4);
                    const float g[4] = {eg.x, eg.y, eg.z, eg.w};
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const float o = fmaf(g[k] * fs, __uint_as_float(a[4 * q + k]), fu * __uint_as_float(e[4 * q + k]));
                        asm volatile("st.shared.f32 [%0], %1;" ::"r"(rows + (part * 16 + q * 4 + k) * (D * 4) + col * 4), "f"(o) : "memory");
                    }
                }
            }
            tc_fence_before();
            bar_sync(2, 128);
            mbar_arrive_if(bar(O_FREE), lane == 0);
            mbar_arrive_if(bar(IN_EMPTY + (c & 1)), lane == 0);
#pragma unroll
            for (int i0 = 0; i0 < C / 4; i0 += ROWS) {      // eight rows at a time: their sums go through the lanes together
                f32x2 o[ROWS][2];
                float ss[ROWS];
#pragma unroll
                for (int k = 0; k < ROWS; ++k) {
                    const float4 v = lds4(rows + ((i0 + k) * 4 + ow) * (D * 4) + lane * 16);
                    o[k][0] = pair(v.x, v.y);
                    o[k][1] = pair(v.z, v.w);
                    const float2 q = both(fma2(o[k][0], o[k][0], mul2(o[k][1], o[k][1])));
                    ss[k] = q.x + q.y;
                }
                const float mine = rsqrtf(sums8(ss, lane) * (1.f / D) + p.eps);
#pragma unroll
                for (int k = 0; k < ROWS; ++k) {
                    const uint2 g = z[i0 + k];
                    const float r = __shfl_sync(0xffffffffu, mine, 4 * k);
                    const float2 a = both(mul2(mul2(mul2(o[k][0], pair(r, r)), gain0), silu2(two_of(g.x)))), e = both(mul2(mul2(mul2(o[k][1], pair(r, r)), gain1), silu2(two_of(g.y))));
                    const uint2 v = make_uint2(pack_bf16(a.x, a.y), pack_bf16(e.x, e.y));
                    const int t = (i0 + k) * 4 + ow;
                    __nv_bfloat16* dst = p.out + (size_t)(row0 + t) * p.out_row + h * D + lane * 4;
                    if (t < n && ok && out_aligned) *reinterpret_cast<uint2*>(dst) = v;
                    if (t < n && ok && !out_aligned) {
                        dst[0] = __ushort_as_bfloat16(v.x & 0xffff); dst[1] = __ushort_as_bfloat16(v.x >> 16);
                        dst[2] = __ushort_as_bfloat16(v.y & 0xffff); dst[3] = __ushort_as_bfloat16(v.y >> 16);
                    }
                }
            }
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(REGS_REST));
        if (warp == 12 && elect_one()) {
            // ------------------------------ copies ------------------------------
            const int ks = h % p.n_k;
            auto load = [&](int full, int empty, uint32_t parity, int bytes) {
                if (!mbar_wait(bar(empty), parity ^ 1, abort_flag)) return false;
                mbar_arrive_expect_tx(bar(full), bytes);
                return true;
            };
            for (int c = 0; c < nc; ++c) {
                const uint8_t *key = key_chunk(cp, u_ws + c, ks), *head = head_chunk(cp, u_ws + c, h);
                const int in = IN_FULL + (c & 1);
                if (!load(in, IN_EMPTY + (c & 1), phase(c), STAGE_BYTES)) break;
                bulk_load(stage(c), key + OFF_KHI, 2 * IMG, bar(in));
                bulk_load(stage(c) + ST_T, head + OFF_THI, 2 * TRI, bar(in));
                bulk_load(stage(c) + ST_VEC, head + OFF_VEC, VEC_BYTES, bar(in));
                if (!load(V_FULL, V_EMPTY, c & 1, VALS)) break;
                bulk_load(base + SM_V, head + OFF_V, VALS, bar(V_FULL));
                if (!load(Q_FULL, Q_EMPTY, c & 1, 2 * IMG)) break;
                bulk_load(base + SM_Q, key + OFF_QHI, 2 * IMG, bar(Q_FULL));
                if (!load(P_FULL, P_EMPTY, c & 1, 2 * TRI)) break;
                bulk_load(base + SM_P, head + OFF_PHI, 2 * TRI, bar(P_FULL));
            }
        } else if (warp == 13 && elect_one()) {
            // ------------------------------ products ------------------------------
            constexpr uint32_t MN = 1u << 16;               // right operand with its rows along K
            for (int c = 0; c < nc; ++c) {
                uint32_t tm = tmem, sm = base;
                asm volatile("" : "+r"(tm), "+r"(sm));      // addresses are added up where they are used, not kept from one chunk to the next
                const uint32_t key = sm + (c & 1) * STAGE_BYTES, tri = key + ST_T, q = sm + SM_Q, pt = sm + SM_P;
                if (!mbar_wait(bar(IN_FULL + (c & 1)), phase(c), abort_flag) || !mbar_wait(bar(S_RDY), c & 1, abort_flag)) break;
                tc_fence_after();
                // (a descriptor counts 16 bytes: what lies in one image is reached by addition)
                auto with_rows = [&](uint32_t d, uint32_t a, uint32_t img, int half, bool first_one) {        // [128 columns x d] [64 rows x d]^T, d from 32 half and 64 + 32 half on
                    const uint64_t desc = smem_desc_sw128(img) + 4 * half;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int at = (k >> 1) * 4 + (k & 1);
                        mma_f16_ts(tm + d, tm + a + (at + 2 * half) * 8, desc + (k >> 1) * (IMG / 2 / 16) + 2 * (k & 1), idesc(C), !first_one || k > 0 ? 1u : 0u);
                    }
                };
                // [128 columns x 64 rows] times a lower triangle's transpose.  All of one shape and accumulator, zeros above the diagonal included: only such products are
                // promised to run in the order in which they are issued, and each adds to what the one before left
                auto with_tri = [&](uint32_t d, uint32_t a, uint32_t img, bool first_one) {
                    const uint64_t desc = smem_desc_sw128(img);
#pragma unroll
                    for (int k = 0; k < 4; ++k) mma_f16_ts(tm + d, tm + a + k * 8, desc + 2 * k, idesc(C), !first_one || k > 0 ? 1u : 0u);
                };
                auto with_keys = [&](uint32_t a, uint32_t img, bool first_one) {                  // [128 columns x 64 rows] [64 rows x d]
                    const uint64_t desc = smem_desc_mn_sw128(img, IMG / 2);
#pragma unroll
                    for (int k = 0; k < 4; ++k)
                        mma_f16_ts(tm + T_DS, tm + a + k * 8, desc + k * (16 * 128 / 16), idesc(D) | MN, !first_one || k > 0 ? 1u : 0u);
                };
                with_rows(T_KS, T_SHI, key, 0, true);
                with_rows(T_KS, T_SLO, key, 0, false);
                with_rows(T_KS, T_SHI, key + IMG, 0, false);
                if (!mbar_wait(bar(S_RDY + 1), c & 1, abort_flag)) break;
                tc_fence_after();
                with_rows(T_KS, T_SHI, key, 1, false);
                with_rows(T_KS, T_SLO, key, 1, false);
                with_rows(T_KS, T_SHI, key + IMG, 1, false);
                mma_commit(bar(KS_DONE));
                if (!mbar_wait(bar(Q_FULL), c & 1, abort_flag) || (c > 0 && !mbar_wait(bar(O_FREE), (c - 1) & 1, abort_flag))) break;
                tc_fence_after();
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    with_rows(T_QS, T_SHI, q, half, half == 0);
                    with_rows(T_QS, T_SLO, q, half, false);
                    with_rows(T_QS, T_SHI, q + IMG, half, false);
                }
                mma_commit(bar(Q_EMPTY));
                if (!mbar_wait(bar(R_RDY), c & 1, abort_flag)) break;
                tc_fence_after();
                with_tri(T_KS, T_RHI, tri, true);
                with_tri(T_KS, T_RLO, tri, false);
                with_tri(T_KS, T_RHI, tri + TRI, false);
                mma_commit(bar(U_DONE));
                if (!mbar_wait(bar(U_RDY), c & 1, abort_flag)) break;
                tc_fence_after();
                with_keys(T_RHI, key, true);
                with_keys(T_RLO, key, false);
                with_keys(T_RHI, key + IMG, false);
                mma_commit(bar(DS_DONE));
                if (!mbar_wait(bar(P_FULL), c & 1, abort_flag) || !mbar_wait(bar(UO_RDY), c & 1, abort_flag)) break;
                tc_fence_after();
                with_tri(T_PU, T_UHI, pt, true);
                with_tri(T_PU, T_ULO, pt, false);
                with_tri(T_PU, T_UHI, pt + TRI, false);
                mma_commit(bar(IN_EMPTY + (c & 1)));
                mma_commit(bar(P_EMPTY));
                mma_commit(bar(O_DONE));
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    teardown(abort_flag, tid, cp.status);
    if (warp == 13) asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
}

}  // namespace gdc

// Bytes of workspace that a pass over `units` chunks takes
size_t gdn_chunk_bytes(int units, int n_k, int n_v) {
    return (size_t)units * ((size_t)(n_k < n_v ? n_k : n_v) * gdc::KEY_BYTES + (size_t)n_v * gdc::HEAD_BYTES);
}

cudaError_t launch_gdn_chunk(const GdnParams& g, void* workspace, size_t bytes, int* status, int& launches, cudaStream_t st) {
    launches = 0;
    if (g.n_seqs == 0 || g.n_rows == 0) return cudaSuccess;
    if (g.d != gdc::D || (reinterpret_cast<uintptr_t>(workspace) & 1023)) return cudaErrorInvalidValue;
    const int total = g.n_seqs == 1 ? (g.n_rows + gdc::C - 1) / gdc::C : g.n_rows / gdc::C + g.n_seqs;       // no fewer than the sequences' chunks
    const size_t most = bytes / gdn_chunk_bytes(1, g.n_k, g.n_v);
    if (most < 1) return cudaErrorInvalidValue;
    gdc::ChunkParams p = {};
    p.g = g; p.ws = static_cast<uint8_t*>(workspace); p.status = status;
    p.n_ks = g.n_k < g.n_v ? g.n_k : g.n_v;
    auto fits = [](const void* x, size_t row, int off) { return (reinterpret_cast<uintptr_t>(x) & 7) == 0 && row % 4 == 0 && off % 4 == 0; };
    p.in_aligned = fits(g.in, g.in_row, g.z_off);
    p.out_aligned = fits(g.out, g.out_row, 0);
    const auto prep = g.K == 4 && p.in_aligned && (reinterpret_cast<uintptr_t>(g.conv_w) & 15) == 0 ? gdc::gdn_chunk_prep_kernel<true> : gdc::gdn_chunk_prep_kernel<false>;
    cudaError_t e = tc5::raise_smem(prep, gdc::PREP_SMEM);
    if (e == cudaSuccess) e = tc5::raise_smem(gdc::gdn_chunk_scan_kernel, gdc::SCAN_SMEM);
    if (e != cudaSuccess) return e;
    // One sequence's scan takes n_v SMs and leaves the others idle, so the next chunks are prepared beside it, in the other half of the workspace; the first
    // pass is what one wave of blocks prepares.  (8192 rows of 48 heads, when it was taken: 945 us one after the other, 719 so.)  The scans of several sequences run side by side instead, as long as the
    // workspace holds all chunks.
    const int wave = 2 * sm_count() / p.n_ks > 0 ? 2 * sm_count() / p.n_ks : 1;
    const bool beside = total > wave && most > 1 && (g.n_seqs == 1 || (size_t)total > most);
    size_t room = beside ? most / 2 : most;
    if (room > 65535) room = 65535;
    const int head = beside && (size_t)wave < room ? wave : (int)room;
    const int more = total > head ? (total - head + (int)room - 1) / (int)room : 0;          // passes behind the first
    const int each = more ? (total - head + more - 1) / more : 0;
    for (int u0 = 0, pass = 0; u0 < total; u0 += p.units, ++pass) {
        p.u0 = u0;
        p.ws = static_cast<uint8_t*>(workspace) + (beside && (pass & 1) ? room * gdn_chunk_bytes(1, g.n_k, g.n_v) : 0);
        p.units = pass ? each : head;
        if (p.units > total - u0) p.units = total - u0;
        const dim3 grid(p.n_ks, p.units);
        p.first = pass == 0;
        if (beside || pass == 0) e = launch_pdl(prep, grid, dim3(gdc::PREP_THREADS), gdc::PREP_SMEM, st, p);
        else { prep<<<grid, gdc::PREP_THREADS, gdc::PREP_SMEM, st>>>(p); e = cudaGetLastError(); }
        if (e != cudaSuccess) return e;
        // (blocks of a scan that come up early help a single pass, 37 rows: 34.8 -> 30.8 us, and are in the way of the passes beside each other, 8192 rows: 620 -> 668 us)
        const dim3 scans(g.n_v, g.n_seqs);
        if (beside) { gdc::gdn_chunk_scan_kernel<<<scans, gdc::THREADS, gdc::SCAN_SMEM, st>>>(p); e = cudaGetLastError(); }
        else e = launch_pdl(gdc::gdn_chunk_scan_kernel, scans, dim3(gdc::THREADS), gdc::SCAN_SMEM, st, p);
        if (e != cudaSuccess) return e;
        launches += 2;
    }
    return cudaSuccess;
}

LLM_DEFINE_BOUNDS_STATUS_READER(bounds_status_gdn_chunk)

}  // namespace llm
