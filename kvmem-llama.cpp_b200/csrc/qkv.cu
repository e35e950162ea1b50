// The two row-wise passes around the attention of a step: norms of the query
// and key heads with the position rotation (qk_kernel), and the append of new
// keys and values to a paged cache with the rotation on the way
// (append_kernel). Both read and write every value once; the bound is HBM
// for chunks of tokens and the launch for single ones.
//
// One row layout serves both. A head row of D elements is held by D / 16
// lanes; lane j has elements 8j .. 8j + 7 of each half, so that
//   - loads and stores are 16 bytes a lane and whole rows a warp,
//   - both elements of every rotation pair (i, i + D / 2) are in one lane,
//   - a block of 32 elements (the quantisers' unit) is four neighbouring
//     lanes' lower or upper octets: its maximum takes two shuffles,
//   - the Hadamard butterflies of strides 1, 2, 4 and D / 2 stay in the lane
//     and strides 8 .. D / 4 are one shuffle each.
// Compiled with -fmad=false: rotation, butterflies and quantisers round step
// by step like the library's other rotations, so a key appended here has the
// bits that the window assembly gives the same key at the same position.
#include "qkv.cuh"

#include <cuda_bf16.h>

#include <algorithm>
#include <cmath>

#include "kvmret.h"
#include "quant.cuh"

namespace kvmret {
namespace {

constexpr int kThreads = 256, kAppendThreads = 128;

template <int D>
struct Row {
    static constexpr int lanes = D / 16;  // lanes of a head row
};

__device__ __forceinline__ void unpack_f16(const uint4 &w, float (&x)[8]) {
    const __half2 *h = reinterpret_cast<const __half2 *>(&w);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float2 f = __half22float2(h[e]);
        x[2 * e] = f.x;
        x[2 * e + 1] = f.y;
    }
}
__device__ __forceinline__ uint4 pack_f16(const float (&x)[8]) {
    uint4 w;
    __half2 *h = reinterpret_cast<__half2 *>(&w);
#pragma unroll
    for (int e = 0; e < 4; ++e) h[e] = __floats2half2_rn(x[2 * e], x[2 * e + 1]);
    return w;
}

// Eight consecutive activations as they lie in memory, and their values.
template <typename T>
struct Octet;
template <>
struct Octet<uint16_t> {  // f16
    uint4 w;
    __device__ __forceinline__ void load(const uint16_t *p) {
        w = __ldg(reinterpret_cast<const uint4 *>(p));
    }
    __device__ __forceinline__ void get(float (&x)[8]) const { unpack_f16(w, x); }
};
template <>
struct Octet<__nv_bfloat16> {
    uint4 w;
    __device__ __forceinline__ void load(const __nv_bfloat16 *p) {
        w = __ldg(reinterpret_cast<const uint4 *>(p));
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        const uint32_t *u = reinterpret_cast<const uint32_t *>(&w);
#pragma unroll
        for (int e = 0; e < 4; ++e) {  // a bf16 is the upper half of a float
            x[2 * e] = __uint_as_float(u[e] << 16);
            x[2 * e + 1] = __uint_as_float(u[e] & 0xffff0000u);
        }
    }
};
template <>
struct Octet<float> {
    float4 a, b;
    __device__ __forceinline__ void load(const float *p) {
        a = __ldg(reinterpret_cast<const float4 *>(p));
        b = __ldg(reinterpret_cast<const float4 *>(p) + 1);
    }
    __device__ __forceinline__ void get(float (&x)[8]) const {
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
};

// RoPE of lane j's pairs 8j .. with the token's table (angles()).
template <int D>
__device__ __forceinline__ void rotate(float (&lo)[8], float (&hi)[8], const float2 *cs, uint32_t j) {
#pragma unroll
    for (int e = 0; e < 8; e += 2) {
        const float4 t = reinterpret_cast<const float4 *>(cs)[e / 2 * Row<D>::lanes + j];
        float a = lo[e], b = hi[e];
        lo[e] = __fsub_rn(__fmul_rn(a, t.x), __fmul_rn(b, t.y));
        hi[e] = __fadd_rn(__fmul_rn(a, t.y), __fmul_rn(b, t.x));
        a = lo[e + 1];
        b = hi[e + 1];
        lo[e + 1] = __fsub_rn(__fmul_rn(a, t.z), __fmul_rn(b, t.w));
        hi[e + 1] = __fadd_rn(__fmul_rn(a, t.w), __fmul_rn(b, t.z));
    }
}

// Orthonormal Hadamard transform of a head row: scale, then butterflies of
// strides 1, 2, 4, ... D / 2. Every lane of the warp takes part.
template <int D>
__device__ __forceinline__ void hadamard(float (&lo)[8], float (&hi)[8], float scale) {
    const uint32_t lane = threadIdx.x & 31;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        lo[e] = __fmul_rn(lo[e], scale);
        hi[e] = __fmul_rn(hi[e], scale);
    }
#pragma unroll
    for (int h = 1; h < 8; h *= 2)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            if (e & h) continue;
            float a = lo[e], b = lo[e + h];
            lo[e] = __fadd_rn(a, b);
            lo[e + h] = __fsub_rn(a, b);
            a = hi[e];
            b = hi[e + h];
            hi[e] = __fadd_rn(a, b);
            hi[e + h] = __fsub_rn(a, b);
        }
#pragma unroll
    for (int h = 1; h < Row<D>::lanes; h *= 2) {  // stride 8h: the other lane's octets
        const bool upper = lane & h;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float a = __shfl_xor_sync(0xffffffffu, lo[e], h);
            const float b = __shfl_xor_sync(0xffffffffu, hi[e], h);
            lo[e] = upper ? __fsub_rn(a, lo[e]) : __fadd_rn(lo[e], a);
            hi[e] = upper ? __fsub_rn(b, hi[e]) : __fadd_rn(hi[e], b);
        }
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float a = lo[e], b = hi[e];
        lo[e] = __fadd_rn(a, b);
        hi[e] = __fsub_rn(a, b);
    }
}

// The {cos, sin} table of a CTA's tokens in shared memory: of each token first
// pairs 8j, 8j + 1 of every lane j, then 8j + 2, 8j + 3 and so on, so that the
// lanes of a row read 16 neighbouring bytes each. (In pair order four lanes
// met in a bank, and the L1 bound a chunk of 2048 tokens at 27 us, now 22.)
template <int D>
__device__ __forceinline__ void angles(float2 *cs, const int32_t *pos, uint32_t n,
                                       const Theta &th) {
    for (uint32_t i = threadIdx.x; i < n * (D / 2); i += blockDim.x) {
        const uint32_t t = i / (D / 2), p = i % (D / 2);
        const uint32_t at = (p % 8 / 2 * Row<D>::lanes + p / 8) * 2 + p % 2;
        cs[t * (D / 2) + at] = rope_cs(pos[t], th.v[p]);
    }
}

// y = x / sqrt(mean(x^2) + eps) * w per head row, f32 throughout (the sum of
// squares per lane, then over the row's lanes by shuffles), rounded once into
// each wanted output. CTA = tokens x a range of heads; a thread has the octets
// of kFly rows on their way at a time, the first ones while the CTA's cosines
// and sines are computed (double precision, about 1 us).
constexpr int kFly = 2;
template <int D, typename T, bool FWHT>
__global__ void __launch_bounds__(kThreads)
    qk_kernel(const __grid_constant__ QkNormRope a, uint32_t tokens, uint32_t heads,
              float fwht_scale) {
    constexpr uint32_t L = Row<D>::lanes, G = kThreads / L;
    __shared__ __align__(16) float2 cs[256];  // tokens * D / 2 <= 256
    __shared__ __align__(16) float ws[2][D];  // weights of q, k: lane by lane like cs
    const uint32_t t0 = blockIdx.x * tokens, nt = min(tokens, a.n_tok - t0);
    const uint32_t h0 = blockIdx.y * heads, nh = min(heads, a.n_head + a.n_head_kv - h0);
    const uint32_t j = threadIdx.x % L, rows = nt * nh;
    struct Place {
        uint32_t dt, hh;
        bool is_q;
    };
    auto place = [&](uint32_t r) {
        const uint32_t dt = nt == 1 ? 0 : r / nh, h = h0 + r - dt * nh;
        return Place{dt, h < a.n_head ? h : h - a.n_head, h < a.n_head};
    };
    Octet<T> u[kFly], v[kFly];
    auto load = [&](uint32_t r0) {
#pragma unroll
        for (int f = 0; f < kFly; ++f) {
            const uint32_t r = r0 + f * G;
            if (r >= rows) break;
            const Place p = place(r);
            const uint64_t t = t0 + p.dt;
            const T *src = (p.is_q ? static_cast<const T *>(a.q) + t * a.q_stride
                                   : static_cast<const T *>(a.k) + t * a.k_stride) +
                           static_cast<uint64_t>(p.hh) * D + 8 * j;
            u[f].load(src);
            v[f].load(src + D / 2);
        }
    };
    const uint32_t first = threadIdx.x / L;
    load(first);
    for (uint32_t i = threadIdx.x; i < 2 * D; i += kThreads) {
        const uint32_t c = i % D, o = c % (D / 2);  // octet o / 8 of its half
        const float *w = i < D ? a.q_weight : a.k_weight;
        ws[i / D][((c / (D / 2) * 2 + o % 8 / 4) * L + o / 8) * 4 + o % 4] = w ? __ldg(w + c) : 1.0f;
    }
    angles<D>(cs, a.pos + t0, nt, a.theta);
    __syncthreads();
    // (whole warps take part in the shuffles: the bound is the CTA's)
    for (uint32_t rb = 0; rb < rows; rb += kFly * G) {
        if (rb) load(rb + first);
#pragma unroll
        for (int f = 0; f < kFly; ++f) {
            if (rb + f * G >= rows) break;
            const uint32_t r = rb + f * G + first;
            const bool act = r < rows;
            const Place p = place(act ? r : 0);
            float lo[8] = {}, hi[8] = {};
            if (act) {
                u[f].get(lo);
                v[f].get(hi);
            }
            float ss = 0.0f;
#pragma unroll
            for (int e = 0; e < 8; ++e) ss += lo[e] * lo[e] + hi[e] * hi[e];
#pragma unroll
            for (uint32_t o = L / 2; o >= 1; o /= 2) ss += __shfl_xor_sync(0xffffffffu, ss, o);
            const float inv = __frsqrt_rn(ss * (1.0f / D) + a.eps);
            const float4 *w = reinterpret_cast<const float4 *>(ws[p.is_q ? 0 : 1]) + j;
#pragma unroll
            for (int e = 0; e < 8; e += 4) {
                const float4 wl = w[e / 4 * L], wh = w[(2 + e / 4) * L];
                lo[e] *= inv * wl.x;
                lo[e + 1] *= inv * wl.y;
                lo[e + 2] *= inv * wl.z;
                lo[e + 3] *= inv * wl.w;
                hi[e] *= inv * wh.x;
                hi[e + 1] *= inv * wh.y;
                hi[e + 2] *= inv * wh.z;
                hi[e + 3] *= inv * wh.w;
            }
            const uint64_t o =
                ((t0 + p.dt) * static_cast<uint64_t>(p.is_q ? a.n_head : a.n_head_kv) + p.hh) * D + 8 * j;
            uint16_t *raw = p.is_q ? a.q_raw : a.k_raw, *rot = p.is_q ? a.q_rot : a.k_rot;
            if (act && raw) {
                *reinterpret_cast<uint4 *>(raw + o) = pack_f16(lo);
                *reinterpret_cast<uint4 *>(raw + o + D / 2) = pack_f16(hi);
            }
            rotate<D>(lo, hi, cs + p.dt * (D / 2), j);
            if constexpr (FWHT) hadamard<D>(lo, hi, fwht_scale);
            if (act && rot) {
                *reinterpret_cast<uint4 *>(rot + o) = pack_f16(lo);
                *reinterpret_cast<uint4 *>(rot + o + D / 2) = pack_f16(hi);
            }
        }
    }
}

// A lane's octet of a 32-element block (quarter `q` of it) as q8_0 bytes into
// the block at `b` of a shared-memory staging row: d = amax / 127, round
// half away, as the library's other q8_0 writers.
__device__ __forceinline__ void put_q8_0(uint8_t *b, uint32_t q, const float (&x)[8]) {
    float amax = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; ++e) amax = fmaxf(amax, fabsf(x[e]));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 1));
    amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, 2));
    const float d = div127_rn(amax);
    const float id = d != 0.0f ? __frcp_rn(d) : 0.0f;
    uint16_t *p = reinterpret_cast<uint16_t *>(b + 2 + 8 * q);
#pragma unroll
    for (int e = 0; e < 8; e += 2)
        p[e / 2] = static_cast<uint16_t>(
            (round_away_int(__fmul_rn(x[e], id)) & 0xff) |
            ((round_away_int(__fmul_rn(x[e + 1], id)) & 0xff) << 8));
    if (q == 0) *reinterpret_cast<uint16_t *>(b) = f2h(d);
}

// The same as q4_0: d = v / -8 with v the first element of largest magnitude;
// byte i of the block holds element i and, in its upper half, element i + 16,
// so the lanes of quarters 0 and 1 collect those of quarters 2 and 3.
__device__ __forceinline__ void put_q4_0(uint8_t *b, uint32_t q, const float (&x)[8]) {
    float v = x[0];
#pragma unroll
    for (int e = 1; e < 8; ++e)
        if (fabsf(v) < fabsf(x[e])) v = x[e];
#pragma unroll
    for (uint32_t o = 1; o <= 2; o *= 2) {
        const float u = __shfl_xor_sync(0xffffffffu, v, o);
        const bool mine_first = !(q & o);
        if (mine_first ? fabsf(v) < fabsf(u) : !(fabsf(u) < fabsf(v))) v = u;
    }
    if (v == 0.0f) v = 0.0f;  // a block of zeros of either sign has d = -0
    const float d = __fmul_rn(v, -0.125f);  // = v / -8, the same rounding
    const float id = d != 0.0f ? __frcp_rn(d) : 0.0f;
    uint32_t n = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const int i = min(__float2int_rz(__fadd_rn(__fmul_rn(x[e], id), 8.5f)), 15);
        n |= static_cast<uint32_t>(i & 15) << (4 * e);
    }
    const uint32_t up = __shfl_xor_sync(0xffffffffu, n, 2);
    if (q < 2) {
        uint16_t *p = reinterpret_cast<uint16_t *>(b + 2 + 8 * q);
#pragma unroll
        for (int e = 0; e < 8; e += 2)
            p[e / 2] = static_cast<uint16_t>(
                ((n >> (4 * e)) & 15) | (((up >> (4 * e)) & 15) << 4) |
                (((n >> (4 * e + 4)) & 15) << 8) | (((up >> (4 * e + 4)) & 15) << 12));
        if (q == 0) *reinterpret_cast<uint16_t *>(b) = f2h(d);
    }
}

template <int TYPE>
struct Fmt {
    static constexpr uint32_t block = TYPE == KVMRET_TYPE_F16 ? 64
                                      : TYPE == KVMRET_TYPE_Q8_0 ? 34 : 18;  // bytes of 32
};

// A warp's span of up to 512 elements of one token row (whole heads), each
// lane's octets lo / hi, into `dst` (16-byte aligned; span_bytes of it).
template <int D, int TYPE>
__device__ __forceinline__ void store_span(uint8_t *dst, uint8_t *stage, uint32_t span_elems,
                                           bool act, const float (&lo)[8], const float (&hi)[8]) {
    const uint32_t lane = threadIdx.x & 31, j = lane % Row<D>::lanes, g = lane / Row<D>::lanes;
    if constexpr (TYPE == KVMRET_TYPE_F16) {
        if (act) {
            uint4 *p = reinterpret_cast<uint4 *>(dst + 2 * (g * D + 8 * j));
            p[0] = pack_f16(lo);
            p[D / 16] = pack_f16(hi);
        }
    } else {
        constexpr uint32_t B = Fmt<TYPE>::block;
        uint8_t *b = stage + (g * (D / 32) + j / 4) * B;
        if constexpr (TYPE == KVMRET_TYPE_Q8_0) {
            put_q8_0(b, j % 4, lo);
            put_q8_0(b + D / 64 * B, j % 4, hi);
        } else {
            put_q4_0(b, j % 4, lo);
            put_q4_0(b + D / 64 * B, j % 4, hi);
        }
        __syncwarp();
        const uint32_t n16 = span_elems / 32 * B / 16;  // whole: E is a multiple of 256
        for (uint32_t c = lane; c < n16; c += 32)
            reinterpret_cast<uint4 *>(dst)[c] = reinterpret_cast<const uint4 *>(stage)[c];
        __syncwarp();
    }
}

// CTA = `tokens` tokens; each warp takes spans of 512 elements of their K and
// V rows. K: rotate, transform, format; V: format.
template <int D, int KT, int VT>
__global__ void __launch_bounds__(kAppendThreads)
    append_kernel(const __grid_constant__ PagedAppend a, uint32_t tokens, float fwht_scale) {
    constexpr uint32_t L = Row<D>::lanes, SPAN = 512;
    __shared__ __align__(16) float2 cs[256];  // tokens * D / 2 <= 256
    __shared__ __align__(16) uint8_t stage[kAppendThreads / 32][SPAN / 32 * 34];
    const uint32_t t0 = blockIdx.x * tokens, nt = min(tokens, a.n_tok - t0);
    const uint32_t lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const uint32_t E = a.pages.n_head_kv * D, spans = (E + SPAN - 1) / SPAN, n_items = 2 * nt * spans;
    const uint32_t g = lane / L, j = lane % L;
    uint4 u = make_uint4(0, 0, 0, 0), v = u;
    int32_t cell = -1;
    auto load = [&](uint32_t i) {
        const uint32_t s = i >> 1, dt = spans == 1 ? s : s / spans, e0 = (s - dt * spans) * SPAN;
        const uint64_t t = t0 + dt;
        cell = __ldg(a.cells + t);
        if (e0 + (g + 1) * D <= E) {
            const uint16_t *p = (i & 1 ? a.v + t * a.v_stride : a.k + t * a.k_stride) + e0 + g * D + 8 * j;
            u = __ldg(reinterpret_cast<const uint4 *>(p));
            v = __ldg(reinterpret_cast<const uint4 *>(p + D / 2));
        }
    };
    if (warp < n_items) load(warp);  // on its way while the angles are computed
    if (a.pos) {
        angles<D>(cs, a.pos + t0, nt, a.theta);
        __syncthreads();
    }
    for (uint32_t i = warp; i < n_items; i += kAppendThreads / 32) {
        if (i != warp) load(i);
        const bool is_v = i & 1;
        const uint32_t s = i >> 1, dt = spans == 1 ? s : s / spans, e0 = (s - dt * spans) * SPAN;
        if (cell < 0 || static_cast<uint32_t>(cell) >= a.pages.n_pages * a.pages.page_tokens)
            continue;  // no such cell: nothing is written
        const uint32_t page = static_cast<uint32_t>(cell) / a.pages.page_tokens;
        const uint32_t off = static_cast<uint32_t>(cell) - page * a.pages.page_tokens;
        const bool act = e0 + (g + 1) * D <= E;
        const uint32_t n = min(SPAN, E - e0);
        float lo[8] = {}, hi[8] = {};
        if (act) {
            unpack_f16(u, lo);
            unpack_f16(v, hi);
        }
        if (is_v) {
            uint8_t *dst = a.pages.v + page * a.pages.v_page + off * a.pages.v_row +
                           e0 / 32 * Fmt<VT>::block;
            store_span<D, VT>(dst, stage[warp], n, act, lo, hi);
        } else {
            if (a.pos) rotate<D>(lo, hi, cs + dt * (D / 2), j);
            if (a.fwht_n) hadamard<D>(lo, hi, fwht_scale);
            uint8_t *dst = a.pages.k + page * a.pages.k_page + off * a.pages.k_row +
                           e0 / 32 * Fmt<KT>::block;
            store_span<D, KT>(dst, stage[warp], n, act, lo, hi);
        }
    }
}

float fwht_scale(uint32_t n) {
    return n ? 1.0f / std::sqrt(static_cast<float>(n)) : 0.0f;
}

// Many tokens: a CTA takes all heads of a few (enough rows to fill its threads
// kFly times), so that a token's angles are computed once. Few: a CTA takes one
// pass of rows of one token, so that there are CTAs for the SMs. (64 + 8 heads
// of 128, bf16 in, four outputs: 256 tokens 5.1 us split, 7.2 us not; 512 tokens
// 10.0 and 7.3 us; 2048 tokens 31 and 22 us = 5.1 TB/s.)
template <int D, typename T>
cudaError_t launch_qk_t(const QkNormRope &a, cudaStream_t st) {
    constexpr uint32_t G = kThreads / Row<D>::lanes;
    const uint32_t heads_all = a.n_head + a.n_head_kv;
    const bool many = a.n_tok >= 512;
    const uint32_t fill = std::max<uint32_t>(256 / D, (kFly * G + heads_all - 1) / heads_all);
    const uint32_t tokens = many ? std::min<uint32_t>(kThreads / (D / 2), fill) : 1;
    const uint32_t heads = many ? heads_all : G;
    const dim3 grid((a.n_tok + tokens - 1) / tokens, (heads_all + heads - 1) / heads);
    const float s = fwht_scale(a.fwht_n);
    if (a.fwht_n)
        qk_kernel<D, T, true><<<grid, kThreads, 0, st>>>(a, tokens, heads, s);
    else
        qk_kernel<D, T, false><<<grid, kThreads, 0, st>>>(a, tokens, heads, s);
    return cudaGetLastError();
}

template <int D>
cudaError_t launch_qk_d(const QkNormRope &a, cudaStream_t st) {
    if (a.type == kTypeF32) return launch_qk_t<D, float>(a, st);
    if (a.type == kTypeBF16) return launch_qk_t<D, __nv_bfloat16>(a, st);
    return launch_qk_t<D, uint16_t>(a, st);
}

// Four warps with a token's spans: 8 tokens of 1024 + 1024 elements take 2.0 us
// (q8_0 + q4_0: 2.9), 2048 tokens 4.9 us (8.0); with four tokens to eight warps
// 3.2 (4.9) and 5.2 us (8.6).
template <int D, int KT, int VT>
cudaError_t launch_append_t(const PagedAppend &a, cudaStream_t st) {
    const uint32_t spans = (a.pages.n_head_kv * D + 511) / 512;
    const uint32_t tokens = std::min<uint32_t>(256 / (D / 2), std::max<uint32_t>(1, kAppendThreads / 64 / spans));
    append_kernel<D, KT, VT><<<(a.n_tok + tokens - 1) / tokens, kAppendThreads, 0, st>>>(
        a, tokens, fwht_scale(a.fwht_n));
    return cudaGetLastError();
}

template <int D, int KT>
cudaError_t launch_append_k(const PagedAppend &a, cudaStream_t st) {
    if (a.pages.v_type == KVMRET_TYPE_F16) return launch_append_t<D, KT, KVMRET_TYPE_F16>(a, st);
    if (a.pages.v_type == KVMRET_TYPE_Q8_0) return launch_append_t<D, KT, KVMRET_TYPE_Q8_0>(a, st);
    return launch_append_t<D, KT, KVMRET_TYPE_Q4_0>(a, st);
}

template <int D>
cudaError_t launch_append_d(const PagedAppend &a, cudaStream_t st) {
    if (a.pages.k_type == KVMRET_TYPE_F16) return launch_append_k<D, KVMRET_TYPE_F16>(a, st);
    if (a.pages.k_type == KVMRET_TYPE_Q8_0) return launch_append_k<D, KVMRET_TYPE_Q8_0>(a, st);
    return launch_append_k<D, KVMRET_TYPE_Q4_0>(a, st);
}

}  // namespace

cudaError_t launch_qk_norm_rope(const QkNormRope &a, cudaStream_t st) {
    if (a.d_head == 64) return launch_qk_d<64>(a, st);
    if (a.d_head == 128) return launch_qk_d<128>(a, st);
    return launch_qk_d<256>(a, st);
}

cudaError_t launch_paged_append(const PagedAppend &a, cudaStream_t st) {
    if (a.pages.d_head == 64) return launch_append_d<64>(a, st);
    if (a.pages.d_head == 128) return launch_append_d<128>(a, st);
    return launch_append_d<256>(a, st);
}

}  // namespace kvmret
