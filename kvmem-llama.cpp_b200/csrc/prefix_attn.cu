// Attention of a batch over a shared prefix and each sequence's own tail.
//
// For query row t (head h, KV head g = h / (n_head / n_head_kv)) of sequence s:
//   out = sum_j p_j v_j / sum_j p_j,  p_j = exp(scale * q . k_j - max)
// over the prefix tokens and the tail tokens up to the row's own (the last
// new token of a sequence sees its whole tail, the one before it one token
// less). Rows that see nothing give zeros and an lse of -inf; rows of no
// sequence are left as they were.
//
// One CTA per (row, head): each warp takes 32 keys at a time (a lane a key
// for the scores, a lane D / 32 dimensions for the values) with a running
// maximum and sum, the warps are joined at the end.
#include "prefix_attn.cuh"

#include <cmath>

#include "kvmret.h"
#include "quant.cuh"

namespace kvmret {
namespace {

constexpr int kWarps = 4;

// element e of a row of the given format
__device__ __forceinline__ float element(const uint8_t *row, int32_t type, uint32_t e) {
    if (type == KVMRET_TYPE_F16) return h2f(reinterpret_cast<const uint16_t *>(row)[e]);
    if (type == KVMRET_TYPE_Q8_0) {
        const uint8_t *b = row + (e / 32) * 34;
        return static_cast<float>(static_cast<int8_t>(b[2 + e % 32])) *
               h2f(*reinterpret_cast<const uint16_t *>(b));
    }
    const uint8_t *b = row + (e / 32) * 18;
    const uint32_t i = e % 32, x = b[2 + (i & 15)];
    return static_cast<float>(static_cast<int>(i < 16 ? x & 15 : x >> 4) - 8) *
           h2f(*reinterpret_cast<const uint16_t *>(b));
}

// K or V row of token i of a list, null when the list has no such token.
__device__ __forceinline__ bool locate(const KeyList &l, uint32_t list, uint32_t i, uint32_t &page,
                                       uint32_t &off) {
    const uint32_t T = l.pages.page_tokens, at = i / T;
    off = i - at * T;
    if (at >= l.n_list) return false;
    const uint64_t slot = static_cast<uint64_t>(list) * l.n_list + at;
    const int32_t p = l.table ? l.table[slot] : static_cast<int32_t>(at);
    if (p < 0 || static_cast<uint32_t>(p) >= l.pages.n_pages) return false;
    page = static_cast<uint32_t>(p);
    return !l.ntok || off < l.ntok[slot];
}

template <int D>
__global__ void __launch_bounds__(32 * kWarps) attn_kernel(const __grid_constant__ PrefixAttn a) {
    constexpr int E = D / 32;
    __shared__ float q[D];
    __shared__ float pm[kWarps], pl[kWarps], po[kWarps][D];
    const uint32_t t = blockIdx.x, h = blockIdx.y, g = h / (a.n_head / a.n_head_kv);
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint32_t seq = 0, seen = 0;
    if (a.n_seq) {
        bool found = false;
        for (uint32_t s = 0; s < a.n_seq && !found; ++s)
            if (static_cast<int32_t>(t) >= a.q_start[s] && static_cast<int32_t>(t) < a.q_start[s + 1]) {
                seq = s;
                found = true;
            }
        if (!found) return;
        const int32_t len = min(a.tail.len[seq], static_cast<int32_t>(a.tail.max_len));
        seen = static_cast<uint32_t>(max(0, len - (a.q_start[seq + 1] - static_cast<int32_t>(t)) + 1));
    }
    uint32_t np = a.prefix.max_len;
    if (np && a.prefix.len) np = static_cast<uint32_t>(min(max(*a.prefix.len, 0), static_cast<int32_t>(np)));
    for (uint32_t e = threadIdx.x; e < D; e += blockDim.x)
        q[e] = h2f(a.q[t * a.q_stride + h * D + e]) * a.scale;
    __syncthreads();
    float m = -INFINITY, l = 0.0f, o[E] = {};
    for (uint32_t i0 = warp * 32; i0 < np + seen; i0 += 32 * kWarps) {
        const uint32_t i = i0 + lane;
        const bool pre = i < np;
        const KeyList &kl = pre ? a.prefix : a.tail;
        uint32_t page = 0, off = 0;
        const bool ok = i < np + seen && locate(kl, pre ? 0 : seq, pre ? i : i - np, page, off);
        float s = -INFINITY;
        if (ok) {
            const uint8_t *row = kl.pages.k + page * kl.pages.k_page + off * kl.pages.k_row;
            s = 0.0f;
            for (uint32_t e = 0; e < D; ++e) s += q[e] * element(row, kl.pages.k_type, g * D + e);
        }
        float top = s;
        for (int x = 16; x; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        if (top == -INFINITY) continue;
        const float mn = fmaxf(m, top), c = expf(m - mn), p = expf(s - mn);
        float sum = p;
        for (int x = 16; x; x >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
        l = l * c + sum;
        m = mn;
        for (int e = 0; e < E; ++e) o[e] *= c;
        for (int j = 0; j < 32; ++j) {
            if (!__shfl_sync(0xffffffffu, static_cast<int>(ok), j)) continue;
            const float pj = __shfl_sync(0xffffffffu, p, j);
            const uint32_t pg = __shfl_sync(0xffffffffu, page, j), of = __shfl_sync(0xffffffffu, off, j);
            const KeyList &vl = i0 + j < np ? a.prefix : a.tail;
            const uint8_t *row = vl.pages.v + pg * vl.pages.v_page + of * vl.pages.v_row;
            for (int e = 0; e < E; ++e)
                o[e] += pj * element(row, vl.pages.v_type, g * D + lane * E + e);
        }
    }
    if (lane == 0) {
        pm[warp] = m;
        pl[warp] = l;
    }
    for (int e = 0; e < E; ++e) po[warp][lane * E + e] = o[e];
    __syncthreads();
    float top = -INFINITY, sum = 0.0f;
    for (int w = 0; w < kWarps; ++w) top = fmaxf(top, pm[w]);
    float c[kWarps];
    for (int w = 0; w < kWarps; ++w) {
        c[w] = top == -INFINITY ? 0.0f : expf(pm[w] - top);
        sum += c[w] * pl[w];
    }
    const uint64_t r = static_cast<uint64_t>(t) * a.n_head + h;
    for (uint32_t e = threadIdx.x; e < D; e += blockDim.x) {
        float x = 0.0f;
        for (int w = 0; w < kWarps; ++w) x += c[w] * po[w][e];
        a.out[r * D + e] = f2h(sum > 0.0f ? x / sum : 0.0f);
    }
    if (a.lse && threadIdx.x == 0) a.lse[r] = sum > 0.0f ? top + logf(sum) : -INFINITY;
}

}  // namespace

cudaError_t launch_prefix_attn_rows(const PrefixAttn &a, cudaStream_t st) {
    const dim3 grid(a.n_q, a.n_head);
    if (a.d_head == 64)
        attn_kernel<64><<<grid, 32 * kWarps, 0, st>>>(a);
    else if (a.d_head == 128)
        attn_kernel<128><<<grid, 32 * kWarps, 0, st>>>(a);
    else
        attn_kernel<256><<<grid, 32 * kWarps, 0, st>>>(a);
    return cudaGetLastError();
}

}  // namespace kvmret
