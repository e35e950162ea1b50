// Attention of a batch over a shared prefix and each sequence's own tail, on
// the tcgen05 tensor cores.
//
// For query row t (head h, KV head g = h / (n_head / n_head_kv)) of sequence s:
//   out = sum_j p_j v_j / sum_j p_j,  p_j = 2^(c q . k_j - m),  c = scale log2 e
// over the prefix tokens and the tail tokens up to the row's own. One pass
// over the keys with a running maximum m and sum (f32); the output is kept
// unnormalised in tensor memory and rescaled only when the maximum has grown
// by more than 8 (a factor of 2^8), so p stays below 2^8 and exact in its
// ratio; p is rounded to f16 for the second product, the sum is not.
//
// A CTA (one per SM) walks its pieces (prefix_attn_plan.cuh). Warps:
//   0      producer: page list, the tile's mask of valid keys, TMA loads of K
//          and V tiles into a ring of shared-memory stages (128-byte swizzle,
//          no multicast);
//   1      one lane issues the products: S = Q K^T (both in shared memory)
//          and O += P V (P in tensor memory over its S, V as it lies: keys
//          along K, MN-major);
//   4-7    softmax of stream 0, a thread a row; also loads Q, rescales and
//          hands on O;
//   8-11   the same for stream 1 (head size 256 has one stream: its output
//          takes half of the tensor memory).
// With more than 128 rows the two streams are two tiles of rows over the same
// key tiles; otherwise they are the same rows over every other key tile, each
// with its own output. While one stream is in its softmax the other one's
// products run. P and S of a stream share columns, so its next S waits until
// the product that reads P has completed.
// Cells without a token may hold anything, NaN too: their scores are replaced
// after the product, their V rows zeroed in shared memory before it.
// Every wait is bounded; on a timeout the outputs become NaN (the join).
#include "prefix_attn.cuh"

#include <cuda_fp16.h>

#include <algorithm>
#include <cmath>

#include "kvmret.h"
#include "prefix_attn_plan.cuh"
#include "quant.cuh"
#include "tc.cuh"

namespace kvmret {
namespace {

template <int D>
struct Cfg {
    static constexpr int NS = D == 256 ? 1 : 2;     // streams
    static constexpr int BN = D == 256 ? 64 : 128;  // keys of a tile
    static constexpr int PR = 128 * NS;             // rows of a unit
    static constexpr int threads = 128 + 128 * NS;
    static constexpr uint32_t stage = BN * D * 2;   // one K or V tile
    static constexpr int stages = D == 64 ? 8 : 5;
    static constexpr uint32_t q_bytes = 128 * D * 2;
    static constexpr uint32_t smem = NS * q_bytes + stages * stage + 1024;
    static __host__ __device__ constexpr uint32_t s_col(int s) { return s * 128; }
    static __host__ __device__ constexpr uint32_t o_col(int s) { return 256 + s * (D == 64 ? 64 : 128); }
};
constexpr uint32_t kAttnTmem = 512;
constexpr int kMeta = 8;  // tiles whose masks are held (more than the ring reaches back)

struct AttnLaunch {
    PrefixAttn a;
    CUtensorMap map[4];  // prefix K, V, tail K, V
    Plan *plan;
    uint32_t *fail;      // [CTA] 1: a wait gave up, or more pieces than slots
    uint64_t *seq_tile;  // [n_seq] first tile of each sequence on the tails' line
    uint32_t *seq_pair;  // [n_seq] its first row pair
    float2 *ml;          // [slot][stream][128]
    float4 *o;           // [slot][stream][D / 4][128]
    uint32_t max_slots;
};

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_h2(float a, float b) {
    const __half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void tmem_ld32_nowait(uint32_t taddr, uint32_t *r) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32"
        " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15,"
        " %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31},"
        " [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
          "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]),
          "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}

// Instruction descriptor: D f32, A and B f16, M = 128, N; B K-major or MN-major.
__host__ __device__ constexpr uint32_t idesc(uint32_t n, bool b_mn) {
    return (1u << 4) | (b_mn ? 1u << 16 : 0u) | ((n >> 3) << 17) | ((128u >> 4) << 24);
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t id,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(id), "r"(accumulate), "r"(0u)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, {%5, %5, %5, %5}, p;\n\t}" ::"r"(d),
        "r"(a), "l"(b), "r"(id), "r"(accumulate), "r"(0u)
        : "memory");
}

// Block-wide plan of the split, in every CTA alike; CTA 0 also leaves it and
// the sequences' offsets in the workspace for the join. `start` receives the
// sequence that holds the CTA's first tail tile.
struct Start {
    uint32_t seq, pair;
    uint64_t tile;
};
template <int D>
__device__ void make_plan(const AttnLaunch &l, Plan &p, Start &start, uint32_t &fail,
                          uint64_t (&red)[2][16]) {
    constexpr int BN = Cfg<D>::BN, PR = Cfg<D>::PR;
    const PrefixAttn &a = l.a;
    const uint32_t tid = threadIdx.x, nthr = blockDim.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t G = a.n_head / a.n_head_kv, H = a.n_head_kv;
    const TileGeom<BN> tg(a.n_seq ? a.tail.pages.page_tokens : BN);
    auto shape = [&](uint32_t s, uint64_t &tiles, uint32_t &pairs) {
        const SeqShape sh = seq_shape(a, s);
        pairs = (sh.q_len * G + PR - 1) / PR;
        tiles = static_cast<uint64_t>(sh.q_len ? tg.tiles(sh.len) : 0) * pairs * H;
    };
    // totals of the tails; the last listed page that holds tokens
    uint64_t tiles = 0, pairs = 0;
    for (uint32_t s = tid; s < a.n_seq; s += nthr) {
        uint64_t t;
        uint32_t n;
        shape(s, t, n);
        tiles += t;
        pairs += n;
    }
    uint32_t held = a.prefix.max_len ? a.prefix.n_list : 0;
    if (held && a.prefix.ntok) {
        held = 0;
        for (uint32_t i = tid; i < a.prefix.n_list; i += nthr)
            if (__ldg(a.prefix.ntok + i)) held = i + 1;
    }
    for (int o = 16; o; o >>= 1) {
        tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
        pairs += __shfl_xor_sync(0xffffffffu, pairs, o);
        held = max(held, __shfl_xor_sync(0xffffffffu, held, o));
    }
    if (lane == 0) {
        red[0][warp] = tiles;
        red[1][warp] = pairs << 32 | held;
    }
    __syncthreads();
    if (tid == 0) {
        tiles = pairs = 0;
        held = 0;
        for (uint32_t w = 0; w < nthr / 32; ++w) {
            tiles += red[0][w];
            pairs += red[1][w] >> 32;
            held = max(held, static_cast<uint32_t>(red[1][w]));
        }
        p.p_len = 0;
        p.np = 0;
        if (a.prefix.max_len) {
            const uint64_t most = static_cast<uint64_t>(held) * a.prefix.pages.page_tokens;
            uint32_t len = a.prefix.max_len;
            if (a.prefix.len)
                len = min(len, static_cast<uint32_t>(max(__ldg(a.prefix.len), 0)));
            p.p_len = most < len ? static_cast<uint32_t>(most) : len;
            p.np = TileGeom<BN>(a.prefix.pages.page_tokens).tiles(p.p_len);
        }
        p.q0 = 0;
        uint32_t q1 = a.n_q;
        if (a.n_seq) {
            const int32_t n = static_cast<int32_t>(a.n_q);
            p.q0 = static_cast<uint32_t>(min(max(__ldg(a.q_start), 0), n));
            q1 = static_cast<uint32_t>(min(max(__ldg(a.q_start + a.n_seq), static_cast<int32_t>(p.q0)), n));
        }
        p.rows = (q1 - p.q0) * G;
        p.n_pair = (p.rows + PR - 1) / PR;
        // 8 CTAs side by side leave at most 4 % of the 148 SMs without a group
        p.n_pg = (p.n_pair + 7) / 8;
        p.gs = p.n_pg ? (p.n_pair + p.n_pg - 1) / p.n_pg : 1;
        if (p.gs > gridDim.x) {
            p.gs = gridDim.x;
            p.n_pg = (p.n_pair + p.gs - 1) / p.gs;
        }
        p.groups = gridDim.x / p.gs;
        p.p_total = static_cast<uint64_t>(p.np) * p.n_pg * H;
        p.t_total = tiles;
        p.t_slot0 = (p.n_pg * H + p.groups) * p.gs;
        const uint64_t slots = p.t_slot0 + pairs * H + gridDim.x;
        if (slots > l.max_slots) {  // q_start was not ascending
            fail = 1;
            p.p_total = p.t_total = 0;
        }
    }
    __syncthreads();
    uint64_t x, x1, y, y1;
    Walk<BN, PR>::ranges(p, blockIdx.x, gridDim.x, x, x1, y, y1);
    if (y >= y1 && blockIdx.x != 0) return;  // no tails here
    uint64_t base_t = 0;
    uint32_t base_p = 0;
    for (uint32_t s0 = 0; s0 < a.n_seq; s0 += nthr) {
        const uint32_t s = s0 + tid;
        uint64_t t = 0;
        uint32_t n = 0;
        if (s < a.n_seq) shape(s, t, n);
        uint64_t ti = t, pi = n;
        for (int o = 1; o < 32; o <<= 1) {
            const uint64_t u = __shfl_up_sync(0xffffffffu, ti, o), v = __shfl_up_sync(0xffffffffu, pi, o);
            if (lane >= o) {
                ti += u;
                pi += v;
            }
        }
        if (lane == 31) {
            red[0][warp] = ti;
            red[1][warp] = pi;
        }
        __syncthreads();
        uint64_t before_t = base_t, before_p = base_p, all_t = 0, all_p = 0;
        for (uint32_t w = 0; w < nthr / 32; ++w) {
            if (w < warp) {
                before_t += red[0][w];
                before_p += red[1][w];
            }
            all_t += red[0][w];
            all_p += red[1][w];
        }
        ti += before_t - t;
        pi += before_p - n;
        if (s < a.n_seq) {
            if (y >= ti && y < ti + t) start = {s, static_cast<uint32_t>(pi), ti};
            if (blockIdx.x == 0) {
                l.seq_tile[s] = ti;
                l.seq_pair[s] = static_cast<uint32_t>(pi);
            }
        }
        base_t += all_t;
        base_p += static_cast<uint32_t>(all_p);
        __syncthreads();
    }
}

template <int D>
__global__ void __launch_bounds__(Cfg<D>::threads, 1)
    attn_tc_kernel(const __grid_constant__ AttnLaunch l) {
    using C = Cfg<D>;
    constexpr int BN = C::BN, PR = C::PR, NS = C::NS, ST = C::stages;
    constexpr uint32_t KB = BN * 128, QB = 128 * 128;  // bytes of a 64-column block of K / V, of Q
    extern __shared__ uint8_t smem_raw[];
    __shared__ Plan plan;
    __shared__ Start start;
    __shared__ uint64_t red[2][16];
    __shared__ uint64_t bars[2 * ST + kMeta + 4 * NS + 1];
    __shared__ uint32_t s_mask[kMeta][4];
    __shared__ uint32_t s_tmem, s_fail;

    const PrefixAttn &a = l.a;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(smem_raw) + 1023u) & ~1023u;  // the swizzle atom
    const uint32_t ring = base + NS * C::q_bytes;
    const uint32_t bar0 = smem_u32(bars);
    auto full = [&](uint32_t i) { return bar0 + 8u * i; };
    auto empty = [&](uint32_t i) { return bar0 + 8u * (ST + i); };
    auto meta = [&](uint32_t i) { return bar0 + 8u * (2 * ST + i); };
    auto q_ready = [&](uint32_t s) { return bar0 + 8u * (2 * ST + kMeta + s); };
    auto s_full = [&](uint32_t s) { return bar0 + 8u * (2 * ST + kMeta + NS + s); };
    auto p_ready = [&](uint32_t s) { return bar0 + 8u * (2 * ST + kMeta + 2 * NS + s); };
    auto pv_done = [&](uint32_t s) { return bar0 + 8u * (2 * ST + kMeta + 3 * NS + s); };
    const uint32_t drain = bar0 + 8u * (2 * ST + kMeta + 4 * NS);
    auto failed = [&] { return *static_cast<volatile uint32_t *>(&s_fail) != 0; };

    if (threadIdx.x == 0) {
        s_fail = 0;
        start = {0, 0, 0};
        for (int i = 0; i < 2 * ST + kMeta; ++i) mbar_init(bar0 + 8u * i, 1);
        mbar_init(drain, 1);
        for (int s = 0; s < NS; ++s) {
            mbar_init(q_ready(s), 4);
            mbar_init(s_full(s), 1);
            mbar_init(p_ready(s), 4);
            mbar_init(pv_done(s), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (int i = a.prefix.max_len ? 0 : 2; i < (a.n_seq ? 4 : 2); ++i)
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&l.map[i]))
                         : "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&s_tmem)),
                     "r"(kAttnTmem)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    make_plan<D>(l, plan, start, s_fail, red);
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = s_tmem;
    Walk<BN, PR> walk(a, plan, start.seq, start.tile, start.pair);
    Seg g;

    if (warp == 0) {  // ---- producer ----
        uint32_t q = 0, j = 0;  // stages and tiles so far
        bool stop = false;
        while (!stop && walk.next(g)) {
            const KeyList &kl = g.tail ? a.tail : a.prefix;
            const CUtensorMap *mk = &l.map[g.tail ? 2 : 0], *mv = mk + 1;
            const TileGeom<BN> geom(kl.pages.page_tokens);
            const uint32_t T = geom.T, box = min(T, static_cast<uint32_t>(BN));
            const uint64_t list = g.tail ? static_cast<uint64_t>(g.seq) * kl.n_list : 0;
            const uint32_t len = g.tail ? min(static_cast<uint32_t>(max(__ldg(a.tail.len + g.seq), 0)),
                                              a.tail.max_len)
                                        : plan.p_len;
            for (uint32_t i = 0; i < g.n; ++i, ++j) {
                // lane p < ppt: page p of the tile, and how many of its tokens count
                uint32_t page, off;
                geom.locate(g.tile0 + i, page, off);
                int32_t id = -1;
                uint32_t held = 0;
                if (lane < geom.ppt && page + lane < kl.n_list) {
                    const uint32_t at = page + lane;
                    id = kl.table ? __ldg(kl.table + list + at) : static_cast<int32_t>(at);
                    if (id >= 0 && static_cast<uint32_t>(id) < kl.pages.n_pages) {
                        held = kl.ntok ? min(__ldg(kl.ntok + at), T) : T;
                        held = min(held, at * T < len ? len - at * T : 0);
                    }
                }
                const bool use = held > off;
                uint32_t mask = 0;  // lane w keeps word w
#pragma unroll
                for (uint32_t w = 0; w < BN / 32; ++w) {
                    const uint32_t key = 32 * w + lane, pk = T < BN ? key / T : 0;
                    const uint32_t h = __shfl_sync(0xffffffffu, held, pk);
                    const uint32_t o = T < BN ? key - pk * T : off + key;
                    const uint32_t b = __ballot_sync(0xffffffffu, pk < geom.ppt && o < h);
                    if (lane == w) mask = b;
                }
                const uint32_t n_use = __popc(__ballot_sync(0xffffffffu, use));
                const uint32_t bytes = n_use * box * D * 2;
#pragma unroll
                for (uint32_t v = 0; v < 2; ++v, ++q) {  // K, then V
                    const uint32_t st = q % ST, round = q / ST;
                    const bool ok = round == 0 || mbar_wait(empty(st), (round - 1) & 1u);
                    if (!__all_sync(0xffffffffu, ok) || failed()) {
                        stop = true;
                        break;
                    }
                    if (v == 0) {
                        if (lane < BN / 32) s_mask[j % kMeta][lane] = mask;
                        __syncwarp();
                        if (lane == 0) mbar_arrive(meta(j % kMeta));
                    }
                    if (lane == 0) mbar_expect_tx(full(st), bytes);
                    __syncwarp();
                    if (use) {
                        const uint32_t dst = ring + st * C::stage + lane * T * 128;
#pragma unroll
                        for (uint32_t b = 0; b < D / 64; ++b)
                            tma_load_4d(dst + b * KB, v ? mv : mk, static_cast<int32_t>(64 * b),
                                        static_cast<int32_t>(g.h), static_cast<int32_t>(off), id,
                                        full(st));
                    }
                }
                if (stop) break;
            }
        }
        if (stop) {  // gave up: drain the loads already issued (bounded)
            if (lane == 0) atomicExch(&s_fail, 1u);
            for (uint32_t i = q > ST ? q - ST : 0; i < q; ++i) mbar_wait(full(i % ST), (i / ST) & 1u);
        }
    } else if (warp == 1) {
        if (lane == 0) {  // ---- products ----
            constexpr uint32_t id_s = idesc(BN, false), id_o = idesc(D, true);
            uint32_t j = 0;  // tiles before this piece
            uint32_t nq[2] = {0, 0}, np[2] = {0, 0}, npv[2] = {0, 0};
            bool stop = false;
            auto wait = [&](uint32_t bar, uint32_t parity) {
                if (!mbar_wait(bar, parity) || failed()) stop = true;
                return !stop;
            };
            while (!stop && walk.next(g)) {
                const bool both = g.rows > 128;  // two row tiles, the same keys
                uint32_t n[2] = {g.n, both ? g.n : 0};
                if (NS == 2 && !both) {
                    n[0] = (g.n + 1) / 2;
                    n[1] = g.n / 2;
                }
                auto tile = [&](uint32_t s, uint32_t i) { return j + (NS == 2 && !both ? 2 * i + s : i); };
                auto scores = [&](uint32_t s, uint32_t i) {
                    const uint32_t k = 2 * tile(s, i), st = k % ST;
                    if (!wait(full(st), (k / ST) & 1u)) return;
                    tc_fence_after();
                    const uint64_t da = sw128_desc(base + s * C::q_bytes);
                    const uint64_t db = sw128_desc(ring + st * C::stage);
#pragma unroll
                    for (uint32_t c = 0; c < D / 16; ++c)  // 16 columns: 32 bytes of a block
                        mma_ss(tmem + C::s_col(s), da + (c / 4) * (QB / 16) + 2 * (c % 4),
                               db + (c / 4) * (KB / 16) + 2 * (c % 4), id_s, c != 0);
                    if (!both || s == 1) mma_commit(empty(st));
                    mma_commit(s_full(s));
                };
                for (uint32_t s = 0; s < NS && !stop; ++s)
                    if (n[s]) {
                        if (!wait(q_ready(s), nq[s]++ & 1u)) break;
                        tc_fence_after();
                        scores(s, 0);
                    }
                for (uint32_t i = 0; i < n[0] && !stop; ++i)
                    for (uint32_t s = 0; s < NS && !stop; ++s) {
                        if (i >= n[s]) continue;
                        const uint32_t v = 2 * tile(s, i) + 1, st = v % ST;
                        if (!wait(p_ready(s), np[s]++ & 1u) || !wait(full(st), (v / ST) & 1u)) break;
                        tc_fence_after();
                        const uint64_t db = sw128_desc_mn(ring + st * C::stage, KB);
#pragma unroll
                        for (uint32_t c = 0; c < BN / 16; ++c)  // 16 keys: 8 columns of P, 2 KiB of V
                            mma_ts(tmem + C::o_col(s), tmem + C::s_col(s) + 8 * c, db + 128 * c, id_o,
                                   i != 0 || c != 0);
                        if (!both || s == 1) mma_commit(empty(st));
                        mma_commit(pv_done(s));
                        ++npv[s];
                        if (i + 1 < n[s]) {  // S over P: after the product that reads it
                            if (!wait(pv_done(s), (npv[s] - 1) & 1u)) break;
                            tc_fence_after();
                            scores(s, i + 1);
                        }
                    }
                j += g.n;
            }
            // on the regular path the softmax waits for the last products; here the
            // issuer does, before the memory they use is given back
            if (stop) {
                atomicExch(&s_fail, 1u);
                mma_commit(drain);
                mbar_wait(drain, 0);
            }
        }
    } else if (warp >= 4) {  // ---- softmax, a thread a row ----
        const uint32_t s = (warp - 4) >> 2, qd = warp & 3, r = 32 * qd + lane;
        const uint32_t tid = threadIdx.x & 127;
        const uint32_t G = a.n_head / a.n_head_kv;
        const float c = fabsf(a.scale) * 1.44269504f;
        const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;  // a negative scale turns Q
        const uint32_t ts = tmem + ((32 * qd) << 16) + C::s_col(s);
        const uint32_t to = tmem + ((32 * qd) << 16) + C::o_col(s);
        uint32_t j = 0, ns = 0, npv = 0;
        bool stop = false;
        auto wait = [&](uint32_t bar, uint32_t parity) {
            const bool ok = mbar_wait(bar, parity) && !failed();
            if (!__all_sync(0xffffffffu, ok)) stop = true;
            return !stop;
        };
        while (!stop && walk.next(g)) {
            const bool both = g.rows > 128;
            const uint32_t first = NS == 2 && both ? 128 * s : 0;  // of the unit's rows
            const uint32_t n = NS == 1 || both ? g.n : (g.n + 1 - s) / 2;
            const uint32_t rows = g.rows - first < 128 ? g.rows - first : 128;
            const uint32_t j0 = j;
            j += g.n;
            if (n == 0) {  // a piece of one tile: nothing from the second stream
                if (r < rows)
                    l.ml[(static_cast<uint64_t>(g.slot) * NS + s) * 128 + r] = make_float2(-INFINITY, 0.0f);
                continue;
            }
            // Q, in the swizzled layout; rows past the last are zeros
            for (uint32_t i = tid; i < 128 * (D / 8); i += 128) {
                const uint32_t qr = i / (D / 8), ch = i % (D / 8);
                uint4 w = make_uint4(0, 0, 0, 0);
                if (qr < rows) {
                    const uint32_t rr = g.row0 + first + qr, t = rr / G;
                    w = __ldg(reinterpret_cast<const uint4 *>(
                        a.q + static_cast<uint64_t>(g.q0 + t) * a.q_stride +
                        static_cast<uint64_t>(g.h * G + rr - t * G) * D + 8 * ch));
                    w.x ^= sign;
                    w.y ^= sign;
                    w.z ^= sign;
                    w.w ^= sign;
                }
                const uint32_t at = base + s * C::q_bytes + (ch / 8) * QB + qr * 128 +
                                    (((ch % 8) ^ (qr % 8)) * 16);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(w.x), "r"(w.y),
                             "r"(w.z), "r"(w.w)
                             : "memory");
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready(s));

            // how far the row sees into the list
            uint32_t seen = 0xffffffffu;
            const TileGeom<BN> geom((g.tail ? a.tail : a.prefix).pages.page_tokens);
            if (g.tail) {
                const SeqShape sh = seq_shape(a, g.seq);
                const uint32_t i = (g.row0 + first + min(r, rows - 1)) / G;
                seen = tail_seen(sh, i);
            }
            float m = -INFINITY, sum = 0.0f;  // of c q . k
            for (uint32_t i = 0; i < n; ++i) {
                const uint32_t tj = NS == 2 && !both ? 2 * i + s : i;  // of the piece
                const uint32_t jj = j0 + tj;
                if (!wait(s_full(s), ns++ & 1u) || !wait(meta(jj % kMeta), (jj / kMeta) & 1u)) break;
                tc_fence_after();
                uint32_t mask[BN / 32], all = 0xffffffffu;
#pragma unroll
                for (int w = 0; w < BN / 32; ++w) {
                    mask[w] = s_mask[jj % kMeta][w];
                    all &= mask[w];
                }
                uint32_t page, off;
                geom.locate(g.tile0 + tj, page, off);
                const uint32_t pos0 = page * geom.T + off;
                const uint32_t lim = seen > pos0 ? min(seen - pos0, static_cast<uint32_t>(BN)) : 0;
                const bool whole = all == 0xffffffffu;
                if (!whole) {  // V rows of cells without a token become zeros
                    const uint32_t k = 2 * jj + 1;
                    if (!wait(full(k % ST), (k / ST) & 1u)) break;
                    for (uint32_t x = tid; x < BN * (D / 64); x += 128) {
                        const uint32_t key = x % BN;
                        if (s_mask[jj % kMeta][key / 32] >> (key % 32) & 1u) continue;
                        const uint32_t at = ring + (k % ST) * C::stage + (x / BN) * KB + key * 128;
#pragma unroll
                        for (uint32_t z = 0; z < 128; z += 16)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at + z), "r"(0u)
                                         : "memory");
                    }
                    fence_async_smem();
                }
                uint32_t v[BN];
#pragma unroll
                for (int w = 0; w < BN / 32; ++w) tmem_ld32_nowait(ts + 32 * w, v + 32 * w);
                tmem_ld_wait();
                const bool clear = __all_sync(0xffffffffu, whole && lim >= BN);
                float top = -INFINITY;
                if (!clear) {
#pragma unroll
                    for (int k = 0; k < BN; ++k)
                        if (!(mask[k / 32] >> (k % 32) & 1u) || k >= lim) v[k] = 0xff800000u;
                }
#pragma unroll
                for (int k = 0; k < BN; k += 4)
                    top = fmaxf(top, fmaxf(fmaxf(__uint_as_float(v[k]), __uint_as_float(v[k + 1])),
                                           fmaxf(__uint_as_float(v[k + 2]), __uint_as_float(v[k + 3]))));
                // a score of c q . k; c = 0 makes 0 of every finite one, and a masked one stays -inf
                top = top == -INFINITY ? top : top * c;
                if (__any_sync(0xffffffffu, top > m + 8.0f)) {
                    const float mn = fmaxf(m, top);
                    const float f = m == -INFINITY ? 0.0f : ex2(m - mn);
                    m = mn;
                    sum *= f;
                    if (i != 0) {  // the product before has completed: S came after it
#pragma unroll 1
                        for (uint32_t col = 0; col < D; col += 32) {
                            uint32_t o[32];
                            tmem_ld32_nowait(to + col, o);
                            tmem_ld_wait();
#pragma unroll
                            for (int k = 0; k < 32; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                            tmem_st32(to + col, o);
                        }
                    }
                }
                const float neg = m == -INFINITY ? 0.0f : -m;
                float s0 = 0.0f, s1 = 0.0f;
                if (c == 0.0f && !clear) {  // -inf * 0
#pragma unroll
                    for (int k = 0; k < BN; ++k)
                        v[k] = __float_as_uint(v[k] == 0xff800000u ? -INFINITY : neg);
                } else {
#pragma unroll
                    for (int k = 0; k < BN; ++k)
                        v[k] = __float_as_uint(__fmaf_rn(__uint_as_float(v[k]), c, neg));
                }
#pragma unroll
                for (int w = 0; w < BN / 64; ++w) {
                    uint32_t pk[32];
#pragma unroll
                    for (int k = 0; k < 32; ++k) {
                        const float x = ex2(__uint_as_float(v[64 * w + 2 * k]));
                        const float y = ex2(__uint_as_float(v[64 * w + 2 * k + 1]));
                        s0 += x;
                        s1 += y;
                        pk[k] = pack_h2(x, y);
                    }
                    tmem_st32(ts + 32 * w, pk);
                }
                sum += s0 + s1;
                tmem_st_wait();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready(s));
                ++npv;
            }
            if (stop || !wait(pv_done(s), (npv - 1) & 1u)) break;
            tc_fence_after();
            const uint64_t slot = static_cast<uint64_t>(g.slot) * NS + s;
            if (r < rows) l.ml[slot * 128 + r] = make_float2(m, sum);
#pragma unroll 1
            for (uint32_t col = 0; col < D; col += 32) {
                uint32_t o[32];
                tmem_ld32_nowait(to + col, o);
                tmem_ld_wait();
                if (r < rows) {
#pragma unroll
                    for (uint32_t k = 0; k < 8; ++k)
                        l.o[(slot * (D / 4) + col / 4 + k) * 128 + r] =
                            make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                                        __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
                }
            }
            tc_fence_before();
        }
        if (stop && lane == 0) atomicExch(&s_fail, 1u);
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x == 0) {
        l.fail[blockIdx.x] = s_fail;
        if (blockIdx.x == 0) *l.plan = plan;
    }
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"(kAttnTmem)
                     : "memory");
    }
}

// The join: a row's pieces of the prefix and of its tail, weighted by
// 2^(m_piece - m), in a fixed order. 8 rows a CTA, a thread per row and four
// dimensions: reads of 128 bytes (8 rows of one float4 column).
constexpr uint32_t kJoinRows = 8, kMaxCtas = 160;
struct JoinRow {
    uint64_t x0[2], x1[2];    // the row's unit on its line: prefix, tail
    uint64_t total[2];
    uint32_t parts[2], first[2], n[2];  // ranges of the line; the first and how many meet the unit
    uint32_t slot0[2], step[2];         // workspace slot of range i: slot0 + i * step
    uint32_t row[2];                    // within the slot's stream
    uint32_t stream[2], both[2];        // the row tile; whether the streams are row tiles
    bool write;
};

template <int D>
__global__ void __launch_bounds__(kJoinRows *D / 4)
    attn_join_kernel(const __grid_constant__ AttnLaunch l, uint32_t n_cta) {
    using C = Cfg<D>;
    constexpr int PR = C::PR, NS = C::NS;
    constexpr uint32_t kList = 4 * kMaxCtas;  // two lines, two streams
    __shared__ JoinRow rows[kJoinRows];
    __shared__ uint32_t s_id[kJoinRows][kList];
    __shared__ float s_w[kJoinRows][kList];
    __shared__ uint32_t s_n[kJoinRows];
    __shared__ float s_inv[kJoinRows];
    const PrefixAttn &a = l.a;
    const uint32_t G = a.n_head / a.n_head_kv, H = a.n_head_kv;
    const uint64_t row0 = static_cast<uint64_t>(blockIdx.x) * kJoinRows;
    cudaGridDependencySynchronize();
    uint32_t bad = 0;
    for (uint32_t i = threadIdx.x; i < n_cta; i += blockDim.x) bad |= l.fail[i];
    if (threadIdx.x < kJoinRows) {
        const Plan &p = *l.plan;
        JoinRow d{};
        const uint64_t x = row0 + threadIdx.x;
        const uint32_t t = static_cast<uint32_t>(x / a.n_head);
        const uint32_t head = static_cast<uint32_t>(x - static_cast<uint64_t>(t) * a.n_head);
        const uint32_t h = head / G, gq = head - h * G;
        uint32_t seq = 0;
        d.write = t < a.n_q;
        if (d.write && a.n_seq) {
            // the last sequence that starts at or before t
            uint32_t lo = 0, hi = a.n_seq + 1;
            while (lo < hi) {
                const uint32_t mid = (lo + hi) / 2;
                if (a.q_start[mid] <= static_cast<int32_t>(t))
                    lo = mid + 1;
                else
                    hi = mid;
            }
            d.write = lo >= 1 && lo <= a.n_seq;
            seq = lo - 1;
        }
        if (d.write && p.np && t >= p.q0 && (t - p.q0) * G + gq < p.rows) {
            const uint32_t r = (t - p.q0) * G + gq, pair = r / PR, pg = pair / p.gs;
            const uint64_t u = static_cast<uint64_t>(pg) * H + h;
            d.total[0] = p.gs == 1 ? p.p_total + p.t_total : p.p_total;
            d.parts[0] = p.gs == 1 ? n_cta : p.groups;
            d.x0[0] = u * p.np;
            d.x1[0] = d.x0[0] + p.np;
            d.slot0[0] = static_cast<uint32_t>(u) * p.gs + pair - pg * p.gs;
            d.step[0] = p.gs;
            d.both[0] = p.rows - pair * PR > 128 && NS == 2;
            d.row[0] = r % 128;
            d.stream[0] = r % PR / 128;
        }
        if (d.write && a.n_seq) {
            const SeqShape sh = seq_shape(a, seq);
            const TileGeom<C::BN> tg(a.tail.pages.page_tokens);
            const uint32_t tiles = tg.tiles(sh.len), i = t - sh.q0;
            if (t >= sh.q0 && i < sh.q_len && tiles && p.t_total) {
                const uint32_t r = i * G + gq, pair = r / PR, u = pair * H + h;
                const uint64_t base = p.gs == 1 ? p.p_total : 0;
                d.total[1] = base + p.t_total;
                d.parts[1] = n_cta;
                d.x0[1] = base + l.seq_tile[seq] + static_cast<uint64_t>(u) * tiles;
                d.x1[1] = d.x0[1] + min(tiles, pair_tiles<C::BN, PR>(sh, tg, pair, G));
                d.slot0[1] = p.t_slot0 + l.seq_pair[seq] * H + u;
                d.step[1] = 1;
                d.both[1] = sh.q_len * G - pair * PR > 128 && NS == 2;
                d.row[1] = r % 128;
                d.stream[1] = r % PR / 128;
            }
        }
        for (int k = 0; k < 2; ++k)
            if (d.x1[k] > d.x0[k]) {
                d.first[k] = owner(d.x0[k], d.total[k], d.parts[k]);
                d.n[k] = owner(d.x1[k] - 1, d.total[k], d.parts[k]) + 1 - d.first[k];
            }
        rows[threadIdx.x] = d;
    }
    bad = __syncthreads_or(bad);
    // a warp lists a row's pieces and weighs them
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    for (uint32_t w = warp; w < kJoinRows; w += blockDim.x / 32) {
        const JoinRow &d = rows[w];
        uint32_t n = 0;
        float top = -INFINITY;
        for (int k = 0; k < 2; ++k) {
            const uint32_t per = NS == 2 && !d.both[k] ? 2 : 1;
            for (uint32_t i0 = 0; i0 < d.n[k] * per; i0 += 32) {
                const uint32_t i = i0 + lane, part = d.first[k] + i / per;
                bool ok = i < d.n[k] * per;
                // a range may be empty when there are fewer tiles than CTAs
                ok = ok && max(d.x0[k], cut(d.total[k], part, d.parts[k])) <
                               min(d.x1[k], cut(d.total[k], part + 1, d.parts[k]));
                uint32_t id = 0;
                float m = -INFINITY;
                if (ok) {
                    id = ((d.slot0[k] + part * d.step[k]) * NS + (per == 2 ? i % 2 : d.stream[k])) * 128 +
                         d.row[k];
                    m = l.ml[id].x;
                    ok = m != -INFINITY;
                }
                const uint32_t have = __ballot_sync(0xffffffffu, ok);
                if (ok) {
                    const uint32_t at = n + __popc(have & ((1u << lane) - 1));
                    s_id[w][at] = id;
                    s_w[w][at] = m;
                    top = fmaxf(top, m);
                }
                n += __popc(have);
            }
        }
        for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        __syncwarp();
        float sum = 0.0f;
        for (uint32_t i = lane; i < n; i += 32) {
            const float f = ex2(s_w[w][i] - top);
            sum += f * l.ml[s_id[w][i]].y;
            s_w[w][i] = f;
        }
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            s_n[w] = n;
            s_inv[w] = bad ? NAN : n ? 1.0f / sum : 0.0f;
            if (a.lse && d.write)
                a.lse[row0 + w] = bad ? NAN : n ? (top + log2f(sum)) * 0.693147181f : -INFINITY;
        }
    }
    __syncthreads();
    const uint32_t r = threadIdx.x % kJoinRows, col = threadIdx.x / kJoinRows;
    if (!rows[r].write) return;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const uint32_t n = s_n[r];
#pragma unroll 4
    for (uint32_t i = 0; i < n; ++i) {
        const uint32_t id = s_id[r][i];
        const float f = s_w[r][i];
        const float4 o = l.o[(static_cast<uint64_t>(id / 128) * (D / 4) + col) * 128 + id % 128];
        acc.x = __fmaf_rn(f, o.x, acc.x);
        acc.y = __fmaf_rn(f, o.y, acc.y);
        acc.z = __fmaf_rn(f, o.z, acc.z);
        acc.w = __fmaf_rn(f, o.w, acc.w);
    }
    const float inv = s_inv[r];
    *reinterpret_cast<uint2 *>(a.out + (row0 + r) * D + 4 * col) =
        make_uint2(pack_h2(acc.x * inv, acc.y * inv), pack_h2(acc.z * inv, acc.w * inv));
}

// 4-D f16 tensor {D, heads, tokens, pages}; box {64, 1, tokens of a tile, 1}.
cudaError_t encode_pages(CUtensorMap *map, const uint8_t *at, uint64_t row, uint64_t page,
                         const PageView &v, uint32_t bn) {
    const EncodeTiledFn fn = encode_fn();
    if (!fn) return cudaErrorNotSupported;
    const cuuint64_t dims[4] = {v.d_head, v.n_head_kv, v.page_tokens, v.n_pages};
    const cuuint64_t strides[3] = {v.d_head * 2ull, row, page};
    const cuuint32_t box[4] = {64, 1, std::min(v.page_tokens, bn), 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4, const_cast<uint8_t *>(at), dims,
                          strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                          CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

uint32_t attn_ctas() {
    int dev = 0, n = 0;
    if (cudaGetDevice(&dev) != cudaSuccess ||
        cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0)
        n = 148;
    return std::min<uint32_t>(static_cast<uint32_t>(n), kMaxCtas);
}

uint64_t up256(uint64_t v) { return (v + 255) / 256 * 256; }

// The workspace: plan, one word per CTA, the sequences' offsets, the pieces.
struct WsLayout {
    uint64_t fail, seq_tile, seq_pair, ml, o, bytes, slots;
    WsLayout(uint32_t n_q, uint32_t n_head, uint32_t n_head_kv, uint32_t d, uint32_t n_seq) {
        const uint64_t pr = d == 256 ? 128 : 256, ns = pr / 128;
        const uint64_t rows = static_cast<uint64_t>(n_q) * (n_head / n_head_kv);
        const uint64_t pairs = (rows + pr - 1) / pr, pg = (pairs + 7) / 8;
        // prefix: n_pg * gs <= pairs + n_pg units a KV head, and a range each;
        // tails: a pair per sequence more than whole pairs of the rows
        slots = (pairs + pg) * n_head_kv + 2 * kMaxCtas +
                (n_seq ? (n_seq + rows / pr) * n_head_kv : 0);
        fail = up256(sizeof(Plan));
        seq_tile = fail + up256(kMaxCtas * 4);
        seq_pair = seq_tile + up256(8ull * n_seq);
        ml = seq_pair + up256(4ull * n_seq);
        o = ml + up256(slots * ns * 128 * 8);
        bytes = o + slots * ns * 128 * d * 4;
    }
};

template <int D>
cudaError_t launch_t(const AttnLaunch &l, cudaStream_t st) {
    const uint32_t n_cta = attn_ctas();
    cudaError_t e = cudaFuncSetAttribute(
        attn_tc_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(Cfg<D>::smem));
    if (e != cudaSuccess) return e;
    attn_tc_kernel<D><<<n_cta, Cfg<D>::threads, Cfg<D>::smem, st>>>(l);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    const uint64_t rows = static_cast<uint64_t>(l.a.n_q) * l.a.n_head;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(static_cast<uint32_t>((rows + kJoinRows - 1) / kJoinRows));
    cfg.blockDim = dim3(kJoinRows * D / 4);
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, attn_join_kernel<D>, l, n_cta);
}

}  // namespace

size_t prefix_attn_ws_bytes(uint32_t n_q, uint32_t n_head, uint32_t n_head_kv, uint32_t d_head,
                            uint32_t n_seq) {
    return WsLayout(n_q, n_head, n_head_kv, d_head, n_seq).bytes;
}

cudaError_t launch_prefix_attn_rows(const PrefixAttn &a, cudaStream_t st);

cudaError_t launch_prefix_attn(const PrefixAttn &a, void *ws, cudaStream_t st) {
    for (const KeyList *kl : {&a.prefix, &a.tail})
        if (kl->max_len && (kl->pages.k_type != KVMRET_TYPE_F16 || kl->pages.v_type != KVMRET_TYPE_F16))
            return launch_prefix_attn_rows(a, st);
    const WsLayout w(a.n_q, a.n_head, a.n_head_kv, a.d_head, a.n_seq);
    uint8_t *b = static_cast<uint8_t *>(ws);
    AttnLaunch l{};
    l.a = a;
    l.plan = reinterpret_cast<Plan *>(b);
    l.fail = reinterpret_cast<uint32_t *>(b + w.fail);
    l.seq_tile = reinterpret_cast<uint64_t *>(b + w.seq_tile);
    l.seq_pair = reinterpret_cast<uint32_t *>(b + w.seq_pair);
    l.ml = reinterpret_cast<float2 *>(b + w.ml);
    l.o = reinterpret_cast<float4 *>(b + w.o);
    l.max_slots = static_cast<uint32_t>(w.slots);
    const uint32_t bn = a.d_head == 256 ? 64 : 128;
    const KeyList *lists[2] = {&a.prefix, &a.tail};
    for (int i = 0; i < 2; ++i) {
        const PageView &v = lists[i]->pages;
        if (!lists[i]->max_len) continue;
        cudaError_t e = encode_pages(&l.map[2 * i], v.k, v.k_row, v.k_page, v, bn);
        if (e == cudaSuccess) e = encode_pages(&l.map[2 * i + 1], v.v, v.v_row, v.v_page, v, bn);
        if (e != cudaSuccess) return e;
    }
    if (a.d_head == 64) return launch_t<64>(l, st);
    if (a.d_head == 128) return launch_t<128>(l, st);
    return launch_t<256>(l, st);
}

}  // namespace kvmret
