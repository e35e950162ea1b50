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
//          no multicast), or of quant blocks into raw tiles;
//   2      plans, walks the pieces and leaves each in a short ring for the others;
//   3      notes for the join where each row's pieces lie;
//   1      an elected lane issues the products: S = Q K^T (both in shared memory)
//          and O += P V (P in tensor memory, V as it lies: keys along K, MN-major);
//   4-7    softmax of stream 0, a thread a row; also loads Q, rescales and
//          hands on O;
//   8-11   f16, head sizes 64 and 128: the same for stream 1;
//   8-15   quantised K or V: four warps turn K blocks into f16 tiles, four V.
// Tiles of 128 keys (head size 256: 64), 128 rows a stream.
//   Two streams (f16): with more than 128 rows they are two tiles of rows over
//     the same key tiles, otherwise the same rows over every other key tile,
//     each with its own output. While one stream is in its softmax the other
//     one's products run. P lies over its S, so a stream's next S waits until
//     the product that reads P has completed.
//   One stream (quantised, whose converting warps take the other one's registers;
//     head size 256, whose output takes its tensor memory): S has two tiles and
//     P columns of its own, so the next scores are issued before this softmax
//     ends, and the softmax can be a loop of 64 keys.
// Cells without a token may hold anything, NaN too: their scores are replaced
// after the product, their V rows zeroed in shared memory before it.
// Every wait is bounded; on a timeout the outputs become NaN (the join).
//
// What bounds it. Memory asks 24 us of 16 rows by 8 heads over 32,768 f16 tokens
// and their tails, the call takes 43: 5 us until the first scores (plan, pages,
// queries, first tiles, each a dependent read), 4 us for the join, between them
// a chain of softmax and product per tile that reads at 4.5 TB/s. With 256 rows a
// unit the chain is about 4000 clocks for 2 * 128 x 128 scores: 2048 exponentials
// a scheduler, the products of one stream during the softmax of the other (tensor
// pipe active 47 %): 2048 rows by 64 heads over 32,768 tokens take 2.18 to 2.5 ms
// as the clock stands, 0.9 to 1.04 PFLOP/s. Quantised: 54 us for the first shape (10 by
// its bytes), bound by the same chain of one stream, 3000 clocks a tile.
// The instruction caches count: conversions as straight code of a tile were 12 %
// slower than a loop over blocks (68 and 61 us), the softmax of one stream as
// straight code of 128 keys 10 % (61 and 55).
// Tried and no better: 64-key tiles with two S tiles for both streams (3.6 ms
// against 2.2; a 64-key product takes 58 clocks, a 128-key one 64); exponentials of
// 1/8 to 3/8 of the keys as polynomials (2.5 to 2.6 against 2.4 ms); a warp for S
// and one for P V (2.28 to 2.38 against 2.15 to 2.25 ms); the products' warp asking
// for all it needs at once (the same); one converting warpgroup and two streams
// (75 us against 55).
#include "prefix_attn.cuh"

#include <cuda_fp16.h>

#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "kvmret.h"
#include "prefix_attn_plan.cuh"
#include "quant.cuh"
#include "tc.cuh"

namespace kvmret {
namespace {

// QUANT: some K or V rows are q8_0 or q4_0 blocks.
template <int D, bool QUANT>
struct Cfg {
    static constexpr int NS = D == 256 || QUANT ? 1 : 2;  // streams
    static constexpr int NB = 3 - NS;               // S tiles of a stream
    static constexpr int BN = D == 256 ? 64 : 128;  // keys of a tile
    static constexpr int PR = 128 * NS;             // rows of a unit
    static constexpr int parts = NS;                // parts of a tile that P is handed on in
    static constexpr int threads = 128 + 128 * NS + (QUANT ? 256 : 0);
    static constexpr uint32_t stage = BN * D * 2;   // one K or V tile
    static constexpr int stages = QUANT ? (D == 64 ? 8 : D == 128 ? 4 : 3) : D == 64 ? 8 : 5;
    static constexpr uint32_t q_bytes = 128 * D * 2;
    // tiles of quant blocks as they lie in memory, on their way: two of K, one or
    // two of V as their formats leave room (AttnLaunch)
    static constexpr int raws = QUANT ? 2 : 0;
    static constexpr uint32_t raw0 = NS * q_bytes + stages * stage;
    static constexpr uint32_t raw_bytes = QUANT ? 3 * BN * (D == 64 ? 80 : D == 128 ? 144 : 272) + 2048 : 0;
    static constexpr uint32_t tiles = raw0 + raw_bytes;
    static __host__ __device__ constexpr uint32_t s_col(int s) { return s * 128; }
    static __host__ __device__ constexpr uint32_t o_col(int s) { return 256 + s * (D == 64 ? 64 : 128); }
    // P of S tile b: one stream leaves columns for it, two put it over its S
    static __host__ __device__ constexpr uint32_t p_col(int s, uint32_t b) {
        return NS == 2 ? s_col(s) : (D == 256 ? 128 : 384) + b * (BN / 2);
    }
    // The stage of the K or V tile of tile t, and how often it was used before.
    // TMA fills one ring in the order K0 V0 K1 V1 ..; the converting warps have
    // a ring each, so that a K does not wait for the P V of another tile.
    static constexpr int k_stages = D == 64 ? 4 : 2, v_stages = D == 64 ? 4 : D == 128 ? 2 : 1;
    static_assert(!QUANT || stages == k_stages + v_stages, "stages");
    static __device__ __forceinline__ uint32_t k_stage(uint32_t t) { return QUANT ? t % k_stages : 2 * t % stages; }
    static __device__ __forceinline__ uint32_t k_round(uint32_t t) { return QUANT ? t / k_stages : 2 * t / stages; }
    static __device__ __forceinline__ uint32_t v_stage(uint32_t t) {
        return QUANT ? k_stages + t % v_stages : (2 * t + 1) % stages;
    }
    static __device__ __forceinline__ uint32_t v_round(uint32_t t) {
        return QUANT ? t / v_stages : (2 * t + 1) / stages;
    }
};
// Bytes of the box that holds a head's row of quant blocks: it starts on a
// 16-byte boundary at or up to 12 bytes before the row.
template <int D>
__host__ __device__ constexpr uint32_t raw_box(int32_t type) {
    return D == 64 ? (type == KVMRET_TYPE_Q8_0 ? 80 : 48) : D == 128 ? (type == KVMRET_TYPE_Q8_0 ? 144 : 80)
                                                        : (type == KVMRET_TYPE_Q8_0 ? 272 : 144);
}
constexpr uint32_t kAttnTmem = 512;
constexpr int kSegs = 4;  // pieces ahead
constexpr int kMeta = 16;  // tiles whose masks are held (more than the ring reaches back)

// Where one row's pieces lie among the workspace's rows: the first at row id, the
// i-th of n at rest + i * step.
struct RowPieces {
    uint32_t id, rest, step, n;
    __device__ __forceinline__ uint32_t at(uint32_t i) const { return i ? rest + i * step : id; }
};
// A row's output in the workspace: rows by eights, so that both a warp with a row
// a lane and the join with eight rows of one column move whole 128-byte lines.
template <int D>
__device__ __forceinline__ uint64_t out_at(uint32_t id, uint32_t col) {
    return static_cast<uint64_t>(id >> 3) * (D / 4 * 8) + col * 8 + (id & 7);
}

struct AttnLaunch {
    PrefixAttn a;
    CUtensorMap map[4];  // prefix K, V, tail K, V
    uint32_t *fail;  // [CTA] 1: a wait gave up, or q_start was not ascending
    RowPieces *at;   // [n_q * n_head][2] pieces of the prefix, of the tail
    float2 *ml;      // [row] maximum and sum
    float4 *o;       // [row / 8][D / 4][8]
    Rooms rooms;
    uint32_t raw_k, raw_v, n_raw_v;  // bytes of a raw K, V tile; raw V tiles
    Divs by;
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
__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32"
        " {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
          "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                   "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
                   "+r"(r[14]), "+r"(r[15])
                 :
                 : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0],"
        " {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(taddr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
// Two products and two sums at a time (each rounded like the scalar operation).
__device__ __forceinline__ void fma_pair(uint32_t &x, uint32_t &y, float a, float b) {
    asm("{\n\t.reg .b64 p, q, r;\n\t"
        "mov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %2};\n\tmov.b64 r, {%3, %3};\n\t"
        "fma.rn.f32x2 p, p, q, r;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "+r"(x), "+r"(y)
        : "f"(a), "f"(b));
}
__device__ __forceinline__ void add_pair(float &x, float &y, float a, float b) {
    asm("{\n\t.reg .b64 p, q;\n\t"
        "mov.b64 p, {%0, %1};\n\tmov.b64 q, {%2, %3};\n\t"
        "add.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "+f"(x), "+f"(y)
        : "f"(a), "f"(b));
}
// The wait for loads under way; it names the registers, so that nothing that
// reads them can be moved before it.
__device__ __forceinline__ void tmem_ld_wait(uint32_t *r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;"
                 : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]),
                   "+r"(r[7]), "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]),
                   "+r"(r[14]), "+r"(r[15]), "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]),
                   "+r"(r[20]), "+r"(r[21]), "+r"(r[22]), "+r"(r[23]), "+r"(r[24]), "+r"(r[25]),
                   "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]), "+r"(r[30]), "+r"(r[31])
                 :
                 : "memory");
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
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d), "l"(a), "l"(b),
        "r"(id), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t id,
                                       uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d), "r"(a), "l"(b),
        "r"(id), "r"(accumulate)
        : "memory");
}
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(p));
    return p;
}

// One key's NB quant blocks at shared address `src` (4-byte aligned), eight columns
// at a time to put(chunk, x), beginning with block `first` (which spreads the
// lanes over the banks). The loop stays one: the code of a tile would not fit
// the instruction caches beside the softmax's. A block's payload starts two
// bytes after its start, so its words straddle those of memory: in even blocks
// (which start on a word) by their upper half, in odd ones (which start between)
// by none.
template <int NB, int TYPE, typename Put>
__device__ __forceinline__ void convert_row(uint32_t src, uint32_t first, Put put) {
    constexpr uint32_t BLOCK = TYPE == KVMRET_TYPE_Q8_0 ? 34 : 18, NW = (BLOCK - 2) / 4;
#pragma unroll 1
    for (uint32_t i = 0; i < NB; ++i) {
        const uint32_t b = (i + first) % NB, at = src + b * BLOCK / 4 * 4;
        const uint32_t sel = b & 1 ? 0x7654 : 0x5432;
        uint32_t w[NW + 1];
#pragma unroll
        for (uint32_t k = 0; k <= NW; ++k) asm volatile("ld.shared.b32 %0, [%1];" : "=r"(w[k]) : "r"(at + 4 * k));
        const uint32_t dd = __byte_perm(w[0], 0, b & 1 ? 0x3232 : 0x1010);
        const __half2 d = *reinterpret_cast<const __half2 *>(&dd);
#pragma unroll
        for (uint32_t k = 0; k < NW; ++k) w[k] = __byte_perm(w[k], w[k + 1], sel);
        // halves of bytes 2k, 2k + 1 of u, less `bias`, times d
        auto pair = [&](uint32_t u, uint32_t k, uint32_t bias) {
            const uint32_t h = __byte_perm(u, 0x64646464u, k ? 0x4342 : 0x4140);
            const __half2 x = __hmul2(__hsub2(*reinterpret_cast<const __half2 *>(&h),
                                              *reinterpret_cast<const __half2 *>(&bias)), d);
            return *reinterpret_cast<const uint32_t *>(&x);
        };
#pragma unroll
        for (uint32_t c = 0; c < 4; ++c) {
            uint32_t u0, u1, bias;
            if constexpr (TYPE == KVMRET_TYPE_Q8_0) {
                u0 = w[2 * c] ^ 0x80808080u;
                u1 = w[2 * c + 1] ^ 0x80808080u;
                bias = 0x64806480u;
            } else {  // lower halves: columns 0 .. 15, upper: 16 .. 31
                u0 = (w[2 * (c % 2)] >> (c < 2 ? 0 : 4)) & 0x0f0f0f0fu;
                u1 = (w[2 * (c % 2) + 1] >> (c < 2 ? 0 : 4)) & 0x0f0f0f0fu;
                bias = 0x64086408u;
            }
            const uint32_t x[4] = {pair(u0, 0, bias), pair(u0, 1, bias), pair(u1, 0, bias), pair(u1, 1, bias)};
            put(4 * b + c, x);
        }
    }
}

// The plan of the split, by one warp, in every CTA alike. `start` receives the
// sequence that holds the CTA's first tail tile. False when q_start descends.
struct Start {
    uint32_t seq, tile;
};
// inclusive sums over the warp's lanes
__device__ __forceinline__ uint32_t scan(uint32_t x) {
    const uint32_t lane = threadIdx.x & 31;
    for (uint32_t o = 1; o < 32; o <<= 1) {
        const uint32_t u = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += u;
    }
    return x;
}

template <int D, bool QUANT>
__device__ bool make_plan(const AttnLaunch &l, Plan &p, Start &start) {
    constexpr int BN = Cfg<D, QUANT>::BN, PR = Cfg<D, QUANT>::PR;
    const PrefixAttn &a = l.a;
    const uint32_t lane = threadIdx.x & 31;
    const uint32_t G = l.by.G.d, H = a.n_head_kv;
    const TileGeom<BN> tg(l.by.list[1]);
    bool ok = true;
    auto shape = [&](uint32_t s) -> uint32_t {  // tiles of sequence s
        if (s >= a.n_seq) return 0;
        ok = ok && __ldg(a.q_start + s) <= __ldg(a.q_start + s + 1);
        const SeqShape sh = seq_shape(a, s);
        const uint32_t n = sh.q_len ? tg.tiles(sh.len) : 0;
        return (n ? n + kUnit<BN> : 0) * ((sh.q_len * G + PR - 1) / PR) * H;
    };
    const bool pre = a.prefix.max_len != 0;
    const int32_t len0 = pre && a.prefix.len ? __ldg(a.prefix.len) : 0x7fffffff;
    const int32_t q_first = a.n_seq ? __ldg(a.q_start) : 0;
    const int32_t q_last = a.n_seq ? __ldg(a.q_start + a.n_seq) : static_cast<int32_t>(a.n_q);
    // totals of the tails
    uint32_t t0 = shape(lane), tiles = t0;
#pragma unroll 4
    for (uint32_t s = 32 + lane; s < a.n_seq; s += 32) tiles += shape(s);
    ok = __all_sync(0xffffffffu, ok);
    // the last listed page with tokens, and how many the pages hold
    uint32_t held = pre ? a.prefix.n_list : 0, all = 0;
    const uint32_t T = a.prefix.pages.page_tokens;
    const bool partial = held && a.prefix.ntok;
    auto page_holds = [&](uint32_t i) {
        const uint32_t n = min(__ldg(a.prefix.ntok + i), T);
        return !a.prefix.table || static_cast<uint32_t>(__ldg(a.prefix.table + i)) < a.prefix.pages.n_pages ? n : 0;
    };
    if (partial) {
        held = 0;
#pragma unroll 8
        for (uint32_t i = lane; i < a.prefix.n_list; i += 32) {
            const uint32_t n = page_holds(i);
            if (n) held = i + 1;
            all += n;
        }
    }
    for (int o = 16; o; o >>= 1) {
        tiles += __shfl_xor_sync(0xffffffffu, tiles, o);
        held = max(held, __shfl_xor_sync(0xffffffffu, held, o));
        all += __shfl_xor_sync(0xffffffffu, all, o);
    }
    p.p_len = 0;
    p.np = 0;
    if (pre) {
        // p_len is a place of the list (page * T + offset): that behind the last token
        const uint64_t most = static_cast<uint64_t>(held) * T;
        const uint32_t len = min(a.prefix.max_len, static_cast<uint32_t>(max(len0, 0)));
        if (!partial) {
            p.p_len = most < len ? static_cast<uint32_t>(most) : len;
        } else if (len >= all) {
            p.p_len = static_cast<uint32_t>(most);
        } else if (len) {  // the page that holds token len - 1
            uint32_t before = 0;
            for (uint32_t i0 = 0; i0 < a.prefix.n_list; i0 += 32) {
                const uint32_t n = i0 + lane < a.prefix.n_list ? page_holds(i0 + lane) : 0;
                const uint32_t upto = scan(n);
                const uint32_t sum = __shfl_sync(0xffffffffu, upto, 31);
                const uint32_t hit = __ballot_sync(0xffffffffu, before + upto >= len);
                if (hit) {
                    const int w = __ffs(hit) - 1;
                    p.p_len = (i0 + w) * T + len - (before + __shfl_sync(0xffffffffu, upto - n, w));
                    break;
                }
                before += sum;
            }
        }
        p.np = TileGeom<BN>(l.by.list[0]).tiles(p.p_len);
    }
    const int32_t nq = static_cast<int32_t>(a.n_q);
    p.q0 = static_cast<uint32_t>(min(max(q_first, 0), nq));
    p.rows = (min(max(q_last, static_cast<int32_t>(p.q0)), nq) - p.q0) * G;
    p.n_pair = (p.rows + PR - 1) / PR;
    // 8 CTAs side by side leave at most 5 % of the 148 SMs without a group
    p.n_pg = (p.n_pair + 7) / 8;
    p.gs = p.n_pg > 1 ? (p.n_pair + p.n_pg - 1) / p.n_pg : max(p.n_pair, 1u);
    if (p.gs > gridDim.x) {
        p.gs = gridDim.x;
        p.n_pg = (p.n_pair + p.gs - 1) / p.gs;
    }
    p.groups = p.gs == 1 ? gridDim.x : gridDim.x / p.gs;
    p.p_total = p.np * p.n_pg * H;
    p.t_total = tiles;
    ok = ok && (p.n_pg * H + p.groups) * p.gs <= l.rooms.n_pre;  // (so it always is)
    p.ok = ok;
    if (!ok) p.p_total = p.t_total = 0;
    if (p.gs == 1) {
        p.pre.set(p.p_total + p.t_total, l.by.ctas);
        p.own = p.pre;
    } else {
        p.pre.set(p.p_total, p.groups);
        p.own.set(p.t_total, l.by.ctas);
    }
    start = {0, 0};
    uint32_t x, x1, y, y1;
    Walk<BN, PR>::ranges(p, blockIdx.x, x, x1, y, y1);
    if (y >= y1) return ok;  // no tails here
    uint32_t base_t = 0;
    for (uint32_t s0 = 0; s0 < a.n_seq; s0 += 32) {
        if (s0) t0 = shape(s0 + lane);
        uint32_t ti = scan(t0);
        const uint32_t all_t = __shfl_sync(0xffffffffu, ti, 31);
        ti += base_t - t0;
        const uint32_t hit = __ballot_sync(0xffffffffu, y >= ti && y < ti + t0);
        if (hit) {
            const int w = __ffs(hit) - 1;
            start.seq = s0 + w;
            start.tile = __shfl_sync(0xffffffffu, ti, w);
            break;
        }
        base_t += all_t;
    }
    return ok;
}

// Where the pieces of every row lie, for the join: by one warp of each CTA, a
// lane a row, the CTAs taking blocks of 32 rows in turn.
template <int D, bool QUANT>
__device__ void note_rows(const AttnLaunch &l, const Plan &p) {
    constexpr int BN = Cfg<D, QUANT>::BN, PR = Cfg<D, QUANT>::PR;
    const PrefixAttn &a = l.a;
    const Rooms &rooms = l.rooms;
    const uint32_t lane = threadIdx.x & 31, n_cta = gridDim.x;
    const uint32_t G = l.by.G.d, H = a.n_head_kv;
    // rows of the tokens [q0, q0 + q_len); tails from tile `tile` on
    auto note = [&](uint32_t q0, uint32_t q_len, const SeqShape *sh, uint32_t tile) {
        const TileGeom<BN> tg(l.by.list[1]);
        const uint32_t tiles = sh ? tg.tiles(sh->len) : 0;
        const uint32_t begin = q0 * a.n_head, end = begin + q_len * a.n_head;
        uint32_t b = begin / 32;
        b += (blockIdx.x + n_cta - b % n_cta) % n_cta;  // the first block of this CTA
        for (; b * 32 < end; b += n_cta) {
            const uint32_t x = 32 * b + lane;
            if (x < begin || x >= end) continue;
            const uint32_t t = x / a.n_head, head = x - t * a.n_head, h = l.by.G(head), gq = head - h * G;
            RowPieces r[2] = {};
            // the first piece's range; the number of pieces
            auto cut = [&](RowPieces &e, const Cuts &cuts, uint32_t x0, uint32_t n) {
                const uint32_t first = cuts.owner(x0);
                e.n = cuts.owner(x0 + n - 1) + 1 - first;
                return first;
            };
            if (p.np) {
                const uint32_t row = (t - p.q0) * G + gq, pair = row / PR, pg = pair / p.gs, u = pg * H + h;
                const uint32_t first = cut(r[0], p.pre, u * p.np, p.np);
                r[0].step = p.gs * rooms.cap;
                r[0].id = r[0].rest = ((u + first) * p.gs + pair - pg * p.gs) * rooms.cap + row % PR;
            }
            if (tiles) {
                const uint32_t row = (t - q0) * G + gq, pair = row / PR, u = pair * H + h;
                const uint32_t n = min(tiles, pair_tiles<BN, PR>(*sh, tg, pair, l.by.G));
                if (n) {
                    const uint32_t first = cut(r[1], p.own, (p.gs == 1 ? p.p_total : 0) + tile +
                                               u * (tiles + kUnit<BN>) + kUnit<BN>, n);
                    r[1].id = rooms.tail + ((q0 - p.q0) * H + h * q_len) * G + row;
                    r[1].step = rooms.cap;
                    r[1].rest = rooms.over + first * rooms.cap + row % PR;
                }
            }
            l.at[2 * x] = r[0];
            l.at[2 * x + 1] = r[1];
        }
    };
    if (!a.n_seq) {
        note(0, a.n_q, nullptr, 0);
        return;
    }
    const TileGeom<BN> tg(l.by.list[1]);
    uint32_t base_t = 0;
    for (uint32_t s0 = 0; s0 < a.n_seq; s0 += 32) {
        SeqShape sh = {};
        if (s0 + lane < a.n_seq) sh = seq_shape(a, s0 + lane);
        const uint32_t pairs = (sh.q_len * G + PR - 1) / PR, n = sh.q_len ? tg.tiles(sh.len) : 0;
        const uint32_t tiles = (n ? n + kUnit<BN> : 0) * pairs * H;
        const uint32_t ti = scan(tiles);
        for (uint32_t w = 0; w < min(32u, a.n_seq - s0); ++w) {
            SeqShape one;
            one.q0 = __shfl_sync(0xffffffffu, sh.q0, w);
            one.q_len = __shfl_sync(0xffffffffu, sh.q_len, w);
            one.len = __shfl_sync(0xffffffffu, sh.len, w);
            note(one.q0, one.q_len, &one, base_t + __shfl_sync(0xffffffffu, ti - tiles, w));
            __syncwarp();
        }
        base_t += __shfl_sync(0xffffffffu, ti, 31);
    }
}

// A tile as the converting warps need it.
struct TileInfo {
    int32_t page[8];  // -1: nothing of it counts
    uint32_t off, h;  // first token within the page, KV head
    uint32_t kind;    // 0 prefix, 1 tail, 2 no more tiles
    uint32_t pad;
};

// What a CTA keeps in shared memory behind the tiles.
template <int D, bool QUANT>
struct Small {
    using C = Cfg<D, QUANT>;
    static constexpr int NS = C::NS;
    alignas(16) uint32_t mask[kMeta][4];  // valid keys of a tile
    float2 ml[NS][128];                   // statistics on their way to the other stream
    uint64_t bars[2 * C::stages + kMeta + 2 * kSegs + (7 + C::NB) * NS + 2 + 4 * C::raws + (QUANT ? kMeta : 0)];
    TileInfo tile[QUANT ? kMeta : 1];
    Plan plan;
    Seg seg[kSegs];
    uint32_t tmem, fail;
};
static_assert(Cfg<128, false>::tiles + sizeof(Small<128, false>) <= 227 * 1024, "shared memory");
static_assert(Cfg<128, true>::tiles + sizeof(Small<128, true>) <= 227 * 1024, "shared memory");
static_assert(Cfg<256, true>::tiles + sizeof(Small<256, true>) <= 227 * 1024, "shared memory");

template <int D, bool QUANT>
__global__ void __launch_bounds__(Cfg<D, QUANT>::threads, 1)
    attn_tc_kernel(const __grid_constant__ AttnLaunch l) {
    using C = Cfg<D, QUANT>;
    constexpr int BN = C::BN, PR = C::PR, NS = C::NS, NB = C::NB, ST = C::stages, RS = C::raws;
    constexpr uint32_t KB = BN * 128, QB = 128 * 128;  // bytes of a 64-column block of K / V, of Q
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    Small<D, QUANT> &sm = *reinterpret_cast<Small<D, QUANT> *>(smem_raw + C::tiles);
    Plan &plan = sm.plan;

    const PrefixAttn &a = l.a;
    const uint32_t warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem_raw);
    if (base & 1023u) {  // the tiles must lie on the swizzle's atoms
        if (threadIdx.x == 0) l.fail[blockIdx.x] = 1;
        return;
    }
    const uint32_t ring = base + NS * C::q_bytes;
    const uint32_t bar0 = smem_u32(sm.bars);
    auto full = [&](uint32_t i) { return bar0 + 8u * i; };
    auto empty = [&](uint32_t i) { return bar0 + 8u * (ST + i); };
    auto meta = [&](uint32_t i) { return bar0 + 8u * (2 * ST + i); };
    auto seg_full = [&](uint32_t i) { return bar0 + 8u * (2 * ST + kMeta + i); };
    auto seg_empty = [&](uint32_t i) { return bar0 + 8u * (2 * ST + kMeta + kSegs + i); };
    constexpr uint32_t SB = 2 * ST + kMeta + 2 * kSegs;
    auto q_ready = [&](uint32_t s) { return bar0 + 8u * (SB + s); };
    // one for each S tile of a stream; P has one for each S tile, or each part of it
    auto s_full = [&](uint32_t s, uint32_t b) { return bar0 + 8u * (SB + NS + NB * s + b); };
    auto p_ready = [&](uint32_t s, uint32_t i) { return bar0 + 8u * (SB + (1 + NB) * NS + 2 * s + i); };
    constexpr uint32_t SP = SB + (3 + NB) * NS;
    auto pv_half = [&](uint32_t s) { return bar0 + 8u * (SP + 3 * NS + s); };
    auto pv_done = [&](uint32_t s) { return bar0 + 8u * (SP + s); };
    auto o_done = [&](uint32_t s) { return bar0 + 8u * (SP + NS + s); };
    auto o_read = [&](uint32_t s) { return bar0 + 8u * (SP + 2 * NS + s); };
    const uint32_t drain = bar0 + 8u * (SP + 4 * NS), planned = drain + 8;
    // raw tiles i of K (v = 0), V
    auto raw_full = [&](uint32_t v, uint32_t i) { return drain + 16 + 8u * (v * RS + i); };
    auto raw_empty = [&](uint32_t v, uint32_t i) { return drain + 16 + 8u * (2 * RS + v * RS + i); };
    auto meta_empty = [&](uint32_t i) { return drain + 16 + 8u * (4 * RS + i); };
    auto raw_tile = [&](uint32_t v, uint32_t i) {
        return base + C::raw0 + (v ? 2 * l.raw_k + i * l.raw_v : i * l.raw_k);
    };
    auto raw_count = [&](uint32_t v) { return v ? l.n_raw_v : 2u; };

    if (threadIdx.x == 0) {
        sm.fail = 0;
        for (int i = 0; i < ST; ++i) {
            mbar_init(full(i), QUANT ? 4 : 1);
            mbar_init(empty(i), NS);  // one arrival per stream
        }
        for (int i = 0; i < kMeta; ++i) mbar_init(meta(i), 1);
        for (int i = 0; i < kSegs; ++i) {
            mbar_init(seg_full(i), 1);
            mbar_init(seg_empty(i), 1 + NS + 4 * NS);  // producer, products, softmax warps
        }
        for (int s = 0; s < NS; ++s) {
            mbar_init(q_ready(s), 4);
            for (int b = 0; b < NB; ++b) mbar_init(s_full(s, b), 1);
            for (int i = 0; i < 2; ++i) mbar_init(p_ready(s, i), 4);
            mbar_init(pv_half(s), 1);
            mbar_init(pv_done(s), 1);
            mbar_init(o_done(s), 4);
            mbar_init(o_read(s), 4);
        }
        mbar_init(drain, 1);
        mbar_init(planned, 1);
        for (int i = 0; i < RS; ++i)
            for (int v = 0; v < 2; ++v) {
                mbar_init(raw_full(v, i), 1);
                mbar_init(raw_empty(v, i), 4);
            }
        if constexpr (QUANT)
            for (int i = 0; i < kMeta; ++i) mbar_init(meta_empty(i), 4);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                         smem_u32(&sm.tmem)),
                     "r"(kAttnTmem)
                     : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = __shfl_sync(0xffffffffu, sm.tmem, 0);
    bool stop = false;
    // a whole warp's wait; false once it has given up (the warps that wait for
    // this one then do too)
    auto wait = [&](uint32_t bar, uint32_t parity) {
        if (!__all_sync(0xffffffffu, mbar_wait_clk(bar, parity))) stop = true;
        return !stop;
    };

    if (warp == 2) {  // ---- the pieces ----
        Start start;
        Plan p;
        if (!make_plan<D, QUANT>(l, p, start)) stop = true;
        if (lane == 0) {
            plan = p;
            mbar_arrive(planned);
        }
        __syncwarp();
        Walk<BN, PR> walk(a, plan, l.by, l.rooms, start.seq, start.tile);
        uint32_t j = 0;
        for (uint32_t i = 0;; ++i) {
            Seg g = {};
            if (!stop && walk.next(g)) {
                g.j0 = j;
                j += g.n;
            }
            // This wait lasts as long as a whole piece, which a very long list makes
            // longer than the limit: it goes on as long as no other warp gave up.
            bool room = i < kSegs;
            for (uint32_t t = 0; !room && t < 64; ++t) {
                room = __all_sync(0xffffffffu, mbar_wait_clk(seg_empty(i % kSegs), (i / kSegs - 1) & 1u));
                if (__any_sync(0xffffffffu, *static_cast<volatile uint32_t *>(&sm.fail))) break;
            }
            if (!room) {
                stop = true;
                break;
            }
            if (lane == 0) {
                sm.seg[i % kSegs] = g;
                mbar_arrive(seg_full(i % kSegs));
            }
            __syncwarp();
            if (g.n == 0) break;
        }
    } else if (warp == 3) {  // ---- the join's notes ----
        if (wait(planned, 0) && plan.ok) note_rows<D, QUANT>(l, plan);
    } else if (warp == 0) {  // ---- producer ----
        if (lane < 4 && (lane < 2 ? a.prefix.max_len != 0 : a.n_seq != 0))
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&l.map[lane]))
                         : "memory");
        uint32_t q = 0, j = 0;  // stages and tiles so far
        uint32_t nr[2] = {0, 0};  // raw tiles of K, V
        // The raw tile of a K (v = 0) or V operand that is in quant blocks.
        auto load_raw = [&](uint32_t kind, uint32_t v, uint32_t h, uint32_t off, int32_t id, bool use) {
            const PageView &pv = (kind ? a.tail : a.prefix).pages;
            const int32_t type = v ? pv.v_type : pv.k_type;
            if (type == KVMRET_TYPE_F16) return;  // the converting warps fetch it
            const uint32_t n = raw_count(v), slot = nr[v] % n, round = nr[v] / n;
            if (round && !wait(raw_empty(v, slot), (round - 1) & 1u)) return;
            ++nr[v];
            const uint32_t T = pv.page_tokens, bx = raw_box<D>(type);
            const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, use)) * min(T, static_cast<uint32_t>(BN)) * bx;
            if (lane == 0) mbar_expect_tx(raw_full(v, slot), bytes);
            __syncwarp();
            const uint32_t row = D / 32 * (type == KVMRET_TYPE_Q8_0 ? 34 : 18);
            if (use)
                tma_load_3d(raw_tile(v, slot) + lane * T * bx, &l.map[2 * kind + v],
                            static_cast<int32_t>(h * row / 16 * 8), static_cast<int32_t>(off), id,
                            raw_full(v, slot));
        };
        uint32_t k_kind = 2, k_h = 0, k_off = 0;  // the tile before
        int32_t k_id = -1;
        bool k_use = false;
        for (uint32_t sg = 0; !stop; ++sg) {
            if (!wait(seg_full(sg % kSegs), (sg / kSegs) & 1u)) break;
            const Seg g = sm.seg[sg % kSegs];
            if (g.n == 0) break;
            __syncwarp();
            if (lane == 0) mbar_arrive(seg_empty(sg % kSegs));
            const KeyList &kl = g.tail ? a.tail : a.prefix;
            const CUtensorMap *mk = &l.map[g.tail ? 2 : 0], *mv = mk + 1;
            const TileGeom<BN> geom(l.by.list[g.tail]);
            const uint32_t T = geom.c.T, box = min(T, static_cast<uint32_t>(BN));
            const uint64_t list = g.tail ? static_cast<uint64_t>(g.seq) * kl.n_list : 0;
            for (uint32_t i = 0; i < g.n && !stop; ++i, ++j) {
                // lane p < ppt: page p of the tile, and how many of its tokens count
                uint32_t page, off;
                geom.locate(g.tile0 + i, page, off);
                int32_t id = -1;
                uint32_t held = 0;
                if (lane < geom.c.ppt && page + lane < kl.n_list) {
                    const uint32_t at = page + lane;
                    id = kl.table ? __ldg(kl.table + list + at) : static_cast<int32_t>(at);
                    if (id >= 0 && static_cast<uint32_t>(id) < kl.pages.n_pages) {
                        held = kl.ntok ? min(__ldg(kl.ntok + at), T) : T;
                        held = min(held, at * T < g.len ? g.len - at * T : 0);
                    }
                }
                const bool use = held > off;
                uint32_t mask = 0;  // lane w keeps word w
#pragma unroll
                for (uint32_t w = 0; w < BN / 32; ++w) {
                    const uint32_t key = 32 * w + lane, pk = T < BN ? key / T : 0;
                    const uint32_t h = __shfl_sync(0xffffffffu, held, pk);
                    const uint32_t o = T < BN ? key - pk * T : off + key;
                    const uint32_t b = __ballot_sync(0xffffffffu, pk < geom.c.ppt && o < h);
                    if (lane == w) mask = b;
                }
                if constexpr (QUANT) {
                    const uint32_t slot = j % kMeta;
                    if (j >= kMeta && !wait(meta_empty(slot), (j / kMeta - 1) & 1u)) break;
                    if (lane < BN / 32) sm.mask[slot][lane] = mask;
                    if (lane < 8) sm.tile[slot].page[lane] = use ? id : -1;
                    if (lane == 0) {
                        sm.tile[slot].off = off;
                        sm.tile[slot].h = g.h;
                        sm.tile[slot].kind = g.tail;
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(meta(slot));
                    load_raw(g.tail, 0, g.h, off, id, use);
                    if (!stop && k_kind < 2) load_raw(k_kind, 1, k_h, k_off, k_id, k_use);
                    k_kind = g.tail;
                    k_h = g.h;
                    k_off = off;
                    k_id = id;
                    k_use = use;
                    continue;
                }
                const uint32_t bytes = __popc(__ballot_sync(0xffffffffu, use)) * box * D * 2;
#pragma unroll
                for (uint32_t v = 0; v < 2; ++v) {  // K, then V
                    const uint32_t st = q % ST, round = q / ST;
                    if (round && !wait(empty(st), (round - 1) & 1u)) break;
                    if (v == 0) {
                        if (lane < BN / 32) sm.mask[j % kMeta][lane] = mask;
                        __syncwarp();
                        if (lane == 0) mbar_arrive(meta(j % kMeta));
                    }
                    if (lane == 0) mbar_expect_tx(full(st), bytes);
                    __syncwarp();
                    ++q;
                    if (use) {
                        const uint32_t dst = ring + st * C::stage + lane * T * 128;
#pragma unroll
                        for (uint32_t b = 0; b < D / 64; ++b)
                            tma_load_4d(dst + b * KB, v ? mv : mk, static_cast<int32_t>(64 * b),
                                        static_cast<int32_t>(g.h), static_cast<int32_t>(off), id,
                                        full(st));
                    }
                }
            }
        }
        if constexpr (QUANT) {
            if (!stop && k_kind < 2) load_raw(k_kind, 1, k_h, k_off, k_id, k_use);
            if (!stop && (j < kMeta || wait(meta_empty(j % kMeta), (j / kMeta - 1) & 1u))) {
                if (lane == 0) {
                    sm.tile[j % kMeta].kind = 2;
                    mbar_arrive(meta(j % kMeta));
                }
            }
        }
        if (stop) {  // gave up: drain the loads already issued (bounded)
            if (lane == 0) atomicExch(&sm.fail, 1u);
            for (uint32_t i = q > ST ? q - ST : 0; i < q; ++i) mbar_wait_clk(full(i % ST), (i / ST) & 1u);
            for (uint32_t v = 0; QUANT && v < 2; ++v)
                for (uint32_t n = raw_count(v), i = nr[v] > n ? nr[v] - n : 0; i < nr[v]; ++i)
                    mbar_wait_clk(raw_full(v, i % n), (i / n) & 1u);
        }
    } else if (warp == 1) {  // ---- products ----
        // Tiles are taken in the CTA's order: the stream whose current tile is
        // first gets its P V product and, once that has read P, its next scores.
        // While it waits for its softmax the other stream's turn comes, so the two
        // stay half a period apart. (Both products of a turn being issued as soon
        // as they could be, in any order, lets the streams fall into step: 2048 rows over
        // 32,768 tokens took a fifth longer.)
        constexpr uint32_t id_s = idesc(BN, false), id_o = idesc(D, true);
        // Upper halves of the descriptors (tc.cuh): 8-row atoms every 1024 bytes, 128-byte
        // swizzle. V is MN-major: rows of 64 dimensions, one a key, and in the leading
        // offset the bytes to the next 64 dimensions.
        constexpr uint32_t kHi = 64u | (1u << 14) | (2u << 29);
        const uint32_t ubase = __shfl_sync(0xffffffffu, base, 0);
        auto desc = [](uint32_t lo) { return static_cast<uint64_t>(kHi) << 32 | lo; };
        Share<NS> sh[2];
        uint32_t sg[2] = {0, 0}, tiles[2] = {0, 0};  // pieces taken up, tiles finished
        bool live[2] = {true, NS == 2}, fresh[2] = {true, true};
        auto open = [&](uint32_t s) {  // the stream's next piece with a tile for it
            for (;;) {
                if (!wait(seg_full(sg[s] % kSegs), (sg[s] / kSegs) & 1u)) return;
                const Seg &g = sm.seg[sg[s] % kSegs];
                const bool end = g.n == 0;
                if (!end) sh[s].set(g, s);
                __syncwarp();
                if (end) {
                    live[s] = false;
                    return;
                }
                if (lane == 0) mbar_arrive(seg_empty(sg[s] % kSegs));
                ++sg[s];
                if (sh[s].any()) break;
            }
            fresh[s] = true;
        };
        uint32_t nq[2] = {0, 0}, cur[2] = {0, 0};
        // a stage is free once each stream has passed it: a tile of one stream
        // alone counts for both
        auto release = [&](uint32_t s, uint32_t st) {
            mma_commit(empty(st));
            if (NS == 2 && !sh[s].both) mma_commit(empty(st));
        };
        // Scores of the stream's current tile, its n-th, into S tile n % NB. With one
        // S tile, `after`: once the product before, which reads the P that S will
        // overwrite, has completed (the last wait, so that the issue follows it).
        auto scores = [&](uint32_t s, uint32_t n, bool after) {
            if (fresh[s] && !wait(q_ready(s), nq[s]++ & 1u)) return;
            const uint32_t st = __shfl_sync(0xffffffffu, C::k_stage(sh[s].tile), 0);
            if (!wait(full(st), C::k_round(sh[s].tile) & 1u)) return;
            if (after && !wait(pv_done(s), (n - 1) & 1u)) return;
            tc_fence_after();
            if (elect_one()) {
                const uint32_t la = ((ubase + s * C::q_bytes) >> 4) | (1u << 16);
                const uint32_t lb = ((ubase + NS * C::q_bytes + st * C::stage) >> 4) | (1u << 16);
                const uint32_t to = tmem + C::s_col(s) + n % NB * BN;
#pragma unroll
                for (uint32_t c = 0; c < D / 16; ++c)  // 16 columns: 32 bytes of a block
                    mma_ss(to, desc(la + (c / 4) * (QB / 16) + 2 * (c % 4)),
                           desc(lb + (c / 4) * (KB / 16) + 2 * (c % 4)), id_s, c != 0);
                mma_commit(s_full(s, n % NB));
                release(s, st);
            }
            __syncwarp();
        };
#pragma unroll
        for (uint32_t s = 0; s < NS; ++s) {
            if (!stop) open(s);
            if (!stop && live[s]) scores(s, 0, false);
            cur[s] = sh[s].tile;
        }
        auto turn = [&](uint32_t s) {
            const uint32_t n = tiles[s]++, st = __shfl_sync(0xffffffffu, C::v_stage(cur[s]), 0);
            const uint32_t add = !fresh[s];
            const bool both = sh[s].both;
            fresh[s] = false;
            sh[s].tile += sh[s].step;
            const bool same = sh[s].any();
            // with two S tiles the next scores come first, if their K is there (a new
            // piece's Q comes only after this tile's P)
            bool ahead = false;
            if (NB == 2) {
                if (same) {
                    const uint32_t t = sh[s].tile;
                    ahead = __all_sync(0xffffffffu, mbar_try(full(C::k_stage(t)), C::k_round(t) & 1u));
                    if (ahead) scores(s, n + 1, false);
                }
            }
            if (stop || !wait(full(st), C::v_round(cur[s]) & 1u)) return;
#pragma unroll
            for (uint32_t h = 0; h < C::parts; ++h) {
                const bool got = NS == 2 ? wait(p_ready(s, h), n & 1u) : wait(p_ready(s, n & 1u), (n >> 1) & 1u);
                if (!got) return;
                tc_fence_after();
                if (elect_one()) {
                    const uint32_t lb = ((ubase + NS * C::q_bytes + st * C::stage) >> 4) | (KB / 16) << 16;
                    const uint32_t p = tmem + C::p_col(s, n % NB);
#pragma unroll
                    for (uint32_t i = 0; i < BN / 16 / C::parts; ++i) {  // 16 keys: 8 columns of P, 2 KiB of V
                        const uint32_t c = h * (BN / 16 / C::parts) + i;
                        mma_ts(tmem + C::o_col(s), p + 8 * c, desc(lb + 128 * c), id_o, c ? 1u : add);
                    }
                    if (h + 1 < C::parts) {
                        mma_commit(pv_half(s));
                    } else {
                        mma_commit(empty(st));
                        if (NS == 2 && !both) mma_commit(empty(st));
                        mma_commit(pv_done(s));
                    }
                }
                __syncwarp();
            }
            if (!same) open(s);
            if (!stop && live[s] && !ahead) scores(s, n + 1, NB == 1);
            cur[s] = sh[s].tile;
        };
        uint32_t last = 1;
        while (!stop && (live[0] || (NS == 2 && live[1]))) {
            const bool one = NS == 2 && live[1] &&
                             (!live[0] || cur[1] < cur[0] || (cur[1] == cur[0] && last == 0));
            last = one;
            if (NS == 2 && one)
                turn(1);
            else
                turn(0);
        }
        // on the regular path the softmax waits for the last products; here the
        // issuer does, before the memory they use is given back
        if (stop) {
            if (lane == 0) {
                atomicExch(&sm.fail, 1u);
                mma_commit(drain);
            }
            __syncwarp();
            mbar_wait(drain, 0);
        }
    } else if (QUANT && warp >= 4 + 4 * NS) {  // ---- conversion of quant blocks ----
        // The first four of these warps have K, the others V. A thread a key's row
        // (head size 256: half of it): blocks from the raw tile to f16(d * q) in the
        // stage's swizzled layout. Whole numbers become halves by their bits
        // (0x6400 + u is 1024 + u), one subtraction and one product by d, rounded
        // once to the tensor cores' type: outputs are 2.9e-4 to 6e-4 off in the mean
        // instead of the 2.9e-4 of f16 pages (most of which P's and the output's own
        // rounding make). d * q whole would take two f16 tiles each for K and V, twice
        // the products, and leave them one stage each. Operands in f16 go to their
        // stage by TMA, issued by the first warp. Each of the four warps waits for the
        // stage and arrives on it, whatever the tile's type: so none can fall a phase
        // of `empty` behind or get one ahead (its parity would then name another
        // phase), and none still reads a tile's entry when that is written anew.
        const uint32_t tid = threadIdx.x & 127, wq = (warp - 4 - 4 * NS) & 3, v = (warp - 4 - 4 * NS) >> 2;
        const uint32_t key = tid % BN, half = tid / BN;  // half: 0 unless the head size is 256
        uint32_t nr = 0;                                 // raw tiles so far
        uint32_t flight = 0;                             // the tile after the last f16 load
        auto unit = [&](uint32_t j) {
            const TileInfo &ti = sm.tile[j % kMeta];
            const PageView &pv = (ti.kind ? a.tail : a.prefix).pages;
            const int32_t type = v ? pv.v_type : pv.k_type;
            const uint32_t st = v ? C::v_stage(j) : C::k_stage(j), round = v ? C::v_round(j) : C::k_round(j);
            if (round && !wait(empty(st), (round - 1) & 1u)) return;
            const uint32_t stage = ring + st * C::stage;
            if (type == KVMRET_TYPE_F16) {
                if (wq != 0) {
                    __syncwarp();  // every lane has read the tile's entry
                    if (lane == 0) mbar_arrive(full(st));
                    return;
                }
                const uint32_t T = pv.page_tokens, box = min(T, static_cast<uint32_t>(BN));
                const int32_t id = lane < 8 ? ti.page[lane] : -1;
                const int32_t h = static_cast<int32_t>(ti.h), off = static_cast<int32_t>(ti.off);
                const CUtensorMap *const map = &l.map[2 * ti.kind + v];
                const uint32_t n = __popc(__ballot_sync(0xffffffffu, id >= 0));
                if (lane == 0) mbar_expect_tx(full(st), n * box * D * 2);
                __syncwarp();
                if (id >= 0)
#pragma unroll
                    for (uint32_t b = 0; b < D / 64; ++b)
                        tma_load_4d(stage + b * KB + lane * T * 128, map, static_cast<int32_t>(64 * b), h, off,
                                    id, full(st));
                flight = j + 1;
                return;
            }
            const uint32_t n_raw = raw_count(v), slot = nr % n_raw;
            if (!wait(raw_full(v, slot), (nr / n_raw) & 1u)) return;
            ++nr;
            const bool q8 = type == KVMRET_TYPE_Q8_0;
            const uint32_t block = q8 ? 34 : 18, row = D / 32 * block;
            const uint32_t src = raw_tile(v, slot) + key * raw_box<D>(type) +
                                 (ti.h * row) % 16 + half * 4 * block;
            constexpr uint32_t blocks = D < 128 ? D / 32 : 4;
            const uint32_t dst = stage + key * 128;
            auto put = [&](uint32_t chunk, const uint32_t(&x)[4]) {  // 8 columns
                const uint32_t ch = half * 16 + chunk;
                const uint32_t at = dst + (ch / 8) * KB + (((ch % 8) ^ (key % 8)) * 16);
                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at), "r"(x[0]), "r"(x[1]),
                             "r"(x[2]), "r"(x[3])
                             : "memory");
            };
            if (q8)
                convert_row<blocks, KVMRET_TYPE_Q8_0>(src, key / 8, put);
            else
                convert_row<blocks, KVMRET_TYPE_Q4_0>(src, key / 8, put);
            fence_async_smem();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(full(st));
                mbar_arrive(raw_empty(v, slot));
            }
        };
        for (uint32_t j = 0;; ++j) {
            if (!wait(meta(j % kMeta), (j / kMeta) & 1u) || sm.tile[j % kMeta].kind == 2) break;
            unit(j);
            if (stop) break;
            // K of tile j in its stage: P V of tile j - 8 is past, its mask read
            if (v == 0 && j >= 8 && lane == 0) mbar_arrive(meta_empty((j - 8) % kMeta));
            __syncwarp();
        }
        if (stop) {
            if (lane == 0) atomicExch(&sm.fail, 1u);
            if (wq == 0)  // the f16 loads under way
                for (uint32_t t = flight > 4 ? flight - 4 : 0; t < flight; ++t)
                    mbar_wait_clk(full(v ? C::v_stage(t) : C::k_stage(t)),
                                  (v ? C::v_round(t) : C::k_round(t)) & 1u);
        }
    } else if (warp >= 4) {  // ---- softmax, a thread a row ----
        const uint32_t s = (warp - 4) >> 2, qd = warp & 3, r = 32 * qd + lane;
        const uint32_t tid = threadIdx.x & 127;
        const uint32_t G = l.by.G.d;
        // (above zero, so that -inf stays -inf; a scale of zero gives equal scores all the same)
        const float c = fmaxf(fabsf(a.scale) * 1.44269504f, 1e-37f);
        const uint32_t sign = a.scale < 0.0f ? 0x80008000u : 0u;  // a negative scale turns Q
        const uint32_t ts0 = tmem + ((32 * qd) << 16) + C::s_col(s);
        const uint32_t to = tmem + ((32 * qd) << 16) + C::o_col(s);
        constexpr uint32_t kRows = 128 / (D / 8);  // rows that one pass of the Q load covers
        const uint32_t step_t = l.by.G(kRows), step_h = kRows - step_t * G;
        uint32_t ns = 0, sg = 0;  // tiles and pieces so far
        uint32_t joins = 0;       // outputs joined with the other stream's
        bool owed = false;        // it may still be reading this one's
        Seg g = {};
        Share<NS> sh = {};
        auto row_first = [&] { return sh.both ? 128 * s : 0u; };  // of the unit's rows
        auto row_count = [&] { return min(128u, g.rows - row_first()); };
        // the stream's next piece: Q in the swizzled layout, rows past the last zeros
        auto open = [&] {
            for (;;) {
                if (!wait(seg_full(sg % kSegs), (sg / kSegs) & 1u)) return false;
                g = sm.seg[sg % kSegs];
                if (g.n == 0) return false;
                __syncwarp();
                if (lane == 0) mbar_arrive(seg_empty(sg % kSegs));
                ++sg;
                sh.set(g, s);
                if (sh.any()) break;  // else the other stream has the piece's only tile
            }
            const uint32_t rows = row_count(), at0 = g.row0 + row_first();
            constexpr uint32_t CH = D / 8, RS = 128 / CH;  // 16-byte chunks of a row; rows a pass
            const uint32_t ch = tid % CH, q1 = tid / CH;
            const uint16_t *const q = a.q + static_cast<uint64_t>(g.q0) * a.q_stride +
                                      static_cast<uint64_t>(g.h) * G * D + 8 * ch;
            uint32_t t = l.by.G(at0 + q1), hg = at0 + q1 - t * G;
            // n passes: all loads first. Only warps that hold a row look at their
            // scores, so rows past the last one of 32 stay as they are.
            auto load = [&](uint32_t i0, auto n) {
                constexpr uint32_t N = decltype(n)::value;
                uint4 w[N];
#pragma unroll
                for (uint32_t i = 0; i < N; ++i) {
                    w[i] = make_uint4(0, 0, 0, 0);
                    if (q1 + (i0 + i) * RS < rows)
                        w[i] = __ldg(reinterpret_cast<const uint4 *>(
                            q + static_cast<uint64_t>(t) * a.q_stride + hg * D));
                    t += step_t;
                    hg += step_h;
                    if (hg >= G) {
                        hg -= G;
                        ++t;
                    }
                }
#pragma unroll
                for (uint32_t i = 0; i < N; ++i) {
                    const uint32_t qr = q1 + (i0 + i) * RS;
                    const uint32_t at = base + s * C::q_bytes + (ch / 8) * QB + qr * 128 +
                                        (((ch % 8) ^ (qr % 8)) * 16);
                    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(at),
                                 "r"(w[i].x ^ sign), "r"(w[i].y ^ sign), "r"(w[i].z ^ sign),
                                 "r"(w[i].w ^ sign)
                                 : "memory");
                }
            };
            if (rows <= 32) {
                load(0, std::integral_constant<uint32_t, 32 / RS>());
            } else {
                constexpr uint32_t QL = CH < 16 ? CH : 16;  // loads in flight
#pragma unroll
                for (uint32_t i0 = 0; i0 < CH; i0 += QL) load(i0, std::integral_constant<uint32_t, QL>());
            }
            fence_async_smem();
            __syncwarp();
            if (lane == 0) mbar_arrive(q_ready(s));
            return true;
        };
        bool more = open();
        while (more) {
            const uint32_t rows = row_count();
            // two streams over the same rows: their outputs are joined here, half of
            // the columns by each
            const bool two = NS == 2 && !sh.both && g.n > 1;
            const uint32_t id = g.room + row_first() + r;  // the row in the workspace
            const bool idle = 32 * qd >= rows;  // no row of this warp: P may be anything
            // how far the row sees into the list
            uint32_t seen = 0xffffffffu;
            if (g.tail) seen = tail_seen(g.len, g.q_len, l.by.G(g.row0 + row_first() + min(r, rows - 1)));
            const uint32_t tile0 = g.tile0 - g.j0;
            float m = -INFINITY, sum = 0.0f;  // of c q . k
            for (bool begin = true; sh.any(); sh.tile += sh.step, begin = false) {
                const uint32_t jj = sh.tile, n = ns++, ts = ts0 + n % NB * BN;  // its n-th tile
                // what the tile's mask says, while the scores are on their way (behind
                // their wait this takes 4 to 8 % of a long call)
                if (!wait(meta(jj % kMeta), (jj / kMeta) & 1u)) break;
                const uint4 mw = *reinterpret_cast<const uint4 *>(sm.mask[jj % kMeta]);
                const bool whole = (mw.x & mw.y & (BN == 128 ? mw.z & mw.w : 0xffffffffu)) == 0xffffffffu;
                // a tile's first token is at most tile * BN: all of it seen?
                const bool clear = whole && __all_sync(0xffffffffu, (tile0 + jj + 1) * BN <= seen);
                // a new piece's output begins with this tile's product: the other
                // stream must have read the last one
                if (begin && owed) {
                    if (!wait(o_read(1 - s), (joins - 1) & 1u)) break;
                    owed = false;
                }
                if (!wait(s_full(s, n % NB), (n / NB) & 1u)) break;
                tc_fence_after();
                // With two S tiles these scores did not wait for the product before: its
                // end, without which O may still change and the phases of pv_done and of
                // the V stage may be one further back than their parities tell.
                auto past = [&] { return NB == 1 || n == 0 || wait(pv_done(s), (n - 1) & 1u); };
                uint32_t x[32];
                if (!clear) {
                    // the S columns of keys that do not count become -inf, the V rows of
                    // cells without a token zeros
                    if (!whole) {
                        const uint32_t st = C::v_stage(jj);
                        if (!past() || !wait(full(st), C::v_round(jj) & 1u)) break;
                        for (uint32_t i = tid; i < BN * 8; i += 128) {  // a lane 16 bytes
                            const uint32_t key = i / 8;
                            if (sm.mask[jj % kMeta][key / 32] >> (key % 32) & 1u) continue;
                            const uint32_t at = ring + st * C::stage + i * 16;
#pragma unroll
                            for (uint32_t z = 0; z < D / 64; ++z)
                                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(at + z * KB),
                                             "r"(0u)
                                             : "memory");
                        }
                        fence_async_smem();
                    }
                    const TileGeom<BN> geom(l.by.list[g.tail]);
                    uint32_t page, off;
                    geom.locate(tile0 + jj, page, off);
                    const uint32_t pos0 = page * geom.c.T + off;
                    const uint32_t lim = seen > pos0 ? min(seen - pos0, static_cast<uint32_t>(BN)) : 0;
#pragma unroll 1
                    for (uint32_t w = 0; w < BN / 32 && !idle; ++w) {
                        const uint32_t left = lim > 32 * w ? lim - 32 * w : 0;
                        const uint32_t mask = sm.mask[jj % kMeta][w] &
                                              (left >= 32 ? 0xffffffffu : (1u << left) - 1);
                        tmem_ld32_nowait(ts + 32 * w, x);
                        tmem_ld_wait(x);
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            if (!(mask >> k & 1u)) x[k] = 0xff800000u;
                        tmem_st32(ts + 32 * w, x);
                    }
                    tmem_st_wait();
                }
                // One pass with the maximum as it stands: p and the keys' own maximum
                // together, 32 columns at a time with the next ones on their way (a
                // piece's first tile starts with that of its first columns). Only when a
                // row's maximum has moved by more than 8 the pass is repeated with the
                // new one; S still stands. Two streams hand the halves of P on one by
                // one, so that the first half's product runs during the second half's
                // softmax (2048 rows over 32,768 tokens took 4 % longer in one piece, 16 rows 7 %).
                constexpr int KEYS = BN / C::parts, STEP = KEYS < 64 ? KEYS : 64;
#pragma unroll 1
                for (uint32_t h = 0; h < C::parts && !idle; ++h) {
                    uint32_t y[32], pk[STEP / 2];
                    const uint32_t tp = tmem + ((32 * qd) << 16) + C::p_col(s, n % NB) + h * (KEYS / 2);
                    const uint32_t tk = ts + h * KEYS;
                    float top = -INFINITY, s0, s1;
                    auto column_max = [&](const uint32_t *v) {
#pragma unroll
                        for (int k = 0; k < 32; k += 2)
                            top = fmaxf(top, fmaxf(__uint_as_float(v[k]), __uint_as_float(v[k + 1])));
                    };
                    auto pass = [&](bool first) {
                        float neg = m == -INFINITY ? 0.0f : -m;
                        s0 = s1 = 0.0f;
                        top = -INFINITY;
                        tmem_ld32_nowait(tk, x);
#pragma unroll 1
                        for (int w0 = 0; w0 < KEYS / 32; w0 += STEP / 32) {
#pragma unroll
                            for (int w = 0; w < STEP / 32; ++w) {
                                uint32_t *const v = w & 1 ? y : x;
                                tmem_ld_wait(v);
                                if (w + 1 < STEP / 32 || w0 + w + 1 < KEYS / 32)
                                    tmem_ld32_nowait(tk + 32 * (w0 + w + 1), w & 1 ? x : y);
                                column_max(v);
                                if (w == 0 && w0 == 0 && first) {
                                    m = top * c;
                                    neg = m == -INFINITY ? 0.0f : -m;
                                }
#pragma unroll
                                for (int k = 0; k < 16; ++k) {
                                    uint32_t e0 = v[2 * k], e1 = v[2 * k + 1];
                                    fma_pair(e0, e1, c, neg);
                                    const float p0 = ex2(__uint_as_float(e0)), p1 = ex2(__uint_as_float(e1));
                                    add_pair(s0, s1, p0, p1);
                                    pk[16 * w + k] = pack_h2(p0, p1);
                                }
                            }
                            if (NS == 1) tmem_st32(tp + 16 * w0, *reinterpret_cast<const uint32_t(*)[32]>(pk));
                        }
                    };
                    bool first = begin && h == 0;
#pragma unroll 1
                    for (;;) {
                        pass(first);
                        first = false;
                        if (!__any_sync(0xffffffffu, top * c > m + 8.0f)) break;
                        // (a row's own maximum decides: what it gets depends on no other row)
                        const float mn = top * c > m + 8.0f ? top * c : m;
                        const float f = m == -INFINITY ? 0.0f : ex2(m - mn);
                        m = mn;
                        sum *= f;
                        if (h == 0 ? begin : !wait(pv_half(s), n & 1u)) {
                            if (stop) break;
                            continue;
                        }
                        if (h == 0 && !past()) break;
                        tc_fence_after();
#pragma unroll 1
                        for (uint32_t col = 0; col < D; col += 16) {
                            uint32_t o[16];
                            tmem_ld16(to + col, o);
#pragma unroll
                            for (int k = 0; k < 16; ++k) o[k] = __float_as_uint(__uint_as_float(o[k]) * f);
                            tmem_st16(to + col, o);
                        }
                    }
                    if (stop) break;
                    sum += s0 + s1;
                    if (NS == 2) tmem_st32(tp, *reinterpret_cast<const uint32_t(*)[32]>(pk));
                    tmem_st_wait();
                    if (h + 1 < C::parts) {
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive(p_ready(s, h));
                    }
                }
                if (stop) break;
                if (idle && C::parts == 2 && lane == 0) mbar_arrive(p_ready(s, 0));
                // (at the piece's last tile, whose product is waited for below)
                if (sh.tile + sh.step >= sh.end && !past()) break;
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(p_ready(s, NS == 2 ? 1 : n & 1u));
            }
            if (stop) break;
            // the last scores are in: Q may be replaced while the last product runs
            more = open();
            if (!wait(pv_done(s), (ns - 1) & 1u)) break;
            tc_fence_after();
            float f0 = 1.0f, f1 = 0.0f;  // weights of this stream's and the other's output
            if (two) {
                sm.ml[s][r] = make_float2(m, sum);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(o_done(s));
                if (!wait(o_done(1 - s), joins & 1u)) break;
                tc_fence_after();
                const float2 other = sm.ml[1 - s][r];
                const float top = fmaxf(m, other.x);
                f0 = m == -INFINITY ? 0.0f : ex2(m - top);
                f1 = other.x == -INFINITY ? 0.0f : ex2(other.x - top);
                m = top;
                sum = f0 * sum + f1 * other.y;
            }
            if (!idle) {
                if (r < rows && (s == 0 || !two)) l.ml[id] = make_float2(m, sum);
                const uint32_t tx = tmem + ((32 * qd) << 16) + C::o_col(NS - 1 - s);
                const uint32_t c0 = two ? s * (D / 2) : 0, c1 = two ? c0 + D / 2 : D;
#pragma unroll 1
                for (uint32_t col = c0; col < c1; col += 32) {
                    uint32_t o[32];
                    tmem_ld32_nowait(to + col, o);
                    tmem_ld_wait(o);
                    if (two) {
                        uint32_t e[32];
                        tmem_ld32_nowait(tx + col, e);
                        tmem_ld_wait(e);
#pragma unroll
                        for (int k = 0; k < 32; ++k)
                            o[k] = __float_as_uint(f0 * __uint_as_float(o[k]) + f1 * __uint_as_float(e[k]));
                    }
                    if (r < rows) {
#pragma unroll
                        for (uint32_t k = 0; k < 8; ++k)
                            l.o[out_at<D>(id, col / 4 + k)] =
                                make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]),
                                            __uint_as_float(o[4 * k + 2]), __uint_as_float(o[4 * k + 3]));
                    }
                }
            }
            if (two) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(o_read(s));
                ++joins;
                owed = true;
            }
            tc_fence_before();
        }
    }
    if (stop && lane == 0) atomicExch(&sm.fail, 1u);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (threadIdx.x == 0) l.fail[blockIdx.x] = sm.fail;
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem),
                     "r"(kAttnTmem)
                     : "memory");
    }
}

// The join: a row's pieces of the prefix and of its tail, weighted by
// 2^(m_piece - m), in a fixed order. 8 rows a CTA (neighbouring heads of a
// token), a thread per row and four dimensions: reads of 128 bytes (8 rows of
// one float4 column), 16 pieces at a time. What bounds it is three dependent
// reads (where the pieces lie, their statistics, the pieces).
constexpr uint32_t kJoinRows = 8, kMaxCtas = 160;

template <int D>
__global__ void __launch_bounds__(kJoinRows *D / 4)
    attn_join_kernel(const __grid_constant__ AttnLaunch l, uint32_t n_cta) {
    constexpr uint32_t NT = kJoinRows * D / 4, kList = 2 * kMaxCtas;  // a piece per CTA and line at most
    __shared__ uint32_t s_id[kJoinRows][kList];
    __shared__ float s_w[kJoinRows][kList];
    __shared__ uint32_t s_n[kJoinRows];
    __shared__ float s_inv[kJoinRows];
    const PrefixAttn &a = l.a;
    const uint32_t tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const uint32_t row0 = blockIdx.x * kJoinRows, n_rows = a.n_q * a.n_head;
    // the rows of a sequence
    uint32_t begin = 0, end = n_rows;
    if (a.n_seq) {
        const int32_t n = static_cast<int32_t>(a.n_q);
        begin = static_cast<uint32_t>(min(max(__ldg(a.q_start), 0), n)) * a.n_head;
        end = static_cast<uint32_t>(min(max(__ldg(a.q_start + a.n_seq), 0), n)) * a.n_head;
    }
    cudaGridDependencySynchronize();
    uint32_t bad = 0;
    for (uint32_t i = tid; i < n_cta; i += NT) bad |= l.fail[i];
    bad = __syncthreads_or(bad);
    if (bad) {  // every row of the batch NaN
        for (uint32_t i = tid; i < kJoinRows * D; i += NT)
            if (row0 + i / D >= begin && row0 + i / D < end)
                a.out[static_cast<uint64_t>(row0) * D + i] = 0x7fff;
        if (a.lse && tid < kJoinRows && row0 + tid >= begin && row0 + tid < end) a.lse[row0 + tid] = NAN;
        return;
    }
    // a warp lists a row's pieces and weighs them
    for (uint32_t w = warp; w < kJoinRows; w += NT / 32) {
        const uint32_t row = row0 + w;
        if (row < begin || row >= end) continue;
        const RowPieces e0 = l.at[2 * static_cast<uint64_t>(row)], e1 = l.at[2 * static_cast<uint64_t>(row) + 1];
        const uint32_t n_all = e0.n + e1.n;
        uint32_t n = 0;
        float top = -INFINITY, sum = 0.0f;
        for (uint32_t i0 = 0; i0 < n_all; i0 += 32) {
            const uint32_t i = i0 + lane;
            const uint32_t id = i < e0.n ? e0.at(i) : e1.at(i - e0.n);
            const float2 ml = i < n_all ? l.ml[id] : make_float2(-INFINITY, 0.0f);
            // a piece without keys has a sum of zero; one whose scores are all NaN has
            // no maximum either, but a NaN sum
            const bool held = ml.x != -INFINITY || ml.y != 0.0f;
            const uint32_t have = __ballot_sync(0xffffffffu, held);
            float mt = ml.x;
            for (int o = 16; o; o >>= 1) mt = fmaxf(mt, __shfl_xor_sync(0xffffffffu, mt, o));
            mt = fmaxf(mt, top);
            // the weights so far, and this lane's, against the new maximum
            const float f = top == -INFINITY ? 0.0f : ex2(top - mt);
            for (uint32_t j = lane; j < n; j += 32) s_w[w][j] *= f;
            sum *= f;
            top = mt;
            if (held) {
                const uint32_t at = n + __popc(have & ((1u << lane) - 1));
                const float e = ex2(ml.x - top);
                s_id[w][at] = id;
                s_w[w][at] = e;
                sum += e * ml.y;
            }
            n += __popc(have);
            __syncwarp();
        }
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) {
            s_n[w] = n;
            s_inv[w] = n ? 1.0f / sum : 0.0f;
            if (a.lse) a.lse[row] = n ? (top + log2f(sum)) * 0.693147181f : -INFINITY;
        }
    }
    __syncthreads();
    const uint32_t r = tid % kJoinRows, col = tid / kJoinRows;
    if (row0 + r < begin || row0 + r >= end) return;
    float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    const uint32_t n = s_n[r];
    for (uint32_t i0 = 0; i0 < n; i0 += 16) {
        float4 o[16];
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) {
            o[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (i0 + i < n) {
                o[i] = l.o[out_at<D>(s_id[r][i0 + i], col)];
            }
        }
#pragma unroll
        for (uint32_t i = 0; i < 16; ++i) {
            const float f = i0 + i < n ? s_w[r][i0 + i] : 0.0f;
            acc.x = __fmaf_rn(f, o[i].x, acc.x);
            acc.y = __fmaf_rn(f, o[i].y, acc.y);
            acc.z = __fmaf_rn(f, o[i].z, acc.z);
            acc.w = __fmaf_rn(f, o[i].w, acc.w);
        }
    }
    const float inv = s_inv[r];
    *reinterpret_cast<uint2 *>(a.out + static_cast<uint64_t>(row0 + r) * D + 4 * col) =
        make_uint2(pack_h2(acc.x * inv, acc.y * inv), pack_h2(acc.z * inv, acc.w * inv));
}

// Tensor map of a page list's K or V rows. f16: 4-D {D, heads, tokens, pages},
// box {64, 1, tokens of a tile, 1}, 128-byte swizzle. Quant blocks: 3-D
// {row bytes / 2, tokens, pages}, box {raw_box / 2, tokens of a tile, 1}.
template <int D>
cudaError_t encode_pages(CUtensorMap *map, const uint8_t *at, uint64_t row, uint64_t page, int32_t type,
                         const PageView &v) {
    const EncodeTiledFn fn = encode_fn();
    if (!fn) return cudaErrorNotSupported;
    const bool f16 = type == KVMRET_TYPE_F16;
    const cuuint32_t tok = std::min<uint32_t>(v.page_tokens, Cfg<D, false>::BN);
    const cuuint64_t dims[4] = {f16 ? D : row / 2, f16 ? v.n_head_kv : v.page_tokens,
                                f16 ? v.page_tokens : v.n_pages, v.n_pages};
    const cuuint64_t strides[3] = {f16 ? D * 2ull : row, f16 ? row : page, page};
    const cuuint32_t box[4] = {f16 ? 64 : raw_box<D>(type) / 2, f16 ? 1 : tok, f16 ? tok : 1, 1};
    const cuuint32_t estr[4] = {1, 1, 1, 1};
    const CUresult r = fn(map, f16 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT16,
                          f16 ? 4 : 3, const_cast<uint8_t *>(at), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE,
                          f16 ? CU_TENSOR_MAP_SWIZZLE_128B : CU_TENSOR_MAP_SWIZZLE_NONE,
                          CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    return r == CUDA_SUCCESS ? cudaSuccess : cudaErrorInvalidValue;
}

// CTAs of a launch: the current device's SMs, asked for once a device.
uint32_t attn_ctas() {
    static std::atomic<uint32_t> known[64];
    int dev = 0, sm = 0;
    const bool one = cudaGetDevice(&dev) == cudaSuccess && dev >= 0 && dev < 64;
    uint32_t n = one ? known[dev].load(std::memory_order_relaxed) : 0;
    if (n) return n;
    if (cudaDeviceGetAttribute(&sm, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sm <= 0) sm = 148;
    n = std::min<uint32_t>(static_cast<uint32_t>(sm), kMaxCtas);
    if (one) known[dev].store(n, std::memory_order_relaxed);
    return n;
}

uint64_t up256(uint64_t v) { return (v + 255) / 256 * 256; }

// The workspace: one word per CTA, the rows' notes, the pieces' rows (Rooms).
struct WsLayout {
    uint64_t at, ml, o, bytes, rows;
    Rooms rooms[2];  // units of 128 rows; of 256 (f16 pages, heads of 64 and 128)
    WsLayout(uint32_t n_q, uint32_t n_head, uint32_t n_head_kv, uint32_t d, uint32_t n_seq) {
        const uint64_t mine = static_cast<uint64_t>(n_q) * (n_head / n_head_kv);
        const uint64_t own = n_seq ? (mine * n_head_kv + 7) / 8 * 8 : 0;
        rows = 0;  // of whichever units take more
        for (uint64_t pr = 128; pr <= (d == 256 ? 128u : 256u); pr *= 2) {
            // the prefix has n_pg * gs <= pairs + n_pg units a KV head, and each CTA a
            // range that may begin in a unit's middle
            const uint64_t pairs = (mine + pr - 1) / pr, cap = std::min<uint64_t>(pr, (mine + 7) / 8 * 8);
            const uint64_t n_pre = (pairs + (pairs + 7) / 8) * n_head_kv + kMaxCtas;
            Rooms &r = rooms[pr / 256];
            r.cap = static_cast<uint32_t>(cap);
            r.n_pre = static_cast<uint32_t>(n_pre);
            r.tail = static_cast<uint32_t>(n_pre * cap);
            r.over = static_cast<uint32_t>(n_pre * cap + own);
            rows = std::max(rows, n_pre * cap + own + (n_seq ? kMaxCtas * cap : 0));
        }
        at = up256(kMaxCtas * 4);
        ml = at + up256(2ull * n_q * n_head * sizeof(RowPieces));
        o = ml + up256(rows * 8);
        bytes = o + rows * d * 4;
    }
};

template <int D, bool QUANT>
cudaError_t launch_main(const AttnLaunch &l, uint32_t n_cta, cudaStream_t st) {
    const size_t smem = Cfg<D, QUANT>::tiles + sizeof(Small<D, QUANT>);
    // (at every launch: a context made after a device reset does not know it)
    const cudaError_t e = cudaFuncSetAttribute(
        attn_tc_kernel<D, QUANT>, cudaFuncAttributeMaxDynamicSharedMemorySize, static_cast<int>(smem));
    if (e != cudaSuccess) return e;
    attn_tc_kernel<D, QUANT><<<n_cta, Cfg<D, QUANT>::threads, smem, st>>>(l);
    return cudaGetLastError();
}

template <int D>
cudaError_t launch_t(AttnLaunch &l, const WsLayout &w, cudaStream_t st) {
    const uint32_t n_cta = attn_ctas();
    const KeyList *lists[2] = {&l.a.prefix, &l.a.tail};
    bool quant = false;
    cudaError_t e = cudaSuccess;
    for (int i = 0; i < 2; ++i) {
        const PageView &v = lists[i]->pages;
        if (!lists[i]->max_len) continue;
        quant = quant || v.k_type != KVMRET_TYPE_F16 || v.v_type != KVMRET_TYPE_F16;
        e = encode_pages<D>(&l.map[2 * i], v.k, v.k_row, v.k_page, v.k_type, v);
        if (e == cudaSuccess)
            e = encode_pages<D>(&l.map[2 * i + 1], v.v, v.v_row, v.v_page, v.v_type, v);
        if (e != cudaSuccess) return e;
    }
    l.by.G.set(l.a.n_head / l.a.n_head_kv);
    l.by.H.set(l.a.n_head_kv);
    l.by.ctas.set(n_cta);
    for (int i = 0; i < 2; ++i)
        l.by.list[i].set(lists[i]->max_len ? lists[i]->pages.page_tokens : Cfg<D, false>::BN, Cfg<D, false>::BN);
    l.rooms = w.rooms[quant || D == 256 ? 0 : 1];
    if (quant) {
        int32_t worst[2] = {KVMRET_TYPE_Q4_0, KVMRET_TYPE_Q4_0};
        for (const KeyList *kl : lists)
            for (int v = 0; v < 2; ++v)
                if (kl->max_len && (v ? kl->pages.v_type : kl->pages.k_type) == KVMRET_TYPE_Q8_0)
                    worst[v] = KVMRET_TYPE_Q8_0;
        l.raw_k = Cfg<D, true>::BN * raw_box<D>(worst[0]);
        l.raw_v = Cfg<D, true>::BN * raw_box<D>(worst[1]);
        l.n_raw_v = std::min<uint32_t>(2, (Cfg<D, true>::raw_bytes - 2 * l.raw_k) / l.raw_v);
    }
    e = quant ? launch_main<D, true>(l, n_cta, st) : launch_main<D, false>(l, n_cta, st);
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

cudaError_t launch_prefix_attn(const PrefixAttn &a, void *ws, cudaStream_t st) {
    const WsLayout w(a.n_q, a.n_head, a.n_head_kv, a.d_head, a.n_seq);
    uint8_t *b = static_cast<uint8_t *>(ws);
    AttnLaunch l{};
    l.a = a;
    l.fail = reinterpret_cast<uint32_t *>(b);
    l.at = reinterpret_cast<RowPieces *>(b + w.at);
    l.ml = reinterpret_cast<float2 *>(b + w.ml);
    l.o = reinterpret_cast<float4 *>(b + w.o);
    if (a.d_head == 64) return launch_t<64>(l, w, st);
    if (a.d_head == 128) return launch_t<128>(l, w, st);
    return launch_t<256>(l, w, st);
}

}  // namespace kvmret
