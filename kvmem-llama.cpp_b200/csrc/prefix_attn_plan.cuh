// Work split of the shared-prefix attention, computed on the device from the
// lengths.
//
// Rows: the G = n_head / n_head_kv query heads of a KV head stand as rows
// r = token * G + head beside one another, so one tile of keys serves all of
// them. A unit is (KV head, up to PR rows) against one key list; its keys go by
// tiles of BN. The units' tiles, laid end to end, are cut into equal
// contiguous ranges, one per CTA, so a long list is shared by many CTAs and a
// short one by none; each (unit, CTA) piece leaves its unnormalised output,
// maximum and sum in rows of the workspace (Rooms), and the join adds a row's pieces
// in a fixed order, so results repeat run to run. Where a row's pieces lie is written
// down by a spare warp of the attention kernel.
//   Prefix: when a KV head has more than PR rows (n_pair > 1), `gs` CTAs walk
//     the same keys side by side, one row pair each, so that all but one of
//     them find the tile in L2; the ranges are then per group of gs CTAs.
//   Tails: units (sequence, row pair, KV head) in that order; each stands on the
//     line with kUnit tiles more than it has, in front of them, for what a piece
//     costs beside its tiles (its queries, its output, the first tile's latency).
// With gs == 1 prefix and tails form one line; otherwise each has its own.
#pragma once

#include "prefix_attn.cuh"

namespace kvmret {
namespace {

// Tiles of BN keys for what a piece costs beside its tiles, about 128 keys' worth.
// Sixteen sequences over 32,768 shared tokens, tails of 1 to 700: 44.1 us with
// this, 52.2 with none, 44.7 with 256 (q8_0 / q4_0: 54.5, 69.0, 55.6); heads of 256
// (tiles of 64 keys) over q8_0 / q4_0: 54.3 us with this, 63.5 with none, 55.3 with 64,
// 57.0 with 256. 32 sequences of up to five rows: 138.0, 139.0 with none, 136.4 with
// 256 (medians, the builds in turn on one box).
template <int BN>
constexpr uint32_t kUnit = 128 / BN;

// Division by a number that the host knows: n / d = (mulhi(n, m) + n) >> s with
// s = ceil(log2 d), m = floor(2^32 (2^s - d) / d) + 1, exact for every n below 2^32
// (Granlund and Montgomery 1994). The plan is a chain of some twenty divisions,
// before which no CTA has work.
struct Div {
    uint32_t d, m, s;
    void set(uint32_t by) {
        d = by;
        for (s = 0; (1ull << s) < by; ++s) {}
        m = static_cast<uint32_t>((((1ull << s) - by) << 32) / by) + 1;
    }
    __device__ __forceinline__ uint32_t operator()(uint32_t n) const {
        return static_cast<uint32_t>((static_cast<uint64_t>(__umulhi(n, m)) + n) >> s);
    }
};

// Key tiles of a list with pages of T tokens: a page of at least BN tokens is
// ceil(T / BN) tiles, else BN / T whole pages make one.
struct PageTiles {
    uint32_t T, tpp, ppt;  // page tokens, tiles per page (T >= BN), pages per tile (T < BN)
    Div whole, pages;      // by the tokens of whole pages (T >= BN: one) of a tile, by tpp
    void set(uint32_t t, uint32_t bn) {
        T = t;
        tpp = t >= bn ? (t - 1) / bn + 1 : 1;
        ppt = t >= bn ? 1 : bn / t;
        whole.set(ppt * t);
        pages.set(tpp);
    }
};
// What the host knows of a call's divisions.
struct Divs {
    Div G, H, ctas;  // query heads a KV head, KV heads, CTAs
    PageTiles list[2];  // of the prefix, the tails
};
template <int BN>
struct TileGeom {
    const PageTiles &c;
    __device__ __forceinline__ explicit TileGeom(const PageTiles &of) : c(of) {}
    __device__ __forceinline__ uint32_t tiles(uint32_t len) const {
        const uint32_t full = c.whole(len), rem = len - full * c.whole.d;
        return c.T < BN ? full + (rem != 0) : full * c.tpp + (rem + BN - 1) / BN;
    }
    __device__ __forceinline__ void locate(uint32_t tile, uint32_t &page, uint32_t &off) const {
        if (c.T < BN) {
            page = tile * c.ppt;
            off = 0;
        } else {
            page = c.pages(tile);
            off = (tile - page * c.tpp) * BN;
        }
    }
};

// A line of tiles cut into `parts` ranges: the first r of them hold q + 1.
struct Cuts {
    uint32_t q, r;
    __device__ __forceinline__ void set(uint32_t total, uint32_t parts) {
        q = total / parts;
        r = total - q * parts;
    }
    __device__ __forceinline__ void set(uint32_t total, const Div &parts) {
        q = parts(total);
        r = total - q * parts.d;
    }
    __device__ __forceinline__ uint32_t at(uint32_t i) const { return q * i + min(i, r); }
    // the range that holds tile x of the line
    __device__ __forceinline__ uint32_t owner(uint32_t x) const {
        const uint32_t head = (q + 1) * r;
        return x < head ? x / (q + 1) : r + (x - head) / q;
    }
};

// The workspace's rows, as the host knows them. A piece of the prefix has a room of
// `cap` rows by its unit and range; of a tail's unit the first piece has the unit's
// own rows (each row of the batch has one) and every further one a room by its CTA,
// which begins at most one unit in its middle. So the rows follow those of the
// batch, however few of them a unit has: 1024 sequences of one row, 64 query and 8 KV
// heads of 128 take 0.12 GB (a tile of 256 rows for each piece would be 1.2 GB).
struct Rooms {
    uint32_t cap;    // rows of a room: a unit's, or all of a KV head's if they are fewer
    uint32_t n_pre;  // rooms of the prefix, from row 0 on
    uint32_t tail;   // first row of the tails' units
    uint32_t over;   // first room of the tails' further pieces
};

// The split, alike in every CTA. (Tile counts fit 32 bits: the host checks their
// bound.)
struct Plan {
    uint32_t p_total, t_total;  // tiles of the prefix line and of the tails
    Cuts pre, own;              // their ranges (gs == 1: of the joint line)
    uint32_t np;                // tiles of the prefix
    uint32_t p_len;             // its tokens (with partly filled pages: the place behind the last)
    uint32_t q0, rows;          // first row token; rows of a KV head (all sequences)
    uint32_t n_pair, n_pg, gs, groups;
    uint32_t ok;                // 0: q_start descends somewhere, nothing is done
};

// Rows and keys of one sequence, all cut to what the host's bounds allow.
struct SeqShape {
    uint32_t q0, q_len, len;
};
__device__ __forceinline__ SeqShape seq_shape(const PrefixAttn &a, uint32_t s) {
    SeqShape r;
    const int32_t n = static_cast<int32_t>(a.n_q);
    const int32_t q0 = min(max(__ldg(a.q_start + s), 0), n);
    const int32_t q1 = min(max(__ldg(a.q_start + s + 1), q0), n);
    r.q0 = static_cast<uint32_t>(q0);
    r.q_len = static_cast<uint32_t>(q1 - q0);
    r.len = min(static_cast<uint32_t>(max(__ldg(a.tail.len + s), 0)), a.tail.max_len);
    return r;
}
// tail tokens that row token i of the sequence sees
__device__ __forceinline__ uint32_t tail_seen(uint32_t len, uint32_t q_len, uint32_t i) {
    const uint32_t after = q_len - 1 - i;
    return len > after ? len - after : 0;
}
// tiles of a tail that the rows of a pair reach
template <int BN, int PR>
__device__ __forceinline__ uint32_t pair_tiles(const SeqShape &s, const TileGeom<BN> &g,
                                               uint32_t pair, const Div &G) {
    const uint32_t last = min(s.q_len - 1, G(pair * PR + PR - 1));
    return g.tiles(tail_seen(s.len, s.q_len, last));
}

// One piece of work of a CTA.
struct Seg {
    uint32_t tail, seq, h;
    uint32_t q0, row0, rows;  // rows [row0, row0 + rows) of the unit's tokens from q0
    uint32_t len, q_len;      // the list's tokens; a tail's new ones
    uint32_t tile0, n;        // key tiles (n == 0: no more pieces)
    uint32_t j0;              // tiles of the CTA's pieces before this one
    uint32_t room;  // first of its rows in the workspace
};

template <int BN, int PR>
struct Walk {
    const PrefixAttn &a;
    const Plan &p;  // in shared memory
    const Divs &by;
    const Rooms &rooms;
    uint32_t cta;
    uint32_t x, x1;       // prefix line: next tile, end
    uint32_t part, lane;  // the range and the CTA's place in its group
    uint32_t y, y1;       // tails' line
    uint32_t seq;         // the sequence that holds y, its first tile
    uint32_t seq_tile;
    SeqShape sh;
    bool fresh;

    __device__ __forceinline__ Walk(const PrefixAttn &a_, const Plan &p_, const Divs &by_,
                                    const Rooms &r, uint32_t s, uint32_t tile)
        : a(a_), p(p_), by(by_), rooms(r), cta(blockIdx.x), seq(s), seq_tile(tile), fresh(true) {
        ranges(p, cta, x, x1, y, y1);
        part = p.gs == 1 ? cta : cta / p.gs;
        lane = cta - part * p.gs;
    }
    static __device__ __forceinline__ void ranges(const Plan &p, uint32_t cta, uint32_t &x,
                                                  uint32_t &x1, uint32_t &y, uint32_t &y1) {
        if (p.gs == 1) {
            const uint32_t b = p.pre.at(cta), e = p.pre.at(cta + 1);
            x = min(b, p.p_total);
            x1 = min(e, p.p_total);
            y = max(b, p.p_total) - p.p_total;
            y1 = max(e, p.p_total) - p.p_total;
        } else {
            const uint32_t part = cta / p.gs;
            x = part < p.groups ? p.pre.at(part) : 0;
            x1 = part < p.groups ? p.pre.at(part + 1) : 0;
            y = p.own.at(cta);
            y1 = p.own.at(cta + 1);
        }
    }

    __device__ __forceinline__ bool next(Seg &g) {
        while (x < x1) {
            const uint32_t u = x / p.np, t = x - u * p.np, n = min(x1 - x, p.np - t);
            x += n;
            const uint32_t pg = by.H(u), pair = pg * p.gs + lane;
            if (pair >= p.n_pair) continue;
            g.tail = 0;
            g.seq = 0;
            g.len = p.p_len;
            g.q_len = 0;
            g.h = u - pg * a.n_head_kv;
            g.q0 = p.q0;
            g.row0 = pair * PR;
            g.rows = min(static_cast<uint32_t>(PR), p.rows - g.row0);
            g.tile0 = t;
            g.n = n;
            g.room = ((u + part) * p.gs + lane) * rooms.cap;
            return true;
        }
        const TileGeom<BN> geom(by.list[1]);
        while (y < y1 && seq < a.n_seq) {
            if (fresh) sh = seq_shape(a, seq);
            fresh = false;
            const uint32_t tiles = sh.q_len ? geom.tiles(sh.len) : 0;
            const uint32_t pairs = (sh.q_len * by.G.d + PR - 1) / PR;
            const uint32_t mine = (tiles ? tiles + kUnit<BN> : 0) * pairs * a.n_head_kv;
            if (y >= seq_tile + mine) {
                seq_tile += mine;
                ++seq;
                fresh = true;
                continue;
            }
            const uint32_t at = y - seq_tile, all = tiles + kUnit<BN>, u = at / all;
            uint32_t t = at - u * all, n = min(y1 - y, all - t);
            y += n;
            if (t + n <= kUnit<BN>) continue;
            n -= t < kUnit<BN> ? kUnit<BN> - t : 0;
            t = t < kUnit<BN> ? 0 : t - kUnit<BN>;
            const uint32_t pair = by.H(u);
            const uint32_t lim = pair_tiles<BN, PR>(sh, geom, pair, by.G);
            if (t >= lim) continue;
            n = min(n, lim - t);
            g.tail = 1;
            g.seq = seq;
            g.len = sh.len;
            g.q_len = sh.q_len;
            g.h = u - pair * a.n_head_kv;
            g.q0 = sh.q0;
            g.row0 = pair * PR;
            g.rows = min(static_cast<uint32_t>(PR), sh.q_len * by.G.d - g.row0);
            g.tile0 = t;
            g.n = n;
            g.room = t ? rooms.over + cta * rooms.cap
                       : rooms.tail + ((sh.q0 - p.q0) * a.n_head_kv + g.h * sh.q_len) * by.G.d + g.row0;
            return true;
        }
        return false;
    }
};

// The tiles of a piece that stream s takes: with more than 128 rows both streams
// take every tile (a row tile each), otherwise stream s takes those whose number
// in the CTA's order has parity s. Two tiles in a row of one stream are then at
// most two apart in that order.
template <int NS>
struct Share {
    uint32_t tile, step, end;  // in the CTA's order
    bool both;
    __device__ __forceinline__ void set(const Seg &g, uint32_t s) {
        both = NS == 2 && g.rows > 128;
        step = NS == 1 || both ? 1 : 2;
        tile = step == 1 ? g.j0 : g.j0 + ((g.j0 ^ s) & 1u);
        end = g.j0 + g.n;
    }
    __device__ __forceinline__ bool any() const { return tile < end; }
};

}  // namespace
}  // namespace kvmret
