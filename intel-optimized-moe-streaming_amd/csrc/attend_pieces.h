// attend_pieces.h -- how attention over 4-bit caches shares its keys out: tiles of rows
// times splits of their sequence's keys, of about the same number of blocks each.
#pragma once

#include <initializer_list>
#include <type_traits>

#include "attend.h"
#include "fp4.h"

namespace mqh {

// the pieces of each row joined (where p.part_rows says that there may be several)
hipError_t launch_pieces_join(const AttendParams& p, hipStream_t s);

// sums, or the largest, over the lanes up to this one
template <class T, class F>
__device__ __forceinline__ T scan_lanes(T x, T none, F op) {
    const int n = __builtin_bit_cast(int, none);
    const auto step = [&](auto moved) { x = op(x, __builtin_bit_cast(T, moved)); };
    step(__builtin_amdgcn_update_dpp(n, __builtin_bit_cast(int, x), 0x111, 0xf, 0xf, false));   // from 1, 2, 4, 8 lanes
    step(__builtin_amdgcn_update_dpp(n, __builtin_bit_cast(int, x), 0x112, 0xf, 0xf, false));   // below, of 16
    step(__builtin_amdgcn_update_dpp(n, __builtin_bit_cast(int, x), 0x114, 0xf, 0xf, false));
    step(__builtin_amdgcn_update_dpp(n, __builtin_bit_cast(int, x), 0x118, 0xf, 0xf, false));
    step(__builtin_amdgcn_update_dpp(n, __builtin_bit_cast(int, x), 0x142, 0xa, 0xf, false));   // the 16's last to the next
    step(__builtin_amdgcn_update_dpp(n, __builtin_bit_cast(int, x), 0x143, 0xc, 0xf, false));   // the 32's to the others
    return x;
}
template <class T>
__device__ __forceinline__ T last_lane(T x) {
    return __builtin_bit_cast(T, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), 63));
}

struct Piece {
    int b, tile, split, splits, first;   // first: the tile's first piece
    int per;                             // blocks of a piece
    SeqRange seq;
    bool live;
};

// The piece of a workgroup: blocks of `block` keys
__device__ __forceinline__ Piece piece_found(const AttendParams& p, int piece, int block, bool report) {
    Piece r{};
    const int lane = threadIdx.x & 63;
    if (!p.even) {
        // every tile a piece of its own, and nothing to sum: tiles of sequence b begin at
        // starts[b] / tile_tokens + b, which leaves room for its partial tiles
        int b = piece;
        if (p.starts) {
            // the last sequence that begins at this piece or before it: of those between b
            // and `past` every lane looks at one, evenly spaced
            int past = p.seqs;
            b = -1;
            while (past - b > 1) {
                const int step = (past - b - 1 + 63) >> 6, i = b + (lane + 1) * step;
                const int begin = min(max(p.starts[min(i, p.seqs - 1)], 0), p.tokens);
                const int here = __builtin_popcountll(__ballot(i < past && begin / p.tile_tokens + i <= piece));
                past = min(b + (here + 1) * step, past);
                b += here * step;
            }
            if (report) {
                bool bad = false;
                for (int i = lane; i < p.seqs; i += 64) bad |= clamped_range(p, i, r.seq);
                if (bad) atomicOr(&p.flags[FLAG_BAD_ID], 1);
            }
            if (b < 0) return r;
        }
        r.b = b = __builtin_amdgcn_readfirstlane(b);
        if (clamped_range(p, b, r.seq) && lane == 0) atomicOr(&p.flags[FLAG_BAD_ID], 1);
        r.tile = p.starts ? piece - (r.seq.first / p.tile_tokens + b) : 0;
        r.splits = 1;
        r.first = piece;
        r.per = 1 << 30;
        r.live = r.tile >= 0 && (int64_t)r.tile * p.tile_tokens < r.seq.count;
        return r;
    }
    // ---- blocks of all sequences, and of the longest
    SeqRange seq{};
    int longest = 0, all_tiles = 0;
    float total = 0.0f;
    bool bad = false;
    for (int i0 = 0; i0 < p.seqs; i0 += 64) {
        seq = SeqRange{};
        if (i0 + lane < p.seqs) bad |= clamped_range(p, i0 + lane, seq);
        const int tiles = (seq.count + p.tile_tokens - 1) / p.tile_tokens, blocks = (seq.length + block - 1) / block;
        total += (float)tiles * (float)blocks;
        all_tiles += tiles;
        longest = max(longest, blocks);
    }
    if (report && bad) atomicOr(&p.flags[FLAG_BAD_ID], 1);
    const auto add = [](auto a, auto b) { return a + b; };
    total = last_lane(scan_lanes(total, 0.0f, add));
    all_tiles = last_lane(scan_lanes(all_tiles, 0, add));
    longest = last_lane(scan_lanes(longest, 0, [](int a, int b) { return max(a, b); }));
    // (a tile's last piece is half full on average; the total is off by less than 80 * 2^-24)
    const int want = max(max(p.even / p.kv_heads - all_tiles / 2, p.even / p.kv_heads / 2), 1);
    int per = (int)fminf(total * 1.00001f / (float)want, 1e9f) + 1;
    per = max(per, (longest + PIECE_SPLITS_MAX - 1) / PIECE_SPLITS_MAX);
    r.per = longest <= p.whole ? p.whole : max((per + 3) & ~3, p.least);
    // ---- this piece's sequence
    int before = 0;
    for (int i0 = 0; i0 < p.seqs; i0 += 64) {
        if (p.seqs > 64) {   // (else the first loop's values are still here)
            seq = SeqRange{};
            if (i0 + lane < p.seqs) clamped_range(p, i0 + lane, seq);
        }
        const int tiles = (seq.count + p.tile_tokens - 1) / p.tile_tokens, blocks = (seq.length + block - 1) / block;
        const int splits = max((blocks + r.per - 1) / r.per, 1);
        const int mine = tiles * splits;
        const int sum = scan_lanes(mine, 0, add);
        const int at = piece - before - (sum - mine);
        const uint64_t hit = __ballot(at >= 0 && at < mine);
        if (hit) {
            const int who = __builtin_ctzll(hit);
            r.b = i0 + who;
            r.splits = __builtin_amdgcn_readlane(splits, who);
            const int local = __builtin_amdgcn_readlane(at, who);
            r.tile = local / r.splits;
            r.split = local - r.tile * r.splits;
            r.first = piece - r.split;
            r.seq.first = __builtin_amdgcn_readlane(seq.first, who);
            r.seq.count = __builtin_amdgcn_readlane(seq.count, who);
            r.seq.length = __builtin_amdgcn_readlane(seq.length, who);
            r.live = true;
            return r;
        }
        before += __builtin_amdgcn_readlane(sum, 63);
    }
    return r;
}

// the same in scalar registers
__device__ __forceinline__ Piece piece_of(const AttendParams& p, int piece, int block, bool report) {
    Piece r = piece_found(p, piece, block, report);
    for (int* x : {&r.b, &r.tile, &r.split, &r.splits, &r.first, &r.per, &r.seq.first, &r.seq.count, &r.seq.length})
        *x = __builtin_amdgcn_readfirstlane(*x);
    r.live = __builtin_amdgcn_readfirstlane(r.live);
    return r;
}

}  // namespace mqh
