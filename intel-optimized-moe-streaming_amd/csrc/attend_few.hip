// attend_few.hip -- attention of few rows over the paged 4-bit cache: single new
// tokens and short drafts, up to 16 rows (tokens times the query heads of a kv
// head) at a time.
//
// The formula and its one pass are those of attend.hip.  What bounds it is the
// cache, read once: 4.25 bits a value, so little that a workgroup's start (the
// lengths, the page table, the first keys: three round trips) weighs as much as
// hundreds of keys.  The keys are therefore shared out evenly, in pieces of about
// as many blocks of 32 as one round of workgroups needs: every wave sums the
// sequences' blocks (a lane a sequence), finds the size of a piece and the
// sequence, tile and split of its own.  Long sequences get more pieces than short
// ones; rows of several are joined by attend_join.hip.
//
// A workgroup takes one kv head of one piece; its four waves take blocks of 32 keys
// in turn, each with a running sum of its own, joined in LDS at the end.  The rows
// are the 16 columns of 16x16x32 matrix instructions.  K goes from memory into
// operand registers: a lane holds 32 channels (one scale) of a key and the
// product's channels are taken in that order.  V becomes FP16 and passes through
// LDS of the wave's own (no barriers), 128 channels at a time, to be read
// transposed; 16-byte pieces are exchanged so that neither the writes (16 lanes: four
// keys' pieces) nor the transposing reads (eight keys) meet in a bank (half of the bank
// conflicts that there are with pieces exchanged for two and four keys).
//
// 64 ragged sequences of up to 8,192 keys, 32 heads of 128 over 8: 63 us, 4.5 TB/s, and
// 4.8 to join.  One sequence of 32,771 keys, 16 heads of 256 over 2: 12.2 us and 4.0, a
// chain of round trips: 1.5 us from a workgroup's start to its piece, 2.4 to its first
// keys, 3.3 for two blocks a wave, 1.9 to join the waves.

#include "attend_pieces.h"

namespace mqh {

constexpr int FEW_BLOCK = 32;   // keys

template <int DIM, int QT>
__global__ __launch_bounds__(256, DIM == 256 ? 2 : 4) void k_attend_few(AttendParams p) {
    using M = MixMath<MIX_F4>;
    typedef typename M::vec8 vec8;
    typedef typename M::vec4 vec4;
    constexpr int KW = DIM == 64 ? 2 : 4;             // dwords of a lane's load of a key
    constexpr int SECTIONS = DIM == 256 ? 2 : 1, SEC = DIM / SECTIONS;   // channels at a time through LDS
    constexpr int KK = DIM / 32, DB = SEC / 16;
    constexpr int ROW = SEC * 2;                      // bytes of a key in LDS
    constexpr int CODES = DIM / 2, SCALES = DIM / 32; // bytes of a key in the cache
    constexpr int PAD = DIM + 4;
    typedef uint32_t load_t __attribute__((ext_vector_type(KW)));

    extern __shared__ __align__(16) uint8_t lds[];    // [4 waves][32 keys x SEC] FP16, then [4][rows][PAD] FP32
    __shared__ float s_m[4][16], s_l[4][16];
    __shared__ int s_nan[4][DIM / 32];                // the first key some rows do not see whose block is not finite

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % p.kv_heads, piece = blockIdx.x / p.kv_heads;
    const Piece w = piece_of(p, piece, FEW_BLOCK, blockIdx.x == 0 && wave == 0);
    if (!w.live) return;
    const SeqRange seq = w.seq;
    const int i0 = w.tile * p.tile_tokens, n_tok = min(p.tile_tokens, seq.count - i0);
    const int first_pos = seq.length - seq.count + i0;   // position of the tile's first token (negative: it sees nothing)
    const int r_tok = col / p.group, r_head = kvh * p.group + col - r_tok * p.group;
    const bool row_live = r_tok < n_tok;
    const int seen = row_live ? first_pos + r_tok : -1;  // last key this column sees
    const int keys = max(first_pos + n_tok, 0), full = first_pos + 1;   // keys any row sees, every row sees
    const int blocks = (keys + FEW_BLOCK - 1) / FEW_BLOCK;
    const int block0 = w.split * w.per, block1 = min(block0 + min(w.per, blocks), blocks);
    const int page_mask = (1 << p.page_shift) - 1;
    if (lane < DIM / 32) s_nan[wave][lane] = 0x7fffffff;

    // ---- pages of this wave's blocks: lane i has those of its blocks i (mod 64)
    int page_a = 0, page_b = 0;   // of a block's first and last 16 keys
    auto load_pages = [&](int first) {
        const int key = (first + 4 * lane) * FEW_BLOCK, last = max(keys - 1, 0);
        const int32_t* row = p.table + (int64_t)w.b * p.table_stride;
        page_a = row[min(key, last) >> p.page_shift];
        page_b = row[min(key + 16, last) >> p.page_shift];
        if ((unsigned)page_a >= (unsigned)p.pages || (unsigned)page_b >= (unsigned)p.pages) {
            atomicOr(&p.flags[FLAG_BAD_ID], 1);
            page_a = (unsigned)page_a >= (unsigned)p.pages ? 0 : page_a;
            page_b = (unsigned)page_b >= (unsigned)p.pages ? 0 : page_b;
        }
    };

    int block = block0 + wave;
    if (block < block1) load_pages(block);

    // ---- loads: 16 keys of a half block, K with key `col` and piece g, V with key
    // lane / 4 and piece lane % 4 (of a section's four)
    load_t kr[2][SECTIONS], vr[2][SECTIONS];
    uint8_t kf[2][SECTIONS], vf[2][SECTIONS];   // scale bytes
    const uint32_t k_at = col * CODES + g * 4 * KW, kf_at = col * SCALES + (KW == 2 ? g >> 1 : g);
    const int v_key = lane >> 2, v_piece = lane & 3;
    const uint32_t v_at = v_key * CODES + v_piece * 4 * KW, vf_at = v_key * SCALES + (KW == 2 ? v_piece >> 1 : v_piece);
    int64_t rows[2];   // the first row of each half in the cache
    auto rows_of = [&](int block, int it) {
        const int pa = __builtin_amdgcn_readlane(page_a, it & 63), pb = __builtin_amdgcn_readlane(page_b, it & 63);
        rows[0] = (((int64_t)pa * p.kv_heads + kvh) << p.page_shift) + ((block * FEW_BLOCK) & page_mask);
        rows[1] = (((int64_t)pb * p.kv_heads + kvh) << p.page_shift) + ((block * FEW_BLOCK + 16) & page_mask);
    };
    // (the offsets kept from the compiler, that they stay 32 bits beside an address in scalar registers)
    auto load_k = [&]() {
        uint32_t at = k_at, f_at = kf_at;
        asm("" : "+v"(at), "+v"(f_at));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint8_t* codes = (const uint8_t*)p.kc + rows[j] * CODES;
            const uint8_t* scales = (const uint8_t*)p.ks + rows[j] * SCALES;
#pragma unroll
            for (int s = 0; s < SECTIONS; ++s) {
                kr[j][s] = *(const load_t*)(codes + at + 64 * s);
                kf[j][s] = scales[f_at + 4 * s];
            }
        }
    };
    auto load_v = [&]() {
        uint32_t at = v_at, f_at = vf_at;
        asm("" : "+v"(at), "+v"(f_at));
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uint8_t* codes = (const uint8_t*)p.vc + rows[j] * CODES;
            const uint8_t* scales = (const uint8_t*)p.vs + rows[j] * SCALES;
#pragma unroll
            for (int s = 0; s < SECTIONS; ++s) {
                vr[j][s] = *(const load_t*)(codes + at + 64 * s);
                vf[j][s] = scales[f_at + 4 * s];
            }
        }
    };

    // ---- the queries: channels of product kk of this lane's quarter (converted behind the first keys' loads)
    uintx4 raw[KK];
    {
        const uint16_t* qp = (const uint16_t*)p.q + (int64_t)(seq.first + i0 + (row_live ? r_tok : 0)) * p.q_token +
                             (int64_t)(row_live ? r_head : kvh * p.group) * p.q_head;
#pragma unroll
        for (int kk = 0; kk < KK; ++kk)
            raw[kk] = load_any<uintx4>(qp + 32 * KW * (kk / KW) + 8 * KW * g + 8 * (kk % KW));
    }
    if (block < block1) {
        rows_of(block, 0);
        load_k();
        load_v();
    }
    vec8 qf[KK];
    float q_scale = 1.0f;
    {
        if constexpr (QT == MIX_BF16) {
            // to FP16 by a power of two per row that brings its largest value to [1, 2)
            uint32_t top = 0;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = max(top, max(raw[kk][i] << 16 & 0x7fffffffu, raw[kk][i] & 0x7fff0000u));
            top = max(top, (uint32_t)__shfl_xor((int)top, 16));
            top = max(top, (uint32_t)__shfl_xor((int)top, 32));
            int e = (int)(top >> 23);
            e = min(max(e, 2), 252);
            const float down = __uint_as_float((uint32_t)(254 - e) << 23);
            q_scale = __uint_as_float((uint32_t)e << 23);
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    qf[kk][2 * i] = (_Float16)(__uint_as_float(raw[kk][i] << 16) * down);
                    qf[kk][2 * i + 1] = (_Float16)(__uint_as_float(raw[kk][i] & 0xffff0000u) * down);
                }
        } else {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) qf[kk] = bits_as<vec8>(raw[kk]);
        }
    }
    // (never 0: a hidden key's score stays -infinity; at most 2^86: products of 2^40 at the
    // most stay finite, and such a softmax is its largest score's already)
    const float c = fminf(fmaxf(q_scale * p.scale_log2, 0x1p-126f), 0x1p86f);

    // ---- the V tile: which 16-byte pieces of a key are exchanged (xor), and this lane's places
    auto swap = [](int key) { return DIM == 64 ? (key & 6) | (key >> 1 & 1) : (key & 7) << 1 | (key >> 1 & 1); };
    uint8_t* vt = lds + wave * FEW_BLOCK * ROW;
    const int ka = 4 * g + ((lane & 15) >> 2);
    uint8_t* to[KW];
    const uint8_t* from[DB];
#pragma unroll
    for (int x = 0; x < KW; ++x) to[x] = vt + v_key * ROW + ((v_piece * KW + x) ^ swap(v_key)) * 16;
#pragma unroll
    for (int d = 0; d < DB; ++d)
        from[d] = vt + ka * ROW + ((2 * d + ((lane & 3) >> 1)) ^ swap(ka)) * 16 + (lane & 1) * 8;

    floatx4 o[SECTIONS][DB];
#pragma unroll
    for (int s = 0; s < SECTIONS; ++s)
#pragma unroll
        for (int d = 0; d < DB; ++d) o[s][d] = floatx4{0};
    float m = -INFINITY, l = 0.0f;

    if (block < block1) {
        for (int it = 0; block < block1; ++it, block += 4) {
            // (past the last block its keys are read once more: with the loads under a
            // condition the compiler waits for all of them where it needs the oldest)
            const bool more = block + 4 < block1;
            const int next = more ? block + 4 : block, base = block * FEW_BLOCK;
            if (more && ((it + 1) & 63) == 0) load_pages(next);
            rows_of(next, more ? it + 1 : it);
            const bool edge = base + FEW_BLOCK > full;
            // S^T = K Q^T
            floatx4 s[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                s[j] = floatx4{0};
#pragma unroll
                for (int i = 0; i < SECTIONS; ++i) {
                    const float f = f4_factor(kf[j][i]);
#pragma unroll
                    for (int x = 0; x < KW; ++x)
                        s[j] = M::mfma16(bits_as<vec8>(f4_to_half(kr[j][i][x], f)), qf[KW * i + x], s[j]);
                }
            }
            load_k();
            if (edge) {
                asm volatile("");   // (a branch: few blocks are)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e)
                        if (base + 16 * j + 4 * g + e > seen) s[j][e] = -INFINITY;
            }
            float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])),
                             fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3]))) * c;
            if (__any(mx - m > ATTEND_GROWTH)) {
                mx = fmaxf(mx, __shfl_xor(mx, 16));
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const float mn = fmaxf(m, mx);
                const float a = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= a;
#pragma unroll
                for (int i = 0; i < SECTIONS; ++i)
#pragma unroll
                    for (int d = 0; d < DB; ++d)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[i][d][e] *= a;
            }
            if (__any(exponent_far(m))) {
                const bool far = exponent_far(m);
                const float back = 1.0f / c;   // (the exponential's argument multiplies by c again)
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[j][e] = far ? score_from(s[j][e], c, m) * back : s[j][e];
            }
            const float ref = exponent_base<M>(m);
            vec8 pb;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float pr = __builtin_amdgcn_exp2f(fmaf(s[j][e], c, -ref));
                    l += pr;
                    pb[4 * j + e] = (typename M::elem)pr;
                }
            // V: blocks that are not finite, where some row does not see them, are taken out
            // and put back at the end for the rows that do; past the end there are zeros
            float f[2][SECTIONS];
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int i = 0; i < SECTIONS; ++i) {
                    uint32_t scale = vf[j][i];
                    if (edge) {
                        asm volatile("");
                        const int key = base + 16 * j + v_key;
                        if (scale == F4_NONE && key < keys)
                            atomicMin(&s_nan[wave][4 * i + (KW == 2 ? v_piece >> 1 : v_piece)], key);
                        if (scale == F4_NONE || key >= keys) scale = 0;
                    }
                    f[j][i] = f4_factor(scale);
                }
            // O^T += V^T P^T (LDS of one wave is in order; the fences are the compiler's)
#pragma unroll
            for (int i = 0; i < SECTIONS; ++i) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int x = 0; x < KW; ++x)
                        *(uintx4*)(to[x] + j * 16 * ROW) = f4_to_half(vr[j][i][x], f[j][i]);
                asm volatile("" ::: "memory");
                if (i == SECTIONS - 1) load_v();
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const vec4 lo = lds_transposed<vec4>(from[d]), hi = lds_transposed<vec4>(from[d] + 16 * ROW);
                    o[i][d] = M::mfma16(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), pb, o[i][d]);
                }
                asm volatile("" ::: "memory");
            }
        }
    }

    // ---- the four waves joined
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (g == 0) {
        s_m[wave][col] = m;
        s_l[wave][col] = l;
    }
    const int n_rows = n_tok * p.group, R = p.tile_tokens * p.group;
    float* po = (float*)lds;
    constexpr int LANES = DIM / 4;   // of an output row
    __syncthreads();   // (the waves' V tiles are done with)
    if (col < n_rows) {
#pragma unroll
        for (int i = 0; i < SECTIONS; ++i)
#pragma unroll
            for (int d = 0; d < DB; ++d) *(floatx4*)(po + (wave * R + col) * PAD + SEC * i + 16 * d + 4 * g) = o[i][d];
    }
    __syncthreads();
    for (int r = tid / LANES; r < n_rows; r += 256 / LANES) {
        const int ch = (tid % LANES) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int x = 0; x < 4; ++x) top = fmaxf(top, s_m[x][r]);
        const float ref = top == -INFINITY ? 0.0f : top;
        floatx4 sum = {0, 0, 0, 0};
        float total = 0.0f;
        int bad = 0x7fffffff;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            bad = min(bad, s_nan[x][ch / 32]);
            if (s_m[x][r] == -INFINITY && s_l[x][r] == 0.0f) continue;   // a wave without keys
            const float a = __builtin_amdgcn_exp2f(s_m[x][r] - ref);
            total = fmaf(a, s_l[x][r], total);
            const floatx4 v = *(const floatx4*)(po + (x * R + r) * PAD + ch);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = fmaf(a, v[e], sum[e]);
        }
        const int t = r / p.group, h = kvh * p.group + r - t * p.group;
        top = exponent_seen(top, total, block0 < block1 && block0 * FEW_BLOCK <= first_pos + t);
        if (bad <= first_pos + t) sum = floatx4{NAN, NAN, NAN, NAN};
        if (w.splits > 1) {
            const int64_t at = ((int64_t)piece * p.kv_heads + kvh) * R + r;
            *(floatx4*)(p.part_o + at * DIM + ch) = sum;
            if (ch == 0) {
                p.part_ml[2 * at] = top;
                p.part_ml[2 * at + 1] = total;
            }
            continue;
        }
        const float inv = inverse_sum(top, total);
        bool finite = true;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            sum[e] *= inv;
            finite &= fits<QT>(sum[e]);
        }
        uint16_t* out = (uint16_t*)p.out + ((int64_t)(seq.first + i0 + t) * p.heads + h) * DIM + ch;
        if constexpr (QT == MIX_F16)
            *(half4*)out = half4{(_Float16)sum[0], (_Float16)sum[1], (_Float16)sum[2], (_Float16)sum[3]};
        else
            *(bfloat4*)out = bfloat4{(__bf16)sum[0], (__bf16)sum[1], (__bf16)sum[2], (__bf16)sum[3]};
        if (!finite) atomicOr(&p.flags[FLAG_NONFINITE], 1);
    }
    // where the tile's rows are to be joined from
    if (p.part_rows && w.split == 0 && tid < n_tok)
        p.part_rows[(int64_t)(seq.first + i0 + tid) * p.kv_heads + kvh] = int4{w.first, w.splits, tid, 0};
}

template <int DIM, int QT>
static hipError_t launch_few_of(const AttendParams& p, hipStream_t s) {
    constexpr int SEC = DIM == 256 ? 128 : DIM;
    const int bytes = std::max(4 * FEW_BLOCK * SEC * 2, 4 * p.tile_tokens * p.group * (DIM + 4) * 4);
    hipLaunchKernelGGL((k_attend_few<DIM, QT>), dim3((unsigned)(p.pieces * p.kv_heads)), dim3(256), bytes, s, p);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? launch_pieces_join(p, s) : e;
}

template <int DIM>
static hipError_t launch_few_dim(const AttendParams& p, hipStream_t s) {
    return p.q_type == MIX_F16 ? launch_few_of<DIM, MIX_F16>(p, s) : launch_few_of<DIM, MIX_BF16>(p, s);
}

hipError_t launch_attend_few(const AttendParams& p, hipStream_t s) {
    switch (p.dim) {
        case 64: return launch_few_dim<64>(p, s);
        case 128: return launch_few_dim<128>(p, s);
        case 256: return launch_few_dim<256>(p, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace mqh
