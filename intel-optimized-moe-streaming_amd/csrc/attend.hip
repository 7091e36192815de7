// attend.hip -- attention of new tokens over the paged cache, many query rows at
// a time (chunks of prompts, drafts).
//
// For query i of a sequence with n new tokens and L cached ones (the new ones
// included), position p = L - n + i:
//   out = sum_{j <= p} e^{scale q.k_j - m} v_j / sum_{j <= p} e^{scale q.k_j - m}
// in one pass over the keys with a running reference exponent m and sum; zeros
// where p < 0.  Query head h reads kv head h / group.
//
// A workgroup takes 128 query rows (256 at dim 256) of one kv head (all heads of
// its group, so a key tile serves them all), 32 rows a wave.  Both products are computed
// transposed, S^T = K Q^T and O^T = V^T P^T, on 32x32x16 matrix instructions: a
// lane then holds scores of ONE query row, so maximum, exponential and sum need
// no lane exchange, and the probabilities already lie in the second product's
// operand layout once its keys are taken in the order the first one leaves them
// (slot e of half h: key 8 (e / 4) + 4 h + e % 4 of 16).  V is read from LDS by
// transposing loads in that order.
//
// Keys go by in steps of 64 (32 at dim 256) through two LDS buffers: the next
// step's rows are loaded into registers while this one is multiplied, converted
// (8-bit codes to FP16) and stored behind it; one barrier a step.  Rows are padded
// in LDS so that neither the operand loads of K nor the transposing ones of V meet
// in a bank.
//
// The reference exponent moves only when a score passes it by 2^8: the sums are
// rescaled a few times a row instead of once a step.  8-bit caches: a key's scale
// multiplies its score; the value's scale vs enters as log2(vs) in the exponent,
// so the product p vs is what is rounded and multiplied by the codes, and the
// sum takes p vs / vs.
//
// Only steps that some row does not see whole test positions.  There, values
// that are not finite are taken out of the product (0 x infinity would reach rows
// that do not see the key) and put back per channel at the end for the rows that
// see them.
//
// A prompt of 8,192 tokens, 32 heads of 128 over 8, BF16: 587 us, 936 TFLOP/s (a
// large library product reaches 1184), the matrix unit 46 % busy beside the
// exponentials and the LDS loads; four ragged chunks of 2,048 tokens in all after up to
// 16,384, 16 heads of 256 over 2, 8-bit cache: 575 us, 750 TFLOP/s, and 18 to join (the
// splits are equal in number, not in keys: the busiest CU goes 296 steps where an equal
// share is 205).

#include <type_traits>

#include "attend.h"

namespace mqh {

template <int DIM, int CACHE, int QT>
__global__ __launch_bounds__(attend_threads(DIM), 2) void k_attend(AttendParams p) {
    using M = MixMath<CACHE>;
    typedef typename M::vec8 vec8;
    typedef typename M::vec4 vec4;
    constexpr bool Q8 = CACHE == MIX_Q8;
    constexpr int STEP = attend_step(DIM);
    constexpr int KROW = attend_krow(DIM), VROW = attend_vrow(DIM);
    constexpr int KTILE = STEP * KROW, BUFFER = KTILE + STEP * VROW;
    constexpr int PIECES = Q8 ? DIM / 16 : DIM / 8;    // 16-byte pieces of a cache row
    constexpr int THREADS = attend_threads(DIM);
    constexpr int PASS = THREADS / PIECES;             // keys of one load of every thread
    constexpr int LOADS = STEP / PASS;
    constexpr int KB = STEP / 32, DB = DIM / 32, KK = DIM / 16;
    // at dim 256 the queries' second half stays in LDS: a wave then fits 256
    // registers and a SIMD holds two
    constexpr int KR = DIM == 256 ? KK / 2 : KK;

    extern __shared__ __align__(16) uint8_t lds[];     // [2][K tile | V tile], then the waves' query operands
    __shared__ __align__(16) float s_kscale[2][STEP];  // 8-bit caches
    __shared__ __align__(16) float s_vlog[2][STEP];    // log2(vs)
    __shared__ __align__(16) float s_vinv[2][STEP];    // 1 / vs
    __shared__ int s_bad[3][DIM];                      // first visible key of a channel that is +inf, -inf, NaN
    __shared__ int s_any_bad;

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;

    // ---- the tile: kv head fastest (blocks go round the 8 XCDs: a head's keys
    // stay in few L2s), tiles with the most keys first
    const int kvh = blockIdx.x % p.kv_heads, split = blockIdx.y;
    const int tile = p.tiles - 1 - blockIdx.x / p.kv_heads;
    if (p.starts && blockIdx.x == 0 && split == 0) {
        // (starts out of order may leave a sequence without a workgroup that looks at it)
        bool bad = false;
        for (int i = tid; i < p.seqs; i += THREADS) {
            const int a = p.starts[i], z = p.starts[i + 1];
            bad |= a < 0 || z < a || z > p.tokens;
        }
        if (bad) atomicOr(&p.flags[FLAG_BAD_ID], 1);
    }
    int b = -1;
    {
        // tiles of sequence b begin at starts[b] / tile_tokens + b, which leaves room
        // for its partial tiles and needs no prefix sum
        for (int i0 = 0; i0 < p.seqs; i0 += 64) {
            const int i = i0 + lane;
            bool le = false;
            if (i < p.seqs) {
                const int s = p.starts ? p.starts[i] : i;
                le = (int64_t)(min(max(s, 0), p.tokens) / p.tile_tokens) + i <= tile;
            }
            b += __builtin_popcountll(__ballot(le));
        }
    }
    if (b < 0) return;
    b = __builtin_amdgcn_readfirstlane(b);
    const SeqRange seq = sequence_range(p, b, tid == 0);
    const int i0 = (tile - (seq.first / p.tile_tokens + b)) * p.tile_tokens;
    if (i0 >= seq.count || i0 < 0) return;
    const int n_tok = min(p.tile_tokens, seq.count - i0);
    const int before = seq.length - seq.count;             // position of query 0 (negative: it sees nothing)
    const int row = wave * 32 + col;
    const int r_tok = row / p.group;
    const bool row_live = r_tok < n_tok;
    const int r_head = kvh * p.group + (row - r_tok * p.group);
    const int seen = row_live ? before + i0 + r_tok : -1;  // last key this row sees
    const int keys = max(before + i0 + n_tok, 0);          // keys any row sees
    const int full = before + i0 + 1;                      // keys every row sees
    const int n_steps = (keys + STEP - 1) / STEP;
    const int per = max((n_steps + p.splits - 1) / p.splits, 512 / STEP);   // (short sequences: fewer splits)
    const int step0 = split * per, step1 = min(step0 + per, n_steps);
    const bool wave_live = wave * 32 < n_tok * p.group;

    if (tid == 0) s_any_bad = 0;
    for (int i = tid; i < 3 * DIM; i += THREADS) (&s_bad[0][0])[i] = 0x7fffffff;

    // ---- the query rows as operands: column `col`, d = 16 kk + 8 half + e
    vec8 qf[KR];
    uintx4* q_rest = (uintx4*)(lds + 2 * BUFFER) + wave * (KK - KR) * 64 + lane;
    float q_scale = 1.0f;   // 8-bit caches with BF16 queries: what the FP16 operands were multiplied by, inverted
    {
        const int64_t at = (int64_t)(seq.first + i0 + (row_live ? r_tok : 0)) * p.q_token +
                           (int64_t)(row_live ? r_head : kvh * p.group) * p.q_head;
        if constexpr (Q8 && QT == MIX_BF16) {
            // BF16 to FP16 by a power of two per row that brings its largest value to
            // [1, 2): exact down to 2^-17 of it
            uint32_t top = 0;
            uintx4 raw[KK];
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                raw[kk] = load_any<uintx4>((const uint16_t*)p.q + at + 16 * kk + 8 * half);
#pragma unroll
                for (int i = 0; i < 4; ++i) top = max(top, max(raw[kk][i] << 16 & 0x7fffffffu, raw[kk][i] & 0x7fff0000u));
            }
            top = max(top, (uint32_t)__shfl_xor((int)top, 32));
            int e = (int)(top >> 23);                   // biased exponent of the largest
            e = min(max(e, 2), 252);
            const float down = __uint_as_float((uint32_t)(254 - e) << 23);
            q_scale = __uint_as_float((uint32_t)e << 23);
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                vec8 v;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[2 * i] = (_Float16)(__uint_as_float(raw[kk][i] << 16) * down);
                    v[2 * i + 1] = (_Float16)(__uint_as_float(raw[kk][i] & 0xffff0000u) * down);
                }
                if (kk < KR) qf[kk] = v;
                else q_rest[(kk - KR) * 64] = __builtin_bit_cast(uintx4, v);
            }
        } else {
#pragma unroll
            for (int kk = 0; kk < KK; ++kk) {
                const uintx4 v = load_any<uintx4>((const uint16_t*)p.q + at + 16 * kk + 8 * half);
                if (kk < KR) qf[kk] = bits_as<vec8>(v);
                else q_rest[(kk - KR) * 64] = v;
            }
        }
    }

    // ---- loading a step: piece tid % PIECES of keys tid / PIECES + PASS i
    const int piece = tid % PIECES, key_in = tid / PIECES;
    const int page_mask = (1 << p.page_shift) - 1;
    const int wave_key = __builtin_amdgcn_readfirstlane(key_in) & ~15;   // the 16 keys a wave's loads fall into
    // lane i holds the page of 16-key group i (mod 64) counted from the split's first
    // key, and that of the group 64 further on, so no address waits for the table
    int pages_now = 0, pages_next = 0;
    auto load_pages = [&](int group) {
        const int key = step0 * STEP + (group + lane) * 16;
        int page = p.table[(int64_t)b * p.table_stride + (min(key, keys - 1) >> p.page_shift)];
        if ((unsigned)page >= (unsigned)p.pages) {
            atomicOr(&p.flags[FLAG_BAD_ID], 1);
            page = 0;
        }
        return page;
    };
    uintx4 kr[LOADS], vr[LOADS];
    float sk = 0, sv = 0;
    auto load_step = [&](int step) {
        const int base = step * STEP, group = (step - step0) * (STEP / 16);
        if (group && (group & 63) == 0) {
            pages_now = pages_next;
            pages_next = load_pages(group + 64);
        }
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int page = __builtin_amdgcn_readlane(pages_now, (group + ((wave_key + PASS * i) >> 4)) & 63);
            const int key = min(base + key_in + PASS * i, keys - 1);
            const int64_t at = ((((int64_t)page * p.kv_heads + kvh) << p.page_shift) + (key & page_mask)) * PIECES + piece;
            kr[i] = ((const uintx4*)p.kc)[at];
            vr[i] = ((const uintx4*)p.vc)[at];
        }
        if constexpr (Q8) {
            const int page = __shfl(pages_now, (group + (lane >> 4)) & 63);   // (with every lane: it reads all of them)
            if (wave == 0 && lane < STEP) {
                const int key = min(base + lane, keys - 1);
                const int64_t at = (((int64_t)page * p.kv_heads + kvh) << p.page_shift) + (key & page_mask);
                sk = ((const float*)p.ks)[at];
                sv = ((const float*)p.vs)[at];
            }
        }
    };
    auto store_step = [&](int step, int buf) {
        const int base = step * STEP;
        const bool edge = base + STEP > full;
        uint8_t* kt = lds + buf * BUFFER;
        uint8_t* vt = kt + KTILE;
#pragma unroll
        for (int i = 0; i < LOADS; ++i) {
            const int key = key_in + PASS * i;
            if constexpr (Q8) {
                // (codes are finite, and a key past the end has probability 0)
                const uintx2 a = codes_to_half(kr[i][0]), b2 = codes_to_half(kr[i][1]);
                const uintx2 c = codes_to_half(kr[i][2]), d = codes_to_half(kr[i][3]);
                const uintx2 e = codes_to_half(vr[i][0]), f = codes_to_half(vr[i][1]);
                const uintx2 g = codes_to_half(vr[i][2]), h = codes_to_half(vr[i][3]);
                uint8_t* ko = kt + key * KROW + piece * 32;
                uint8_t* vo = vt + key * VROW + piece * 32;
                *(uintx4*)ko = uintx4{a[0], a[1], b2[0], b2[1]};
                *(uintx4*)(ko + 16) = uintx4{c[0], c[1], d[0], d[1]};
                *(uintx4*)vo = uintx4{e[0], e[1], f[0], f[1]};
                *(uintx4*)(vo + 16) = uintx4{g[0], g[1], h[0], h[1]};
            } else {
                *(uintx4*)(kt + key * KROW + piece * 16) = kr[i];
                if (edge) {
                    const bool there = base + key < keys;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        uint32_t x = there ? vr[i][w] : 0u;
#pragma unroll
                        for (int hh = 0; hh < 2; ++hh) {
                            const uint32_t v = (x >> (16 * hh)) & 0xffffu;
                            if ((v & M::EXPONENT) == M::EXPONENT) {
                                const bool nan = v & (M::EXPONENT ^ 0x7fffu);
                                atomicMin(&s_bad[nan ? 2 : v >> 15][8 * piece + 2 * w + hh], base + key);
                                s_any_bad = 1;
                                x &= hh ? 0x0000ffffu : 0xffff0000u;
                            }
                        }
                        vr[i][w] = x;
                    }
                }
                *(uintx4*)(vt + key * VROW + piece * 16) = vr[i];
            }
        }
        if constexpr (Q8) {
            if (wave == 0 && lane < STEP) {
                const float vs = sv >= KV_MIN_SCALE ? sv : ATTEND_ZERO_SCALE;   // (NaN: the logarithm stays NaN)
                s_kscale[buf][lane] = sk * p.scale_log2;
                s_vlog[buf][lane] = sv != sv ? sv : __builtin_log2f(vs);
                s_vinv[buf][lane] = 1.0f / vs;
            }
        }
    };

    floatx16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = floatx16{0};
    float m = -INFINITY, l = 0.0f;   // reference exponent (log2), this lane's part of the sum

    if (step0 < step1) {
        pages_now = load_pages(0);
        pages_next = load_pages(64);
        load_step(step0);
    }
    __syncthreads();   // (s_bad)
    if (step0 < step1) store_step(step0, 0);
    __syncthreads();

    // where this lane points for the transposing loads: key 4 half + i / 4, channels
    // 16 (lane / 16 % 2) + 4 (i % 4) of 32
    const int v_at = (4 * half + ((lane & 15) >> 2)) * VROW + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
    // Operand addresses of a buffer: with the buffer a constant they are offsets
    auto compute = [&](int step, auto which) {
        constexpr int buf = decltype(which)::value;
        const bool more = step + 1 < step1;
        if (more) load_step(step + 1);
        if (wave_live) {
            const uint8_t* kt = lds + buf * BUFFER + col * KROW + half * 16;
            const uint8_t* vt = lds + buf * BUFFER + KTILE + v_at;
            // (at dim 256 a wave's products go before the other wave's exponentials: 631 us
            // without, 601 with for four chunks over 8-bit caches; at 128 it costs 2 %)
            if constexpr (DIM == 256) __builtin_amdgcn_s_setprio(1);
            // S^T = K Q^T
            floatx16 s[KB];
#pragma unroll
            for (int j = 0; j < KB; ++j) {
                s[j] = floatx16{0};
#pragma unroll
                for (int kk = 0; kk < KK; ++kk) {
                    const vec8 a = bits_as<vec8>(*(const uintx4*)(kt + 32 * j * KROW + 32 * kk));
                    const vec8 q = kk < KR ? qf[kk < KR ? kk : 0] : bits_as<vec8>(q_rest[(kk - KR) * 64]);
                    s[j] = M::mfma32(a, q, s[j]);
                }
            }
            if constexpr (DIM == 256) __builtin_amdgcn_s_setprio(0);
            // 8-bit caches: scores in log2 with the keys' scales and log2(vs) (else the
            // softmax scale goes into the exponential's argument)
            const int base = step * STEP;
            const float c = Q8 ? 1.0f : p.scale_log2;
            if constexpr (Q8) {
#pragma unroll
                for (int j = 0; j < KB; ++j)
#pragma unroll
                    for (int r4 = 0; r4 < 4; ++r4) {
                        const int k0 = 32 * j + 8 * r4 + 4 * half;
                        const floatx4 ks4 = *(const floatx4*)&s_kscale[buf][k0], vl4 = *(const floatx4*)&s_vlog[buf][k0];
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const float t = QT == MIX_BF16 ? s[j][4 * r4 + e] * q_scale : s[j][4 * r4 + e];
                            s[j][4 * r4 + e] = fmaf(t, ks4[e], vl4[e]);
                        }
                    }
            }
            if (base + STEP > full) {
#pragma unroll
                for (int j = 0; j < KB; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r)
                        if (base + 32 * j + 8 * (r >> 2) + 4 * half + (r & 3) > seen) s[j][r] = -INFINITY;
            }
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < KB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, s[j][r]);
            mx *= c;
            if (__any(mx - m > ATTEND_GROWTH)) {
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const float mn = fmaxf(m, mx);
                const float a = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= a;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int r = 0; r < 16; ++r) o[d][r] *= a;
            }
            if (__any(exponent_far(m))) {
                const bool far = exponent_far(m);
                const float back = 1.0f / c;   // (the exponential's argument multiplies by c again)
#pragma unroll
                for (int j = 0; j < KB; ++j)
#pragma unroll
                    for (int r = 0; r < 16; ++r) s[j][r] = far ? score_from(s[j][r], c, m) * back : s[j][r];
            }
            const float ref = exponent_base<M>(m);
            vec8 probs[STEP / 16];
#pragma unroll
            for (int t = 0; t < STEP / 16; ++t) {
#pragma unroll
                for (int e4 = 0; e4 < 2; ++e4) {
                    const int k0 = 16 * t + 8 * e4 + 4 * half;
                    floatx4 vi4;
                    if constexpr (Q8) vi4 = *(const floatx4*)&s_vinv[buf][k0];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const float pr = __builtin_amdgcn_exp2f(fmaf(s[t / 2][8 * (t & 1) + 4 * e4 + e], c, -ref));
                        if constexpr (Q8) l = fmaf(pr, vi4[e], l);
                        else l += pr;
                        probs[t][4 * e4 + e] = (typename M::elem)pr;
                    }
                }
            }
            // O^T += V^T P^T
            if constexpr (DIM == 256) __builtin_amdgcn_s_setprio(1);
#pragma unroll
            for (int t = 0; t < STEP / 16; ++t)
#pragma unroll
                for (int d = 0; d < DB; ++d) {
                    const vec4 lo = lds_transposed<vec4>(vt + 16 * t * VROW + 64 * d);
                    const vec4 hi = lds_transposed<vec4>(vt + (16 * t + 8) * VROW + 64 * d);
                    const vec8 va = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
                    o[d] = M::mfma32(va, probs[t], o[d]);
                }
            if constexpr (DIM == 256) __builtin_amdgcn_s_setprio(0);
        }
        if (more) store_step(step + 1, buf ^ 1);
        __syncthreads();
    };
    for (int step = step0; step < step1; step += 2) {
        compute(step, std::integral_constant<int, 0>());
        if (step + 1 < step1) compute(step + 1, std::integral_constant<int, 1>());
    }

    // ---- the rows out: this lane's channels 32 d + 8 r4 + 4 half + e
    if (!row_live) return;
    l += __shfl_xor(l, 32);   // (both halves of a row are live or neither)
    m = exponent_seen(m, l, step0 < step1 && step0 * STEP <= seen);
    if (s_any_bad) {
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int c = 32 * d + 8 * (r >> 2) + 4 * half + (r & 3);
                const bool pos = s_bad[0][c] <= seen, neg = s_bad[1][c] <= seen, nan = s_bad[2][c] <= seen;
                if (nan || (pos && neg)) o[d][r] = __uint_as_float(0x7fc00000u);
                else if (pos) o[d][r] += INFINITY;
                else if (neg) o[d][r] -= INFINITY;
            }
    }
    const int64_t out_row = (int64_t)(seq.first + i0 + r_tok) * p.heads + r_head;
    if (p.splits > 1) {
        const int64_t at = (int64_t)split * p.tokens * p.heads + out_row;
        float* po = p.part_o + at * DIM;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4)
                *(floatx4*)(po + 32 * d + 8 * r4 + 4 * half) =
                    floatx4{o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]};
        if (half == 0) {
            p.part_ml[2 * at] = m;
            p.part_ml[2 * at + 1] = l;
        }
        return;
    }
    const float inv = inverse_sum(m, l);
    uint16_t* out = (uint16_t*)p.out + out_row * DIM;
    bool finite = true;
#pragma unroll
    for (int d = 0; d < DB; ++d)
#pragma unroll
        for (int r4 = 0; r4 < 4; ++r4) {
            float y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[e] = o[d][4 * r4 + e] * inv;
                finite &= fits<QT>(y[e]);
            }
            const int c = 32 * d + 8 * r4 + 4 * half;
            if constexpr (QT == MIX_F16)
                *(half4*)(out + c) = half4{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
            else
                *(bfloat4*)(out + c) = bfloat4{(__bf16)y[0], (__bf16)y[1], (__bf16)y[2], (__bf16)y[3]};
        }
    if (!finite) atomicOr(&p.flags[FLAG_NONFINITE], 1);
}

// The splits of a row joined: the sums brought to the largest reference exponent
// and added in split order.  A wave takes a row: lane i first reads split i's
// exponent and sum (one round trip for all of them), then every lane its channels
// of eight splits at a time.
template <int DIM, int QT>
__global__ __launch_bounds__(256) void k_attend_join(AttendParams p) {
    constexpr int N = DIM / 64;   // channels of a lane
    typedef float vec __attribute__((ext_vector_type(N)));
    const int64_t rows = (int64_t)p.tokens * p.heads;
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= rows) return;
    if (p.starts) {   // rows of no sequence stay as they were
        const int t = (int)(row / p.heads);
        if (t < p.starts[0] || t >= p.starts[p.seqs]) return;
    }
    const float2* ml = (const float2*)p.part_ml + row;
    const float2 none = {-INFINITY, 0.0f};
    const float2 a = lane < p.splits ? ml[lane * rows] : none, b = lane + 64 < p.splits ? ml[(lane + 64) * rows] : none;
    float top = fmaxf(a.x, b.x);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) top = fmaxf(top, __shfl_xor(top, d));
    const float ref = top == -INFINITY ? 0.0f : top;
    // (a split without keys for this row weighs nothing)
    const float wa = a.x == -INFINITY && a.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(a.x - ref);
    const float wb = b.x == -INFINITY && b.y == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(b.x - ref);
    float l = fmaf(wa, a.y, wb * b.y);
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) l += __shfl_xor(l, d);

    const vec* part = (const vec*)(p.part_o + row * DIM) + lane;
    const int64_t step = rows * 64;   // of a split, in vecs
    vec sum = {};
    for (int s0 = 0; s0 < p.splits; s0 += 8) {
        vec v[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) v[i] = part[min(s0 + i, p.splits - 1) * step];
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int s = s0 + i;
            const float w = __shfl(s < 64 ? wa : wb, s & 63);
            if (s < p.splits)   // (also where w is 0: infinity and NaN stay so; a split without keys left zeros)
#pragma unroll
                for (int e = 0; e < N; ++e) sum[e] = fmaf(w, v[i][e], sum[e]);
        }
    }
    const float inv = inverse_sum(top, l);
    bool finite = true;
    uint16_t* out = (uint16_t*)p.out + row * DIM + lane * N;
    uint16_t y[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        const float x = sum[e] * inv;
        finite &= fits<QT>(x);
        if constexpr (QT == MIX_F16) y[e] = __builtin_bit_cast(uint16_t, (_Float16)x);
        else y[e] = __builtin_bit_cast(uint16_t, (__bf16)x);
    }
    __builtin_memcpy(__builtin_assume_aligned(out, 2 * N), y, 2 * N);
    if (!finite) atomicOr(&p.flags[FLAG_NONFINITE], 1);
}

template <int DIM, int CACHE, int QT>
static hipError_t launch_attend_of(const AttendParams& p, hipStream_t s) {
    constexpr int threads = attend_threads(DIM);
    constexpr int bytes = 2 * attend_step(DIM) * (attend_krow(DIM) + attend_vrow(DIM)) + (DIM == 256 ? threads / 64 * 8 * 1024 : 0);
    hipLaunchKernelGGL((k_attend<DIM, CACHE, QT>), dim3((unsigned)(p.tiles * p.kv_heads), (unsigned)p.splits),
                       dim3(threads), bytes, s, p);
    return hipGetLastError();
}

template <int DIM>
static hipError_t launch_attend_dim(const AttendParams& p, hipStream_t s) {
    if (p.cache_type == MIX_F16) return launch_attend_of<DIM, MIX_F16, MIX_F16>(p, s);
    if (p.cache_type == MIX_BF16) return launch_attend_of<DIM, MIX_BF16, MIX_BF16>(p, s);
    if (p.q_type == MIX_F16) return launch_attend_of<DIM, MIX_Q8, MIX_F16>(p, s);
    return launch_attend_of<DIM, MIX_Q8, MIX_BF16>(p, s);
}

hipError_t launch_attend(const AttendParams& p, hipStream_t s) {
    switch (p.dim) {
        case 64: return launch_attend_dim<64>(p, s);
        case 128: return launch_attend_dim<128>(p, s);
        case 256: return launch_attend_dim<256>(p, s);
    }
    return hipErrorInvalidValue;
}

template <int DIM>
static hipError_t launch_join_dim(const AttendParams& p, hipStream_t s) {
    const dim3 grid((unsigned)(((int64_t)p.tokens * p.heads + 3) / 4));
    if (p.q_type == MIX_F16) hipLaunchKernelGGL((k_attend_join<DIM, MIX_F16>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((k_attend_join<DIM, MIX_BF16>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

hipError_t launch_attend_join(const AttendParams& p, hipStream_t s) {
    switch (p.dim) {
        case 64: return launch_join_dim<64>(p, s);
        case 128: return launch_join_dim<128>(p, s);
        case 256: return launch_join_dim<256>(p, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace mqh
