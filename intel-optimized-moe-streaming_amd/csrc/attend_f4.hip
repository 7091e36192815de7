// attend_f4.hip -- attention of many rows (prompts, chunks) over the paged 4-bit
// cache.
//
// The formula, the transposed products, their operands' layouts and the running
// reference exponent are those of attend.hip; 4-bit codes become FP16 numbers on
// their way into LDS, exactly.  A workgroup takes 256 query rows of one kv head, 32 rows
// a wave.
//
// What bounds it is the matrix unit and the vector unit together: a step's products
// and its exponentials take a wave about equally long, and two waves of a SIMD that go
// in step wait for the same one.  So the workgroup's halves (a wave of each on every
// SIMD) take turns, a barrier between: one multiplies and loads, the other computes its
// probabilities and stores the keys of the steps to come.  Two buffers of keys and of
// values in LDS suffice.
//
// A prompt of 8,192 tokens, 32 heads of 128 over 8: 508 us, 1080 TFLOP/s (a large library
// product reaches 1170 to 1210), the matrix unit 52 % busy at 2.0 GHz: beside the
// exponentials the chip lowers its clock (2.4 GHz with the products alone, 1.8 where the
// stores into LDS are left out), so fewer cycles no longer are less time.  Four ragged
// chunks of 2,048 tokens in all after up to 16,384, 16 heads of 256 over 2: 460 us, 937
// TFLOP/s, and 17 to join; there is no register for operands read ahead.
//
// Steps that some row does not see whole test positions and come last; blocks of
// values that are not finite are taken out there and put back at the end for the
// rows that see them.

#include "attend_pieces.h"

namespace mqh {

// kinds of instructions, as the scheduler numbers them
constexpr int SCHED_MFMA = 0x8, SCHED_DS_READ = 0x100, SCHED_DS_WRITE = 0x200, SCHED_EXP = 0x400;

template <int DIM, int QT>
__global__ __launch_bounds__(F4_THREADS, 2) void k_attend_f4(AttendParams p) {
    using M = MixMath<MIX_F4>;
    typedef typename M::vec8 vec8;
    typedef typename M::vec4 vec4;
    constexpr int STEP = attend_step(DIM);
    constexpr int KROW = attend_krow(DIM), VROW = attend_vrow(DIM);
    constexpr int KTILE = STEP * KROW, VTILE = STEP * VROW;
    constexpr int PIECES = F4_THREADS / STEP, PW = DIM / PIECES / 8;   // pieces of a key, a thread each; dwords of one
    typedef uint32_t load_t __attribute__((ext_vector_type(PW)));
    constexpr int KB = STEP / 32, DB = DIM / 32, KK = DIM / 16, TB = STEP / 16;
    // at dim 256 the queries' second half stays in LDS: a wave then fits 256
    // registers and a SIMD holds two
    constexpr int KR = DIM == 256 ? KK / 2 : KK;

    extern __shared__ __align__(16) uint8_t lds[];      // [2][K tile], [2][V tile], then the waves' query operands
    __shared__ int s_nan[DIM / 32];                     // first key some rows do not see whose block is not finite

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 31, half = lane >> 5;
    const int kvh = blockIdx.x % p.kv_heads;
    const int piece = p.pieces - 1 - blockIdx.x / p.kv_heads;   // (later tiles have more keys: they go first)
    const Piece w = piece_of(p, piece, STEP, blockIdx.x == 0 && wave == 0);
    if (!w.live) return;
    const SeqRange seq = w.seq;
    const int i0 = w.tile * p.tile_tokens, n_tok = min(p.tile_tokens, seq.count - i0);
    const int before = seq.length - seq.count;             // position of query 0 (negative: it sees nothing)
    const int row = wave * 32 + col;
    const int r_tok = row / p.group;
    const bool row_live = r_tok < n_tok;
    const int r_head = kvh * p.group + (row - r_tok * p.group);
    const int seen = row_live ? before + i0 + r_tok : -1;  // last key this row sees
    const int keys = max(before + i0 + n_tok, 0);          // keys any row sees
    const int full = before + i0 + 1;                      // keys every row sees
    const int n_steps = (keys + STEP - 1) / STEP;
    const int step0 = w.split * w.per, step1 = min(step0 + min(w.per, n_steps), n_steps);
    const bool wave_live = wave * 32 < n_tok * p.group;
    if (tid < DIM / 32) s_nan[tid] = 0x7fffffff;

    // ---- the query rows as operands: column `col`, d = 16 kk + 8 half + e
    vec8 qf[KR];
    uintx4* q_rest = (uintx4*)(lds + 2 * (KTILE + VTILE)) + wave * (KK - KR) * 64 + lane;
    float q_scale = 1.0f;   // BF16 queries: what the FP16 operands were multiplied by, inverted
    {
        const int64_t at = (int64_t)(seq.first + i0 + (row_live ? r_tok : 0)) * p.q_token +
                           (int64_t)(row_live ? r_head : kvh * p.group) * p.q_head;
        uintx4 raw[KK];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) raw[kk] = load_any<uintx4>((const uint16_t*)p.q + at + 16 * kk + 8 * half);
        float down = 1.0f;
        if constexpr (QT == MIX_BF16) {
            // BF16 to FP16 by a power of two per row that brings its largest value to [1, 2)
            uint32_t top = 0;
#pragma unroll
            for (int kk = 0; kk < KK; ++kk)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = max(top, max(raw[kk][i] << 16 & 0x7fffffffu, raw[kk][i] & 0x7fff0000u));
            top = max(top, (uint32_t)__shfl_xor((int)top, 32));
            const int e = min(max((int)(top >> 23), 2), 252);
            down = __uint_as_float((uint32_t)(254 - e) << 23);
            q_scale = __uint_as_float((uint32_t)e << 23);
        }
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            vec8 v = bits_as<vec8>(raw[kk]);
            if constexpr (QT == MIX_BF16) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    v[2 * i] = (_Float16)(__uint_as_float(raw[kk][i] << 16) * down);
                    v[2 * i + 1] = (_Float16)(__uint_as_float(raw[kk][i] & 0xffff0000u) * down);
                }
            }
            if (kk < KR) qf[kk] = v;
            else q_rest[(kk - KR) * 64] = __builtin_bit_cast(uintx4, v);
        }
    }
    // (never 0: a hidden key's score stays -infinity; at most 2^86: products of 2^40 at the
    // most stay finite, and such a softmax is its largest score's already)
    const float c = fminf(fmaxf(q_scale * p.scale_log2, 0x1p-126f), 0x1p86f);

    // ---- loading: piece tid % PIECES of key tid / PIECES
    const int part = tid % PIECES, key_in = tid / PIECES;
    const int page_mask = (1 << p.page_shift) - 1;
    const int wave_key = __builtin_amdgcn_readfirstlane(key_in) >> 4;   // which 16 keys a wave's loads fall into
    // lane i holds the page of 16-key group i (mod 64) counted from the piece's first
    // key, and that of the group 64 further on, so no address waits for the table
    int pages_now = 0, pages_next = 0, window = 0;
    auto load_pages = [&](int group) {
        const int key = step0 * STEP + (group + lane) * 16;
        int page = p.table[(int64_t)w.b * p.table_stride + (min(key, keys - 1) >> p.page_shift)];
        if ((unsigned)page >= (unsigned)p.pages) {
            atomicOr(&p.flags[FLAG_BAD_ID], 1);
            page = 0;
        }
        return page;
    };
    load_t kr, vr;
    uint8_t kf, vf;   // scales of the pieces' blocks
    // the key's page in the cache (in scalar registers, for a wave's keys share it) and its place there
    auto place = [&](int step, uint32_t& at) {
        const int group = (step - step0) * TB + wave_key;
        const int page = __builtin_amdgcn_readlane(group < window + 64 ? pages_now : pages_next, group & 63);
        at = (uint32_t)(min(step * STEP + key_in, keys - 1) & page_mask) * PIECES + part;
        return ((int64_t)page * p.kv_heads + kvh) << p.page_shift;
    };
    auto load_k = [&](int step) {
        uint32_t at;
        const int64_t first = place(step, at);
        kr = *(const load_t*)((const uint8_t*)p.kc + first * (DIM / 2) + at * (4 * PW));
        kf = ((const uint8_t*)p.ks + first * (DIM / 32))[at / (4 / PW)];
    };
    auto load_v = [&](int step) {
        uint32_t at;
        const int64_t first = place(step, at);
        vr = *(const load_t*)((const uint8_t*)p.vc + first * (DIM / 2) + at * (4 * PW));
        vf = ((const uint8_t*)p.vs + first * (DIM / 32))[at / (4 / PW)];
    };
    uint8_t* const k_to = lds + key_in * KROW + part * (16 * PW);
    uint8_t* const v_to = lds + 2 * KTILE + key_in * VROW + part * (16 * PW);
    auto store_k = [&](int buf) {
        const float f = f4_factor(kf);
#pragma unroll
        for (int x = 0; x < PW; ++x) *(uintx4*)(k_to + buf * KTILE + 16 * x) = f4_to_half(kr[x], f);
    };
    // values of a step that some row does not see whole: blocks that are not finite are noted and taken out
    auto test_v = [&](int step) {
        if (step * STEP + STEP > full) {
            const int key = step * STEP + key_in;
            if (vf == F4_NONE && key < keys) atomicMin(&s_nan[part * PW / 4], key);
            if (vf == F4_NONE || key >= keys) vf = 0;
        }
    };
    auto store_v = [&](int buf) {
        const float f = f4_factor(vf);
#pragma unroll
        for (int x = 0; x < PW; ++x) *(uintx4*)(v_to + buf * VTILE + 16 * x) = f4_to_half(vr[x], f);
    };

    floatx16 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = floatx16{0};
    float m = -INFINITY, l[4] = {0.0f, 0.0f, 0.0f, 0.0f};   // reference exponent (log2), this lane's parts of the sum

    // operand addresses: K row `col`, channels 8 half; V as the transposing loads take it (key
    // 4 half + i / 4, channels 16 (lane / 16 % 2) + 4 (i % 4) of 32)
    const uint8_t* const k_from = lds + col * KROW + half * 16;
    const uint8_t* const v_from = lds + 2 * KTILE + (4 * half + ((lane & 15) >> 2)) * VROW + ((lane >> 4) & 1) * 32 + (lane & 3) * 8;
    auto query = [&](int kk) { return kk < KR ? qf[kk < KR ? kk : 0] : bits_as<vec8>(q_rest[(kk - KR) * 64]); };

    floatx16 s[KB];      // scores, then of the next step
    vec8 probs[TB];
    // product i of O^T += V^T P^T, of S^T = K Q^T
    auto value = [&](int buf, int i) {
        const int t = i / DB, d = i % DB;
        const uint8_t* at = v_from + buf * VTILE + 16 * t * VROW + 64 * d;
        const vec4 lo = lds_transposed<vec4>(at), hi = lds_transposed<vec4>(at + 8 * VROW);
        o[d] = M::mfma32(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), probs[t], o[d]);
    };
    auto score = [&](int buf, int i) {
        const int kk = i / KB, j = i % KB;
        if (kk == 0) s[j] = floatx16{0};
        s[j] = M::mfma32(bits_as<vec8>(*(const uintx4*)(k_from + buf * KTILE + 32 * j * KROW + 32 * kk)), query(kk), s[j]);
    };
    constexpr int PRODUCTS = TB * DB;   // of each
    static_assert(PRODUCTS == KB * KK, "as many products of values as of keys");
    // step t's reference exponent
    auto reference = [&](int t) {
        const int base = (step0 + t) * STEP;
        if (base + STEP > full) {
#pragma unroll
            for (int j = 0; j < KB; ++j)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (base + 32 * j + 8 * (r >> 2) + 4 * half + (r & 3) > seen) s[j][r] = -INFINITY;
        }
        float part_mx[4];   // (four chains: a wave alone on its vector unit waits for each result)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            part_mx[i] = s[0][4 * i];
#pragma unroll
            for (int j = 0; j < KB; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) part_mx[i] = fmaxf(part_mx[i], s[j][4 * i + e]);
        }
        float mx = fmaxf(fmaxf(part_mx[0], part_mx[1]), fmaxf(part_mx[2], part_mx[3])) * c;
        if (__any(mx - m > ATTEND_GROWTH)) {
            mx = fmaxf(mx, __shfl_xor(mx, 32));
            const float mn = fmaxf(m, mx);
            const float a = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
#pragma unroll
            for (int i = 0; i < 4; ++i) l[i] *= a;
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
    };
    auto probabilities = [&]() {
        const float ref = exponent_base<M>(m);
#pragma unroll
        for (int t = 0; t < TB; ++t)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float pr = __builtin_amdgcn_exp2f(fmaf(s[t / 2][8 * (t & 1) + e], c, -ref));
                l[e & 3] += pr;
                probs[t][e] = (typename M::elem)pr;
            }
    };

    // The waves' halves take turns: in a slot of time one multiplies (the values of
    // its last step, the keys of its next) and loads, the other puts what it loaded into
    // LDS and computes its probabilities; the second half is a slot behind.  Each half
    // moves half the keys: those of step t + 1 and the values of step t are whole when the
    // first half begins to multiply the keys of step t + 1.
    const int n = step1 - step0, behind = wave >> 2;
    auto at_most = [&](int t) { return step0 + min(t, n - 1); };
    auto store = [&](int t) {
        store_k((t + 1 + behind) & 1);
        store_v((t + behind) & 1);
    };
    auto load = [&](int t) {
        load_k(at_most(t + 1 + behind));
        load_v(at_most(t + behind));
    };
    auto turn_pages = [&](int t) {   // loads from step t's on are of these groups or later ones
        if ((at_most(t + behind) - step0) * TB >= window + 64) {
            window += 64;
            pages_now = pages_next;
            pages_next = load_pages(window + 64);
        }
    };
    if (n > 0) {
        pages_now = load_pages(0);
        pages_next = load_pages(64);
        load_k(at_most(0));
    }
    __syncthreads();   // (s_nan)
    if (n > 0) {
        store_k(0);
        behind ? (load_k(at_most(1)), load_v(at_most(0))) : load(0);
        __syncthreads();
        if (behind) {
            test_v(at_most(0));
            store(-1);
            load(0);
            __syncthreads();
        }
        if (wave_live)
#pragma unroll
            for (int i = 0; i < PRODUCTS; ++i) score(0, i);
        __syncthreads();
        for (int t = 0; t < n; ++t) {
            turn_pages(t + 1);
            test_v(at_most(t + behind));
            if (wave_live) {
                reference(t);
                store(t);
                probabilities();
                // LDS is busy with the other half's operands: the stores go among the exponentials
#pragma unroll
                for (int i = 0; i < 2 * PW; ++i) {
                    __builtin_amdgcn_sched_group_barrier(SCHED_EXP, 2, 1);
                    __builtin_amdgcn_sched_group_barrier(SCHED_DS_WRITE, 1, 1);
                }
            } else {
                store(t);
            }
            __syncthreads();
            if (wave_live) {
                __builtin_amdgcn_s_setprio(1);
                // (scores past the last step: of keys that are there, for nothing)
                if constexpr (DIM == 256) {
                    // (no registers for more: 465 us for four chunks of 2,048 rows in all, 476 with
                    // the two products' instructions in turn, 707 with six reads ahead)
#pragma unroll
                    for (int i = 0; i < PRODUCTS; ++i) value(t & 1, i);
#pragma unroll
                    for (int i = 0; i < PRODUCTS; ++i) score((t + 1) & 1, i);
                    load(t + 1);
                } else {
#pragma unroll
                    for (int i = 0; i < PRODUCTS; ++i) {
                        value(t & 1, i);
                        score((t + 1) & 1, i);
                    }
                    load(t + 1);
                    // operands are read ahead of the products that they are for (a prompt of 8,192
                    // tokens 502 us, 517 in the compiler's order)
                    __builtin_amdgcn_sched_group_barrier(SCHED_DS_READ, 8, 0);
#pragma unroll
                    for (int i = 0; i < PRODUCTS; ++i) {
                        __builtin_amdgcn_sched_group_barrier(SCHED_MFMA, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(SCHED_DS_READ, 2, 0);
                        __builtin_amdgcn_sched_group_barrier(SCHED_MFMA, 1, 0);
                        __builtin_amdgcn_sched_group_barrier(SCHED_DS_READ, 1, 0);
                    }
                }
                __builtin_amdgcn_s_setprio(0);
            } else {
                load(t + 1);
            }
            __syncthreads();
        }
        if (!behind) __syncthreads();
    }

    // ---- the rows out: this lane's channels 32 d + 8 r4 + 4 half + e
    if (p.part_rows && w.split == 0)
        for (int i = tid; i < n_tok; i += F4_THREADS)
            p.part_rows[(int64_t)(seq.first + i0 + i) * p.kv_heads + kvh] = int4{w.first, w.splits, i, 0};
    if (!row_live) return;
    float sum = (l[0] + l[1]) + (l[2] + l[3]);
    sum += __shfl_xor(sum, 32);   // (both halves of a row are live or neither)
    m = exponent_seen(m, sum, n > 0 && step0 * STEP <= seen);
#pragma unroll
    for (int d = 0; d < DB; ++d)
        if (s_nan[d] <= seen)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[d][r] = NAN;
    if (w.splits > 1) {
        const int64_t at = ((int64_t)piece * p.kv_heads + kvh) * (p.tile_tokens * p.group) + row;
        float* po = p.part_o + at * DIM;
#pragma unroll
        for (int d = 0; d < DB; ++d)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4)
                *(floatx4*)(po + 32 * d + 8 * r4 + 4 * half) =
                    floatx4{o[d][4 * r4], o[d][4 * r4 + 1], o[d][4 * r4 + 2], o[d][4 * r4 + 3]};
        if (half == 0) {
            p.part_ml[2 * at] = m;
            p.part_ml[2 * at + 1] = sum;
        }
        return;
    }
    const float inv = inverse_sum(m, sum);
    uint16_t* out = (uint16_t*)p.out + ((int64_t)(seq.first + i0 + r_tok) * p.heads + r_head) * DIM;
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
            const int ch = 32 * d + 8 * r4 + 4 * half;
            if constexpr (QT == MIX_F16)
                *(half4*)(out + ch) = half4{(_Float16)y[0], (_Float16)y[1], (_Float16)y[2], (_Float16)y[3]};
            else
                *(bfloat4*)(out + ch) = bfloat4{(__bf16)y[0], (__bf16)y[1], (__bf16)y[2], (__bf16)y[3]};
        }
    if (!finite) atomicOr(&p.flags[FLAG_NONFINITE], 1);
}

template <int DIM, int QT>
static hipError_t launch_f4_of(const AttendParams& p, hipStream_t s) {
    constexpr int bytes = 2 * attend_step(DIM) * (attend_krow(DIM) + attend_vrow(DIM)) + (DIM == 256 ? F4_THREADS / 64 * 8 * 1024 : 0);
    hipLaunchKernelGGL((k_attend_f4<DIM, QT>), dim3((unsigned)(p.pieces * p.kv_heads)), dim3(F4_THREADS), bytes, s, p);
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? launch_pieces_join(p, s) : e;
}

template <int DIM>
static hipError_t launch_f4_dim(const AttendParams& p, hipStream_t s) {
    return p.q_type == MIX_F16 ? launch_f4_of<DIM, MIX_F16>(p, s) : launch_f4_of<DIM, MIX_BF16>(p, s);
}

hipError_t launch_attend_f4(const AttendParams& p, hipStream_t s) {
    switch (p.dim) {
        case 64: return launch_f4_dim<64>(p, s);
        case 128: return launch_f4_dim<128>(p, s);
        case 256: return launch_f4_dim<256>(p, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace mqh
