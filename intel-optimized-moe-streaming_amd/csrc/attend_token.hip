// attend_token.hip -- attention of single new tokens over the paged cache: one
// query a sequence, up to 16 query heads a kv head.
//
// The same one-pass formula as for many rows (reference exponent, sums in FP32,
// products transposed).  What bounds it is the cache, read once: a workgroup
// takes one kv head of one sequence and one split of its keys, and its four
// waves take blocks of 32 keys in turn, each with a running sum of its own; the
// waves are joined in LDS, the splits by k_attend_join.  The group's query heads
// are the 16 columns of 16x16x32 matrix instructions, so a key row read serves
// all of them.
//
// K goes from memory straight into operand registers (a lane holds 16 bytes of a
// key; for 8-bit codes the product's channels are taken in the order that gives
// a lane 16 consecutive codes).  V passes through LDS of the wave's own (no
// barriers) to be read transposed.  The loads of the next block are issued as
// soon as this one's registers are consumed.  A lane keeps the page numbers of
// 64 blocks, so no address waits for the page table.
//
// 64 ragged sequences of up to 8,191 keys, 32 heads of 128 over 8, BF16: 200 us, 5.4
// TB/s.  One sequence of 4,099 keys, 16 heads of 256 over 2, 8-bit: 12.1 us, round trips
// (length, pages, keys, the next keys) of 32 workgroups, and 3.9 to join.

#include "attend.h"

namespace mqh {

template <int DIM, int CACHE, int QT>
__global__ __launch_bounds__(256) void k_attend_token(AttendParams p) {
    using M = MixMath<CACHE>;
    typedef typename M::vec8 vec8;
    typedef typename M::vec4 vec4;
    constexpr bool Q8 = CACHE == MIX_Q8;
    constexpr int ROW = DIM * 2;
    constexpr int PIECES = Q8 ? DIM / 16 : DIM / 8;   // 16-byte pieces of a cache row
    constexpr int KK = DIM / 32, DB = DIM / 16;
    constexpr int KL = Q8 ? KK / 2 : KK;              // loads of a key's row by its four lanes
    constexpr int PASS = 64 / PIECES;                 // keys of one load of V by the wave
    constexpr int VL = 32 / PASS;
    constexpr int PAD = DIM + 4;

    extern __shared__ __align__(16) uint8_t lds[];    // [4 waves][32 keys x DIM] 16-bit, then [4][16][PAD] FP32
    __shared__ float s_m[4][16], s_l[4][16];

    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int col = lane & 15, g = lane >> 4;
    const int kvh = blockIdx.x % p.kv_heads, b = blockIdx.x / p.kv_heads, split = blockIdx.y;
    const SeqRange seq = sequence_range(p, b, tid == 0);
    const int keys = seq.length;
    const int blocks = (keys + 31) >> 5;
    const int per = max((blocks + p.splits - 1) / p.splits, 8);   // (short sequences: fewer splits)
    const int block0 = split * per, block1 = min(block0 + per, blocks);
    const int page_mask = (1 << p.page_shift) - 1;

    // ---- the queries: column `col` is head col of the group (heads past it repeat the first)
    vec8 qf[KK];
    float q_scale = 1.0f;
    {
        const int head = kvh * p.group + (col < p.group ? col : 0);
        const uint16_t* qp = (const uint16_t*)p.q + (int64_t)b * p.q_token + (int64_t)head * p.q_head;
        uintx4 raw[KK];
#pragma unroll
        for (int kk = 0; kk < KK; ++kk) {
            const int d = Q8 ? 64 * (kk >> 1) + 16 * g + 8 * (kk & 1) : 32 * kk + 8 * g;
            raw[kk] = load_any<uintx4>(qp + d);
        }
        if constexpr (Q8 && QT == MIX_BF16) {
            // to FP16 by a power of two per head that brings its largest value to [1, 2)
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
    q_scale *= p.scale_log2;

    // ---- pages of this wave's blocks: lane i has those of its blocks i (mod 64)
    int page_a = 0, page_b = 0;   // of a block's first and last 16 keys
    auto load_pages = [&](int first) {
        const int key = (first + 4 * lane) * 32, last = max(keys - 1, 0);
        const int32_t* row = p.table + (int64_t)b * p.table_stride;
        page_a = row[min(key, last) >> p.page_shift];
        page_b = row[min(key + 16, last) >> p.page_shift];
        if ((unsigned)page_a >= (unsigned)p.pages || (unsigned)page_b >= (unsigned)p.pages) {
            atomicOr(&p.flags[FLAG_BAD_ID], 1);
            page_a = (unsigned)page_a >= (unsigned)p.pages ? 0 : page_a;
            page_b = (unsigned)page_b >= (unsigned)p.pages ? 0 : page_b;
        }
    };

    uintx4 kr[2][KL], vr[VL];
    floatx4 ks4[2], vs4[2];
    // the first row of each half of a block in the cache
    auto rows_of = [&](int block, int it, int64_t& ra, int64_t& rb) {
        const int pa = __builtin_amdgcn_readlane(page_a, it & 63), pb = __builtin_amdgcn_readlane(page_b, it & 63);
        ra = (((int64_t)pa * p.kv_heads + kvh) << p.page_shift) + ((block * 32) & page_mask);
        rb = (((int64_t)pb * p.kv_heads + kvh) << p.page_shift) + ((block * 32 + 16) & page_mask);
    };
    auto load_k = [&](int64_t ra, int64_t rb) {
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const uintx4* kp = (const uintx4*)p.kc + ((j ? rb : ra) + col) * PIECES + g;
#pragma unroll
            for (int i = 0; i < KL; ++i) kr[j][i] = kp[4 * i];
            if constexpr (Q8) ks4[j] = *(const floatx4*)((const float*)p.ks + (j ? rb : ra) + 4 * g);
        }
    };
    auto load_v = [&](int64_t ra, int64_t rb) {
        const int piece = lane % PIECES, key = lane / PIECES;
#pragma unroll
        for (int i = 0; i < VL; ++i) {
            const int k = key + PASS * i;   // (PASS divides 16)
            const int64_t r = PASS * i < 16 ? ra + k : rb + (k - 16);
            vr[i] = ((const uintx4*)p.vc)[r * PIECES + piece];
        }
        if constexpr (Q8) {
            vs4[0] = *(const floatx4*)((const float*)p.vs + ra + 4 * g);
            vs4[1] = *(const floatx4*)((const float*)p.vs + rb + 4 * g);
        }
    };

    floatx4 o[DB];
#pragma unroll
    for (int d = 0; d < DB; ++d) o[d] = floatx4{0};
    float m = -INFINITY, l = 0.0f;
    uint8_t* vt = lds + wave * 32 * ROW;

    int block = block0 + wave;
    if (block < block1) {
        load_pages(block);
        int64_t ra, rb;
        rows_of(block, 0, ra, rb);
        load_k(ra, rb);
        load_v(ra, rb);
        for (int it = 0; block < block1; ++it, block += 4) {
            // (past the last block its keys are read once more: with the loads under a
            // condition the compiler waits for all of them where it needs the oldest)
            const bool more = block + 4 < block1;
            const int next = more ? block + 4 : block;
            if (more && ((it + 1) & 63) == 0) load_pages(next);
            rows_of(next, more ? it + 1 : it, ra, rb);
            const bool edge = block * 32 + 32 > keys;
            // S^T = K Q^T
            floatx4 s[2];
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                s[j] = floatx4{0};
#pragma unroll
                for (int i = 0; i < KL; ++i) {
                    if constexpr (Q8) {
                        const uintx2 a = codes_to_half(kr[j][i][0]), c = codes_to_half(kr[j][i][1]);
                        const uintx2 d = codes_to_half(kr[j][i][2]), e = codes_to_half(kr[j][i][3]);
                        s[j] = M::mfma16(bits_as<vec8>(uintx4{a[0], a[1], c[0], c[1]}), qf[2 * i], s[j]);
                        s[j] = M::mfma16(bits_as<vec8>(uintx4{d[0], d[1], e[0], e[1]}), qf[2 * i + 1], s[j]);
                    } else {
                        s[j] = M::mfma16(bits_as<vec8>(kr[j][i]), qf[i], s[j]);
                    }
                }
            }
            floatx4 vinv[2];
            float mx = -INFINITY;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    float t;
                    if constexpr (Q8) {
                        const float sv = vs4[j][e], vs = sv >= KV_MIN_SCALE ? sv : ATTEND_ZERO_SCALE;
                        t = fmaf(s[j][e] * ks4[j][e], q_scale, sv != sv ? sv : __builtin_amdgcn_logf(vs));
                        vinv[j][e] = __builtin_amdgcn_rcpf(vs);
                    } else {
                        t = s[j][e] * q_scale;
                    }
                    if (edge && block * 32 + 16 * j + 4 * g + e >= keys) {
                        t = -INFINITY;
                        if constexpr (Q8) vinv[j][e] = 1.0f;
                    }
                    s[j][e] = t;
                    mx = fmaxf(mx, t);
                }
            load_k(ra, rb);
            // V into LDS (rows past the end as zeros: what is there may be anything)
            {
                const int piece = lane % PIECES, key = lane / PIECES;
#pragma unroll
                for (int i = 0; i < VL; ++i) {
                    const int k = key + PASS * i, sw = swizzle<DIM>(k);
                    if constexpr (Q8) {
                        const uintx2 a = codes_to_half(vr[i][0]), c = codes_to_half(vr[i][1]);
                        const uintx2 d = codes_to_half(vr[i][2]), e = codes_to_half(vr[i][3]);
                        *(uintx4*)(vt + k * ROW + ((2 * piece) ^ sw) * 16) = uintx4{a[0], a[1], c[0], c[1]};
                        *(uintx4*)(vt + k * ROW + ((2 * piece + 1) ^ sw) * 16) = uintx4{d[0], d[1], e[0], e[1]};
                    } else {
                        const bool there = !edge || block * 32 + k < keys;
                        *(uintx4*)(vt + k * ROW + (piece ^ sw) * 16) = there ? vr[i] : uintx4{0, 0, 0, 0};
                    }
                }
            }
            load_v(ra, rb);
            if (__any(mx - m > ATTEND_GROWTH)) {
                mx = fmaxf(mx, __shfl_xor(mx, 16));
                mx = fmaxf(mx, __shfl_xor(mx, 32));
                const float mn = fmaxf(m, mx);
                const float a = mn == -INFINITY ? 1.0f : __builtin_amdgcn_exp2f(m - mn);
                m = mn;
                l *= a;
#pragma unroll
                for (int d = 0; d < DB; ++d)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[d][e] *= a;
            }
            if (__any(exponent_far(m))) {
#pragma unroll
                for (int j = 0; j < 2; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[j][e] = exponent_far(m) ? s[j][e] - m : s[j][e];
            }
            const float ref = exponent_base<M>(m);
            vec8 pb;
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float pr = __builtin_amdgcn_exp2f(s[j][e] - ref);
                    if constexpr (Q8) l = fmaf(pr, vinv[j][e], l);
                    else l += pr;
                    pb[4 * j + e] = (typename M::elem)pr;
                }
            // O^T += V^T P^T (LDS of one wave is in order; the fences are the compiler's)
            asm volatile("" ::: "memory");
            const int i = lane & 15, ka = 4 * g + (i >> 2), kb = 16 + ka;
            const int swa = swizzle<DIM>(ka), swb = swizzle<DIM>(kb);
            const uint8_t* pa = vt + ka * ROW + (i & 1) * 8;
            const uint8_t* pc = vt + kb * ROW + (i & 1) * 8;
#pragma unroll
            for (int d = 0; d < DB; ++d) {
                const int piece = 2 * d + ((i & 3) >> 1);
                const vec4 lo = lds_transposed<vec4>(pa + (piece ^ swa) * 16);
                const vec4 hi = lds_transposed<vec4>(pc + (piece ^ swb) * 16);
                o[d] = M::mfma16(__builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7), pb, o[d]);
            }
            asm volatile("" ::: "memory");
        }
    }

    // ---- the four waves joined
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    __syncthreads();   // (the waves' V tiles are done with)
    float* po = (float*)lds;
#pragma unroll
    for (int d = 0; d < DB; ++d) *(floatx4*)(po + (wave * 16 + col) * PAD + 16 * d + 4 * g) = o[d];
    if (g == 0) {
        s_m[wave][col] = m;
        s_l[wave][col] = l;
    }
    __syncthreads();
    constexpr int LANES = DIM / 4;   // of an output row
    for (int r = tid / LANES; r < p.group; r += 256 / LANES) {
        const int c = (tid % LANES) * 4;
        float top = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) top = fmaxf(top, s_m[w][r]);
        const float ref = top == -INFINITY ? 0.0f : top;
        floatx4 sum = {0, 0, 0, 0};
        float total = 0.0f;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const float f = __builtin_amdgcn_exp2f(s_m[w][r] - ref);
            if (s_m[w][r] == -INFINITY && s_l[w][r] == 0.0f) continue;   // a wave without keys
            total = fmaf(f, s_l[w][r], total);
            const floatx4 v = *(const floatx4*)(po + (w * 16 + r) * PAD + c);
#pragma unroll
            for (int e = 0; e < 4; ++e) sum[e] = fmaf(f, v[e], sum[e]);
        }
        const int64_t out_row = (int64_t)b * p.heads + kvh * p.group + r;
        top = exponent_seen(top, total, block0 < block1);
        if (p.splits > 1) {
            const int64_t at = (int64_t)split * p.tokens * p.heads + out_row;
            *(floatx4*)(p.part_o + at * DIM + c) = sum;
            if (c == 0) {
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
        uint16_t* out = (uint16_t*)p.out + out_row * DIM + c;
        if constexpr (QT == MIX_F16)
            *(half4*)out = half4{(_Float16)sum[0], (_Float16)sum[1], (_Float16)sum[2], (_Float16)sum[3]};
        else
            *(bfloat4*)out = bfloat4{(__bf16)sum[0], (__bf16)sum[1], (__bf16)sum[2], (__bf16)sum[3]};
        if (!finite) atomicOr(&p.flags[FLAG_NONFINITE], 1);
    }
}

template <int DIM, int CACHE, int QT>
static hipError_t launch_token_of(const AttendParams& p, hipStream_t s) {
    constexpr int bytes = 4 * 16 * (DIM + 4) * 4;
    static_assert(bytes >= 4 * 32 * DIM * 2, "the waves' V tiles fit under the joined rows");
    hipLaunchKernelGGL((k_attend_token<DIM, CACHE, QT>), dim3((unsigned)(p.seqs * p.kv_heads), (unsigned)p.splits),
                       dim3(256), bytes, s, p);
    return hipGetLastError();
}

template <int DIM>
static hipError_t launch_token_dim(const AttendParams& p, hipStream_t s) {
    if (p.cache_type == MIX_F16) return launch_token_of<DIM, MIX_F16, MIX_F16>(p, s);
    if (p.cache_type == MIX_BF16) return launch_token_of<DIM, MIX_BF16, MIX_BF16>(p, s);
    if (p.q_type == MIX_F16) return launch_token_of<DIM, MIX_Q8, MIX_F16>(p, s);
    return launch_token_of<DIM, MIX_Q8, MIX_BF16>(p, s);
}

hipError_t launch_attend_token(const AttendParams& p, hipStream_t s) {
    switch (p.dim) {
        case 64: return launch_token_dim<64>(p, s);
        case 128: return launch_token_dim<128>(p, s);
        case 256: return launch_token_dim<256>(p, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace mqh
