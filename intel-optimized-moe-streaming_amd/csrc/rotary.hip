// rotary.hip -- rotary positions of queries and keys: each pair (a, b) of a head's
// first `rotary` channels is turned by its position's angle,
//   (a, b) -> (a cos - b sin, a sin + b cos),  angle = position * frequency,
// pairs being halves (i, i + rotary / 2) or neighbours (2 i, 2 i + 1); before it,
// where weights are given, the head's row goes through x / sqrt(mean x^2 + eps) * w.
// All in FP32, rounded once; rows whose squares may pass FP32 take the norm of numbers
// 2^96 times smaller, in a branch of their own (84 registers at FP32 where 79 were: heads
// of 256 normed 34.5 -> 35.7 us; 16-bit rows are no slower).
//
// An angle far out needs more than FP32 (a million radians in FP32 are off by
// 0.06).  Frequencies are held as turns a position in units of 2^-64, so that the
// 64-bit product with the position drops whole turns by itself; its upper 32 bits
// are the angle to 2^-32 of a turn.  An eighth of a turn either way is left by the
// quadrant, where Taylor's series to the ninth and tenth power are exact to FP32.
//
// Rows of position -1 are what a page table gives to a batch's padding: whatever they
// hold (a layer before may have left them as they were) is turned, but not reported.
//
// Bound by memory: rows are read and written once.  dim / 8 lanes own a row, eight
// channels each; a workgroup takes the same few tokens of several heads, so that
// the sines are computed once for all of them.  16,384 tokens of 32 + 8 heads of 128,
// BF16: 70 us, 4.8 TB/s (a large copy reaches 4.7 to 4.8); 4,099 FP32 tokens of 16 + 2
// heads of 256, normed: 35.5 us, 4.3 TB/s.  64 tokens: 5 us, two round trips and the sines.

#include "mixers.h"

namespace mqh {

__device__ __forceinline__ void cos_sin(int position, uint64_t turns, float& c, float& s) {
    const uint32_t lo = (uint32_t)turns, hi = (uint32_t)(turns >> 32);
    uint32_t t = __umulhi((uint32_t)position, lo) + (uint32_t)position * hi;
    if (position < 0) t -= lo;   // (the product took it as 2^32 more)
    const uint32_t quadrant = (t + 0x20000000u) >> 30;
    const float x = (float)(int32_t)(t - (quadrant << 30)) * 1.4629180792671596e-9f;   // 2 pi / 2^32
    const float y = x * x;
    const float sn = fmaf(x * y, fmaf(y, fmaf(y, fmaf(y, 1.0f / 362880, -1.0f / 5040), 1.0f / 120), -1.0f / 6), x);
    const float cs = fmaf(y, fmaf(y, fmaf(y, fmaf(y, fmaf(y, -1.0f / 3628800, 1.0f / 40320), -1.0f / 720), 1.0f / 24), -0.5f), 1.0f);
    const bool swap = quadrant & 1;
    c = swap ? sn : cs;
    s = swap ? cs : sn;
    if (((quadrant + 1) & 2)) c = -c;
    if (quadrant & 2) s = -s;
}

template <int DIM, int TYPE>
__global__ __launch_bounds__(256) void k_rotary(RotaryParams p) {
    constexpr int LANES = DIM / 8, ROWS = 256 / LANES, N = 4;   // heads in flight
    const int lane = threadIdx.x % LANES, c0 = 8 * lane;
    const int64_t token = (int64_t)blockIdx.x * ROWS + threadIdx.x / LANES;
    const bool live = token < p.tokens;
    const int64_t at = live ? token : p.tokens - 1;
    const int head0 = blockIdx.y * p.per, head1 = min(head0 + p.per, p.heads + p.kv_heads);
    const int half = p.rotary >> 1;
    const bool turned = c0 < p.rotary;
    const int position = p.positions[at];
    // halves: out = x cos + partner * sin (-sin in the first half), the partner's lane
    // rotary / 16 on; neighbours: cos and sin of four pairs, twice
    float cs[8], sn[8];
    int partner = threadIdx.x & 63;
    if (turned) {
        if (p.interleaved) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                cos_sin(position, p.turns[c0 / 2 + i], cs[2 * i], sn[2 * i + 1]);
                cs[2 * i] *= p.amplitude;
                sn[2 * i + 1] *= p.amplitude;
                cs[2 * i + 1] = cs[2 * i];
                sn[2 * i] = -sn[2 * i + 1];
            }
        } else {
            const bool low = c0 < half;
            partner += low ? half / 8 : -(half / 8);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                cos_sin(position, p.turns[c0 - (low ? 0 : half) + i], cs[i], sn[i]);
                cs[i] *= p.amplitude;
                sn[i] *= low ? -p.amplitude : p.amplitude;
            }
        }
    }
    for (int h0 = head0; h0 < head1; h0 += N) {
        float x[N][8];
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int h = min(h0 + n, head1 - 1);
            if (h < p.heads) load8<TYPE>(p.q, at * p.q_token + (int64_t)h * p.q_head + c0, x[n]);
            else load8<TYPE>(p.k, at * p.k_token + (int64_t)(h - p.heads) * p.k_head + c0, x[n]);
        }
#pragma unroll
        for (int n = 0; n < N; ++n) {
            const int h = h0 + n;
            const float* w = h < p.heads ? p.q_weight : p.k_weight;
            if (w && h < head1) {
                float sum = 0.0f;
#pragma unroll
                for (int i = 0; i < 8; ++i) sum = fmaf(x[n][i], x[n][i], sum);
                sum = lane_sum<LANES>(sum);
                float r = 1.0f / sqrtf(sum * (1.0f / DIM) + p.eps);
                // rows whose squares may be past FP32: the same of numbers 2^96 times smaller
                const bool past = !(sum <= 0x1p120f);
                if (__any(past)) {
                    constexpr float DOWN = 0x1p-96f;
                    float part = 0.0f;
#pragma unroll
                    for (int i = 0; i < 8; ++i) part = fmaf(x[n][i] * DOWN, x[n][i] * DOWN, part);
                    part = lane_sum<LANES>(part);
                    part = 1.0f / sqrtf(part * (1.0f / DIM) + p.eps * DOWN * DOWN);
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[n][i] = past ? x[n][i] * part * DOWN : x[n][i];
                    r = past ? 1.0f : r;
                }
                // (by the norm first: its product with a weight may lie where FP32 has no numbers)
#pragma unroll
                for (int i = 0; i < 8; ++i) x[n][i] = x[n][i] * r * w[c0 + i];
            }
            float y[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) y[i] = p.interleaved ? x[n][i ^ 1] : __shfl(x[n][i], partner);
            bool finite = true;
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                if (turned) x[n][i] = fmaf(x[n][i], cs[i], y[i] * sn[i]);
                finite &= fits<TYPE>(x[n][i]);
            }
            if (!live || h >= head1) continue;
            if (h < p.heads) store8<TYPE>(p.q_out, token * p.qo_token + (int64_t)h * p.qo_head + c0, x[n]);
            else store8<TYPE>(p.k_out, token * p.ko_token + (int64_t)(h - p.heads) * p.ko_head + c0, x[n]);
            if (!finite && position != -1) atomicOr(&p.flags[FLAG_NONFINITE], 1);
        }
    }
}

template <int DIM, int TYPE>
static hipError_t launch_rotary_of(RotaryParams p, hipStream_t s) {
    constexpr int ROWS = 256 / (DIM / 8);
    const int groups = (p.tokens + ROWS - 1) / ROWS, total = p.heads + p.kv_heads;
    // heads of a workgroup: enough workgroups for eight a CU, or four heads
    const int parts = std::max(1, std::min((total + 3) / 4, (2048 + groups - 1) / groups));
    p.per = (total + parts - 1) / parts;
    hipLaunchKernelGGL((k_rotary<DIM, TYPE>), dim3((unsigned)groups, (unsigned)((total + p.per - 1) / p.per)), dim3(256), 0,
                       s, p);
    return hipGetLastError();
}

template <int DIM>
static hipError_t launch_rotary_dim(const RotaryParams& p, hipStream_t s) {
    switch (p.type) {
        case MIX_F32: return launch_rotary_of<DIM, MIX_F32>(p, s);
        case MIX_F16: return launch_rotary_of<DIM, MIX_F16>(p, s);
        case MIX_BF16: return launch_rotary_of<DIM, MIX_BF16>(p, s);
    }
    return hipErrorInvalidValue;
}

hipError_t launch_rotary(RotaryParams p, hipStream_t s) {
    switch (p.dim) {
        case 64: return launch_rotary_dim<64>(p, s);
        case 128: return launch_rotary_dim<128>(p, s);
        case 256: return launch_rotary_dim<256>(p, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace mqh
