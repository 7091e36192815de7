// linear_step.hip -- one token of every sequence through linear attention with a
// decay per head, with the delta rule or without:
//   S <- e^gate S;  u = beta (v - S k) or v;  S <- S + u k^T;  out = S q
// for S [value_dim x key_dim] FP32 of each sequence and head, in place.
//
// Bound by memory: the state once in, once out.  key_dim / 4 lanes (a power of
// two of them) own a row, four columns each, so rows are read and written in
// 16-byte pieces and the row stays in registers between.  Both dot products are
// taken of the state as read, S q = e^gate (S q) + u (k q), so one pass of lane
// sums serves them.  A wave takes 16 rows of one head and has all their loads in
// flight.  Everything is FP32; 16-bit q, k and v are exact in it.  64 sequences of 32
// x 128 x 128, FP32: 57 us over changing states, 4.8 TB/s (a large copy: 4.9).

#include "mixers.h"

namespace mqh {

template <int LANES, int TYPE, bool DELTA>
__global__ __launch_bounds__(256) void k_linear_step(LinearParams p) {
    constexpr int AT_ONCE = 64 / LANES;                  // rows a wave reads with one instruction
    constexpr int PASSES = LANES >= 4 ? LANES / 4 : 1;   // 16 rows a wave
    constexpr int ROWS = AT_ONCE * PASSES;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int row_waves = (p.value_dim + ROWS - 1) / ROWS;
    const int64_t unit = (int64_t)blockIdx.x * 4 + wave;   // (sequence, head, 16 rows)
    const int64_t sh = unit / row_waves;
    if (sh >= (int64_t)p.seqs * p.heads) return;
    const int seq = (int)(sh / p.heads), head = (int)(sh - (int64_t)seq * p.heads);
    const int row0 = (int)(unit - sh * row_waves) * ROWS + lane / LANES;
    const int key_head = head / (p.heads / p.key_heads);
    const int col = (lane % LANES) * 4;
    const bool cols = col < p.key_dim;

    floatx4 k4 = {0, 0, 0, 0}, q4 = {0, 0, 0, 0};
    if (cols) {
        k4 = load4<TYPE>(p.k, seq * p.k_token + key_head * p.k_head + col);
        q4 = load4<TYPE>(p.q, seq * p.q_token + key_head * p.q_head + col);
    }
    float* state = p.state + sh * p.value_dim * p.key_dim + col;
    floatx4 s[PASSES];
    float v[PASSES];
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        const int row = min(row0 + AT_ONCE * i, p.value_dim - 1);
        s[i] = cols ? *(const floatx4*)(state + (int64_t)row * p.key_dim) : floatx4{0, 0, 0, 0};
        v[i] = load1<TYPE>(p.v, seq * p.v_token + head * p.v_head + row);
    }
    const float decay = expf(p.gate[seq * p.gate_token + head]);
    const float beta = DELTA ? p.beta[seq * p.beta_token + head] : 1.0f;
    float kq = 0.0f;
#pragma unroll
    for (int e = 0; e < 4; ++e) kq = fmaf(k4[e], q4[e], kq);
    kq = lane_sum<LANES>(kq);
    bool finite = true;
#pragma unroll
    for (int i = 0; i < PASSES; ++i) {
        float sq = 0.0f, sk = 0.0f;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            sq = fmaf(s[i][e], q4[e], sq);
            if constexpr (DELTA) sk = fmaf(s[i][e], k4[e], sk);
        }
        sq = lane_sum<LANES>(sq);
        float u = v[i];
        if constexpr (DELTA) u = beta * (u - decay * lane_sum<LANES>(sk));
#pragma unroll
        for (int e = 0; e < 4; ++e) s[i][e] = fmaf(u, k4[e], s[i][e] * decay);
        const int row = row0 + AT_ONCE * i;
        if (row >= p.value_dim) continue;
        if (cols) *(floatx4*)(state + (int64_t)row * p.key_dim) = s[i];
        if (lane % LANES == 0) {
            const float out = fmaf(u, kq, decay * sq);
            store1<TYPE>(p.out, sh * p.value_dim + row, out);
            finite &= fits<TYPE>(out);
        }
    }
    if (!finite) atomicOr(&p.flags[FLAG_NONFINITE], 1);
}

template <int LANES, int TYPE>
static hipError_t launch_step_of(const LinearParams& p, hipStream_t s) {
    constexpr int ROWS = (64 / LANES) * (LANES >= 4 ? LANES / 4 : 1);
    const int64_t units = (int64_t)p.seqs * p.heads * ((p.value_dim + ROWS - 1) / ROWS);
    const dim3 grid((unsigned)((units + 3) / 4));
    if (p.beta) hipLaunchKernelGGL((k_linear_step<LANES, TYPE, true>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((k_linear_step<LANES, TYPE, false>), grid, dim3(256), 0, s, p);
    return hipGetLastError();
}

template <int TYPE>
static hipError_t launch_step_type(const LinearParams& p, hipStream_t s) {
    if (p.key_dim <= 16) return launch_step_of<4, TYPE>(p, s);
    if (p.key_dim <= 32) return launch_step_of<8, TYPE>(p, s);
    if (p.key_dim <= 64) return launch_step_of<16, TYPE>(p, s);
    if (p.key_dim <= 128) return launch_step_of<32, TYPE>(p, s);
    return launch_step_of<64, TYPE>(p, s);
}

hipError_t launch_linear_step(const LinearParams& p, hipStream_t s) {
    switch (p.type) {
        case MIX_F32: return launch_step_type<MIX_F32>(p, s);
        case MIX_F16: return launch_step_type<MIX_F16>(p, s);
        case MIX_BF16: return launch_step_type<MIX_BF16>(p, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace mqh
