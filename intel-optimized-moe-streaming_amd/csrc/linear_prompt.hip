// linear_prompt.hip -- a prompt through linear attention with a decay per head,
// with the delta rule or without, in chunks of 64 tokens.
//
// With G_i the running sum of the gate in a chunk, S0 the state before it:
//   (1 + L) U = diag(beta) V - diag(beta e^G) K S0^T,  L_ij = beta_i e^(G_i - G_j) k_i.k_j  (j < i)
//   O = diag(e^G) Q S0^T + M U,                        M_ij = e^(G_i - G_j) q_i.k_j          (j <= i)
//   S1 = e^(G_C) S0 + (diag(e^(G_C - G)) U)^T K
// (U = V without the delta rule).  Only U and S1 need the chunks in order, so
// three launches share the work:
//   1 k_linear_solve   chunks in parallel: W = (1 + L)^-1 diag(beta e^G) K and
//                      (1 + L)^-1 diag(beta) V
//   2 k_linear_scan    chunk after chunk, 16 value rows of a head a workgroup:
//                      U = (1 + L)^-1 diag(beta) V - W S0^T, then S1
//   3 k_linear_out     chunks in parallel: O
// Everything is FP32 on FP32 matrix instructions (16x16x4); the sums G are taken
// in double, so that differences of far gates keep their digits, and a gate
// below -1e4 counts as that (its exponential is 0 either way).  The triangular
// system is solved by substitution, block by block of 16 rows: powers of L would
// cancel where keys repeat.
//
// Operand layout.  The 16x16x4 instruction leaves row 4 g + r, column l % 16 of
// its result in register r of lane l = 16 g + l % 16, and takes element (row or
// column l % 16, k = g) of an operand from lane l.  Four instructions that take
// k = 4 g + j (j = 0..3) contract 16 of them, with the operand's four consecutive
// elements in one 16-byte load and, for the right one, register j of a result as
// it stands.  So U goes from result to operand without moving, and so does the
// state: S^T tiles are both the accumulators of S1 and the operand of W S0^T.

#include "mixers.h"

namespace mqh {

constexpr int C = LINEAR_CHUNK;

__device__ __forceinline__ floatx4 mfma4(floatx4 a, floatx4 b, floatx4 c) {
#pragma unroll
    for (int j = 0; j < 4; ++j) c = __builtin_amdgcn_mfma_f32_16x16x4f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

struct ChunkRange {
    int seq, first, count;   // its tokens [first, first + count), count <= 64, 0: none
    int at;                  // its index in the workspace
};

__device__ __forceinline__ void sequence_bounds(const LinearParams& p, int b, int& s0, int& s1, bool report) {
    s0 = 0;
    s1 = p.tokens;
    if (!p.starts) return;
    const int a = p.starts[b], z = p.starts[b + 1];
    s0 = min(max(a, 0), p.tokens);
    s1 = min(max(z, s0), p.tokens);
    if (report && (a < 0 || z < a || z > p.tokens)) atomicOr(&p.flags[FLAG_BAD_ID], 1);
}

// the sequence and tokens of chunk p.chunk0 + at
__device__ __forceinline__ ChunkRange chunk_range(const LinearParams& p, int at) {
    const int lane = threadIdx.x & 63, chunk = p.chunk0 + at;
    ChunkRange r = {0, 0, 0, at};
    if (p.starts) {
        int b = -1;
        for (int i0 = 0; i0 < p.seqs; i0 += 64) {
            const int i = i0 + lane;
            const bool le = i < p.seqs && min(max(p.starts[i], 0), p.tokens) / C + i <= chunk;
            b += __builtin_popcountll(__ballot(le));
        }
        if (b < 0) return r;
        r.seq = __builtin_amdgcn_readfirstlane(b);
    }
    int s0, s1;
    sequence_bounds(p, r.seq, s0, s1, threadIdx.x == 0);
    const int begin = (chunk - (s0 / C + r.seq)) * C;
    r.first = s0 + begin;
    r.count = begin < 0 ? 0 : min(max(s1 - r.first, 0), C);
    return r;
}

// running sums of the gate over the chunk: lane t has token t's (past the end:
// the last one's)
__device__ __forceinline__ double gate_sums(const LinearParams& p, const ChunkRange& c, int head) {
    const int lane = threadIdx.x & 63;
    double g = 0.0;
    if (lane < c.count) {
        const float x = p.gate[(int64_t)(c.first + lane) * p.gate_token + head];
        g = x < -1e4f ? -1e4 : (double)x;
    }
#pragma unroll
    for (int d = 1; d < 64; d <<= 1) {
        const double o = __shfl_up(g, d);
        if (lane >= d) g += o;
    }
    return g;
}

// what the other two kernels read of the gate, by one wave
__device__ __forceinline__ void store_gates(const LinearParams& p, int64_t ch, double g) {
    const int lane = threadIdx.x & 63;
    const double end = __shfl(g, 63);
    p.g[ch * C + lane] = g;
    p.e[ch * 128 + lane] = expf((float)(end - g));
    if (lane == 63) p.e[ch * 128 + 64] = expf((float)end);
}

// without the delta rule: the gates are all there is to prepare
__global__ __launch_bounds__(256) void k_linear_gates(LinearParams p) {
    const int64_t ch = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (ch >= (int64_t)p.chunks * p.heads) return;
    const ChunkRange c = chunk_range(p, (int)(ch / p.heads));
    if (!c.count) return;
    store_gates(p, ch, gate_sums(p, c, (int)(ch % p.heads)));
}

// rows of a chunk into LDS as FP32 [64][KP + 4], zeros past its end and key_dim
template <int KP, int TYPE>
__device__ __forceinline__ void stage_rows(const LinearParams& p, const ChunkRange& c, const void* x, int64_t token,
                                           int64_t head_at, float* to) {
    constexpr int PIECES = KP / 4;
#pragma unroll 4
    for (int i = threadIdx.x; i < C * PIECES; i += 256) {
        const int t = i / PIECES, col = (i % PIECES) * 4;
        floatx4 v = {0, 0, 0, 0};
        if (t < c.count && col < p.key_dim) v = load4<TYPE>(x, (int64_t)(c.first + t) * token + head_at + col);
        *(floatx4*)(to + t * (KP + 4) + col) = v;
    }
}

// tiles (i, j <= i) of a 4 x 4 block triangle, wave w taking the w-th of every four
__device__ __forceinline__ void triangle_tile(int n, int& i, int& j) {
    i = n >= 6 ? 3 : n >= 3 ? 2 : n >= 1 ? 1 : 0;
    j = n - i * (i + 1) / 2;
}

// 16x16 tile (rows 16 i of a, rows 16 j of b) of a b^T, both in LDS
template <int KP>
__device__ __forceinline__ floatx4 tile_product(const float* a, const float* b, int i, int j) {
    const int lane = threadIdx.x & 63, l16 = lane & 15, g = lane >> 4;
    floatx4 acc = {0, 0, 0, 0};
    const float* pa = a + (16 * i + l16) * (KP + 4) + 4 * g;
    const float* pb = b + (16 * j + l16) * (KP + 4) + 4 * g;
#pragma unroll
    for (int k = 0; k < KP; k += 16) acc = mfma4(*(const floatx4*)(pa + k), *(const floatx4*)(pb + k), acc);
    return acc;
}

constexpr int LS = C + 4;   // row stride of the 64 x 64 matrices in LDS

// ---- 1: W and (1 + L)^-1 diag(beta) V of a chunk of a head
template <int KP, int TYPE>
__global__ __launch_bounds__(256) void k_linear_solve(LinearParams p) {
    extern __shared__ __align__(16) float lds[];
    float* sk = lds;                       // [64][KP + 4]
    float* sl = sk + C * (KP + 4);         // [64][LS]: -L
    float* st = sl + C * LS;               // [4][16][20]: inverses of the diagonal blocks of 1 + L
    __shared__ double s_g[C];
    __shared__ __align__(16) float s_beta[C], s_through[C];   // beta, beta e^G

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g = lane >> 4;
    const int64_t ch = blockIdx.x;
    const int head = (int)(ch % p.heads), key_head = head / (p.heads / p.key_heads);
    const ChunkRange c = chunk_range(p, (int)(ch / p.heads));
    if (!c.count) return;

    stage_rows<KP, TYPE>(p, c, p.k, p.k_token, key_head * p.k_head, sk);
    if (wave == 0) {
        const double sum = gate_sums(p, c, head);
        const float beta = lane < c.count ? p.beta[(int64_t)(c.first + lane) * p.beta_token + head] : 0.0f;
        s_g[lane] = sum;
        s_beta[lane] = beta;
        s_through[lane] = beta * expf((float)sum);
        store_gates(p, ch, sum);
    }
    __syncthreads();

    for (int n = wave; n < 10; n += 4) {
        int i, j;
        triangle_tile(n, i, j);
        const floatx4 d = tile_product<KP>(sk, sk, i, j);
        const int tj = 16 * j + l16;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int ti = 16 * i + 4 * g + r;
            sl[ti * LS + tj] = tj < ti ? -s_beta[ti] * expf((float)(s_g[ti] - s_g[tj])) * d[r] : 0.0f;
        }
    }
    __syncthreads();

    // column l16 of the inverse of diagonal block `wave`, by substitution
    {
        float x[16];
        const float* rows = sl + 16 * wave * LS + 16 * wave;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            x[i] = i == l16 ? 1.0f : 0.0f;
#pragma unroll
            for (int j = 0; j < i; ++j) x[i] = fmaf(rows[i * LS + j], x[j], x[i]);
            if (g == 0) st[(wave * 16 + i) * 20 + l16] = x[i];
        }
    }
    __syncthreads();

    // left operands: -L below the diagonal blocks, the diagonal inverses
    floatx4 lo[6], inv[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        inv[i] = *(const floatx4*)(st + (16 * i + l16) * 20 + 4 * g);
#pragma unroll
        for (int j = 0; j < i; ++j)
            lo[i * (i - 1) / 2 + j] = *(const floatx4*)(sl + (16 * i + l16) * LS + 16 * j + 4 * g);
    }
    const int vp = (p.value_dim + 15) & ~15;
    float* w = p.w + ch * C * KP;
    float* u = p.u + ch * C * vp;
    for (int n = wave; n < KP / 16 + vp / 16; n += 4) {
        const bool is_v = n >= KP / 16;
        const int col = 16 * (is_v ? n - KP / 16 : n) + l16;
        floatx4 x[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const floatx4 f = *(const floatx4*)((is_v ? s_beta : s_through) + 16 * i + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * i + 4 * g + r;
                float v = 0.0f;
                if (!is_v) v = sk[t * (KP + 4) + col];
                else if (t < c.count && col < p.value_dim)
                    v = load1<TYPE>(p.v, (int64_t)(c.first + t) * p.v_token + head * p.v_head + col);
                x[i][r] = v * f[r];
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            floatx4 acc = x[i];
#pragma unroll
            for (int j = 0; j < i; ++j) acc = mfma4(lo[i * (i - 1) / 2 + j], x[j], acc);
            x[i] = mfma4(inv[i], acc, floatx4{0, 0, 0, 0});
            if (is_v) *(floatx4*)(u + (int64_t)col * C + 16 * i + 4 * g) = x[i];
            else
#pragma unroll
                for (int r = 0; r < 4; ++r) w[(16 * i + 4 * g + r) * KP + col] = x[i][r];
        }
    }
}

// ---- 2: the state from chunk to chunk, 16 value rows of a head
template <int KP, int TYPE, bool DELTA>
__global__ __launch_bounds__(256, 1) void k_linear_scan(LinearParams p) {
    constexpr int KW = KP / 4;       // key columns of a wave
    constexpr int NB = KW / 16;
    __shared__ __align__(16) floatx4 part[2][4][4][64];   // W S0^T over each wave's columns, by turns

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g = lane >> 4;
    // the value tiles of a head run on one XCD (workgroups go round the eight), so
    // that its W and K are read into one L2
    const int vt = (p.value_dim + 15) / 16;
    const int sh = blockIdx.x / (8 * vt) * 8 + (blockIdx.x & 7), tile = (blockIdx.x / 8) % vt;
    if (sh >= p.seqs * p.heads) return;
    const int b = sh / p.heads, head = sh % p.heads, key_head = head / (p.heads / p.key_heads);
    int s0, s1;
    sequence_bounds(p, b, s0, s1, tid == 0);
    // this pass's chunks of the sequence
    const int base = (p.starts ? s0 / C + b : 0) - p.chunk0, count = (s1 - s0 + C - 1) / C;
    const int n0 = max(0, -base), n1 = min(count, p.chunks - base);
    if (n0 >= n1) return;

    const int row = 16 * tile + l16, vp = 16 * vt;
    const bool row_live = row < p.value_dim;
    const int kc = wave * KW;
    float* state = p.state + ((int64_t)sh * p.value_dim + (row_live ? row : 0)) * p.key_dim;
    floatx4 s[NB];   // S^T: columns kc + 16 n + 4 g + r of row `row`
#pragma unroll
    for (int n = 0; n < NB; ++n) {
        const int col = kc + 16 * n + 4 * g;
        s[n] = row_live && col < p.key_dim ? *(const floatx4*)(state + col) : floatx4{0, 0, 0, 0};
    }

    floatx4 w[DELTA ? 4 : 1][NB], k[4][NB], u[4], e[4];
    float end;
    auto load = [&](int n) {
        const int64_t ch = (int64_t)(base + n) * p.heads + head;
        const int first = s0 + n * C, left = min(s1 - first, C);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            e[i] = *(const floatx4*)(p.e + ch * 128 + 16 * i + 4 * g);
            if constexpr (DELTA) {
                u[i] = *(const floatx4*)(p.u + (ch * vp + row) * C + 16 * i + 4 * g);
#pragma unroll
                for (int m = 0; m < NB; ++m)
                    w[i][m] = *(const floatx4*)(p.w + (ch * C + 16 * i + l16) * KP + kc + 16 * m + 4 * g);
            }
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * i + 4 * g + r;
                const bool there = t < left;
                const int64_t token = first + (there ? t : 0);
                if constexpr (!DELTA) {
                    const float v = load1<TYPE>(p.v, token * p.v_token + head * p.v_head + (row_live ? row : 0));
                    u[i][r] = there && row_live ? v : 0.0f;
                }
#pragma unroll
                for (int m = 0; m < NB; ++m) {
                    const int col = kc + 16 * m + l16;
                    const float v = load1<TYPE>(p.k, token * p.k_token + key_head * p.k_head + (col < p.key_dim ? col : 0));
                    k[i][m][r] = there && col < p.key_dim ? v : 0.0f;
                }
            }
        }
        end = p.e[ch * 128 + 64];
    };
    load(n0);
    for (int n = n0; n < n1; ++n) {
        const int64_t ch = (int64_t)(base + n) * p.heads + head;
        float* kept = p.s0 + (ch * vp + row) * KP + kc + 4 * g;
#pragma unroll
        for (int m = 0; m < NB; ++m) *(floatx4*)(kept + 16 * m) = s[m];
        if constexpr (DELTA) {
            floatx4(*mine)[64] = part[n & 1][wave];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                floatx4 x = {0, 0, 0, 0};
#pragma unroll
                for (int m = 0; m < NB; ++m) x = mfma4(w[i][m], s[m], x);
                mine[i][lane] = x;
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                floatx4 x = part[n & 1][0][i][lane];
#pragma unroll
                for (int v = 1; v < 4; ++v) x += part[n & 1][v][i][lane];
                u[i] -= x;
            }
            // (the waves share the writing of U: 16 tokens each)
            floatx4 own = u[0];
#pragma unroll
            for (int i = 1; i < 4; ++i) own = wave == i ? u[i] : own;
            *(floatx4*)(p.u + (ch * vp + row) * C + 16 * wave + 4 * g) = own;
        }
        floatx4 ue[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) ue[i] = u[i] * e[i];
#pragma unroll
        for (int m = 0; m < NB; ++m) s[m] *= end;
        // (the next chunk's loads go out behind this one's last use of each register)
#pragma unroll
        for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int m = 0; m < NB; ++m) s[m] = mfma4(k[i][m], ue[i], s[m]);
        if (n + 1 < n1) load(n + 1);
    }
    if (row_live)
#pragma unroll
        for (int n = 0; n < NB; ++n) {
            const int col = kc + 16 * n + 4 * g;
            if (col < p.key_dim) *(floatx4*)(state + col) = s[n];
        }
}

// ---- 3: the outputs of a chunk of a head
template <int KP, int TYPE, bool DELTA>
__global__ __launch_bounds__(256) void k_linear_out(LinearParams p) {
    extern __shared__ __align__(16) float lds[];
    float* sq = lds;                    // [64][KP + 4]
    float* sk = sq + C * (KP + 4);      // [64][KP + 4], then M [64][LS]
    __shared__ double s_g[C];
    __shared__ __align__(16) float s_from[C];   // e^G

    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, l16 = lane & 15, g = lane >> 4;
    const int64_t ch = blockIdx.x;
    const int head = (int)(ch % p.heads), key_head = head / (p.heads / p.key_heads);
    const ChunkRange c = chunk_range(p, (int)(ch / p.heads));
    if (!c.count) return;
    stage_rows<KP, TYPE>(p, c, p.q, p.q_token, key_head * p.q_head, sq);
    stage_rows<KP, TYPE>(p, c, p.k, p.k_token, key_head * p.k_head, sk);
    if (wave == 0) {
        const double sum = p.g[ch * C + lane];
        s_g[lane] = sum;
        s_from[lane] = expf((float)sum);
    }
    __syncthreads();
    floatx4 m[3];
#pragma unroll
    for (int n = 0; n < 3; ++n) {
        int i, j;
        if (wave + 4 * n >= 10) break;
        triangle_tile(wave + 4 * n, i, j);
        m[n] = tile_product<KP>(sq, sk, i, j);
    }
    __syncthreads();   // (M goes where K was)
#pragma unroll
    for (int n = 0; n < 3; ++n) {
        int i, j;
        if (wave + 4 * n >= 10) break;
        triangle_tile(wave + 4 * n, i, j);
        const int tj = 16 * j + l16;
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            const int ti = 16 * i + 4 * g + r;
            sk[ti * LS + tj] = tj <= ti ? expf((float)(s_g[ti] - s_g[tj])) * m[n][r] : 0.0f;
        }
    }
    __syncthreads();

    const int vp = (p.value_dim + 15) & ~15;
    const float* state = p.s0 + ch * vp * KP;
    bool finite = true;
    for (int n = wave; n < vp / 16; n += 4) {
        const int row = 16 * n + l16;
        const bool row_live = row < p.value_dim;
        floatx4 acc[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) acc[i] = floatx4{0, 0, 0, 0};
        const float* srow = state + (int64_t)row * KP + 4 * g;
#pragma unroll 4
        for (int k = 0; k < KP; k += 16) {
            const floatx4 s4 = *(const floatx4*)(srow + k);
#pragma unroll
            for (int i = 0; i < 4; ++i)
                acc[i] = mfma4(*(const floatx4*)(sq + (16 * i + l16) * (KP + 4) + k + 4 * g), s4, acc[i]);
        }
        floatx4 u[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (DELTA) {
                u[i] = *(const floatx4*)(p.u + (ch * vp + row) * C + 16 * i + 4 * g);
            } else {
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int t = 16 * i + 4 * g + r;
                    u[i][r] = t < c.count && row_live
                                  ? load1<TYPE>(p.v, (int64_t)(c.first + t) * p.v_token + head * p.v_head + row)
                                  : 0.0f;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            acc[i] *= *(const floatx4*)(s_from + 16 * i + 4 * g);
#pragma unroll
            for (int j = 0; j <= i; ++j)
                acc[i] = mfma4(*(const floatx4*)(sk + (16 * i + l16) * LS + 16 * j + 4 * g), u[j], acc[i]);
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int t = 16 * i + 4 * g + r;
                if (t < c.count && row_live) {
                    store1<TYPE>(p.out, ((int64_t)(c.first + t) * p.heads + head) * p.value_dim + row, acc[i][r]);
                    finite &= __builtin_isfinite(acc[i][r]);
                }
            }
        }
    }
    if (!finite) atomicOr(&p.flags[FLAG_NONFINITE], 1);
}

template <int KP, int TYPE, bool DELTA>
static hipError_t launch_prompt_of(const LinearParams& p, hipStream_t s) {
    const unsigned units = (unsigned)((int64_t)p.chunks * p.heads);
    if constexpr (DELTA) {
        constexpr int bytes = (C * (KP + 4) + C * LS + 4 * 16 * 20) * 4;
        hipLaunchKernelGGL((k_linear_solve<KP, TYPE>), dim3(units), dim3(256), bytes, s, p);
    } else {
        hipLaunchKernelGGL(k_linear_gates, dim3((units + 3) / 4), dim3(256), 0, s, p);
    }
    hipError_t e = hipGetLastError();
    if (e != hipSuccess) return e;
    const unsigned vt = (unsigned)(p.value_dim + 15) / 16, sh = (unsigned)(p.seqs * p.heads);
    hipLaunchKernelGGL((k_linear_scan<KP, TYPE, DELTA>), dim3((sh + 7) / 8 * 8 * vt), dim3(256), 0, s, p);
    if ((e = hipGetLastError()) != hipSuccess) return e;
    constexpr int bytes = 2 * C * (KP + 4) * 4;
    hipLaunchKernelGGL((k_linear_out<KP, TYPE, DELTA>), dim3(units), dim3(256), bytes, s, p);
    return hipGetLastError();
}

template <int KP, int TYPE>
static hipError_t launch_prompt_rule(const LinearParams& p, hipStream_t s) {
    return p.beta ? launch_prompt_of<KP, TYPE, true>(p, s) : launch_prompt_of<KP, TYPE, false>(p, s);
}

template <int TYPE>
static hipError_t launch_prompt_type(const LinearParams& p, hipStream_t s) {
    switch (linear_kp(p.key_dim)) {
        case 64: return launch_prompt_rule<64, TYPE>(p, s);
        case 128: return launch_prompt_rule<128, TYPE>(p, s);
        default: return launch_prompt_rule<256, TYPE>(p, s);
    }
}

hipError_t launch_linear_prompt(const LinearParams& p, hipStream_t s) {
    switch (p.type) {
        case MIX_F32: return launch_prompt_type<MIX_F32>(p, s);
        case MIX_F16: return launch_prompt_type<MIX_F16>(p, s);
        case MIX_BF16: return launch_prompt_type<MIX_BF16>(p, s);
    }
    return hipErrorInvalidValue;
}

}  // namespace mqh
