// dh_vocab.hip -- losses over a vocabulary from hidden states H (N x D) and a table W (V x D),
// without an N x V matrix of logits.
//
//   z = c H W^T (c = the logit scale, or 1 / T),  lse_n = log sum_v exp z_nv
//   cross entropy   loss_n = lse_n - z_nt                    (t = the row's target)
//   distillation    loss_n = T^2 sum_k q_nk (log q_nk - z_nk + lse_n)
//                   (q = softmax of the row's K teacher logits / T, k its K tokens)
//   gradient        G_nv = w_n (exp(z_nv - lse_n) - q_nv), dH = G W, dW = G^T H
//                   (q_nv = 1 at the target, or the teacher's; w_n = the row's loss weight times
//                   c, or times T)
//
// The vocabulary goes by in pieces.  Forward: each 256 x 256 tile of a piece's logits is reduced
// in registers to a maximum and a sum per row and 128 tokens, joined afterwards.  Backward: a
// piece's logits are formed again, and its G goes through a buffer of the piece's size into both
// products.  Rows without a target (padding) are taken out first: the rows that count are packed
// side by side, so padding costs no product and nothing in it, NaN included, reaches a sum.
//
// All four products run on the bf16 matrix cores with fp32 accumulators.  An fp32 operand is
// split into three bf16 parts, x = x1 + x2 + x3 (8 significant bits each, the last remainder is
// exact), and a product takes the six pairs of parts that reach 2^-24 of it, smallest first:
// x3 y1, x2 y2, x1 y3, x2 y1, x1 y2, x1 y1 -- six bf16 products at 16 times the rate of the fp32
// ones.
#include "dh_common.hpp"
#include "dh_gemm_bf16.hpp"

namespace dh {
namespace {

// ---- rows of either type ----------------------------------------------------------------------
typedef float f4a __attribute__((ext_vector_type(4), aligned(4)));
typedef uint16_t h8a __attribute__((ext_vector_type(8), aligned(2)));

// Elements c .. c + 7 of a row of D, zero past its end; any alignment.
__device__ inline void load8(const float* __restrict__ p, int c, int D, float (&v)[8]) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        if (c + 4 * q + 4 <= D) {
            const f4a x = *reinterpret_cast<const f4a*>(p + c + 4 * q);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * q + e] = x[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) v[4 * q + e] = c + 4 * q + e < D ? p[c + 4 * q + e] : 0.f;
        }
    }
}
__device__ inline void load8(const uint16_t* __restrict__ p, int c, int D, float (&v)[8]) {
    if (c + 8 <= D) {
        const h8a x = *reinterpret_cast<const h8a*>(p + c);
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = bf16_bits_to_f32(x[e]);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = c + e < D ? bf16_bits_to_f32(p[c + e]) : 0.f;
    }
}
__device__ inline uint16_t rne_bf16(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }

// x = the sum of three bf16 values, to 24 bits.  Values whose nearest bf16 is infinite are
// truncated instead; infinities and NaN are their own first part.
__device__ inline void split3(float x, uint16_t (&b)[3]) {
    b[0] = rne_bf16(x);
    const bool finite = __builtin_fabsf(x) < INFINITY;
    if (finite && (b[0] & 0x7FFF) == 0x7F80) b[0] = (uint16_t)(__builtin_bit_cast(uint32_t, x) >> 16);
    const float r = finite ? x - bf16_bits_to_f32(b[0]) : 0.f;
    b[1] = rne_bf16(r);
    b[2] = rne_bf16(r - bf16_bits_to_f32(b[1]));
}

typedef uint16_t h8 __attribute__((ext_vector_type(8)));

// 8 values as PLANES bf16 parts at dst, dst + plane, ...  One part: the values are bf16 already.
template <int PLANES>
__device__ inline void store_parts(uint16_t* __restrict__ dst, long long plane, const float (&v)[8]) {
    h8 o[PLANES];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        if constexpr (PLANES == 1) {
            o[0][e] = rne_bf16(v[e]);
        } else {
            uint16_t b[3];
            split3(v[e], b);
#pragma unroll
            for (int p = 0; p < 3; ++p) o[p][e] = b[p];
        }
    }
#pragma unroll
    for (int p = 0; p < PLANES; ++p) *reinterpret_cast<h8*>(dst + p * plane) = o[p];
}

// ---- packing ------------------------------------------------------------------------------------
// What a packed row i is: its row n, target, loss weight and lse (backward).  Arrays are padded
// to whole tiles of rows, so that a tile's epilogue may load past the last row.
struct Rows {
    int* cnt;          // rows that count
    int* row;          // packed -> row
    int* inv;          // row -> packed, or -1
    int* target;
    float *w, *lse;    // backward only
};

__device__ inline bool counts(int target, int V) { return (unsigned)target < (unsigned)V; }

// Work-group b packs rows 64 b .. 64 b + 63: it counts the rows that count before them (the
// targets are few and stay in cache), then copies its own, a wave per row, as bf16 parts with
// zeros up to Dp.  Forward (loss not null) also writes the padding's zeros.
template <typename T, int PLANES>
__global__ void __launch_bounds__(1024) pack_rows(const int* __restrict__ target, int N, int V, int D,
                                                  const T* __restrict__ H, int ldh,
                                                  uint16_t* __restrict__ Hp, int Dp, long long plane,
                                                  Rows rows, float* __restrict__ loss,
                                                  float* __restrict__ lse_out,
                                                  const float* __restrict__ lse_in,
                                                  const float* __restrict__ dloss, float wscale) {
    __shared__ int red[16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int n0 = blockIdx.x * 64;
    int before = 0;
    for (int n = threadIdx.x; n < n0; n += 1024) before += counts(target[n], V);
    for (int m = 1; m < 64; m <<= 1) before += __shfl_xor(before, m, 64);
    if (lane == 0) red[w] = before;
    __syncthreads();
    before = 0;
    for (int x = 0; x < 16; ++x) before += red[x];
    const bool mine = n0 + lane < N && counts(target[n0 + lane], V);
    const uint64_t mask = __ballot(mine);
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == 0) *rows.cnt = before + __popcll(mask);
    for (int r = w; r < 64 && n0 + r < N; r += 16) {
        const int n = n0 + r;
        const bool keep = (mask >> r) & 1;
        const int i = before + __popcll(mask & ((1ull << r) - 1));
        if (lane == 0) {
            rows.inv[n] = keep ? i : -1;
            if (keep) {
                rows.row[i] = n;
                rows.target[i] = target[n];
                if (lse_in) {
                    rows.lse[i] = lse_in[n];
                    rows.w[i] = (dloss ? dloss[n] : 1.f) * wscale;
                }
            } else if (loss) {
                loss[n] = 0.f;
                if (lse_out) lse_out[n] = 0.f;
            }
        }
        if (!keep) continue;
        for (int c = 8 * lane; c < Dp; c += 512) {
            float v[8];
            load8(H + (size_t)n * ldh, c, D, v);
            store_parts<PLANES>(Hp + (size_t)i * Dp + c, plane, v);
        }
    }
}

// Rows v0 .. v0 + R - 1 of the table as bf16 parts with zeros up to Dp, a wave per row.
template <typename T, int PLANES>
__global__ void __launch_bounds__(256) stage_table(const T* __restrict__ W, int ldw, int v0, int R, int D,
                                                   uint16_t* __restrict__ dst, int Dp,
                                                   long long plane) {
    const int lane = threadIdx.x & 63;
    const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= R) return;
    for (int c = 8 * lane; c < Dp; c += 512) {
        float v[8];
        load8(W + (size_t)(v0 + r) * ldw, c, D, v);
        store_parts<PLANES>(dst + (size_t)r * Dp + c, plane, v);
    }
}

// ---- targets -------------------------------------------------------------------------------------
// The K teacher entries of a row: token and logit.  An entry whose token lies outside the table
// or whose logit is -inf is none.
struct Teacher {
    const int* id;
    const float* logit;
    int K;
    float inv_t;   // 1 / T
};
__device__ inline bool entry_counts(const Teacher& t, size_t at, int V) {
    return counts(t.id[at], V) && !(t.logit[at] == -INFINITY);
}

// flag[n] = 0 where row n has an entry, -1 where it has none (padding).  A wave per row.
__global__ void __launch_bounds__(256) teacher_flags(Teacher t, int N, int V, int* __restrict__ flag) {
    const int lane = threadIdx.x & 63;
    const int n = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= N) return;
    bool any = false;
    for (int k = lane; k < t.K; k += 64) any |= entry_counts(t, (size_t)n * t.K + k, V);
    const bool has = __ballot(any) != 0;
    if (lane == 0) flag[n] = has ? 0 : -1;
}

template <typename T>
__device__ inline float row_dot(const T* __restrict__ a, const T* __restrict__ b, int D, int lane) {
    float s = 0.f;
    for (int c = 8 * lane; c < D; c += 512) {
        float x[8], y[8];
        load8(a, c, D, x);
        load8(b, c, D, y);
#pragma unroll
        for (int e = 0; e < 8; ++e) s = __builtin_fmaf(x[e], y[e], s);
    }
    return wave_reduce(s, OpSum());
}

// base[i] = -z at the packed row's target: the row's loss is lse + base.  A wave per row.
template <typename T>
__global__ void __launch_bounds__(256) target_dot(Rows rows, const T* __restrict__ H, int ldh,
                                                  const T* __restrict__ W, int ldw, int D, float c,
                                                  float* __restrict__ base) {
    const int lane = threadIdx.x & 63;
    const int i = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (i >= *rows.cnt) return;
    const float d = row_dot(H + (size_t)rows.row[i] * ldh, W + (size_t)rows.target[i] * ldw, D, lane);
    if (lane == 0) base[i] = -(c * d);
}

// A work-group per packed row: the teacher's probabilities q (N x K, zero where there is no
// entry), the student's logits z at its tokens, and base[i] = sum q (log q - z).
template <typename T>
__global__ void __launch_bounds__(256) teacher_dots(Rows rows, Teacher t, int V,
                                                    const T* __restrict__ H, int ldh,
                                                    const T* __restrict__ W, int ldw, int D,
                                                    float* __restrict__ q, float* __restrict__ z,
                                                    float* __restrict__ base) {
    __shared__ float red[4];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int i = blockIdx.x;
    if (i >= *rows.cnt) return;
    const int n = rows.row[i];
    const size_t at = (size_t)n * t.K, to = (size_t)i * t.K;
    auto all = [&](float v, auto op) {
        v = wave_reduce(v, op);
        __syncthreads();
        if (lane == 0) red[w] = v;
        __syncthreads();
        return op(op(red[0], red[1]), op(red[2], red[3]));
    };
    float mx = -INFINITY;
    for (int k = threadIdx.x; k < t.K; k += 256)
        if (entry_counts(t, at + k, V)) mx = fmaxf(mx, t.logit[at + k]);
    mx = all(mx, OpMax());
    float sum = 0.f;
    for (int k = threadIdx.x; k < t.K; k += 256)
        if (entry_counts(t, at + k, V)) sum += __expf((t.logit[at + k] - mx) * t.inv_t);
    sum = all(sum, OpSum());
    const float log_sum = __logf(sum);
    float part = 0.f;
    for (int k = w; k < t.K; k += 4) {
        float zk = 0.f, qk = 0.f;
        if (entry_counts(t, at + k, V)) {
            const float d = row_dot(H + (size_t)n * ldh, W + (size_t)t.id[at + k] * ldw, D, lane);
            zk = t.inv_t * d;
            const float lq = (t.logit[at + k] - mx) * t.inv_t - log_sum;
            qk = __expf(lq);
            // exp underflows below about -104: the entry's share of the loss is zero there
            if (!(qk == 0.f)) part += qk * (lq - zk);
        }
        if (lane == 0) {
            q[to + k] = qk;
            z[to + k] = zk;
        }
    }
    __syncthreads();   // red[] may still be read
    if (lane == 0) red[w] = part;
    __syncthreads();
    if (threadIdx.x == 0) base[i] = (red[0] + red[1]) + (red[2] + red[3]);
}

// ---- products -------------------------------------------------------------------------------------
// C (M x N) = sum over k of A and B, operands of bf16 parts.  AK: A is stored [m][k], else [k][m];
// BK: B is stored [n][k], else [k][n].  One of M, N and K counts packed rows: its extent is *cnt.
struct Prod {
    const uint16_t *A, *B;
    int lda, ldb;
    long long pa, pb;      // elements between an operand's parts
    int M, N, K;
    int kstages;           // 32-k stages of one split (blockIdx.y)
    const int* cnt;
};
enum { TOK_M, TOK_N, TOK_K };

// One operand's DMA for 32-k stages of a 256-wide tile: as FastOperand, with a resource per stage
// whose base is the stage's first element and whose range ends with the operand's rows, so
// operands of any size keep 32-bit offsets and what lies behind the rows reads as zero.
template <bool KC>
struct Stager {
    FastOperand<KC, 8> f;
    uint32_t last[FastOperand<KC, 8>::PER];   // offsets in the stage that K ends in
    const uint16_t* base;    // the tile's first element
    int ld, rows, K;         // rows: of the tile (KC)
    __device__ void init(const uint16_t* p, int ld_, int t0, int extent, int K_, int wave, int lane) {
        ld = ld_;
        K = K_;
        f.init(ld, 0, 0, wave, lane);
        base = KC ? p + (size_t)t0 * ld : p + t0;
        rows = KC ? min(extent - t0, 256) : t0;
        if (KC) {
#pragma unroll
            for (int t = 0; t < f.PER; ++t) {
                const int c = (lane & 3) ^ ((lane >> 4) & 3);
                // chunks past K (a multiple of 8) lie outside the resource
                last[t] = 8 * c < (K & 31) ? f.off[t] : 0xFFFFFFF0u;
            }
        }
    }
    __device__ void issue(long long plane, int kt, uint16_t* lds, int wave) const {
        const uint16_t* p = base + plane + (KC ? (size_t)kt * 32 : (size_t)kt * 32 * ld);
        const uint32_t bytes =
            KC ? 2u * ((uint32_t)rows * ld - 32u * kt)
               : 2u * ((uint32_t)min(K - 32 * kt, 32) * ld - (uint32_t)rows);
        const u32x4 rs = make_rsrc(p, bytes);
        const uint32_t to = __builtin_amdgcn_readfirstlane(lds_addr(lds) + 1024u * f.PER * wave);
        const bool end = KC && 32 * kt + 32 > K;
#pragma unroll
        for (int t = 0; t < f.PER; ++t)
            lds_dma16_buf_so(KC && end ? last[t] : f.off[t], rs, 0u, to + 1024u * t);
    }
};

// Pairs of parts in the order they are added (see the head of the file).
template <int PLANES>
__device__ inline void pair_of(int s, int& a, int& b) {
    if (PLANES == 1) {
        a = b = 0;
        return;
    }
    constexpr uint32_t PA = 0x210100u, PB = 0x012010u;   // a digit per pair, the first on the left
    a = (PA >> (4 * (5 - s))) & 0xF;
    b = (PB >> (4 * (5 - s))) & 0xF;
}

// 256 x 256 tile, 8 waves of 128 x 64, 32-k stages through a ring of four in LDS filled by
// direct DMA three stages ahead; each stage's two 16-k steps run while the next operands are
// read (the schedule of the bf16 GEMM's 8-wave form).  Epi::run gets the tile's accumulators:
// register r of block (a, b) is row m0 + wm + 32 a + 8 (r / 4) + 4 h + r % 4, column
// n0 + wn + 32 b + l32 (lane = 32 h + l32).
template <bool AK, bool BK, int TOK, int PLANES, class Epi>
__global__ void __launch_bounds__(512) vocab_gemm(Prod g, Epi epi) {
    constexpr int FM = 4, FN = 2, PAIRS = PLANES == 1 ? 1 : 6;
    using OA = FastOperand<AK, 8>;
    using OB = FastOperand<BK, 8>;
    __shared__ __attribute__((aligned(16))) uint16_t ring[FAST_NSTAGE * 2 * FAST_TILE];
    const int cnt = *g.cnt;
    const int M = TOK == TOK_M ? cnt : g.M, N = TOK == TOK_N ? cnt : g.N;
    const int Kall = TOK == TOK_K ? cnt : g.K;
    const int tiles_m = (g.M + 255) / 256, tiles_n = (g.N + 255) / 256;
    int tm, tn;
    xcd_tile_order(blockIdx.x, gridDim.x, tiles_m, tiles_n, 4, tm, tn);
    const int m0 = tm * 256, n0 = tn * 256;
    if (m0 >= M || n0 >= N) return;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = (wave / 4) * 128, wn = (wave % 4) * 64;

    f32x16 acc[FM][FN];
#pragma unroll
    for (int a = 0; a < FM; ++a)
#pragma unroll
        for (int b = 0; b < FN; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;

    const int kt0 = blockIdx.y * g.kstages;
    const int nk = max(0, min((Kall + 31) / 32 - kt0, g.kstages));
    const int total = nk * PAIRS;
    if (total > 0) {
        Stager<AK> sa;
        Stager<BK> sb;
        sa.init(g.A, g.lda, m0, M, Kall, wave, lane);
        sb.init(g.B, g.ldb, n0, N, Kall, wave, lane);
        int ikt = 0, ipair = 0, islot = 0;   // the next stage to fetch
        auto issue = [&]() {
            int pa, pb;
            pair_of<PLANES>(ipair, pa, pb);
            uint16_t* st = ring + islot * 2 * FAST_TILE;
            sa.issue(pa * g.pa, kt0 + ikt, st, wave);
            sb.issue(pb * g.pb, kt0 + ikt, st + FAST_TILE, wave);
            islot = (islot + 1) % FAST_NSTAGE;
            if (++ikt == nk) {
                ikt = 0;
                ++ipair;
            }
        };
        auto stage = [&](int s) { return ring + (s % FAST_NSTAGE) * 2 * FAST_TILE; };
        const int pre = min(total, FAST_NSTAGE - 1);
        for (int s = 0; s < pre; ++s) issue();
        static_assert(OA::PER == 2 && OB::PER == 2, "wait_dma_stages<4>: 4 loads per stage");
        wait_dma_stages<4>(pre - 1);
        __syncthreads();
        bf16x8 f0a[FM], f0b[FN], f1a[FM], f1b[FN];
        load_frags<OA, OB, FM, FN>(stage(0), 0, wm, wn, lane, f0a, f0b);
        for (int s = 0; s < total - 1; ++s) {
            if (s + FAST_NSTAGE - 1 < total) issue();
            load_frags<OA, OB, FM, FN>(stage(s), 1, wm, wn, lane, f1a, f1b);
            __builtin_amdgcn_sched_barrier(0);
            mfma_block<FM, FN>(f0a, f0b, acc);
            __builtin_amdgcn_sched_barrier(0);
            const int ahead = min(total - 1, s + FAST_NSTAGE - 1) - (s + 1);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            wait_dma_stages<4>(ahead);
            __syncthreads();
            load_frags<OA, OB, FM, FN>(stage(s + 1), 0, wm, wn, lane, f0a, f0b);
            __builtin_amdgcn_sched_barrier(0);
            mfma_block<FM, FN>(f1a, f1b, acc);
            __builtin_amdgcn_sched_barrier(0);
        }
        load_frags<OA, OB, FM, FN>(stage(total - 1), 1, wm, wn, lane, f1a, f1b);
        __builtin_amdgcn_sched_barrier(0);
        mfma_block<FM, FN>(f0a, f0b, acc);
        mfma_block<FM, FN>(f1a, f1b, acc);
    }
    epi.template run<FM, FN>(acc, M, N, m0 + wm, n0 + wn, lane);
}

// Row of register r of block a, relative to the wave's first row.
__device__ inline int reg_row(int a, int r, int lane) { return 32 * a + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3); }

// Forward: rows are table rows, columns packed rows.  A lane holds 64 logits of each of its
// columns, the other half's lane the wave's other 64: maximum and sum of exponentials of the
// wave's 128 go to part[128-row block][column].
struct EpiLse {
    float c;
    float2* part;
    int ldp;
    template <int FM, int FN>
    __device__ void run(const f32x16 (&acc)[FM][FN], int M, int N, int row0, int col0, int lane) const {
        if (row0 >= M) return;   // the wave has no table row: its block is not joined either
#pragma unroll
        for (int b = 0; b < FN; ++b) {
            float mx = -INFINITY;
            bool full = row0 + 128 <= M;
#pragma unroll
            for (int a = 0; a < FM; ++a)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (full || row0 + reg_row(a, r, lane) < M) mx = fmaxf(mx, c * acc[a][b][r]);
            mx = fmaxf(mx, xor32(mx));
            const float m = mx == -INFINITY ? 0.f : mx;   // all -inf: a sum of zeros, not of NaN
            float s = 0.f;
#pragma unroll
            for (int a = 0; a < FM; ++a)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (full || row0 + reg_row(a, r, lane) < M) s += __expf(c * acc[a][b][r] - m);
            s += xor32(s);
            const int col = col0 + 32 * b + (lane & 31);
            if (lane < 32 && col < N) part[(size_t)(row0 / 128) * ldp + col] = float2{mx, s};
        }
    }
};

// Backward: rows are packed rows, columns the piece's table rows.  G as bf16 (parts): one
// rounding of each entry of G to the type that the products take (in three parts, to 24 bits).
// Columns past the table's end up to the tile's are zero.
template <int PLANES, bool HARD>
struct EpiG {
    float c;
    const float *lse, *w;
    const int* target;
    int v0;
    uint16_t* G;
    int ldg;
    long long plane;
    template <int FM, int FN>
    __device__ void run(const f32x16 (&acc)[FM][FN], int M, int N, int row0, int col0, int lane) const {
#pragma unroll
        for (int a = 0; a < FM; ++a)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const int row = row0 + reg_row(a, 4 * r4, lane);
                const f32x4 l4 = *reinterpret_cast<const f32x4*>(lse + row);
                const f32x4 w4 = *reinterpret_cast<const f32x4*>(w + row);
                int t4[4];
                if constexpr (HARD)
#pragma unroll
                    for (int e = 0; e < 4; ++e) t4[e] = target[row + e] - v0;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (row + e >= M) continue;
#pragma unroll
                    for (int b = 0; b < FN; ++b) {
                        const int col = col0 + 32 * b + (lane & 31);
                        float p = __expf(__builtin_fmaf(c, acc[a][b][4 * r4 + e], -l4[e]));
                        if constexpr (HARD)
                            if (col == t4[e]) p -= 1.f;
                        const float v = col < N ? w4[e] * p : 0.f;
                        uint16_t* to = G + (size_t)(row + e) * ldg + col;
                        if constexpr (PLANES == 1) {
                            *to = rne_bf16(v);
                        } else {
                            uint16_t x[3];
                            split3(v, x);
#pragma unroll
                            for (int q = 0; q < 3; ++q) to[q * plane] = x[q];
                        }
                    }
                }
            }
    }
};

// dH: fp32 sums over the pieces, one block per split of the piece.
struct EpiAcc {
    float* C;
    int ldc, first;
    long long split;
    template <int FM, int FN>
    __device__ void run(const f32x16 (&acc)[FM][FN], int M, int N, int row0, int col0, int lane) const {
        float* p = C + blockIdx.y * split;
#pragma unroll
        for (int a = 0; a < FM; ++a)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = row0 + reg_row(a, r, lane);
                if (row >= M) continue;
#pragma unroll
                for (int b = 0; b < FN; ++b) {
                    const int col = col0 + 32 * b + (lane & 31);
                    if (col >= N) continue;
                    float* to = p + (size_t)row * ldc + col;
                    *to = first ? acc[a][b][r] : *to + acc[a][b][r];
                }
            }
    }
};

// dW: the piece's rows of the gradient, in its type.
template <typename OT>
struct EpiOut {
    OT* C;
    int ldc, accumulate;
    template <int FM, int FN>
    __device__ void run(const f32x16 (&acc)[FM][FN], int M, int N, int row0, int col0, int lane) const {
#pragma unroll
        for (int a = 0; a < FM; ++a)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = row0 + reg_row(a, r, lane);
                if (row >= M) continue;
#pragma unroll
                for (int b = 0; b < FN; ++b) {
                    const int col = col0 + 32 * b + (lane & 31);
                    if (col >= N) continue;
                    OT* to = C + (size_t)row * ldc + col;
                    float v = acc[a][b][r];
                    if constexpr (sizeof(OT) == 4) {
                        *to = accumulate ? *to + v : v;
                    } else {
                        if (accumulate) v += bf16_bits_to_f32(*to);
                        *to = rne_bf16(v);
                    }
                }
            }
    }
};

// ---- joins ----------------------------------------------------------------------------------------
__device__ inline void lse_merge(float& m, float& s, float m2, float s2) {
    const float mx = fmaxf(m, m2);
    const float ref = mx == -INFINITY ? 0.f : mx;
    s = s * __expf(m - ref) + s2 * __expf(m2 - ref);
    m = mx;
}

// A work-group per 64 packed rows, 16 waves that share the piece's 128-row blocks; their results
// meet in LDS in wave order.  state: what earlier pieces left (first: nothing).  The last piece
// writes lse and loss = factor (lse + base).
__global__ void __launch_bounds__(1024) lse_join(const float2* __restrict__ part, int ldp, int blocks,
                                                 Rows rows, float2* __restrict__ state, int first,
                                                 int last, const float* __restrict__ base, float factor,
                                                 float* __restrict__ loss, float* __restrict__ lse) {
    __shared__ float2 red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int i = blockIdx.x * 64 + lane;
    const int cnt = *rows.cnt;
    if ((int)blockIdx.x * 64 >= cnt) return;
    float m = -INFINITY, s = 0.f;
    if (i < cnt)
        for (int b = w; b < blocks; b += 16) {
            const float2 p = part[(size_t)b * ldp + i];
            lse_merge(m, s, p.x, p.y);
        }
    red[w][lane] = float2{m, s};
    __syncthreads();
    if (w != 0 || i >= cnt) return;
    if (!first) {
        const float2 p = state[i];
        m = p.x;
        s = p.y;
        lse_merge(m, s, red[0][lane].x, red[0][lane].y);
    }
    for (int x = 1; x < 16; ++x) lse_merge(m, s, red[x][lane].x, red[x][lane].y);
    if (!last) {
        state[i] = float2{m, s};
        return;
    }
    const int n = rows.row[i];
    const float l = m + __logf(s);
    if (lse) lse[n] = l;
    loss[n] = factor * (l + base[i]);
}

// The entries of G at the teacher's tokens inside a piece, from the fp32 logits: w (p - q), q
// summed where a token occurs more than once (each of its entries writes the same value).
template <int PLANES>
__global__ void __launch_bounds__(256) teacher_entries(Rows rows, Teacher t, int V, int v0, int R,
                                                       const float* __restrict__ q,
                                                       const float* __restrict__ z,
                                                       uint16_t* __restrict__ G, int ldg,
                                                       long long plane) {
    const int i = blockIdx.x;
    if (i >= *rows.cnt) return;
    const size_t at = (size_t)rows.row[i] * t.K, from = (size_t)i * t.K;
    const float w = rows.w[i], lse = rows.lse[i];
    for (int k = threadIdx.x; k < t.K; k += 256) {
        const int id = t.id[at + k];
        if (id < v0 || id >= v0 + R || !entry_counts(t, at + k, V)) continue;
        float sum = 0.f;
        for (int j = 0; j < t.K; ++j)
            if (t.id[at + j] == id) sum += q[from + j];
        const float v = w * (__expf(z[from + k] - lse) - sum);
        uint16_t* to = G + (size_t)i * ldg + (id - v0);
        if constexpr (PLANES == 1) {
            *to = rne_bf16(v);
        } else {
            uint16_t x[3];
            split3(v, x);
#pragma unroll
            for (int p = 0; p < 3; ++p) to[p * plane] = x[p];
        }
    }
}

// dH (+)= the splits' sums, row by row in the callers' order; zero (or unchanged) for padding.
template <typename OT>
__global__ void __launch_bounds__(256) dh_finish(const int* __restrict__ inv, int N, int D,
                                                 const float* __restrict__ acc, int lda, int splits,
                                                 long long split, OT* __restrict__ dH, int ldd,
                                                 int accumulate) {
    const int lane = threadIdx.x & 63;
    const long long n = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (n >= N) return;
    const int i = inv[n];
    if (i < 0 && accumulate) return;
    for (int c = lane; c < D; c += 64) {
        float v = 0.f;
        if (i >= 0)
            for (int s = 0; s < splits; ++s) v += acc[s * split + (size_t)i * lda + c];
        OT* to = dH + (size_t)n * ldd + c;
        if constexpr (sizeof(OT) == 4) {
            *to = accumulate ? *to + v : v;
        } else {
            if (accumulate) v += bf16_bits_to_f32(*to);
            *to = rne_bf16(v);
        }
    }
}

// The gradient of no rows at all (N = 0).
template <typename OT>
__global__ void __launch_bounds__(256) clear_rows(OT* __restrict__ p, int R, int D, int ld) {
    const int lane = threadIdx.x & 63;
    for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < R; r += 4LL * gridDim.x)
        for (int c = lane; c < D; c += 64) p[(size_t)r * ld + c] = OT(0);
}

// ---- host -----------------------------------------------------------------------------------------
struct Head {
    const char* op;
    int dtype, N, V, D;
    const void* H;
    int ldh;
    const void* W;
    int ldw;
    float c;                // logit scale
    const int* target;      // or null:
    Teacher teacher;
    float factor, wscale;   // loss = factor (lse + base); G's weight = dloss wscale
};

size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// The workspace: a part whose size the shapes give, and a piece whose size is what is left.
struct Plan {
    int planes, Dp, Nt;       // parts of an operand, padded columns, rows padded to whole tiles
    bool direct;              // the table is read in place
    size_t ints, w, lse, base, q, z, state, Hp, acc;
    int splits;
    size_t piece;             // first byte of the piece's buffers
    size_t per_block;         // bytes of a piece per 256 table rows
};

Plan make_plan(int dtype, int N, int V, int D, int K, int backward, const void* W, int ldw) {
    Plan p{};
    p.planes = dtype == DH_F32 ? 3 : 1;
    p.Dp = (D + 31) / 32 * 32;
    p.Nt = (int)(((long long)N + 255) / 256 * 256);
    // In place: whole 16-byte chunks at aligned addresses, 256 rows within 32-bit offsets.
    p.direct = dtype == DH_BF16 && D % 8 == 0 && ldw % 8 == 0 && ldw <= 1 << 22 && ((uintptr_t)W & 15) == 0;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += up256(bytes);
        return here;
    };
    p.ints = take(((size_t)4 * p.Nt + 64) * 4);   // cnt, flags, row, inv, target
    p.w = take((size_t)p.Nt * 4);
    p.lse = take((size_t)p.Nt * 4);
    p.base = take((size_t)p.Nt * 4);
    p.q = take((size_t)N * K * 4);
    p.z = take((size_t)N * K * 4);
    p.Hp = take((size_t)p.planes * N * p.Dp * 2);
    if (backward) {
        const long long tiles = (long long)(p.Nt / 256) * ((D + 255) / 256);
        p.splits = tiles >= 256 ? 1 : (int)(256 / (tiles > 0 ? tiles : 1));
        if (p.splits > 8) p.splits = 8;
        p.acc = take((size_t)p.splits * N * p.Dp * 4);
        p.per_block = (size_t)p.planes * N * 256 * 2;
    } else {
        p.state = take((size_t)p.Nt * 8);
        p.per_block = (size_t)p.Nt * 2 * 8;
    }
    if (!p.direct) p.per_block += (size_t)p.planes * 256 * p.Dp * 2;
    p.piece = at;
    return p;
}

// The workspace that serves any alignment of the operands (staged tables take more).
size_t least_ws(int dtype, int N, int V, int D, int K, int backward) {
    const Plan p = make_plan(dtype, N, V, D, K, backward, nullptr, 1);
    return p.piece + p.per_block + 512;
}

// Table rows of a piece: as many blocks of 256 as fit, the same for every piece.
int piece_rows(const Plan& p, int V, size_t ws_bytes) {
    const long long blocks = (V + 255LL) / 256;
    long long fit = (long long)((ws_bytes - 512 - p.piece) / p.per_block);
    if (fit > blocks) fit = blocks;
    if (fit > 4096) fit = 4096;   // 256 rows of G stay within 32-bit offsets
    const long long pieces = (blocks + fit - 1) / fit;
    return (int)((blocks + pieces - 1) / pieces) * 256;
}

int check_head(const Head& h, int K, const void* ws, size_t ws_bytes, int backward) {
    if (h.dtype != DH_F32 && h.dtype != DH_BF16)
        return set_error(DH_ERR_INVALID, "%s: dtype must be fp32 or bf16", h.op);
    if (h.N < 0 || h.V < 1 || h.D < 1 || K < 0 || h.N > 0x7FFFFE00 || h.V > 0x7FFFFE00 || h.D > 1 << 20)
        return set_error(DH_ERR_INVALID, "%s: shape N=%d V=%d D=%d", h.op, h.N, h.V, h.D);
    if (h.ldh < h.D || h.ldw < h.D)
        return set_error(DH_ERR_INVALID, "%s: leading dimension below D", h.op);
    if (!(h.c > 0.f) || !(h.c < INFINITY) || !(h.factor < INFINITY))
        return set_error(DH_ERR_INVALID, "%s: the scale (temperature) must be finite and > 0", h.op);
    if (h.N == 0) return DH_OK;
    if (!h.H || !h.W || !ws) return set_error(DH_ERR_INVALID, "%s: null pointer", h.op);
    if ((uintptr_t)ws & 15) return set_error(DH_ERR_INVALID, "%s: workspace not 16-byte aligned", h.op);
    const size_t need = least_ws(h.dtype, h.N, h.V, h.D, K, backward);
    if (ws_bytes < need)
        return set_error(DH_ERR_INVALID, "%s: workspace of %zu bytes, %zu needed", h.op, ws_bytes, need);
    return DH_OK;
}

struct Work {
    Plan p;
    Rows rows;
    float *base, *q, *z;
    uint16_t* Hp;
    int* flags;
    char* piece;
};

Work lay_out(const Plan& p, void* ws, int N) {
    char* b = (char*)(((uintptr_t)ws + 255) & ~(uintptr_t)255);
    int* ints = (int*)(b + p.ints);
    Work w{};
    w.p = p;
    w.rows = {ints, ints + 64, ints + 64 + p.Nt, ints + 64 + 2 * (size_t)p.Nt, (float*)(b + p.w),
              (float*)(b + p.lse)};
    w.flags = ints + 64 + 3 * (size_t)p.Nt;
    w.base = (float*)(b + p.base);
    w.q = (float*)(b + p.q);
    w.z = (float*)(b + p.z);
    w.Hp = (uint16_t*)(b + p.Hp);
    w.piece = b + p.piece;
    return w;
}

template <typename T, int PLANES>
int prepare_rows(const Head& h, const Work& w, float* loss, float* lse_out, const float* lse_in,
                 const float* dloss) {
    const int* target = h.target;
    if (!target) {
        teacher_flags<<<(h.N + 3) / 4, 256, 0, stream()>>>(h.teacher, h.N, h.V, w.flags);
        DH_TRY(check_launch(h.op));
        target = w.flags;
    }
    pack_rows<T, PLANES><<<(h.N + 63) / 64, 1024, 0, stream()>>>(
        target, h.N, h.V, h.D, (const T*)h.H, h.ldh, w.Hp, w.p.Dp, (long long)h.N * w.p.Dp, w.rows, loss,
        lse_out, lse_in, dloss, h.wscale);
    DH_TRY(check_launch(h.op));
    if (!h.target)
        teacher_dots<T><<<h.N, 256, 0, stream()>>>(w.rows, h.teacher, h.V, (const T*)h.H, h.ldh,
                                                   (const T*)h.W, h.ldw, h.D, w.q, w.z, w.base);
    else if (loss)
        target_dot<T><<<(h.N + 3) / 4, 256, 0, stream()>>>(w.rows, (const T*)h.H, h.ldh, (const T*)h.W,
                                                           h.ldw, h.D, h.c, w.base);
    return check_launch(h.op);
}

// The table rows of a piece as a product's operand: in place, or staged at `at`.
template <typename T, int PLANES>
int piece_table(const Head& h, const Plan& p, int v0, int R, uint16_t* at, const uint16_t*& W, int& ld,
                long long& plane) {
    if (p.direct) {
        W = (const uint16_t*)h.W + (size_t)v0 * h.ldw;
        ld = h.ldw;
        plane = 0;
        return DH_OK;
    }
    W = at;
    ld = p.Dp;
    plane = (long long)R * p.Dp;
    stage_table<T, PLANES><<<(R + 3) / 4, 256, 0, stream()>>>((const T*)h.W, h.ldw, v0, R, h.D, at, p.Dp,
                                                             plane);
    return check_launch(h.op);
}

template <bool AK, bool BK, int TOK, int PLANES, class Epi>
int product(const char* op, Prod g, int splits, const Epi& epi) {
    const long long tiles = ((g.M + 255LL) / 256) * ((g.N + 255LL) / 256);
    const int stages = (g.K + 31) / 32;
    g.kstages = (stages + splits - 1) / splits;
    vocab_gemm<AK, BK, TOK, PLANES, Epi><<<dim3((unsigned)tiles, splits), 512, 0, stream()>>>(g, epi);
    return check_launch(op);
}

template <typename T, int PLANES>
int forward(const Head& h, float* loss, float* lse, void* ws, size_t ws_bytes) {
    const Plan p = make_plan(h.dtype, h.N, h.V, h.D, h.target ? 0 : h.teacher.K, 0, h.W, h.ldw);
    const Work w = lay_out(p, ws, h.N);
    float2* state = (float2*)((char*)w.piece - p.piece + p.state);
    DH_TRY((prepare_rows<T, PLANES>(h, w, loss, lse, nullptr, nullptr)));
    const int rows = piece_rows(p, h.V, ws_bytes);
    float2* part = (float2*)w.piece;
    uint16_t* staged = (uint16_t*)(w.piece + (size_t)(rows / 128) * p.Nt * 8);
    for (int v0 = 0; v0 < h.V; v0 += rows) {
        const int R = h.V - v0 < rows ? h.V - v0 : rows;
        Prod g{};
        DH_TRY((piece_table<T, PLANES>(h, p, v0, R, staged, g.A, g.lda, g.pa)));
        g.B = w.Hp;
        g.ldb = p.Dp;
        g.pb = (long long)h.N * p.Dp;
        g.M = R;
        g.N = h.N;
        g.K = p.direct ? h.D : p.Dp;
        g.cnt = w.rows.cnt;
        DH_TRY((product<true, true, TOK_N, PLANES>(h.op, g, 1, EpiLse{h.c, part, p.Nt})));
        lse_join<<<p.Nt / 64, 1024, 0, stream()>>>(part, p.Nt, (R + 127) / 128, w.rows, state, v0 == 0,
                                                   v0 + R >= h.V, w.base, h.factor, loss, lse);
        DH_TRY(check_launch(h.op));
        if (h.V - v0 <= rows) break;   // v0 + rows may pass the largest int
    }
    return DH_OK;
}

struct Grads {
    const float *lse, *dloss;
    void* dH;
    int lddh, acc_dH;
    void* dW;
    int lddw, acc_dW, type;
};

template <typename T, int PLANES>
int backward(const Head& h, const Grads& d, void* ws, size_t ws_bytes) {
    const Plan p = make_plan(h.dtype, h.N, h.V, h.D, h.target ? 0 : h.teacher.K, 1, h.W, h.ldw);
    const Work w = lay_out(p, ws, h.N);
    float* acc = (float*)((char*)w.piece - p.piece + p.acc);
    DH_TRY((prepare_rows<T, PLANES>(h, w, nullptr, nullptr, d.lse, d.dloss)));
    const int rows = piece_rows(p, h.V, ws_bytes);
    const long long hplane = (long long)h.N * p.Dp, split = hplane;
    uint16_t* G = (uint16_t*)w.piece;
    const long long gplane = (long long)h.N * rows;
    uint16_t* staged = G + PLANES * gplane;
    for (int v0 = 0; v0 < h.V; v0 += rows) {
        const int R = h.V - v0 < rows ? h.V - v0 : rows;
        const uint16_t* W;
        int ldw;
        long long wplane;
        DH_TRY((piece_table<T, PLANES>(h, p, v0, R, staged, W, ldw, wplane)));
        const int K = p.direct ? h.D : p.Dp;
        Prod g{w.Hp, W, p.Dp, ldw, hplane, wplane, h.N, R, K, 0, w.rows.cnt};
        if (h.target) {
            DH_TRY((product<true, true, TOK_M, PLANES>(
                h.op, g, 1, EpiG<PLANES, true>{h.c, w.rows.lse, w.rows.w, w.rows.target, v0, G, rows, gplane})));
        } else {
            DH_TRY((product<true, true, TOK_M, PLANES>(
                h.op, g, 1, EpiG<PLANES, false>{h.c, w.rows.lse, w.rows.w, nullptr, v0, G, rows, gplane})));
            teacher_entries<PLANES><<<h.N, 256, 0, stream()>>>(w.rows, h.teacher, h.V, v0, R, w.q, w.z, G,
                                                               rows, gplane);
            DH_TRY(check_launch(h.op));
        }
        if (d.dH) {
            Prod gh{G, W, rows, ldw, gplane, wplane, h.N, h.D, R, 0, w.rows.cnt};
            DH_TRY((product<true, false, TOK_M, PLANES>(h.op, gh, p.splits,
                                                        EpiAcc{acc, p.Dp, v0 == 0, split})));
        }
        if (d.dW) {
            Prod gw{G, w.Hp, rows, p.Dp, gplane, hplane, R, h.D, h.N, 0, w.rows.cnt};
            if (d.type == DH_F32)
                DH_TRY((product<false, false, TOK_K, PLANES>(
                    h.op, gw, 1, EpiOut<float>{(float*)d.dW + (size_t)v0 * d.lddw, d.lddw, d.acc_dW})));
            else
                DH_TRY((product<false, false, TOK_K, PLANES>(
                    h.op, gw, 1, EpiOut<uint16_t>{(uint16_t*)d.dW + (size_t)v0 * d.lddw, d.lddw, d.acc_dW})));
        }
        if (h.V - v0 <= rows) break;
    }
    if (d.dH) {
        if (d.type == DH_F32)
            dh_finish<<<(h.N + 3) / 4, 256, 0, stream()>>>(w.rows.inv, h.N, h.D, acc, p.Dp, p.splits, split,
                                                           (float*)d.dH, d.lddh, d.acc_dH);
        else
            dh_finish<<<(h.N + 3) / 4, 256, 0, stream()>>>(w.rows.inv, h.N, h.D, acc, p.Dp, p.splits, split,
                                                           (uint16_t*)d.dH, d.lddh, d.acc_dH);
        DH_TRY(check_launch(h.op));
    }
    return DH_OK;
}

int run_forward(const Head& h, float* loss, float* lse, void* ws, size_t ws_bytes) {
    const int K = h.target ? 0 : h.teacher.K;
    DH_TRY(check_head(h, K, ws, ws_bytes, 0));
    if (h.N > 0 && (!loss || (!h.target && K > 0 && (!h.teacher.id || !h.teacher.logit))))
        return set_error(DH_ERR_INVALID, "%s: null pointer", h.op);
    DH_TRY(ensure_init());
    if (h.N == 0) return DH_OK;
    return h.dtype == DH_F32 ? forward<float, 3>(h, loss, lse, ws, ws_bytes)
                             : forward<uint16_t, 1>(h, loss, lse, ws, ws_bytes);
}

int run_backward(const Head& h, const Grads& d, void* ws, size_t ws_bytes) {
    const int K = h.target ? 0 : h.teacher.K;
    DH_TRY(check_head(h, K, ws, ws_bytes, 1));
    if (d.type != DH_F32 && d.type != h.dtype)
        return set_error(DH_ERR_INVALID, "%s: grad_type must be fp32 or the inputs' type", h.op);
    if ((d.dH && d.lddh < h.D) || (d.dW && d.lddw < h.D))
        return set_error(DH_ERR_INVALID, "%s: leading dimension of a gradient below D", h.op);
    if (h.N > 0 && (!d.lse || (!h.target && K > 0 && (!h.teacher.id || !h.teacher.logit))))
        return set_error(DH_ERR_INVALID, "%s: null pointer", h.op);
    DH_TRY(ensure_init());
    if (!d.dH && !d.dW) return DH_OK;
    if (h.N == 0) {
        if (!d.dW || d.acc_dW) return DH_OK;
        if (d.type == DH_F32)
            clear_rows<<<2048, 256, 0, stream()>>>((float*)d.dW, h.V, h.D, d.lddw);
        else
            clear_rows<<<2048, 256, 0, stream()>>>((uint16_t*)d.dW, h.V, h.D, d.lddw);
        return check_launch(h.op);
    }
    return h.dtype == DH_F32 ? backward<float, 3>(h, d, ws, ws_bytes)
                             : backward<uint16_t, 1>(h, d, ws, ws_bytes);
}

Head xent_head(const char* op, int dtype, int N, int V, int D, float scale, const void* H, int ldh,
               const void* W, int ldw, const int* target) {
    return Head{op, dtype, N, V, D, H, ldh, W, ldw, scale, target, Teacher{}, 1.f, scale};
}
// c = 1 / T; the loss's T^2 and the logits' 1 / T leave G a factor of T.
Head distill_head(const char* op, int dtype, int N, int V, int D, int K, float T, const void* H, int ldh,
                  const void* W, int ldw, const int* id, const float* logit) {
    return Head{op, dtype, N, V, D, H, ldh, W, ldw, 1.f / T, nullptr, Teacher{id, logit, K, 1.f / T}, T * T, T};
}

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" {

size_t dh_linear_xent_workspace(int dtype, int N, int V, int D, int backward) {
    return N < 0 || V < 1 || D < 1 ? 0 : least_ws(dtype, N, V, D, 0, backward);
}

int dh_linear_xent_fwd(int dtype, int N, int V, int D, float scale, const void* H, int ldh, const void* W,
                       int ldw, const int* target, float* loss, float* lse, void* ws, size_t ws_bytes) {
    if (N > 0 && !target) return set_error(DH_ERR_INVALID, "dh_linear_xent_fwd: null pointer");
    return run_forward(xent_head("dh_linear_xent_fwd", dtype, N, V, D, scale, H, ldh, W, ldw, target), loss,
                       lse, ws, ws_bytes);
}

int dh_linear_xent_bwd(int dtype, int N, int V, int D, float scale, const void* H, int ldh, const void* W,
                       int ldw, const int* target, const float* lse, const float* dloss, void* dH, int lddh,
                       int acc_dH, void* dW, int lddw, int acc_dW, int grad_type, void* ws,
                       size_t ws_bytes) {
    if (N > 0 && !target) return set_error(DH_ERR_INVALID, "dh_linear_xent_bwd: null pointer");
    return run_backward(xent_head("dh_linear_xent_bwd", dtype, N, V, D, scale, H, ldh, W, ldw, target),
                        Grads{lse, dloss, dH, lddh, acc_dH, dW, lddw, acc_dW, grad_type}, ws, ws_bytes);
}

size_t dh_linear_distill_workspace(int dtype, int N, int V, int D, int K, int backward) {
    return N < 0 || V < 1 || D < 1 || K < 0 ? 0 : least_ws(dtype, N, V, D, K, backward);
}

int dh_linear_distill_fwd(int dtype, int N, int V, int D, int K, float T, const void* H, int ldh,
                          const void* W, int ldw, const int* top_id, const float* top_logit, float* loss,
                          float* lse, void* ws, size_t ws_bytes) {
    if (K < 0) return set_error(DH_ERR_INVALID, "dh_linear_distill_fwd: K=%d", K);
    return run_forward(distill_head("dh_linear_distill_fwd", dtype, N, V, D, K, T, H, ldh, W, ldw, top_id,
                                    top_logit), loss, lse, ws, ws_bytes);
}

int dh_linear_distill_bwd(int dtype, int N, int V, int D, int K, float T, const void* H, int ldh,
                          const void* W, int ldw, const int* top_id, const float* top_logit,
                          const float* lse, const float* dloss, void* dH, int lddh, int acc_dH, void* dW,
                          int lddw, int acc_dW, int grad_type, void* ws, size_t ws_bytes) {
    if (K < 0) return set_error(DH_ERR_INVALID, "dh_linear_distill_bwd: K=%d", K);
    return run_backward(distill_head("dh_linear_distill_bwd", dtype, N, V, D, K, T, H, ldh, W, ldw, top_id,
                                     top_logit),
                        Grads{lse, dloss, dH, lddh, acc_dH, dW, lddw, acc_dW, grad_type}, ws, ws_bytes);
}

}  // extern "C"
