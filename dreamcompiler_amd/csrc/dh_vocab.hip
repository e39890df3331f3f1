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
// All four products run on the 16-bit matrix cores with fp32 accumulators.  The forward takes bf16
// operands as they are.  Every other operand is scaled by a power of two and held in fp16 parts of 11
// significant bits, one or two, x = hi + 2^-11 lo; a product of two by two is 2^-11 (lo hi + hi lo) +
// hi hi: the cross products are added first, the accumulators scaled by 2^-11 (exactly), then the
// third is added (lo lo, at most 2^-22 of the product, is left out).  Three 16-bit products at 16 times the rate of an fp32 one.
//   fp32 inputs            two parts of all operands
//   bf16, gradients bf16   one part: H and W fit exactly, G is rounded to 11 bits, whose 2^-11 is an eighth
//                          of the result's own rounding (to bf16 G would lose as much as the result
//                          does, and at the targets in one direction); as many products
//   bf16, gradients fp32   one part of H and W, two of G: 1, 2 and 2 products
// A row's weight is w_n = wtop 2^k m with wtop the largest weight and m in [1/2, 1): G has m, and 2^k, which
// is exact, goes to the other operand of dW and to dH's rows, so neither loses rows of small weight.
// With the operand's largest value scaled below 2^15, the others are taken to 2^-23 (one part: 2^-11) of
// themselves or 2^-50 (2^-39) of it, whichever is more.  What the scale is common to: a row
// where k runs along the row (H, and W in the forward), else all of the operand (W in the
// backward, where its rows are summed over; G, whose entries are m (p - q); and 2^k H_n, the other
// operand of dW).
#include <algorithm>
#include <type_traits>

#include "dh_common.hpp"
#include "dh_vocab_range.hpp"

namespace dh {
namespace {

// Launches of more than 2^22 work-groups have a second dimension: a dimension has less than 2^32 threads.
inline dim3 long_grid(long long n) {
    const long long x = 1 << 22;
    return dim3((unsigned)std::min(n, x), (unsigned)((n + x - 1) / x));
}
__device__ inline long long grid_index() { return (long long)blockIdx.y << 22 | blockIdx.x; }

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

typedef uint16_t h8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));

// |x| < 2^16 as two fp16 parts, x = p[0] + 2^-11 p[1]; an infinity or NaN is its own first part.
__device__ inline void split2(float x, uint16_t (&p)[2]) {
    // Holds x to its fp32 value: a product that the compiler folds into the conversion is rounded
    // once there and twice for the remainder, and near a tie hi and the remainder then belong to
    // different neighbours.
    asm("" : "+v"(x));
    const _Float16 hi = (_Float16)x;
    const float r = __builtin_fabsf(x) < INFINITY ? x - (float)hi : 0.f;
    const _Float16 lo = (_Float16)(r * 2048.f);
    p[0] = __builtin_bit_cast(uint16_t, hi);
    p[1] = __builtin_bit_cast(uint16_t, lo);
}
// What the products take of a value: its nearest bf16 (BF), or that many fp16 parts.
constexpr int BF = 0;
constexpr int parts_of(int P) { return P == 2 ? 2 : 1; }
template <int P>
__device__ inline void to_parts(float x, uint16_t (&p)[parts_of(P)]) {
    if constexpr (P == BF) p[0] = rne_bf16(x);
    else if constexpr (P == 1) p[0] = __builtin_bit_cast(uint16_t, (_Float16)x);
    else split2(x, p);
}
template <int P>
__device__ inline void store_parts(uint16_t* __restrict__ dst, long long plane, const float (&v)[8]) {
    constexpr int PARTS = parts_of(P);
    h8 o[PARTS];
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        uint16_t x[PARTS];
        to_parts<P>(v[e], x);
#pragma unroll
        for (int p = 0; p < PARTS; ++p) o[p][e] = x[p];
    }
#pragma unroll
    for (int p = 0; p < PARTS; ++p) *reinterpret_cast<h8*>(dst + p * plane) = o[p];
}

// The scale of an operand whose largest finite value is mx: 2^-e puts it into [2^14, 2^15).  e is
// at least -124, so that 2^-e is finite: what that loses lies below fp32's range.
__device__ inline int scale_of(float mx) {
    return mx > 0.f ? max(__builtin_amdgcn_frexp_expf(mx) - 15, -124) : 0;
}
__device__ inline float larger(float mx, const float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const float a = __builtin_fabsf(x[e]);
        mx = a < INFINITY ? fmaxf(mx, a) : mx;
    }
    return mx;
}

// One row of D values as parts with zeros up to Dp, by one wave.  fp16: OWN, at the row's own
// scale, which is returned; else v 2^-e f (f at most 1 in size, so nothing overflows on the way).
template <typename T, int P, bool OWN>
__device__ inline int convert_row(const T* __restrict__ src, int D, uint16_t* __restrict__ dst, int Dp,
                                  long long plane, int lane, int e = 0, float f = 1.f) {
    if constexpr (P == BF) {
        for (int c = 8 * lane; c < Dp; c += 512) {
            float v[8];
            load8(src, c, D, v);
            store_parts<BF>(dst + c, plane, v);
        }
        return 0;
    } else {
        constexpr int KEEP = OWN ? 4 : 0;   // 2048 columns in registers, the rest is read again
        float v[KEEP + 1][8];
        if constexpr (OWN) {
            float mx = 0.f;
#pragma unroll
            for (int t = 0; t < KEEP; ++t)
                if (8 * lane + 512 * t < Dp) {
                    load8(src, 8 * lane + 512 * t, D, v[t]);
                    mx = larger(mx, v[t]);
                }
            for (int c = 8 * lane + 512 * KEEP; c < Dp; c += 512) {
                float x[8];
                load8(src, c, D, x);
                mx = larger(mx, x);
            }
            e = scale_of(wave_reduce(mx, OpMax()));
        }
        const float scale = __builtin_ldexpf(1.f, -e);
        auto put = [&](int c, float (&x)[8]) {
#pragma unroll
            for (int q = 0; q < 8; ++q) x[q] = OWN ? x[q] * scale : (x[q] * scale) * f;
            store_parts<P>(dst + c, plane, x);
        };
#pragma unroll
        for (int t = 0; t < KEEP; ++t)
            if (8 * lane + 512 * t < Dp) put(8 * lane + 512 * t, v[t]);
        for (int c = 8 * lane + 512 * KEEP; c < Dp; c += 512) {
            float x[8];
            load8(src, c, D, x);
            put(c, x);
        }
        return e;
    }
}

// ---- packing ------------------------------------------------------------------------------------
// What a packed row i is: its row n, target, loss weight and lse (backward), and its scale (fp16).
// Arrays are padded to whole tiles of rows, so that a tile's epilogue may load past the last row.
struct Rows {
    int* cnt;          // rows that count
    int* row;          // packed -> row
    int* target;
    int* hexp;
    float *w, *lse;    // backward only.  w: w_n, from stage_scaled on its m
    float* rest;       // and wtop 2^k
};
// fp16: the scales of the other operands.
struct Exps {
    int* e;            // forward: of the piece's table rows
    int *X, *E;        // backward: of 2^k H_n and of the table
    float* wtop;       // the largest weight
    int* group;        // per group of packed rows, the largest scale that w_n H_n asks for,
    float* gtop;       // and its largest weight
    float* wmax;       // per work-group of the scan, the table's largest value
};
constexpr int SCAN = 1024;   // most work-groups that look for it
constexpr int NO_EXP = -(1 << 20);
__device__ inline int exponent(float x) {   // of a finite value that is not zero
    const float a = __builtin_fabsf(x);
    return a > 0.f && a < INFINITY ? __builtin_amdgcn_frexp_expf(x) : NO_EXP;
}

__device__ inline bool counts(int target, int V) { return (unsigned)target < (unsigned)V; }

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
// Whether row n counts: it has a target, or an entry.
struct Targets {
    const int* target;   // or null: the teacher's
    Teacher t;
    int V;
    __device__ bool has(int n) const {
        if (target) return counts(target[n], V);
        for (int k = 0; k < t.K; ++k)
            if (entry_counts(t, (size_t)n * t.K + k, V)) return true;
        return false;
    }
};

// flag[n] = 0 where row n has an entry, -1 where it has none: for so many entries that pack_rows
// had better not look for them again and again (2048 rows x 32: packing 16.0 us alone, 8.3 with the
// flags, which take 5.1), or for so many of a row that one without entries, which is known only after all,
// holds its group up (200 x 100 entries x 2000 x 256 bf16, 0.3 of the rows padding, forward and gradient 86 us
// without and 66 with flags; without padding 64 and 67).  A wave per row.
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

template <typename OT>
__device__ inline void zero_row(OT* p, int D, int lane) {
    for (int c = lane; c < D; c += 64) p[c] = OT(0);
}

struct Pack {
    Targets targets;
    int N, D;
    const void* H;
    int ldh;
    const void* W;
    int ldw;
    uint16_t* Hp;
    int Dp;
    long long plane;
    Rows rows;
    Exps exps;
    int groups;              // of PACK rows
    const int* counts;       // of count_rows, or null
    float c;
    // forward
    float *loss, *lse_out, *base;
    // backward
    const float *lse_in, *dloss;
    float wscale;
    void* dH;                // its padding rows are cleared here (or null)
    int lddh, dh_f32;
    // work-groups behind the groups
    int tables;              // stage the table's first rows: R of them, 16 a work-group
    int R;
    uint16_t* staged;
    long long wplane;
};
constexpr int PACK = 16;     // rows of a work-group, one per wave

// How many of every COUNT rows count, for N above MANY: every group of pack_rows looking through all
// rows before its own is quadratic in them (forward and gradient of N x 65 x 32 bf16, us, without / with these launches
// and that of scales(): 8192 43.3 / 45.5, 16384 63.4 / 58.8, 65536 283 / 140, 2^20 35598 / 1913).
constexpr int COUNT = 1024, MANY = 10240;
__global__ void __launch_bounds__(COUNT) count_rows(Targets t, int N, int* __restrict__ counts) {
    __shared__ int red[COUNT / 64];
    const int n = blockIdx.x * COUNT + threadIdx.x;
    const uint64_t mask = __ballot(n < N && t.has(n));
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = __popcll(mask);
    __syncthreads();
    if (threadIdx.x != 0) return;
    int sum = 0;
    for (int x = 0; x < COUNT / 64; ++x) sum += red[x];
    counts[blockIdx.x] = sum;
}

// Work-group b < groups packs rows 16 b .. 16 b + 15: it counts the rows that count before them (the
// targets are few and stay in cache), then converts its own.  Forward: also the padding's zeros and,
// for cross entropy, base = -z at the target (the loss is lse + base).  The work-groups behind
// stage table rows (forward), or look for the table's largest value (backward).
template <typename T, int P>
__global__ void __launch_bounds__(1024) pack_rows(Pack a) {
    __shared__ int red[16];
    __shared__ float tops[16];
    __shared__ int own[PACK];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const T* H = (const T*)a.H;
    const T* W = (const T*)a.W;
    const int V = a.targets.V, D = a.D;
    if ((int)blockIdx.x >= a.groups) {
        const int b = blockIdx.x - a.groups;
        if (b < a.tables) {
            const int r = 16 * b + w;
            if (r >= a.R) return;
            const int e = convert_row<T, P, true>(W + (size_t)r * a.ldw, D, a.staged + (size_t)r * a.Dp,
                                                  a.Dp, a.wplane, lane);
            if (P != BF && lane == 0) a.exps.e[r] = e;
            return;
        }
        if constexpr (P != BF) {
            const int scan = gridDim.x - a.groups;
            float mx = 0.f;
            for (long long v = 16LL * b + w; v < V; v += 16LL * scan)
                for (int c = 8 * lane; c < D; c += 512) {
                    float x[8];
                    load8(W + (size_t)v * a.ldw, c, D, x);
                    mx = larger(mx, x);
                }
            mx = wave_reduce(mx, OpMax());
            if (lane == 0) red[w] = __builtin_bit_cast(int, mx);
            __syncthreads();
            if (threadIdx.x != 0) return;
            for (int x = 1; x < 16; ++x) mx = fmaxf(mx, __builtin_bit_cast(float, red[x]));
            a.exps.wmax[b] = mx;
        }
        return;
    }
    const int n0 = blockIdx.x * PACK;
    int before = 0;
    if (a.counts)
        for (int b = threadIdx.x; b < n0 / COUNT; b += 1024) before += a.counts[b];
    for (int n = (a.counts ? n0 / COUNT * COUNT : 0) + threadIdx.x; n < n0; n += 1024) before += a.targets.has(n);
    for (int m = 1; m < 64; m <<= 1) before += __shfl_xor(before, m, 64);
    if (lane == 0) red[w] = before;
    if (threadIdx.x < PACK) own[threadIdx.x] = n0 + (int)threadIdx.x < a.N && a.targets.has(n0 + threadIdx.x);
    __syncthreads();
    before = 0;
    for (int x = 0; x < 16; ++x) before += red[x];
    int count = 0, i = before;
    for (int x = 0; x < PACK; ++x) {
        if (x < w) i += own[x];
        count += own[x];
    }
    if ((int)blockIdx.x == a.groups - 1 && threadIdx.x == 0) *a.rows.cnt = before + count;
    const int n = n0 + w;
    const bool keep = own[w];
    int most = NO_EXP;
    float top = 0.f;   // the weight's size, where finite
    if (keep) {
        const int h = convert_row<T, P, true>(H + (size_t)n * a.ldh, D, a.Hp + (size_t)i * a.Dp, a.Dp, a.plane,
                                              lane);
        const int target = a.targets.target ? a.targets.target[n] : 0;
        if (a.base) {
            const float d = row_dot(H + (size_t)n * a.ldh, W + (size_t)target * a.ldw, D, lane);
            if (lane == 0) a.base[i] = -(a.c * d);
        }
        if (lane == 0) {
            a.rows.row[i] = n;
            a.rows.target[i] = target;
            a.rows.hexp[i] = h;
            if (a.lse_in) {
                const float wn = (a.dloss ? a.dloss[n] : 1.f) * a.wscale, size = __builtin_fabsf(wn);
                a.rows.lse[i] = a.lse_in[n];
                a.rows.w[i] = wn;
                most = exponent(wn) + h;   // |w_n H_n| < 2^(15 + this)
                top = size < INFINITY ? size : 0.f;
            }
        }
    } else if (n < a.N) {
        if (lane == 0 && a.loss) {
            a.loss[n] = 0.f;
            if (a.lse_out) a.lse_out[n] = 0.f;
        }
        if (a.dH) {
            if (a.dh_f32) zero_row((float*)a.dH + (size_t)n * a.lddh, D, lane);
            else zero_row((uint16_t*)a.dH + (size_t)n * a.lddh, D, lane);
        }
    }
    if (P != BF && a.lse_in) {
        __syncthreads();   // red[] has been read
        if (lane == 0) {
            red[w] = most;
            tops[w] = top;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            for (int x = 1; x < 16; ++x) {
                most = max(most, red[x]);
                top = fmaxf(top, tops[x]);
            }
            a.exps.group[blockIdx.x] = most;
            a.exps.gtop[blockIdx.x] = top;
        }
    }
}

// Forward: rows v0 .. v0 + R - 1 of the table as parts, a wave per row.
template <typename T, int P>
__global__ void __launch_bounds__(256) stage_table(const T* __restrict__ W, int ldw, int v0, int R, int D,
                                                   uint16_t* __restrict__ dst, int Dp, long long plane,
                                                   int* __restrict__ exps) {
    const int lane = threadIdx.x & 63;
    const int r = blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= R) return;
    const int e = convert_row<T, P, true>(W + (size_t)(v0 + r) * ldw, D, dst + (size_t)r * Dp, Dp, plane,
                                          lane);
    if (P != BF && lane == 0) exps[r] = e;
}

// Backward: the scales of the table and of 2^k H_n, and the largest weight, from the scan's results and the
// groups', by a work-group of WAVES waves.
template <int WAVES>
__device__ inline void find_scales(const Exps& exps, int groups, int scan, int& E, int& X, float& top) {
    __shared__ float red[3][WAVES];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    float mx = 0.f, x = NO_EXP;   // exponents are exact as floats
    top = 0.f;
    for (int g = threadIdx.x; g < max(scan, groups); g += 64 * WAVES) {   // all loads before the first wait
        if (g < scan) mx = fmaxf(mx, exps.wmax[g]);
        if (g < groups) {
            x = fmaxf(x, (float)exps.group[g]);
            top = fmaxf(top, exps.gtop[g]);
        }
    }
    mx = wave_reduce(mx, OpMax());
    x = wave_reduce(x, OpMax());
    top = wave_reduce(top, OpMax());
    if (lane == 0) {
        red[0][w] = mx;
        red[1][w] = x;
        red[2][w] = top;
    }
    __syncthreads();
    for (int o = 0; o < WAVES; ++o) {
        mx = fmaxf(mx, red[0][o]);
        x = fmaxf(x, red[1][o]);
        top = fmaxf(top, red[2][o]);
    }
    X = (int)x;
    E = scale_of(mx);
    if (!(top > 0.f)) top = 1.f;   // all weights are zero
    X = X - exponent(top) + 1;     // |w_n / top| < 2^(its exponent - top's + 1), and so 2^k at most
}
// For N above MANY: once, instead of by every work-group of stage_scaled.
__global__ void __launch_bounds__(1024) scales(Exps exps, int groups, int scan) {
    int E, X;
    float top;
    find_scales<16>(exps, groups, scan, E, X, top);
    if (threadIdx.x != 0) return;
    *exps.E = E;
    *exps.X = X;
    *exps.wtop = top;
}

// Backward: rows of the table at its scale; the work-groups behind (first piece) convert the packed rows of
// 2^k H_n at theirs, and take the weights apart.  Unless the scales are known, each work-group finds them, and the first one
// writes them down.  HBM-bound: 131072 x 2048 bf16 187 us, 5.7 TB/s (and pack_rows' scan before it 133 us, 4.0 TB/s).
template <typename T, int P>
__global__ void __launch_bounds__(256) stage_scaled(const T* __restrict__ W, int ldw, int v0, int R,
                                                    int D, uint16_t* __restrict__ dst, int Dp,
                                                    long long plane, Exps exps, int groups, int scan, int known,
                                                    int tables, Rows rows, const T* __restrict__ H, int ldh,
                                                    uint16_t* __restrict__ Xp, long long xplane) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    int E, X;
    float top;
    if (known) {
        E = *exps.E;
        X = *exps.X;
        top = *exps.wtop;
    } else {
        find_scales<4>(exps, groups, scan, E, X, top);
        if (blockIdx.x == 0 && threadIdx.x == 0) {
            *exps.E = E;
            *exps.X = X;
            *exps.wtop = top;
        }
    }
    if ((int)blockIdx.x < tables) {
        const int r = blockIdx.x * 4 + w;
        if (r < R)
            convert_row<T, P, false>(W + (size_t)(v0 + r) * ldw, D, dst + (size_t)r * Dp, Dp, plane, lane, E);
        return;
    }
    const int i = (blockIdx.x - tables) * 4 + w;
    if (i >= *rows.cnt) return;
    const int h = rows.hexp[i];
    // A weight of zero (or none: G has the infinity or NaN) takes nothing of H.
    const float share = rows.w[i] / top;
    const int k = exponent(share);
    const bool some = k != NO_EXP;
    convert_row<T, P, false>(H + (size_t)rows.row[i] * ldh, D, Xp + (size_t)i * Dp, Dp, xplane, lane, h,
                             some ? __builtin_ldexpf(1.f, k + h - X) : 0.f);
    if (lane == 0) {
        rows.w[i] = some ? __builtin_ldexpf(share, -k) : share;
        rows.rest[i] = some ? __builtin_ldexpf(top, k) : 1.f;
    }
}

// ---- teachers ------------------------------------------------------------------------------------
// A row's teacher: largest logit and logarithm of the sum of exponentials, by every wave.
__device__ inline void teacher_stats(const Teacher& t, size_t at, int V, float& mx, float& log_sum) {
    const int lane = threadIdx.x & 63;
    mx = -INFINITY;
    for (int k = lane; k < t.K; k += 64)
        if (entry_counts(t, at + k, V)) mx = fmaxf(mx, t.logit[at + k]);
    mx = wave_reduce(mx, OpMax());
    float sum = 0.f;
    for (int k = lane; k < t.K; k += 64)
        if (entry_counts(t, at + k, V)) sum += __expf((t.logit[at + k] - mx) * t.inv_t);
    log_sum = __logf(wave_reduce(sum, OpSum()));
}

// A work-group per packed row: the teacher's probabilities q (N x K, zero where there is no entry), the
// student's logits z at its tokens, and base[i] = sum q (log q - z).  The entries' rows of W lie
// anywhere, so a wave has four of them in flight: 2048 x 32 entries x 1024 bf16 31 us, 4.3 TB/s (two a wave, one
// after the other: 39), 4096 x 100 x 2048 330 us, 5.1 TB/s (360).
constexpr int TEACHER_FLY = 4;
template <typename T>
__global__ void __launch_bounds__(512) teacher_dots(Rows rows, Teacher t, int V,
                                                    const T* __restrict__ H, int ldh,
                                                    const T* __restrict__ W, int ldw, int D,
                                                    float* __restrict__ q, float* __restrict__ z,
                                                    float* __restrict__ base) {
    __shared__ float red[8];
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), waves = blockDim.x >> 6;
    const int i = (int)grid_index();
    if (i >= *rows.cnt) return;
    const int n = rows.row[i];
    const size_t at = (size_t)n * t.K, to = (size_t)i * t.K;
    const T* h = H + (size_t)n * ldh;
    for (int k0 = w; k0 < t.K; k0 += TEACHER_FLY * waves) {
        const T* row[TEACHER_FLY];
        float s[TEACHER_FLY] = {};
#pragma unroll
        for (int f = 0; f < TEACHER_FLY; ++f) {   // no entry: the table's first row, unused
            const int k = k0 + f * waves, id = k < t.K ? t.id[at + k] : -1;
            row[f] = W + (counts(id, V) ? (size_t)id * ldw : 0);
        }
        for (int c = 8 * lane; c < D; c += 512) {
            float x[8], y[TEACHER_FLY][8];
            load8(h, c, D, x);
#pragma unroll
            for (int f = 0; f < TEACHER_FLY; ++f) load8(row[f], c, D, y[f]);
#pragma unroll
            for (int f = 0; f < TEACHER_FLY; ++f)
#pragma unroll
                for (int e = 0; e < 8; ++e) s[f] = __builtin_fmaf(x[e], y[f][e], s[f]);
        }
#pragma unroll
        for (int f = 0; f < TEACHER_FLY; ++f) {
            s[f] = wave_reduce(s[f], OpSum());
            const int k = k0 + f * waves;
            if (lane == 0 && k < t.K) z[to + k] = t.inv_t * s[f];
        }
    }
    // Largest logit and sum of exponentials: every wave for itself, over all entries.
    float mx, log_sum;
    teacher_stats(t, at, V, mx, log_sum);
    __syncthreads();   // z is there
    float part = 0.f;
    for (int k = threadIdx.x; k < t.K; k += blockDim.x) {
        float qk = 0.f;
        if (entry_counts(t, at + k, V)) {
            const float lq = (t.logit[at + k] - mx) * t.inv_t - log_sum;
            qk = __expf(lq);
            // exp underflows below about -104: the entry's share of the loss is zero there
            if (!(qk == 0.f)) part += qk * (lq - z[to + k]);
        }
        q[to + k] = qk;
    }
    part = wave_reduce(part, OpSum());
    if (lane == 0) red[w] = part;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int x = 1; x < waves; ++x) part += red[x];
    base[i] = part;
}

// The probabilities of a row's tokens, for many entries: q[k] of the first entry of a token is the sum over its
// entries, of the others -1.  Sums are integers of 2^-62, so they do not go by the order of the atomics (q below
// 2^-39 is cut there, far below what the products take of it).  A work-group per row; the table's tokens go
// by in ranges of SUM_RANGE, each a look at all entries.  Looking through the row for each entry instead, as
// fewer do, is quadratic in K (forward and gradient of D = 256 bf16, us, that / so: 512 x 32000 of 128 entries 179 / 181,
// 256 215 / 210, 1024 594 / 375, 8192 16755 / 2021; 512 x 131072 of 256 469 / 496, 512 567 / 552, 2048 1838 / 957; 4096 x
// 32000 of 128 710 / 768, 256 931 / 937, 1024 2837 / 1929).
constexpr int SUM_RANGE = 4096, SUM_LEAST = 128;
bool by_sums(int V, int K) { return K > SUM_LEAST && (long long)K * K > 2LL * V; }
__global__ void __launch_bounds__(1024) teacher_sums(const int* __restrict__ cnt, const int* __restrict__ row,
                                                     Teacher t, int V, float* __restrict__ q) {
    __shared__ unsigned long long sum[SUM_RANGE];
    __shared__ int first[SUM_RANGE];
    const int i = (int)grid_index();
    if (cnt && i >= *cnt) return;
    const size_t at = (size_t)(row ? row[i] : i) * t.K, to = (size_t)i * t.K;
    float mx, log_sum;
    teacher_stats(t, at, V, mx, log_sum);
    auto prob = [&](int k) { return __expf((t.logit[at + k] - mx) * t.inv_t - log_sum); };
    const bool sound = log_sum - log_sum == 0.f && mx < INFINITY;   // else every entry's q is NaN
    for (int k = threadIdx.x; k < t.K; k += 1024) q[to + k] = sound ? -1.f : NAN;
    if (!sound) return;
    for (long long v0 = 0; v0 < V; v0 += SUM_RANGE) {
        __syncthreads();   // the range before has been read
        for (int r = threadIdx.x; r < SUM_RANGE; r += 1024) {
            sum[r] = 0;
            first[r] = t.K;
        }
        __syncthreads();
        for (int k = threadIdx.x; k < t.K; k += 1024) {
            const long long r = t.id[at + k] - v0;
            if (r < 0 || r >= SUM_RANGE || !entry_counts(t, at + k, V)) continue;
            atomicAdd(&sum[r], (unsigned long long)(prob(k) * 0x1p62f));
            atomicMin(&first[r], k);
        }
        __syncthreads();
        for (int k = threadIdx.x; k < t.K; k += 1024) {
            const long long r = t.id[at + k] - v0;
            if (r >= 0 && r < SUM_RANGE && first[r] == k) q[to + k] = (float)sum[r] * 0x1p-62f;
        }
    }
}

// ---- products -------------------------------------------------------------------------------------
// C (M x N) = sum over k of A and B, operands of PA and PB fp16 parts (or both BF).  AK: A is stored
// [m][k], else [k][m]; BK: B is stored [n][k], else [k][n].  One of M, N and K counts packed rows: its
// extent is *cnt.
struct Prod {
    const uint16_t *A, *B;
    int lda, ldb;
    long long pa, pb;      // elements between an operand's parts
    int M, N, K;
    int kstages;           // 32-k stages of one split (blockIdx.y)
    const int* cnt;
};
enum { TOK_M, TOK_N, TOK_K };

// One operand's tile of T rows (of m or n) and stages of BK k in LDS, by WAVES waves.  Filled by
// direct DMA in blocks of 1 KB (lane l's 16 bytes land at 16 l), read as MFMA fragments of 32 rows
// and 16 k.  16-byte chunks, swizzled so that neither kind of read meets bank conflicts:
//   KC   [T rows][BK k]: chunk c of row r at c ^ (r / 4 % 4) (BK = 32) or c ^ (r / 2 % 8) (64);
//        a fragment is one 16-byte read
//   else [BK k][T]: chunk c of row k at c ^ 4 (k % 4), for T = 64 (two rows in the 64 banks)
//        c ^ 4 (k / 2 % 2); a fragment is two transposing reads
// Loads go through a buffer resource whose range ends with the operand's last column of the last row
// (dh_vocab_range.hpp), so what lies behind reads as zero; it begins with the tile (KC; the stage's place in
// the rows is a scalar offset) or with the stage, so operands of any size keep 32-bit offsets.
template <bool KC, int T, int BK, int WAVES>
struct Operand {
    static constexpr int PER = T * BK / 512 / WAVES;   // blocks per wave
    static constexpr int CPR = KC ? BK / 8 : T / 8;    // chunks in a row
    static_assert(PER >= 1, "tile shapes");
    uint32_t off[PER];
    u32x4 rs;
    uint32_t soff;
    const uint16_t* base;          // the tile's first element
    long long plane;
    int ld, K, rows;               // rows: of the tile (KC)
    int t0, extent;

    __device__ static int swizzle(int r) {
        if (KC) return BK == 32 ? (r >> 2) & 3 : (r >> 1) & 7;
        return T == 64 ? 4 * ((r >> 1) & 1) : 4 * (r & 3);
    }
    __device__ static int row_of(int t, int wave, int lane) { return 64 / CPR * (PER * wave + t) + lane / CPR; }
    __device__ static int chunk_of(int t, int wave, int lane) {
        return (lane % CPR) ^ swizzle(row_of(t, wave, lane));
    }
    __device__ void init(const uint16_t* p, long long plane_, int ld_, int t0_, int extent_, int K_, int wave,
                         int lane) {
        ld = ld_;
        K = K_;
        t0 = t0_;
        extent = extent_;
        plane = plane_;
        base = KC ? p + (size_t)t0 * ld : p + t0;
        rows = min(extent - t0, T);
#pragma unroll
        for (int t = 0; t < PER; ++t)
            off[t] = 2u * ((uint32_t)row_of(t, wave, lane) * ld + 8 * chunk_of(t, wave, lane));
    }
    // Stage kt of a part is the next one.
    __device__ void start(int part, int kt) {
        rs = make_rsrc(base + part * plane + (KC ? 0 : (size_t)kt * BK * ld),
                       KC ? range_bytes(rows, ld, K, 0) : range_bytes(BK, ld, extent, t0));
#pragma unroll
        for (int e = 0; e < 4; ++e) rs[e] = __builtin_amdgcn_readfirstlane(rs[e]);
        soff = __builtin_amdgcn_readfirstlane(KC ? 2u * BK * kt : 0u);
    }
    __device__ void next() {
        if (KC) {
            soff += 2 * BK;
        } else {
            const uint64_t a = (((uint64_t)rs[1] << 32) | rs[0]) + 2u * BK * ld;
            rs[0] = (uint32_t)a;
            rs[1] = (uint32_t)(a >> 32);
        }
    }
    __device__ void issue_one(uint32_t to, int t) const { lds_dma16_buf_so(off[t], rs, soff, to + 1024u * t); }
    // Of a stage kt that ends behind K: zeros from there on (KC: by whole chunks).
    __device__ void issue_end(uint32_t to, int t, int kt, int wave, int lane) const {
        const int left = K - BK * kt;
        u32x4 r = rs;
        if (!KC) r[2] = range_bytes(min(left, BK), ld, extent, t0);
        lds_dma16_buf_so(!KC || 8 * chunk_of(t, wave, lane) < left ? off[t] : 0xFFFFFFF0u, r, soff, to + 1024u * t);
    }
    // Tile rows o .. o + 31, 16-k step kk of the stage.
    __device__ static bf16x8 frag(const uint16_t* lds, int o, int kk, int lane) {
        const int h = lane >> 5;
        if constexpr (KC) {
            const int r = o + (lane & 31);
            return *reinterpret_cast<const bf16x8*>(lds + r * BK + 8 * ((2 * kk + h) ^ swizzle(r)));
        } else {
            const int i = lane & 15, n = o + 16 * ((lane >> 4) & 1) + 4 * (i & 3);
            s16x4 r[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int k = 16 * kk + 8 * h + 4 * q + (i >> 2);
                r[q] = ds_read_tr(lds + k * T + 8 * ((n >> 3) ^ swizzle(k)) + 4 * ((n >> 2) & 1));
            }
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
};

// The 16-bit products that make one of such operands, in this order: low parts of A by B (two of A),
// A by low parts of B (two of B), high by high.
constexpr int kinds_of(int PA, int PB) { return 1 + (PA == 2) + (PB == 2); }
constexpr int part_a(int PA, int kind) { return PA == 2 && kind == 0; }
constexpr int part_b(int PA, int PB, int kind) { return PB == 2 && kind == (PA == 2); }

template <int PA>
__device__ inline void mfma16(const bf16x8& a, const bf16x8& b, f32x16& acc) {
    if constexpr (PA == BF)
        acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, acc, 0, 0, 0);
    else
        acc = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), acc,
                                                     0, 0, 0);
}
template <int PA, int FM, int FN>
__device__ inline void mfma_parts(const bf16x8 (&fa)[FM], const bf16x8 (&fb)[FN], f32x16 (&acc)[FM][FN]) {
#pragma unroll
    for (int a = 0; a < FM; ++a)
#pragma unroll
        for (int b = 0; b < FN; ++b) mfma16<PA>(fa[a], fb[b], acc[a][b]);
}

// Tiles: 256 x 256 by 8 waves of 128 x 64 and 128 x 128 by 4 waves of 64 x 64, stages of 32 k; 64 x 64
// by 4 waves of 32 x 32, stages of 64 k (few work-groups: half the barriers, and whole 128-byte
// lines of a k-contiguous operand).
template <int T_>
struct Shape {
    static constexpr int T = T_, BK = T == 64 ? 64 : 32, NS = 4;
    static constexpr int DEEP = 3 * T * 64 + NS * T * 32;   // elements of gemm_deep's rings
    static constexpr int WAVES = T == 256 ? 8 : 4;
    static constexpr int WAVES_N = T == 256 ? 4 : 2;
    static constexpr int WM = T * WAVES_N / WAVES, WN = T / WAVES_N;
    static constexpr int FM = WM / 32, FN = WN / 32;
    static constexpr int STAGE = 2 * T * BK;   // elements
    static constexpr int THREADS = 64 * WAVES;
};

// Row of register r of block a, relative to the wave's first row.
__device__ inline int reg_row(int a, int r, int lane) { return 32 * a + 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3); }

typedef int i32x4 __attribute__((ext_vector_type(4)));
constexpr float LOG2E = 1.4426950408889634f;

// 32 rows of a wave's tile of 16-bit values through its piece of LDS, so that they are written as
// 16-byte pieces of rows: element by element (a lane has one column of 16 rows) the stores of a 256 x 256
// tile took 38 us, as much as 40 of its stages.  put(row, chunk column, 8 values) writes a piece.
// The lanes read what others stored, and the next 32 rows go into the same LDS: fences before both.
constexpr int LDS_TILE = 32 * (64 + 8);   // elements; rows 16 bytes longer, so that the halves' banks differ
template <int FN, class Put>
__device__ inline void store_rows(uint16_t* lds, const uint16_t (&v)[FN][16], int row0, int lane, const Put& put) {
    constexpr int LD = 32 * FN + 8, CHUNKS = 4 * FN;
#pragma unroll
    for (int b = 0; b < FN; ++b)
#pragma unroll
        for (int r = 0; r < 16; ++r) lds[reg_row(0, r, lane) * LD + 32 * b + (lane & 31)] = v[b][r];
    wave_fence();
#pragma unroll
    for (int i = 0; i < 32 * CHUNKS / 64; ++i) {
        const int r = 64 / CHUNKS * i + lane / CHUNKS, c = 8 * (lane % CHUNKS);
        put(row0 + r, c, *reinterpret_cast<const h8*>(lds + r * LD + c));
    }
    wave_fence();
}

// One tile of one split: stages of BK k through a ring of four in LDS filled by direct DMA three
// stages ahead; a stage's 16-k steps run while the next operands are read (the schedule of the
// bf16 GEMM's 8-wave form).  Epi::run gets the tile's accumulators: register r of block (a, b) is
// row m0 + wm + 32 a + 8 (r / 4) + 4 h + r % 4, column n0 + wn + 32 b + l32 (lane = 32 h + l32).
template <class S, bool AK, bool BK_, int TOK, int PA, int PB, class Epi>
__device__ inline void gemm_tile(uint16_t* ring, const Prod& g, const Epi& epi, int tile, int tiles,
                                 int split) {
    constexpr int FM = S::FM, FN = S::FN, BK = S::BK, NS = S::NS, STEPS = BK / 16;
    using OA = Operand<AK, S::T, BK, S::WAVES>;
    using OB = Operand<BK_, S::T, BK, S::WAVES>;
    constexpr int BOFF = S::T * BK, LOADS = OA::PER + OB::PER;
    const int cnt = __builtin_amdgcn_readfirstlane(*g.cnt);
    const int M = TOK == TOK_M ? cnt : g.M, N = TOK == TOK_N ? cnt : g.N;
    const int Kall = TOK == TOK_K ? cnt : g.K;
    int tm, tn;
    xcd_tile_order(tile, tiles, (g.M + S::T - 1) / S::T, (g.N + S::T - 1) / S::T, 4, tm, tn);
    const int m0 = tm * S::T, n0 = tn * S::T;
    if (m0 >= M || n0 >= N) return;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = (wave / S::WAVES_N) * S::WM, wn = (wave % S::WAVES_N) * S::WN;

    f32x16 acc[FM][FN];
#pragma unroll
    for (int a = 0; a < FM; ++a)
#pragma unroll
        for (int b = 0; b < FN; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;

    const int kt0 = split * g.kstages;
    const int nk = max(0, min((Kall + BK - 1) / BK - kt0, g.kstages));
    // the last kind, from stage `cross` on, is high by high
    constexpr int KINDS = kinds_of(PA, PB);
    const int total = KINDS * nk, cross = (KINDS - 1) * nk;
    if (total > 0) {
        OA sa;
        OB sb;
        sa.init(g.A, g.pa, g.lda, m0, M, Kall, wave, lane);
        sb.init(g.B, g.pb, g.ldb, n0, N, Kall, wave, lane);
        sa.start(part_a(PA, 0), kt0);
        sb.start(part_b(PA, PB, 0), kt0);
        const int tail = (kt0 + nk) * BK > Kall ? nk - 1 : -1;   // the stage that ends behind K
        constexpr uint32_t RING = 2u * NS * S::STAGE;
        const uint32_t ring0 = lds_addr(ring);
        const uint32_t wave_a = 1024u * OA::PER * wave, wave_b = 2u * BOFF + 1024u * OB::PER * wave;
        int ikt = 0, kind = 0;   // the next stage to fetch
        uint32_t slot = 0;
        auto issue = [&]() {
            const uint32_t to = __builtin_amdgcn_readfirstlane(ring0 + slot);
            if (__builtin_expect(ikt != tail, 1)) {
#pragma unroll
                for (int t = 0; t < OA::PER; ++t) sa.issue_one(to + wave_a, t);
#pragma unroll
                for (int t = 0; t < OB::PER; ++t) sb.issue_one(to + wave_b, t);
            } else {
#pragma unroll
                for (int t = 0; t < OA::PER; ++t) sa.issue_end(to + wave_a, t, kt0 + ikt, wave, lane);
#pragma unroll
                for (int t = 0; t < OB::PER; ++t) sb.issue_end(to + wave_b, t, kt0 + ikt, wave, lane);
            }
            slot = slot == RING - 2u * S::STAGE ? 0u : slot + 2u * S::STAGE;
            sa.next();
            sb.next();
            if (++ikt == nk && KINDS > 1) {
                ikt = 0;
                ++kind;
                sa.start(part_a(PA, kind), kt0);
                sb.start(part_b(PA, PB, kind), kt0);
            }
        };
        auto landed = [&](int ahead) {   // all but the youngest `ahead` stages
            if (ahead >= 2) wait_vmcnt<2 * LOADS>();
            else if (ahead == 1) wait_vmcnt<LOADS>();
            else wait_vmcnt<0>();
        };
        auto scale_cross = [&](int s) {
            if (KINDS > 1 && s == cross)
#pragma unroll
                for (int a = 0; a < FM; ++a)
#pragma unroll
                    for (int b = 0; b < FN; ++b)
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[a][b][r] *= 0x1p-11f;
        };
        auto read = [&](int s, int kk, bf16x8 (&fa)[FM], bf16x8 (&fb)[FN]) {
            const uint16_t* st = ring + (s % NS) * S::STAGE;
#pragma unroll
            for (int x = 0; x < FM; ++x) fa[x] = OA::frag(st, wm + 32 * x, kk, lane);
#pragma unroll
            for (int x = 0; x < FN; ++x) fb[x] = OB::frag(st + BOFF, wn + 32 * x, kk, lane);
            __builtin_amdgcn_sched_barrier(0);
        };
        bf16x8 fa[2][FM], fb[2][FN];
        auto mma = [&](int f) {
            mfma_parts<PA, FM, FN>(fa[f], fb[f], acc);
            __builtin_amdgcn_sched_barrier(0);
        };
        auto inner = [&](int s) {   // all steps but the last, whose operands it reads
            scale_cross(s);
#pragma unroll
            for (int kk = 0; kk < STEPS - 1; ++kk) {
                read(s, kk + 1, fa[(kk + 1) & 1], fb[(kk + 1) & 1]);
                mma(kk & 1);
            }
        };
        const int pre = min(total, NS - 1);
        for (int s = 0; s < pre; ++s) issue();
        landed(pre - 1);
        __syncthreads();
        read(0, 0, fa[0], fb[0]);
        int s = 0;
        for (; s < total - NS + 1; ++s) {
            issue();
            inner(s);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            wait_vmcnt<(NS - 2) * LOADS>();
            __syncthreads();
            read(s + 1, 0, fa[0], fb[0]);
            mma(1);
        }
        for (; s < total - 1; ++s) {   // all is fetched
            inner(s);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            landed(total - 2 - s);
            __syncthreads();
            read(s + 1, 0, fa[0], fb[0]);
            mma(1);
        }
        inner(total - 1);
        mma(1);
    }
    if constexpr (Epi::LDS) __syncthreads();   // the ring is free
    epi.template run<FM, FN>(acc, M, N, m0 + wm, n0 + wn, lane, split, ring + wave * LDS_TILE);
}

// The 256-wide tile with a k-contiguous A: A in 64-k stages (whole 128-byte lines of a row, where 32-k
// stages fetch each half by itself) through a ring of three beside B's 32-k stages in a ring of
// four, 160 KB; the bf16 GEMM's schedule for such operands.  A pair of stages (64 k) at a time:
// pair p of A is fetched in stage 2 p - 4, stage s of B in stage s - 3, and past the end the last
// ones again into slots that nobody reads any more, so that the waits are constants: when stage s
// ends, stage s + 1 has landed and 12 (s even) or 8 (odd) younger loads may be in flight.  An odd
// last stage lies past K and reads as zero.
template <class S, bool BK_, int TOK, int PA, int PB, class Epi>
__device__ inline void gemm_deep(uint16_t* ring, const Prod& g, const Epi& epi, int tile, int tiles, int split) {
    constexpr int FM = S::FM, FN = S::FN, T = S::T;
    using OA = Operand<true, T, 64, S::WAVES>;
    using OB = Operand<BK_, T, 32, S::WAVES>;
    static_assert(OA::PER == 4 && OB::PER == 2, "the waits below");
    const int cnt = __builtin_amdgcn_readfirstlane(*g.cnt);
    const int M = TOK == TOK_M ? cnt : g.M, N = TOK == TOK_N ? cnt : g.N;
    int tm, tn;
    xcd_tile_order(tile, tiles, (g.M + T - 1) / T, (g.N + T - 1) / T, 4, tm, tn);
    const int m0 = tm * T, n0 = tn * T;
    if (m0 >= M || n0 >= N) return;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = (wave / S::WAVES_N) * S::WM, wn = (wave % S::WAVES_N) * S::WN;

    f32x16 acc[FM][FN];
#pragma unroll
    for (int a = 0; a < FM; ++a)
#pragma unroll
        for (int b = 0; b < FN; ++b)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;

    const int p0 = split * g.kstages;   // in pairs
    const int np = max(0, min((g.K + 63) / 64 - p0, g.kstages));
    constexpr int KINDS = kinds_of(PA, PB);
    const int pairs = KINDS * np;
    if (pairs > 0) {
        OA sa;
        OB sb;
        sa.init(g.A, g.pa, g.lda, m0, M, g.K, wave, lane);
        sb.init(g.B, g.pb, g.ldb, n0, N, g.K, wave, lane);
        sa.start(part_a(PA, 0), p0);
        sb.start(part_b(PA, PB, 0), 2 * p0);
        const uint32_t ring_a0 = lds_addr(ring) + 1024u * OA::PER * wave;
        const uint32_t ring_b0 = lds_addr(ring) + 2u * 3 * T * 64 + 1024u * OB::PER * wave;
        uint16_t* const ring_a = ring;
        uint16_t* const ring_b = ring + 3 * T * 64;
        const bool tail = (p0 + np) * 64 > g.K;
        int ap = 0, akind = 0, an = 0;   // the next pair of A, and how many are fetched
        uint32_t aslot = 0;
        // Load t of the next pair; with the last one goes on to the pair behind it.  INSIDE: neither
        // the last pair of the part, nor one that ends behind K.
        auto load_a = [&](int t, auto inside) {
            constexpr bool INSIDE = decltype(inside)::value;
            const uint32_t to = ring_a0 + aslot;
            if (INSIDE || __builtin_expect(!tail || ap != np - 1, 1)) sa.issue_one(to, t);
            else sa.issue_end(to, t, p0 + ap, wave, lane);
            if (t + 1 < OA::PER) return;
            aslot = aslot == 2u * 2 * T * 64 ? 0u : aslot + 2u * T * 64;
            if (INSIDE) {
                sa.next();
            } else if (++an < pairs) {
                sa.next();
                if (++ap == np) {
                    ap = 0;
                    ++akind;
                    sa.start(part_a(PA, akind), p0);
                }
            }
        };
        int bs = 0, bkind = 0, bn = 0;
        uint32_t bslot = 0;
        auto load_b = [&](int t, auto inside) {
            constexpr bool INSIDE = decltype(inside)::value;
            const uint32_t to = ring_b0 + bslot;
            if (INSIDE || __builtin_expect(!tail || bs < 2 * np - 2, 1)) sb.issue_one(to, t);
            else sb.issue_end(to, t, 2 * p0 + bs, wave, lane);
            if (t + 1 < OB::PER) return;
            bslot = (bslot + 2u * T * 32) & (2u * 4 * T * 32 - 1);
            if (INSIDE) {
                sb.next();
            } else if (++bn < 2 * pairs) {
                sb.next();
                if (++bs == 2 * np) {
                    bs = 0;
                    ++bkind;
                    sb.start(part_b(PA, PB, bkind), 2 * p0);
                }
            }
        };
        constexpr std::false_type anywhere{};
        auto issue_a = [&] {
#pragma unroll
            for (int t = 0; t < OA::PER; ++t) load_a(t, anywhere);
        };
        auto issue_b = [&] {
#pragma unroll
            for (int t = 0; t < OB::PER; ++t) load_b(t, anywhere);
        };
        bf16x8 fa[2][FM], fb[2][FN];
        // The products of fragments f, and under each a read of the other ones (16-k step ka of A's
        // slot la, kb of B's lb) and a load: a wave that issues them in a row leaves its SIMD's matrix
        // core idle.
        auto step = [&](int f, const uint16_t* la, int ka, const uint16_t* lb, int kb, auto dma) {
#pragma unroll
            for (int i = 0; i < FM * FN; ++i) {
                const int a = i / FN, b = i % FN;
                mfma16<PA>(fa[f][a], fb[f][b], acc[a][b]);
                if (i < FM) fa[f ^ 1][i] = OA::frag(la, wm + 32 * i, ka, lane);
                else if (i < FM + FN) fb[f ^ 1][i - FM] = OB::frag(lb, wn + 32 * (i - FM), kb, lane);
                dma(i);
                __builtin_amdgcn_sched_barrier(0);
            }
        };
        auto none = [](int) {};
        issue_a();
        issue_b();
        issue_b();
        issue_a();
        issue_b();
        wait_vmcnt<8>();
        __syncthreads();
#pragma unroll
        for (int x = 0; x < FM; ++x) fa[0][x] = OA::frag(ring_a, wm + 32 * x, 0, lane);
#pragma unroll
        for (int x = 0; x < FN; ++x) fb[0][x] = OB::frag(ring_b, wn + 32 * x, 0, lane);
        uint32_t sla = 0, slb = 0;   // elements to the slots of the pair at hand
        auto pair = [&](auto inside) {
            const uint16_t* la = ring_a + sla;
            sla = sla == 2 * T * 64 ? 0 : sla + T * 64;
            const uint16_t* next = ring_a + sla;
            const uint16_t *lb = ring_b + slb, *lb1 = lb + T * 32;
            slb ^= 2 * T * 32;
            const uint16_t* lb2 = ring_b + slb;
            step(0, la, 1, lb, 1, [&](int i) {
                if (i >= 2 && i < 4) load_b(i - 2, inside);
                else if (i >= 4) load_a(i - 4, inside);
            });
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            wait_vmcnt<12>();
            __syncthreads();
            step(1, la, 2, lb1, 0, none);
            step(0, la, 3, lb1, 1, [&](int i) {
                if (i >= 6) load_b(i - 6, inside);
            });
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            wait_vmcnt<8>();
            __syncthreads();
            step(1, next, 0, lb2, 0, none);   // after the last pair: what is there, unused
        };
        for (int kind = 0; kind < KINDS; ++kind) {
            if (KINDS > 1 && kind == KINDS - 1)
#pragma unroll
                for (int a = 0; a < FM; ++a)
#pragma unroll
                    for (int b = 0; b < FN; ++b)
#pragma unroll
                        for (int r = 0; r < 16; ++r) acc[a][b][r] *= 0x1p-11f;
            int p = 0;
            for (; p < np - 3; ++p) pair(std::true_type{});   // fetches pair p + 2 and stage 2 p + 4
            an += p, ap += p, bn += 2 * p, bs += 2 * p;
            for (; p < np; ++p) pair(anywhere);
        }
        wait_vmcnt<0>();   // what was fetched again lands before the LDS is given away
    }
    if constexpr (Epi::LDS) __syncthreads();   // the ring is free
    epi.template run<FM, FN>(acc, M, N, m0 + wm, n0 + wn, lane, split, ring + wave * LDS_TILE);
}

// The 64-wide tile of two parts by two: a stage holds 64 k of both parts of both operands (32 KB, a ring of
// four) and each of its 16-k steps makes all three products, the cross products in accumulators of
// their own.  One chain of stages instead of three, and two thirds of the loads.
template <class S, bool AK, bool BK_, int TOK, class Epi>
__device__ inline void gemm_both(uint16_t* ring, const Prod& g, const Epi& epi, int tile, int tiles,
                                 int split) {
    constexpr int T = S::T, BK = S::BK, NS = S::NS, STEPS = BK / 16, SUB = T * BK;
    static_assert(S::FM == 1 && S::FN == 1, "one block per wave");
    using OA = Operand<AK, T, BK, S::WAVES>;
    using OB = Operand<BK_, T, BK, S::WAVES>;
    constexpr int LOADS = 2 * (OA::PER + OB::PER);
    const int cnt = __builtin_amdgcn_readfirstlane(*g.cnt);
    const int M = TOK == TOK_M ? cnt : g.M, N = TOK == TOK_N ? cnt : g.N;
    const int Kall = TOK == TOK_K ? cnt : g.K;
    int tm, tn;
    xcd_tile_order(tile, tiles, (g.M + T - 1) / T, (g.N + T - 1) / T, 4, tm, tn);
    const int m0 = tm * T, n0 = tn * T;
    if (m0 >= M || n0 >= N) return;
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = (wave / S::WAVES_N) * S::WM, wn = (wave % S::WAVES_N) * S::WN;

    f32x16 acc[1][1], cross;
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[0][0][r] = cross[r] = 0.f;
    const int kt0 = split * g.kstages;
    const int total = max(0, min((Kall + BK - 1) / BK - kt0, g.kstages));
    if (total > 0) {
        OA sa[2];
        OB sb[2];
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            sa[p].init(g.A, g.pa, g.lda, m0, M, Kall, wave, lane);
            sb[p].init(g.B, g.pb, g.ldb, n0, N, Kall, wave, lane);
            sa[p].start(p, kt0);
            sb[p].start(p, kt0);
        }
        const int tail = (kt0 + total) * BK > Kall ? total - 1 : -1;   // the stage that ends behind K
        constexpr uint32_t RING = 2u * NS * 4 * SUB;
        const uint32_t ring0 = lds_addr(ring) + 1024u * OA::PER * wave;
        static_assert(OA::PER == OB::PER, "one offset of the wave");
        int ikt = 0;   // the next stage to fetch
        uint32_t slot = 0;
        auto issue = [&]() {
            const uint32_t to = ring0 + slot;
#pragma unroll
            for (int p = 0; p < 2; ++p)
#pragma unroll
                for (int t = 0; t < OA::PER; ++t) {
                    if (__builtin_expect(ikt != tail, 1)) {
                        sa[p].issue_one(to + 2u * SUB * p, t);
                        sb[p].issue_one(to + 2u * SUB * (2 + p), t);
                    } else {
                        sa[p].issue_end(to + 2u * SUB * p, t, kt0 + ikt, wave, lane);
                        sb[p].issue_end(to + 2u * SUB * (2 + p), t, kt0 + ikt, wave, lane);
                    }
                }
            slot = slot == RING - 2u * 4 * SUB ? 0u : slot + 2u * 4 * SUB;
            ++ikt;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                sa[p].next();
                sb[p].next();
            }
        };
        auto landed = [&](int ahead) {   // all but the youngest `ahead` stages
            if (ahead >= 2) wait_vmcnt<2 * LOADS>();
            else if (ahead == 1) wait_vmcnt<LOADS>();
            else wait_vmcnt<0>();
        };
        f16x8 fa[2][2], fb[2][2];   // [buffer][part]
        auto read = [&](int s, int kk, int f) {
            const uint16_t* st = ring + (s % NS) * 4 * SUB;
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                fa[f][p] = __builtin_bit_cast(f16x8, OA::frag(st + p * SUB, wm, kk, lane));
                fb[f][p] = __builtin_bit_cast(f16x8, OB::frag(st + (2 + p) * SUB, wn, kk, lane));
            }
            __builtin_amdgcn_sched_barrier(0);
        };
        auto mma = [&](int f) {
            cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[f][1], fb[f][0], cross, 0, 0, 0);
            acc[0][0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[f][0], fb[f][0], acc[0][0], 0, 0, 0);
            cross = __builtin_amdgcn_mfma_f32_32x32x16_f16(fa[f][0], fb[f][1], cross, 0, 0, 0);
            __builtin_amdgcn_sched_barrier(0);
        };
        const int pre = min(total, NS - 1);
        for (int s = 0; s < pre; ++s) issue();
        landed(pre - 1);
        __syncthreads();
        read(0, 0, 0);
        for (int s = 0; s < total; ++s) {
            if (s + NS - 1 < total) issue();
#pragma unroll
            for (int kk = 0; kk < STEPS - 1; ++kk) {
                read(s, kk + 1, (kk + 1) & 1);
                mma(kk & 1);
            }
            if (s + 1 < total) {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                landed(min(total - 1, s + NS - 1) - (s + 1));
                __syncthreads();
                read(s + 1, 0, 0);
            }
            mma(1);
        }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) acc[0][0][r] = __builtin_fmaf(cross[r], 0x1p-11f, acc[0][0][r]);
    if constexpr (Epi::LDS) __syncthreads();   // the ring is free
    epi.template run<1, 1>(acc, M, N, m0 + wm, n0 + wn, lane, split, ring + wave * LDS_TILE);
}

// The form that a shape and its operands take, and its LDS in elements.
template <class S, bool AK, int PA, int PB>
constexpr int ring_of() {
    return S::T == 256 && AK ? S::DEEP : S::NS * S::STAGE * (S::T == 64 && PA == 2 && PB == 2 ? 2 : 1);
}
template <class S, bool AK, bool BK, int TOK, int PA, int PB, class Epi>
__device__ inline void gemm_form(uint16_t* ring, const Prod& g, const Epi& epi, int tile, int tiles, int split) {
    if constexpr (S::T == 256 && AK) gemm_deep<S, BK, TOK, PA, PB>(ring, g, epi, tile, tiles, split);
    else if constexpr (S::T == 64 && PA == 2 && PB == 2) gemm_both<S, AK, BK, TOK>(ring, g, epi, tile, tiles, split);
    else gemm_tile<S, AK, BK, TOK, PA, PB>(ring, g, epi, tile, tiles, split);
}

// The four products.  Bound by the matrix cores, at a clock that falls under them (by the cycles counted at most
// 1.55 to 1.71 of 2.4 GHz).  Measured for 8192 rows x 131072 x 2048 bf16, 4.4 TFLOP each, in ms, PFLOP/s and share of
// the cycles that the matrix cores are busy: statistics 3.48 / 1.26 / 76%, G 3.90 / 1.13 / 63% (exponentials, and
// 16-bit G through LDS), dH 3.28 / 1.34 / 82%, dW 3.76 / 1.17 / 67% (both operands by transposing reads, 32-k
// stages); a bf16 product of 8192^3 by the vendor's library reaches 1.23 here.  2048 x 32000 x 1024 fp32,
// 0.134 TFLOP each, in us and TFLOP/s of fp32: 342 / 392, 375 / 358, 329 / 408, 371 / 362; the fp32 matrix
// cores themselves end at 157.
template <class S, bool AK, bool BK, int TOK, int PA, int PB, class Epi>
__global__ void __launch_bounds__(S::THREADS) vocab_gemm(Prod g, Epi epi) {
    __shared__ __attribute__((aligned(16))) uint16_t ring[ring_of<S, AK, PA, PB>()];
    gemm_form<S, AK, BK, TOK, PA, PB>(ring, g, epi, blockIdx.x, gridDim.x, blockIdx.y);
}

// dH and dW of a piece in one launch: the first `first` work-groups are dH's, splits one after the
// other.  H and W in P parts, G in GP.
template <class S, int P, int GP, class EpiH, class EpiW>
__global__ void __launch_bounds__(S::THREADS) vocab_grads(Prod gh, EpiH eh, int tiles_h, int first, Prod gw,
                                                          EpiW ew, int tiles_w) {
    __shared__ __attribute__((aligned(16))) uint16_t ring[ring_of<S, true, GP, P>()];
    const int b = blockIdx.x;
    if (b < first)
        gemm_form<S, true, false, TOK_M, GP, P>(ring, gh, eh, b % tiles_h, tiles_h, b / tiles_h);
    else
        gemm_form<S, false, false, TOK_K, GP, P>(ring, gw, ew, (b - first) % tiles_w, tiles_w,
                                                 (b - first) / tiles_w);
}

// Forward: rows are table rows, columns packed rows.  A lane holds half of the wave's logits of
// each of its columns, lane + 32 the other half: their maximum and sum of exponentials go to
// part[the wave's block of 32 FM rows][column].
template <int P>
struct EpiLse {
    static constexpr bool LDS = false;
    float c;
    const int *e, *h;      // exponents of the table's and the packed rows' scales (fp16)
    float2* part;
    int ldp;
    template <int FM, int FN>
    __device__ void run(f32x16 (&acc)[FM][FN], int M, int N, int row0, int col0, int lane, int,
                        uint16_t*) const {
        if (row0 >= M) return;   // the wave has no table row: its block is not joined either
        const bool full = row0 + 32 * FM <= M;
        // fp16: the logits in place; bf16: they are c times the accumulators, and
        // exp(c (x - mx)) = 2^(k x - k mx) with k = c log2(e), one multiply-add an exponential.
        // -inf past the table's end.
        float kc[FN];
#pragma unroll
        for (int b = 0; b < FN; ++b)
            kc[b] = P == BF ? 1.f : __builtin_ldexpf(c, h[col0 + 32 * b + (lane & 31)]);
        const float k = P == BF ? c * LOG2E : LOG2E;
        if (P != BF || !full)
#pragma unroll
        for (int a = 0; a < FM; ++a)
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const int row = row0 + reg_row(a, 4 * r4, lane);
                i32x4 e4;
                if constexpr (P != BF) e4 = *reinterpret_cast<const i32x4*>(e + row);
#pragma unroll
                for (int q = 0; q < 4; ++q)
#pragma unroll
                    for (int b = 0; b < FN; ++b) {
                        const float z =
                            P == BF ? acc[a][b][4 * r4 + q]
                                       : acc[a][b][4 * r4 + q] * __builtin_ldexpf(kc[b], e4[q]);
                        acc[a][b][4 * r4 + q] = full || row + q < M ? z : -INFINITY;
                    }
            }
#pragma unroll
        for (int b = 0; b < FN; ++b) {
            float mx = -INFINITY;
#pragma unroll
            for (int a = 0; a < FM; ++a)
#pragma unroll
                for (int r = 0; r < 16; ++r) mx = fmaxf(mx, acc[a][b][r]);
            mx = fmaxf(mx, xor32(mx));
            const float m = mx == -INFINITY ? 0.f : mx;   // all -inf: a sum of zeros, not of NaN
            const float km = k * m;
            float s = 0.f;
#pragma unroll
            for (int a = 0; a < FM; ++a)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s += __builtin_amdgcn_exp2f(P == BF ? __builtin_fmaf(k, acc[a][b][r], -km)
                                                           : k * (acc[a][b][r] - m));
            s += xor32(s);
            const int col = col0 + 32 * b + (lane & 31);
            if (lane < 32 && col < N)
                part[(size_t)(row0 / (32 * FM)) * ldp + col] = float2{P == BF ? c * mx : mx, s};
        }
    }
};

// Backward: rows are packed rows, columns the piece's table rows.  G = 2^14 m (p - q) in GP fp16
// parts.  Columns past the table's end up to the tile's are zero.
template <int GP, bool HARD>
struct EpiG {
    static constexpr bool LDS = true;
    float c;
    const float *lse, *w;
    const int *target, *h, *E;
    int v0;
    uint16_t* G;
    int ldg;
    long long plane;
    template <int FM, int FN>
    __device__ void run(const f32x16 (&acc)[FM][FN], int M, int N, int row0, int col0, int lane, int,
                        uint16_t* lds) const {
        const int table = *E, col = col0 + (lane & 31);
        // One part: 2^(k x - log2(e) lse) with the factor log2(e) in k, one multiply-add an exponential.
        const float c1 = GP == 1 ? c * LOG2E : c;
#pragma unroll
        for (int a = 0; a < FM; ++a) {
            uint16_t v[GP][FN][16];
#pragma unroll
            for (int r4 = 0; r4 < 4; ++r4) {
                const int row = row0 + reg_row(a, 4 * r4, lane);
                const f32x4 l4 = *reinterpret_cast<const f32x4*>(lse + row);
                const f32x4 w4 = *reinterpret_cast<const f32x4*>(w + row);
                const i32x4 h4 = *reinterpret_cast<const i32x4*>(h + row);
                i32x4 t4;
                if constexpr (HARD) t4 = *reinterpret_cast<const i32x4*>(target + row);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const float k = __builtin_ldexpf(c1, h4[e] + table);
                    const float l = GP == 1 ? l4[e] * LOG2E : l4[e];
                    const float m = 0x1p14f * w4[e];
#pragma unroll
                    for (int b = 0; b < FN; ++b) {
                        const float x = __builtin_fmaf(k, acc[a][b][4 * r4 + e], -l);
                        float p = __builtin_amdgcn_exp2f(GP == 1 ? x : x * LOG2E);
                        if constexpr (HARD)
                            if (col + 32 * b == t4[e] - v0) p -= 1.f;
                        uint16_t parts[GP];
                        to_parts<GP>(col + 32 * b < N ? m * p : 0.f, parts);
#pragma unroll
                        for (int q = 0; q < GP; ++q) v[q][b][4 * r4 + e] = parts[q];
                    }
                }
            }
#pragma unroll
            for (int q = 0; q < GP; ++q)
                store_rows<FN>(lds, v[q], row0 + 32 * a, lane, [&](int row, int cc, h8 x) {
                    if (row < M) *reinterpret_cast<h8*>(G + q * plane + (size_t)row * ldg + col0 + cc) = x;
                });
        }
    }
};

// fp32 sums over the pieces (dH), one block per split.
struct EpiAcc {
    static constexpr bool LDS = false;
    float* C;
    int ldc, first;
    long long split;
    template <int FM, int FN>
    __device__ void run(const f32x16 (&acc)[FM][FN], int M, int N, int row0, int col0, int lane, int s,
                        uint16_t*) const {
        float* p = C + s * split;
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

// A gradient's rows and their scales: dH's packed rows go to their places, times wtop 2^k 2^(E - 14); dW's
// stay in order, times wtop 2^(X - 14).
template <typename OT>
struct Grad {
    OT* C;
    int ldc, accumulate;
    const int *row, *exp;
    const float* w;
    int own;               // w is the rows', else one for all
    // wtop in two: its power of two goes with the scale, so that a sum of large H and a small weight stay
    // within fp32 between the two steps.
    __device__ int scale() const { return *exp - 14 + (own ? 0 : __builtin_amdgcn_frexp_expf(*w)); }
    __device__ float common() const { return own ? 1.f : __builtin_amdgcn_frexp_mantf(*w); }
    __device__ float weight(int i, float common) const { return own ? w[i] : common; }
    __device__ OT* at(int i) const { return C + (size_t)(row ? row[i] : i) * ldc; }
    __device__ void put(OT* to, float v) const {
        if constexpr (sizeof(OT) == 4) {
            *to = accumulate ? *to + v : v;
        } else {
            if (accumulate) v += bf16_bits_to_f32(*to);
            *to = rne_bf16(v);
        }
    }
};

// A gradient from its only split and piece.  bf16 that is not added to what is there goes through LDS.
template <typename OT>
struct EpiOut {
    static constexpr bool LDS = sizeof(OT) == 2;
    Grad<OT> out;
    template <int FM, int FN>
    __device__ void run(const f32x16 (&acc)[FM][FN], int M, int N, int row0, int col0, int lane, int,
                        uint16_t* lds) const {
        const int s = out.scale();
        const float common = out.common();
        if constexpr (LDS) {
            if (!out.accumulate) {
#pragma unroll
                for (int a = 0; a < FM; ++a) {
                    uint16_t v[FN][16];
#pragma unroll
                    for (int r = 0; r < 16; ++r) {
                        const int row = row0 + reg_row(a, r, lane);
                        const float w = row < M ? out.weight(row, common) : 0.f;
#pragma unroll
                        for (int b = 0; b < FN; ++b) v[b][r] = rne_bf16(__builtin_ldexpf(acc[a][b][r], s) * w);
                    }
                    store_rows<FN>(lds, v, row0 + 32 * a, lane, [&](int row, int cc, h8 x) {
                        if (row >= M || col0 + cc >= N) return;
                        OT* to = out.at(row) + col0 + cc;
                        if (col0 + cc + 8 <= N) {
                            *reinterpret_cast<h8a*>(to) = x;   // at any alignment
                        } else {
#pragma unroll
                            for (int e = 0; e < 8; ++e)
                                if (col0 + cc + e < N) to[e] = x[e];
                        }
                    });
                }
                return;
            }
        }
#pragma unroll
        for (int a = 0; a < FM; ++a)
#pragma unroll
            for (int r = 0; r < 16; ++r) {
                const int row = row0 + reg_row(a, r, lane);
                if (row >= M) continue;
                OT* to = out.at(row);
                const float w = out.weight(row, common);
#pragma unroll
                for (int b = 0; b < FN; ++b) {
                    const int col = col0 + 32 * b + (lane & 31);
                    if (col >= N) continue;
                    out.put(to + col, __builtin_ldexpf(acc[a][b][r], s) * w);
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

// The end of a row's join: what earlier pieces left (first: nothing) merged with this piece's, kept
// for the next, or the row's lse and loss = factor (lse + base) from the last.
struct JoinOut {
    Rows rows;
    float2* state;
    int first, last;
    const float* base;
    float factor;
    float *loss, *lse;
    __device__ void put(int i, float m, float s) const {
        if (!first) {
            const float2 p = state[i];
            float m0 = p.x, s0 = p.y;
            lse_merge(m0, s0, m, s);
            m = m0;
            s = s0;
        }
        if (!last) {
            state[i] = float2{m, s};
            return;
        }
        const int n = rows.row[i];
        const float l = m + __logf(s);
        if (lse) lse[n] = l;
        loss[n] = factor * (l + base[i]);
    }
};

// A work-group per 64 packed rows, 16 waves that share the piece's blocks of table rows; their
// results meet in LDS in wave order.  8192 rows x 1024 blocks: 41 us.
__global__ void __launch_bounds__(1024) lse_join(const float2* __restrict__ part, int ldp, int blocks,
                                                 JoinOut out) {
    __shared__ float2 red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int i = blockIdx.x * 64 + lane;
    const int cnt = *out.rows.cnt;
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
    m = red[0][lane].x;
    s = red[0][lane].y;
    for (int x = 1; x < 16; ++x) lse_merge(m, s, red[x][lane].x, red[x][lane].y);
    out.put(i, m, s);
}

// Up to 512 rows, which are few work-groups of the other kind (forward of 100 x 32000 x 256 bf16 14.9 against
// 24.5 us, of 512 23.4 against 27.2).
// A work-group per packed row, its 256 threads share the blocks.  The lanes' results
// meet at distances 1 to 32, the waves' in wave order.
__global__ void __launch_bounds__(256) lse_join_few(const float2* __restrict__ part, int ldp, int blocks,
                                                    JoinOut out) {
    __shared__ float2 red[4];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int i = blockIdx.x;
    if (i >= *out.rows.cnt) return;
    float m = -INFINITY, s = 0.f;
    for (int b = threadIdx.x; b < blocks; b += 256) {
        const float2 p = part[(size_t)b * ldp + i];
        lse_merge(m, s, p.x, p.y);
    }
    for (int x = 1; x < 64; x <<= 1) {
        const float m2 = __shfl_xor(m, x, 64), s2 = __shfl_xor(s, x, 64);
        lse_merge(m, s, m2, s2);
    }
    if (lane == 0) red[w] = float2{m, s};
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int x = 1; x < 4; ++x) lse_merge(m, s, red[x].x, red[x].y);
    out.put(i, m, s);
}

// The entries of G at the teacher's tokens inside a piece, from the fp32 logits: m (p - q), q
// summed where a token occurs more than once: by its first entry (SUMS: teacher_sums has done it), else each of
// its entries writes the same value.
template <int GP, bool SUMS>
__global__ void __launch_bounds__(256) teacher_entries(Rows rows, Teacher t, int V, int v0, int R,
                                                       const float* __restrict__ q,
                                                       const float* __restrict__ z,
                                                       uint16_t* __restrict__ G, int ldg,
                                                       long long plane) {
    const int i = (int)grid_index();
    if (i >= *rows.cnt) return;
    const size_t at = (size_t)rows.row[i] * t.K, from = (size_t)i * t.K;
    const float m = 0x1p14f * rows.w[i], lse = rows.lse[i];
    for (int k = threadIdx.x; k < t.K; k += 256) {
        const int id = t.id[at + k];
        if (id < v0 || id >= v0 + R || !entry_counts(t, at + k, V)) continue;
        float sum = 0.f;
        if constexpr (SUMS) {
            sum = q[from + k];
            if (sum < 0.f) continue;
        } else {
            for (int j = 0; j < t.K; ++j)
                if (t.id[at + j] == id) sum += q[from + j];
        }
        uint16_t parts[GP];
        to_parts<GP>(m * (__expf(z[from + k] - lse) - sum), parts);
        uint16_t* to = G + (size_t)i * ldg + (id - v0);
#pragma unroll
        for (int p = 0; p < GP; ++p) to[p * plane] = parts[p];
    }
}

// A gradient (+)= the sum of its splits, in their order.  Four columns per thread.
template <typename OT>
struct Finish {
    Grad<OT> out;
    const float* acc;
    int rows, lda, splits;
    long long split;
    const int* cnt;          // rows that count, or null: all
    long long groups;        // work-groups of 256 threads
};
template <typename OT>
__global__ void __launch_bounds__(256) finish(Finish<OT> h, Finish<OT> w, int D) {
    const long long group = grid_index();
    const bool second = group >= h.groups;
    if (group >= h.groups + w.groups) return;
    const Finish<OT>& f = second ? w : h;
    const int quads = (D + 3) / 4;
    const long long t = (group - (second ? h.groups : 0)) * 256 + threadIdx.x;
    const long long i = t / quads;
    const int c = 4 * (int)(t % quads);
    if (i >= (f.cnt ? *f.cnt : f.rows)) return;
    f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
    for (int s = 0; s < f.splits; ++s)
        v += *reinterpret_cast<const f32x4*>(f.acc + s * f.split + (size_t)i * f.lda + c);
    const int e = f.out.scale();
    const float wi = f.out.weight((int)i, f.out.common());
    OT* to = f.out.at((int)i) + c;
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if (c + q < D) f.out.put(to + q, __builtin_ldexpf(v[q], e) * wi);
}

// ---- few rows --------------------------------------------------------------------------------------
// Few rows: bound by reading the table, so it is read as it is, at any alignment, once for
// the forward and twice for the gradient, straight into the fp32 matrix cores (v_mfma_f32_16x16x4:
// at 16 rows they take 17 TB/s of fp32 values or 9 of bf16), with no packing: a row that does not
// count reads as zeros, and its G is zero.  G is fp32, [table row][FEW].
constexpr int FEW = 16;
constexpr int FEW_MAX_V = 1 << 21;

struct Few {
    Targets targets;
    int N, D;
    const void* H;
    int ldh;
    const void* W;
    int ldw;
    float c;
    uint32_t* keep;      // the rows that count, as bits, from few_mark; null: they have a target
    const float* sums;   // of teacher_sums, or null
    float2* part;        // [work-group of few_lse][ldpart]
    int ldpart;
    float* G;
    const float *lse, *dloss;
    float wscale, factor;
    float *loss, *lse_out;
    // dH's splits of the table rows, [split][FEW][Dp]
    float* acc;
    int Dp, splits, rows_per_split, hblocks, hslabs;
    // dW
    int wrows, wslabs, wlanes;   // table rows of a work-group, slabs of columns, lanes of a row
};

// One wave's operands of a step of 32 k: lane l has 8 values from k + 8 (l / 16) of the rows l % 16 of
// RT tiles of the table, and of token l % 16 of TG groups.  The order of k within the step is the same on
// both sides, so it does not matter which instruction takes which.
template <typename T, int RT, int TG> struct FewStep;
template <int RT, int TG> struct FewStep<float, RT, TG> {   // v_mfma_f32_16x16x4_f32: a value of each lane at a time
    static constexpr int AHEAD = 1;
    float x[RT][8], y[TG][8];
    __device__ static void get(const float* p, int k, int D, float (&v)[8]) { load8(p, k, D, v); }
    __device__ void zero(int t) {
#pragma unroll
        for (int e = 0; e < 8; ++e) y[t][e] = 0.f;
    }
    __device__ void mma(f32x4 (&acc)[TG][RT]) const {
#pragma unroll
        for (int e = 0; e < 8; ++e)
#pragma unroll
            for (int t = 0; t < TG; ++t)
#pragma unroll
                for (int a = 0; a < RT; ++a)
                    acc[t][a] = __builtin_amdgcn_mfma_f32_16x16x4f32(x[a][e], y[t][e], acc[t][a], 0, 0, 0);
    }
};
template <int RT, int TG> struct FewStep<uint16_t, RT, TG> {   // v_mfma_f32_16x16x32_bf16: all 8; more ahead
    static constexpr int AHEAD = 3;
    h8 x[RT], y[TG];
    __device__ static void get(const uint16_t* p, int k, int D, h8& v) {
        if (k + 8 <= D) {
            v = *reinterpret_cast<const h8a*>(p + k);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] = k + e < D ? p[k + e] : (uint16_t)0;
        }
    }
    __device__ void zero(int t) { y[t] = h8{}; }
    __device__ void mma(f32x4 (&acc)[TG][RT]) const {
#pragma unroll
        for (int t = 0; t < TG; ++t)
#pragma unroll
            for (int a = 0; a < RT; ++a)
                acc[t][a] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(
                    __builtin_bit_cast(bf16x8, x[a]), __builtin_bit_cast(bf16x8, y[t]), acc[t][a], 0, 0, 0);
    }
};

// 16 RT rows of logits against 16 TG tokens: the work-group's KW waves share the k of all rows (steps of
// 32 k in turn), and their sums meet in LDS in wave order.  Thread t < 64 RT ends with row t / 4,
// tokens 4 (t % 4) .. + 3 of each 16.
template <typename T, int KW, int RT, int TG>
__device__ inline void few_logits(const Few& f, int v0, uint32_t keep, float (*red)[16 * RT][16 * TG], f32x4 (&z)[TG]) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int m = lane & 15, k8 = 8 * (lane >> 4);
    const int V = f.targets.V, D = f.D;
    const T* rows[RT];
#pragma unroll
    for (int a = 0; a < RT; ++a)   // past the end: the last row again, unused
        rows[a] = (const T*)f.W + (size_t)min(v0 + 16 * a + m, V - 1) * f.ldw;
    const T* h = (const T*)f.H + (size_t)m * f.ldh;
    f32x4 acc[TG][RT];
#pragma unroll
    for (int t = 0; t < TG; ++t)
#pragma unroll
        for (int a = 0; a < RT; ++a) acc[t][a] = f32x4{0.f, 0.f, 0.f, 0.f};
    using Step = FewStep<T, RT, TG>;
    constexpr int AHEAD = Step::AHEAD, NB = AHEAD + 1, HOP = 32 * KW;
    Step step[NB];
    auto fetch = [&](int k, Step& st) {
#pragma unroll
        for (int a = 0; a < RT; ++a) Step::get(rows[a], k + k8, D, st.x[a]);
#pragma unroll
        for (int t = 0; t < TG; ++t)
            if ((keep >> (16 * t + m)) & 1) Step::get(h + (size_t)16 * t * f.ldh, k + k8, D, st.y[t]);
            else st.zero(t);
    };
#pragma unroll
    for (int u = 0; u < AHEAD; ++u)
        if (32 * w + HOP * u < D) fetch(32 * w + HOP * u, step[u]);
    for (int k = 32 * w; k < D; k += HOP * NB) {
#pragma unroll
        for (int u = 0; u < NB; ++u) {
            const int here = k + HOP * u;
            if (here >= D) break;
            if (here + HOP * AHEAD < D) fetch(here + HOP * AHEAD, step[(u + AHEAD) % NB]);
            step[u].mma(acc);
        }
    }
#pragma unroll
    for (int t = 0; t < TG; ++t)
#pragma unroll
        for (int a = 0; a < RT; ++a)
#pragma unroll
            for (int r = 0; r < 4; ++r) red[w][16 * a + 4 * (lane >> 4) + r][16 * t + m] = acc[t][a][r];
    __syncthreads();
    const int row = (threadIdx.x % (64 * RT)) >> 2, n4 = 4 * (threadIdx.x & 3);
#pragma unroll
    for (int t = 0; t < TG; ++t) {
        z[t] = *reinterpret_cast<const f32x4*>(&red[0][row][16 * t + n4]);
#pragma unroll
        for (int p = 1; p < KW; ++p) z[t] += *reinterpret_cast<const f32x4*>(&red[p][row][16 * t + n4]);
    }
}

// The rows that count, as bits: a teacher's from a launch of its own, as a row without entries is known
// for one only after all K (16 x 32000 x 1024 fp32, K = 100, forward and gradient: every work-group looking for
// itself 245 us with half of the rows padding, 141 so; without padding 140 and 144).
__global__ void __launch_bounds__(1024) few_mark(Few f) {
    __shared__ uint32_t bits[16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const Teacher& t = f.targets.t;
    uint32_t mine = 0;
    for (int n = w; n < f.N; n += 16) {
        bool any = false;
        for (int k = lane; k < t.K; k += 64) any |= entry_counts(t, (size_t)n * t.K + k, f.targets.V);
        if (__ballot(any)) mine |= 1u << n;
    }
    if (lane == 0) bits[w] = mine;
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int x = 1; x < 16; ++x) mine |= bits[x];
    *f.keep = mine;
}
__device__ inline uint32_t few_keep(const Few& f) {
    if (f.keep) return *f.keep;
    const int lane = threadIdx.x & 63;
    return (uint32_t)__ballot(lane < f.N && counts(f.targets.target[lane < f.N ? lane : 0], f.targets.V));
}

// Reads the table once: 1 x 131072 x 2048 bf16 101 us, 5.3 TB/s; 16 x 41216 x 2357 fp32 (rows at odd
// 4-byte places) 117 us, 3.3 TB/s.
template <typename T, int KW, int RT, int TG>
__global__ void __launch_bounds__(64 * KW) few_lse(Few f) {
    __shared__ float red[KW][16 * RT][16 * TG];
    __shared__ float stat[2][RT][16 * TG];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int v0 = blockIdx.x * 16 * RT, row = threadIdx.x >> 2, n4 = 4 * (threadIdx.x & 3);
    f32x4 z[TG], mx[TG];
    few_logits<T, KW, RT, TG>(f, v0, few_keep(f), red, z);
    const bool own = w < RT, in = v0 + row < f.targets.V;
#pragma unroll
    for (int t = 0; t < TG; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            float m = z[t][q] = in ? f.c * z[t][q] : -INFINITY;
            for (int x = 4; x < 64; x <<= 1) m = fmaxf(m, __shfl_xor(m, x, 64));
            if (own && lane < 4) stat[0][w][16 * t + n4 + q] = m;
        }
    __syncthreads();
#pragma unroll
    for (int t = 0; t < TG; ++t)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
            const int n = 16 * t + n4 + q;
            float m = stat[0][0][n];
            for (int x = 1; x < RT; ++x) m = fmaxf(m, stat[0][x][n]);
            mx[t][q] = m;
            float s = __expf(z[t][q] - (m == -INFINITY ? 0.f : m));
            for (int x = 4; x < 64; x <<= 1) s += __shfl_xor(s, x, 64);
            if (own && lane < 4) stat[1][w][n] = s;
        }
    __syncthreads();
    if (threadIdx.x < 4)
#pragma unroll
        for (int t = 0; t < TG; ++t)
#pragma unroll
            for (int q = 0; q < 4; ++q) {
                const int n = 16 * t + n4 + q;
                float s = stat[1][0][n];
                for (int x = 1; x < RT; ++x) s += stat[1][x][n];
                f.part[(size_t)blockIdx.x * f.ldpart + n] = float2{mx[t][q], s};
            }
}

// A work-group per row: joins the parts, takes the logits at the row's targets and writes loss and
// lse.
template <typename T>
__global__ void __launch_bounds__(1024) few_loss(Few f, int blocks) {
    __shared__ float2 red[16];
    __shared__ float redf[16];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int n = blockIdx.x;
    const Targets& tg = f.targets;
    if (!((few_keep(f) >> n) & 1)) {
        if (threadIdx.x == 0) {
            f.loss[n] = 0.f;
            if (f.lse_out) f.lse_out[n] = 0.f;
        }
        return;
    }
    float m = -INFINITY, s = 0.f;
    for (int b = threadIdx.x; b < blocks; b += 1024) {
        const float2 p = f.part[(size_t)b * f.ldpart + n];
        lse_merge(m, s, p.x, p.y);
    }
    for (int x = 1; x < 64; x <<= 1) {
        const float m2 = __shfl_xor(m, x, 64), s2 = __shfl_xor(s, x, 64);
        lse_merge(m, s, m2, s2);
    }
    const T* h = (const T*)f.H + (size_t)n * f.ldh;
    const T* W = (const T*)f.W;
    float base = 0.f;   // of this wave
    if (tg.target) {
        if (w == 0) base = -(f.c * row_dot(h, W + (size_t)tg.target[n] * f.ldw, f.D, lane));
    } else {
        const size_t at = (size_t)n * tg.t.K;
        float mx, log_sum;
        teacher_stats(tg.t, at, tg.V, mx, log_sum);
        for (int k = w; k < tg.t.K; k += 16)
            if (entry_counts(tg.t, at + k, tg.V)) {
                const float z = f.c * row_dot(h, W + (size_t)tg.t.id[at + k] * f.ldw, f.D, lane);
                const float lq = (tg.t.logit[at + k] - mx) * tg.t.inv_t - log_sum, q = __expf(lq);
                if (!(q == 0.f)) base += q * (lq - z);
            }
    }
    if (lane == 0) {
        red[w] = float2{m, s};
        redf[w] = base;
    }
    __syncthreads();
    if (threadIdx.x != 0) return;
    for (int x = 1; x < 16; ++x) {
        lse_merge(m, s, red[x].x, red[x].y);
        base += redf[x];
    }
    const float l = m + __logf(s);
    if (f.lse_out) f.lse_out[n] = l;
    f.loss[n] = f.factor * (l + base);
}

// G = w (softmax - [target]); what a teacher takes off follows.
template <typename T, int KW, int RT>
__global__ void __launch_bounds__(64 * KW) few_g(Few f) {
    __shared__ float red[KW][16 * RT][FEW];
    const int v0 = blockIdx.x * 16 * RT, v = v0 + (threadIdx.x >> 2), n4 = 4 * (threadIdx.x & 3);
    const uint32_t keep = few_keep(f);
    f32x4 z[1];
    few_logits<T, KW, RT, 1>(f, v0, keep, red, z);
    if (threadIdx.x >= 64 * RT || v >= f.targets.V) return;
    f32x4 g = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int q = 0; q < 4; ++q)
        if ((keep >> (n4 + q)) & 1) {
            const int n = n4 + q;
            float p = __expf(__builtin_fmaf(f.c, z[0][q], -f.lse[n]));
            if (f.targets.target && f.targets.target[n] == v) p -= 1.f;
            g[q] = (f.dloss ? f.dloss[n] : 1.f) * f.wscale * p;
        }
    *reinterpret_cast<f32x4*>(f.G + (size_t)v * FEW + n4) = g;
}

// A work-group per row: the first entry of each token takes off the sum of its entries.
__global__ void __launch_bounds__(256) few_teacher(Few f) {
    const int n = blockIdx.x;
    const Teacher& t = f.targets.t;
    const int V = f.targets.V;
    const size_t at = (size_t)n * t.K;
    const float w = (f.dloss ? f.dloss[n] : 1.f) * f.wscale;
    if (f.sums) {
        for (int k = threadIdx.x; k < t.K; k += 256) {
            const float q = f.sums[at + k];
            if (entry_counts(t, at + k, V) && !(q < 0.f)) f.G[(size_t)t.id[at + k] * FEW + n] -= w * q;
        }
        return;
    }
    float mx, log_sum;
    teacher_stats(t, at, V, mx, log_sum);
    for (int k = threadIdx.x; k < t.K; k += 256) {
        if (!entry_counts(t, at + k, V)) continue;
        const int id = t.id[at + k];
        float q = 0.f;
        bool first = true;
        for (int j = 0; j < t.K; ++j)
            if (t.id[at + j] == id && entry_counts(t, at + j, V)) {
                first &= j >= k;
                q += __expf((t.logit[at + j] - mx) * t.inv_t - log_sum);
            }
        if (first) f.G[(size_t)id * FEW + n] -= w * q;
    }
}

// R values of a row from column c, zero past its end; any alignment.
template <int R, typename T>
__device__ inline void load_piece(const T* __restrict__ p, int c, int D, float* v) {
    typedef T piece __attribute__((ext_vector_type(R), aligned(sizeof(T))));
    if (c + R <= D) {
        const piece x = *reinterpret_cast<const piece*>(p + c);
#pragma unroll
        for (int e = 0; e < R; ++e) {
            if constexpr (sizeof(T) == 4) v[e] = x[e];
            else v[e] = bf16_bits_to_f32(x[e]);
        }
    } else {
#pragma unroll
        for (int e = 0; e < R; ++e) {
            if constexpr (sizeof(T) == 4) v[e] = c + e < D ? p[c + e] : 0.f;
            else v[e] = c + e < D ? bf16_bits_to_f32(p[c + e]) : 0.f;
        }
    }
}

// dH and dW.  Work-groups [0, hblocks): a split of the table rows and a slab of 16 C columns (C = 4
// or 8 values of 16 bytes); its 4 waves take a quarter of the rows each, 4 rows an instruction:
// lane l has G of token l % 16 and C columns of the table at row l / 16, and the products with
// column j of each piece go to accumulator j.  The others: rows of dW by slabs of 64 C' columns, a
// lane's C' columns of all rows of H in registers, G by scalar loads; narrow tables take several rows
// at a time, 1 / lanes of a wave each.
template <typename T, typename OT, int NT>
__global__ void __launch_bounds__(256) few_grads(Few f, const float* __restrict__ G, Grad<OT> dW) {
    constexpr int C = 16 / sizeof(T), CW = 16 / sizeof(OT);
    __shared__ float red[3][FEW][16 * C];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int V = f.targets.V, D = f.D;
    if ((int)blockIdx.x < f.hblocks) {
        const int slab = blockIdx.x % f.hslabs, split = blockIdx.x / f.hslabs;
        const int c0 = 16 * C * slab + C * (lane & 15), r4 = lane >> 4, n = lane & 15;
        const int per = f.rows_per_split / 4;   // a multiple of 4
        const int begin = split * f.rows_per_split + w * per, end = min(begin + per, V);
        const T* W = (const T*)f.W;
        f32x4 acc[C];
#pragma unroll
        for (int j = 0; j < C; ++j) acc[j] = f32x4{0.f, 0.f, 0.f, 0.f};
        constexpr int FLY = 4;
        for (int v0 = begin; v0 < end; v0 += 4 * FLY) {
            float g[FLY], x[FLY][8];
#pragma unroll
            for (int u = 0; u < FLY; ++u) {
                const int v = v0 + 4 * u + r4, at = v < end ? v : begin;
                g[u] = G[(size_t)at * FEW + n];
                if (v >= end) g[u] = 0.f;
                load_piece<C>(W + (size_t)at * f.ldw, c0, D, x[u]);
            }
#pragma unroll
            for (int u = 0; u < FLY; ++u)
#pragma unroll
                for (int j = 0; j < C; ++j)
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x4f32(g[u], x[u][j], acc[j], 0, 0, 0);
        }
        // acc[j][r]: token 4 (lane / 16) + r, column C (lane % 16) + j of the slab
        if (w > 0)
#pragma unroll
            for (int j = 0; j < C; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r) red[w - 1][4 * r4 + r][C * n + j] = acc[j][r];
        __syncthreads();
        if (w > 0) return;
#pragma unroll
        for (int j = 0; j < C; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                float v = acc[j][r];
                for (int p = 0; p < 3; ++p) v += red[p][4 * r4 + r][C * n + j];
                if (c0 + j < D) f.acc[((size_t)split * FEW + 4 * r4 + r) * f.Dp + c0 + j] = v;
            }
        return;
    }
    const int b = blockIdx.x - f.hblocks;
    const int slab = b % f.wslabs, v0 = b / f.wslabs * f.wrows, end = min(v0 + f.wrows, V);
    const int lanes = f.wlanes, each = 64 / lanes;   // lanes of a row, rows of a wave
    const int c0 = 64 * CW * slab + CW * (lane & (lanes - 1));
    const uint32_t keep = few_keep(f);
    float h[NT][CW];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        float x[8] = {};
        if ((keep >> n) & 1) load_piece<CW>((const T*)f.H + (size_t)n * f.ldh, c0, D, x);
#pragma unroll
        for (int j = 0; j < CW; ++j) h[n][j] = x[j];
    }
    auto put = [&](int v, const float* __restrict__ g) {
        float s[CW] = {};
#pragma unroll
        for (int n = 0; n < NT; ++n) {
            const float gn = g[n];
#pragma unroll
            for (int j = 0; j < CW; ++j) s[j] = __builtin_fmaf(gn, h[n][j], s[j]);
        }
        OT* to = dW.at(v) + c0;
        if (!dW.accumulate && c0 + CW <= D) {
            if constexpr (CW == 4) {
                *reinterpret_cast<f4a*>(to) = f4a{s[0], s[1], s[2], s[3]};
            } else {
                h8a x;
#pragma unroll
                for (int j = 0; j < 8; ++j) x[j] = rne_bf16(s[j]);
                *reinterpret_cast<h8a*>(to) = x;
            }
        } else {
#pragma unroll
            for (int j = 0; j < CW; ++j)
                if (c0 + j < D) dW.put(to + j, s[j]);
        }
    };
    if (each == 1) {
        for (int v = v0 + w; v < end; v += 4) put(v, G + (size_t)v * FEW);
    } else {
        for (int v = v0 + w * each + lane / lanes; v < end; v += 4 * each) put(v, G + (size_t)v * FEW);
    }
}

// dH (+)= the sum of its splits: a work-group per row and 64 columns, its 16 waves share the splits
// and meet in LDS in wave order.
template <typename OT>
__global__ void __launch_bounds__(1024) few_finish(Few f, Grad<OT> dH) {
    __shared__ float red[16][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int n = blockIdx.y, c = blockIdx.x * 64 + lane;
    const bool on = (few_keep(f) >> n) & 1;
    if (!on && dH.accumulate) return;
    float v = 0.f;
    if (on && c < f.D)
#pragma unroll 4
        for (int s = w; s < f.splits; s += 16) v += f.acc[((size_t)s * FEW + n) * f.Dp + c];
    red[w][lane] = v;
    __syncthreads();
    if (w != 0 || c >= f.D) return;
    for (int x = 1; x < 16; ++x) v += red[x][lane];
    dH.put(dH.C + (size_t)n * dH.ldc + c, v);
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

// A product's tile.
enum Kind { T256, T128, T64 };
int side(Kind t) { return t == T256 ? 256 : t == T128 ? 128 : 64; }
int wave_rows(Kind t) { return side(t) / 2; }
long long tiles_of(Kind t, long long M, long long N) {
    return ((M + side(t) - 1) / side(t)) * ((N + side(t) - 1) / side(t));
}
// Estimated time of a product in us, the rule that picks its tile and how many splits of K are added
// afterwards: rounds of work-groups (a last round that is not full counts half of what it lacks)
// times their 32-k stages, each of the time measured with one work-group on a CU or with as many as
// fit; the sums of splits are written, read and cost a launch.
double estimate(Kind t, long long M, long long N, long long K, int kinds, int splits) {
    static const double alone[] = {1.0, 0.45, 0.19}, full[] = {1.0, 0.68, 0.30};
    const bool both = t == T64 && kinds == 3;   // gemm_both: three products a stage, one group a CU
    const int fit = t == T256 || both ? 1 : 2;
    const double groups = (double)tiles_of(t, M, N) * splits;
    const double stages = (double)((K + 31) / 32) * (both ? 1 : kinds) / splits + 4;
    double rounds = groups / (256 * fit);
    const double whole = (double)(long long)(rounds + 0.9999);
    rounds = rounds <= 1 ? 1 : (rounds + whole) / 2;
    const double stage = both ? 0.30 : groups <= 256 ? alone[t] : full[t];
    return rounds * stages * stage + (splits > 1 ? 4 + (double)splits * M * N * 8 / 4e6 : 0);
}
struct Choice {
    Kind kind;
    int splits;
};
Choice pick(long long M, long long N, long long K, int kinds, bool split) {
    Choice best{T64, 1};
    double least = estimate(T64, M, N, K, kinds, 1);
    for (Kind t : {T64, T128, T256})
        for (int s = 1; s <= 64 && s * 128 <= std::max(128LL, K); s = s < 8 ? s + 1 : s + 4) {
            const double e = estimate(t, M, N, K, kinds, s);
            if (e < least) {
                least = e;
                best = {t, s};
            }
            if (!split) break;
        }
    return best;
}

// The workspace: a part whose size the shapes give, and a piece whose size is what is left.
struct Plan {
    int parts, gparts;        // of H and W; of G
    int Dp, Nt;               // columns and rows as the workspace holds them
    bool direct;              // the table is read in place
    Kind lse, g, dh, dw;      // the products' tiles
    int splits, wsplits;      // of dH and dW
    size_t ints, w, lses, rest, base, q, z, state, Hp, Xp, acc, wacc;
    size_t piece;             // first byte of the piece's buffers
    size_t per_block;         // bytes of a piece per 256 table rows
};

// gtype: the gradients' type, or a negative one for the forward.
Plan make_plan(int dtype, int gtype, int N, int V, int D, int K, const void* W, int ldw) {
    Plan p{};
    const bool backward = gtype >= 0;
    p.parts = dtype == DH_F32 ? 2 : 1;
    p.gparts = gtype == DH_F32 ? 2 : 1;
    p.Dp = (D + 31) / 32 * 32;
    p.Nt = (int)(((long long)N + 255) / 256 * 256);
    // In place (forward): whole 16-byte chunks at aligned addresses, 256 rows within 32-bit offsets.
    p.direct = !backward && dtype == DH_BF16 && D % 8 == 0 && ldw % 8 == 0 && ldw <= 1 << 22 && ((uintptr_t)W & 15) == 0;
    p.lse = pick(V, N, D, kinds_of(p.parts, p.parts), false).kind;
    p.g = pick(N, V, D, kinds_of(p.parts, p.parts), false).kind;
    const Choice dh = pick(N, D, V, kinds_of(p.gparts, p.parts), true),
                 dw = pick(V, D, N, kinds_of(p.gparts, p.parts), true);
    p.dh = dh.kind;
    p.dw = dw.kind;
    p.splits = dh.splits;
    p.wsplits = dw.splits;
    size_t at = 0;
    auto take = [&](size_t bytes) {
        const size_t here = at;
        at += up256(bytes);
        return here;
    };
    p.ints = take(((size_t)4 * p.Nt + 2 * (p.Nt / PACK) + 64 + SCAN + p.Nt / COUNT + 1) * 4);   // cnt and scales, row, target, ...
    p.w = take((size_t)p.Nt * 4);
    p.lses = take((size_t)p.Nt * 4);
    p.rest = take((size_t)p.Nt * 4);
    p.base = take((size_t)p.Nt * 4);
    p.q = take((size_t)N * K * 4);
    p.z = take((size_t)N * K * 4);
    p.Hp = take((size_t)p.parts * N * p.Dp * 2);
    if (backward) {
        p.acc = take((size_t)p.splits * N * p.Dp * 4);
        p.Xp = take((size_t)p.parts * N * p.Dp * 2);
        p.per_block = (size_t)p.gparts * N * 256 * 2;
        // dW's sums over splits of the rows: a piece's, fp32.
        if (p.wsplits > 1) p.per_block += (size_t)p.wsplits * 256 * p.Dp * 4;
    } else {
        p.state = take((size_t)p.Nt * 8);
        p.per_block = (size_t)p.Nt * (256 / wave_rows(p.lse)) * 8;
        if (p.parts == 2) p.per_block += 1024;
    }
    if (!p.direct) p.per_block += (size_t)p.parts * 256 * p.Dp * 2;
    p.piece = at;
    return p;
}

// Which calls take this form, measured against the form for many rows (us, that one's behind the stroke):
//   forward, up to FEW rows      fp32 16 x 32000 x 1024: under half; bf16 16 x 131072 x 2048 116 / 116,
//                                16 x 50001 x 1001 48 / 60, 1 x 131072 x 2048 107 / 115
//   forward, up to 2 FEW, fp32   as there the table would be staged: 18 x 41216 x 2357 155 / 248; bf16 tables
//                                are read in place or cheap to stage: 32 x 50001 x 1001 63 / 60
//   gradient, up to FEW rows     with its forward fp32 16 x 32000 x 1024 111 / 240; bf16 4 x 131072 x 2048 560 / 825,
//                                16 x 131072 x 2048 738 / 835, 16 x 50001 x 1000 183 / 179, x 1001 250 / 202, 16 x
//                                8000 x 512 38 / 50; bf16 inputs with fp32 gradients 16 x 131072 x 2048 803 / 1056.
//                                Its G is fp32 for any of them: a row more or less does not change how exact they are.
bool is_few(int dtype, int N, int V, int backward) {
    return V <= FEW_MAX_V && N <= (dtype == DH_F32 && !backward ? 2 * FEW : FEW);
}

struct FewPlan {
    int Dp, rows, waves, blocks;   // of few_lse and few_g: table rows and waves of a work-group
    int splits, rows_per_split, hslabs, wslabs, wrows, wlanes;
    size_t G, acc, keep, sums, total;   // the parts of the forward lie at G
};
FewPlan few_plan(int dtype, int grad_type, int N, int V, int D, int K, int backward) {
    FewPlan p{};
    const int C = dtype == DH_F32 ? 4 : 8, CW = grad_type == DH_F32 ? 4 : 8;
    p.Dp = (D + 3) / 4 * 4;
    // 64 rows (32 for two groups of tokens) and 4 waves; few work-groups of those: 16 rows, and a long k shared by 16 waves, which
    // shortens its chain of loads (2000 x 4000 fp32: 41 / 18 us).
    const bool small = V <= 64 * 256;
    p.rows = small ? 16 : N <= FEW ? 64 : 32;
    p.waves = small && D >= 512 ? 16 : 4;
    p.blocks = (V + p.rows - 1) / p.rows;
    if (!backward) {
        p.keep = up256((size_t)p.blocks * (N <= FEW ? FEW : 2 * FEW) * 8);
        p.total = p.keep + 256;
        return p;
    }
    // About 1024 work-groups of 4 waves for dH and 4096 for dW.
    p.hslabs = (D + 16 * C - 1) / (16 * C);
    const int splits = std::max(1, std::min(1024 / p.hslabs, (V + 63) / 64));
    p.rows_per_split = ((V + splits - 1) / splits + 15) / 16 * 16;
    p.splits = (V + p.rows_per_split - 1) / p.rows_per_split;
    p.wslabs = (D + 64 * CW - 1) / (64 * CW);
    p.wlanes = 64;
    while (p.wlanes > 1 && p.wlanes / 2 * CW >= D) p.wlanes /= 2;
    const int least = 16 * (64 / p.wlanes);   // rows of a work-group
    const int chunks = std::max(1, std::min(4096 / p.wslabs, (V + least - 1) / least));
    p.wrows = (V + chunks - 1) / chunks;
    p.acc = up256((size_t)p.blocks * p.rows * FEW * 4);
    p.keep = p.acc + up256((size_t)p.splits * FEW * p.Dp * 4);
    p.sums = p.keep + 256;
    p.total = p.sums + (by_sums(V, K) ? up256((size_t)N * K * 4) : 0);
    return p;
}

// The workspace that serves any alignment of the operands (staged tables take more).
size_t least_ws(int dtype, int N, int V, int D, int K, int backward) {
    if (is_few(dtype, N, V, backward))   // whichever type the gradients have
        return std::max(few_plan(dtype, DH_F32, N, V, D, K, backward).total,
                        few_plan(dtype, dtype, N, V, D, K, backward).total);
    size_t need = 0;
    for (int g : {(int)DH_F32, dtype}) {
        const Plan p = make_plan(dtype, backward ? g : -1, N, V, D, K, nullptr, 1);
        need = std::max(need, p.piece + p.per_block + 512);
    }
    return need;
}

// The most rows that a loss takes, and the most values of H: a launch has less than 2^32 threads in
// a dimension.
constexpr int MOST_ROWS = 1 << 25;
constexpr long long MOST_VALUES = 1LL << 35;

// Table rows of a piece: as many blocks of 256 as fit, the same for every piece.
int piece_rows(const Plan& p, int N, int V, int D, size_t ws_bytes) {
    const long long blocks = (V + 255LL) / 256;
    long long fit = (long long)((ws_bytes - 512 - p.piece) / p.per_block);
    if (fit > blocks) fit = blocks;
    if (fit > 4096) fit = 4096;   // 256 rows of G stay within 32-bit offsets
    // 64-wide tiles of rows x N or D have a thread per 16 values.
    const long long most = (1LL << 34) / std::max(N, D) / 256;   // at least 1, as N <= 2^25
    if (fit > most) fit = most;
    const long long pieces = (blocks + fit - 1) / fit;
    return (int)((blocks + pieces - 1) / pieces) * 256;
}

int check_head(const Head& h, int K, const void* ws, size_t ws_bytes, int backward) {
    if (h.dtype != DH_F32 && h.dtype != DH_BF16)
        return set_error(DH_ERR_INVALID, "%s: dtype must be fp32 or bf16", h.op);
    if (h.N < 0 || h.V < 1 || h.D < 1 || K < 0 || h.N > MOST_ROWS || h.V > 0x7FFFFE00 || h.D > 1 << 20 ||
        (long long)h.N * h.D > MOST_VALUES)
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
    Exps exps;
    int *flags, *counts;
    float *base, *q, *z, *acc;
    float2* state;
    uint16_t *Hp, *Xp;   // Xp: the other operand of dW
    char* piece;
};

Work lay_out(const Plan& p, void* ws) {
    char* b = (char*)(((uintptr_t)ws + 255) & ~(uintptr_t)255);
    int* ints = (int*)(b + p.ints);
    auto array = [&](int k) { return ints + 64 + (size_t)k * p.Nt; };
    Work w{};
    w.p = p;
    w.rows = {ints, array(0), array(1), array(2), (float*)(b + p.w), (float*)(b + p.lses),
              (float*)(b + p.rest)};
    w.flags = array(3);
    const int groups = p.Nt / PACK;
    w.exps = {nullptr, ints + 1, ints + 2, (float*)(ints + 3), array(4), (float*)(array(4) + groups),
              (float*)(array(4) + 2 * groups)};
    w.counts = array(4) + 2 * groups + SCAN;
    w.base = (float*)(b + p.base);
    w.q = (float*)(b + p.q);
    w.z = (float*)(b + p.z);
    w.state = (float2*)(b + p.state);
    w.acc = (float*)(b + p.acc);
    w.Hp = (uint16_t*)(b + p.Hp);
    w.Xp = (uint16_t*)(b + p.Xp);
    w.piece = b + p.piece;
    return w;
}

// Packs the rows; `more` work-groups of the launch stage table rows or scan the table.
template <typename T, int P>
int prepare_rows(const Head& h, const Work& w, Pack a, int more) {
    a.targets = {h.target, h.teacher, h.V};
    if (!h.target && (h.teacher.K > 16 || (long long)h.N * h.teacher.K > 1 << 15)) {
        teacher_flags<<<(h.N + 3) / 4, 256, 0, stream()>>>(h.teacher, h.N, h.V, w.flags);
        DH_TRY(check_launch(h.op));
        a.targets.target = w.flags;
    }
    if (h.N > MANY) {
        count_rows<<<(h.N + COUNT - 1) / COUNT, COUNT, 0, stream()>>>(a.targets, h.N, w.counts);
        DH_TRY(check_launch(h.op));
        a.counts = w.counts;
    }
    a.N = h.N;
    a.D = h.D;
    a.H = h.H;
    a.ldh = h.ldh;
    a.W = h.W;
    a.ldw = h.ldw;
    a.Hp = w.Hp;
    a.Dp = w.p.Dp;
    a.plane = (long long)h.N * w.p.Dp;
    a.rows = w.rows;
    a.exps = w.exps;
    a.groups = (h.N + PACK - 1) / PACK;
    a.c = h.c;
    a.wscale = h.wscale;
    pack_rows<T, P><<<a.groups + more, 1024, 0, stream()>>>(a);
    DH_TRY(check_launch(h.op));
    if (h.target) return DH_OK;
    // Up to 8 waves, with as few idle places in their last turn as that leaves.
    const int turns = std::max(1, (h.teacher.K + 8 * TEACHER_FLY - 1) / (8 * TEACHER_FLY));
    const int waves = std::max(1, (h.teacher.K + TEACHER_FLY * turns - 1) / (TEACHER_FLY * turns));
    teacher_dots<T><<<long_grid(h.N), 64 * waves, 0, stream()>>>(w.rows, h.teacher, h.V, (const T*)h.H, h.ldh, (const T*)h.W,
                                               h.ldw, h.D, w.q, w.z, w.base);
    return check_launch(h.op);
}

template <class S, bool AK, bool BK, int TOK, int PA, int PB, class Epi>
int launch(const char* op, Prod g, int splits, const Epi& epi) {
    const long long tiles = ((g.M + S::T - 1LL) / S::T) * ((g.N + S::T - 1LL) / S::T);
    const int bk = S::T == 256 && AK ? 64 : S::BK;   // gemm_deep counts pairs
    const int stages = (g.K + bk - 1) / bk;
    g.kstages = (stages + splits - 1) / splits;
    vocab_gemm<S, AK, BK, TOK, PA, PB, Epi><<<dim3((unsigned)tiles, splits), S::THREADS, 0, stream()>>>(g, epi);
    return check_launch(op);
}
template <bool AK, bool BK, int TOK, int PA, int PB, class Epi>
int product(const char* op, Kind t, const Prod& g, int splits, const Epi& epi) {
    if (t == T256) return launch<Shape<256>, AK, BK, TOK, PA, PB>(op, g, splits, epi);
    if (t == T128) return launch<Shape<128>, AK, BK, TOK, PA, PB>(op, g, splits, epi);
    return launch<Shape<64>, AK, BK, TOK, PA, PB>(op, g, splits, epi);
}

template <typename T, int P>
int forward(const Head& h, float* loss, float* lse, void* ws, size_t ws_bytes) {
    const Plan p = make_plan(h.dtype, -1, h.N, h.V, h.D, h.target ? 0 : h.teacher.K, h.W, h.ldw);
    Work w = lay_out(p, ws);
    const int rows = piece_rows(p, h.N, h.V, h.D, ws_bytes);
    const int wr = wave_rows(p.lse);
    float2* part = (float2*)w.piece;
    uint16_t* staged = (uint16_t*)(w.piece + (size_t)(rows / wr) * p.Nt * 8);
    w.exps.e = (int*)(staged + (size_t)p.parts * rows * p.Dp);
    const long long wplane = (long long)rows * p.Dp;
    Pack a{};
    a.loss = loss;
    a.lse_out = lse;
    if (h.target) a.base = w.base;
    if (!p.direct) {   // the first piece's table rows go with the packing
        a.R = h.V < rows ? h.V : rows;
        a.tables = (a.R + 15) / 16;
        a.staged = staged;
        a.wplane = wplane;
    }
    DH_TRY((prepare_rows<T, P>(h, w, a, a.tables)));
    for (int v0 = 0;; v0 += rows) {
        const int R = h.V - v0 < rows ? h.V - v0 : rows;
        const bool last = h.V - v0 <= rows;
        Prod g{staged, w.Hp, p.Dp, p.Dp, wplane, (long long)h.N * p.Dp, R, h.N, p.Dp, 0, w.rows.cnt};
        if (p.direct) {
            g.A = (const uint16_t*)h.W + (size_t)v0 * h.ldw;
            g.lda = h.ldw;
            g.K = h.D;
        } else if (v0 > 0) {
            stage_table<T, P><<<(R + 3) / 4, 256, 0, stream()>>>((const T*)h.W, h.ldw, v0, R, h.D, staged, p.Dp,
                                                                    wplane, w.exps.e);
            DH_TRY(check_launch(h.op));
        }
        DH_TRY((product<true, true, TOK_N, P, P>(h.op, p.lse, g, 1,
                                                  EpiLse<P>{h.c, w.exps.e, w.rows.hexp, part, p.Nt})));
        const JoinOut out{w.rows, w.state, v0 == 0, last, w.base, h.factor, loss, lse};
        const int blocks = (R + wr - 1) / wr;
        if (h.N <= 512) lse_join_few<<<h.N, 256, 0, stream()>>>(part, p.Nt, blocks, out);
        else lse_join<<<p.Nt / 64, 1024, 0, stream()>>>(part, p.Nt, blocks, out);
        DH_TRY(check_launch(h.op));
        if (last) return DH_OK;
    }
}

struct Grads {
    const float *lse, *dloss;
    void* dH;
    int lddh, acc_dH;
    void* dW;
    int lddw, acc_dW, type;
};

// dH and dW of a piece, in one launch where both take the same small tile.
template <int P, int GP, class EpiH, class EpiW>
int gradients(const char* op, const Plan& p, const Prod* gh, const EpiH& eh, const Prod* gw, const EpiW& ew) {
    if (gh && gw && p.dh == T64 && p.dw == T64) {
        using S = Shape<64>;
        auto per = [](int K, int splits) { return ((K + S::BK - 1) / S::BK + splits - 1) / splits; };
        Prod a = *gh, b = *gw;
        a.kstages = per(a.K, p.splits);
        b.kstages = per(b.K, p.wsplits);
        const long long th = tiles_of(p.dh, a.M, a.N), tw = tiles_of(p.dw, b.M, b.N);
        vocab_grads<S, P, GP, EpiH, EpiW>
            <<<(unsigned)(th * p.splits + tw * p.wsplits), S::THREADS, 0, stream()>>>(
                a, eh, (int)th, (int)(th * p.splits), b, ew, (int)tw);
        return check_launch(op);
    }
    if (gh) DH_TRY((product<true, false, TOK_M, GP, P>(op, p.dh, *gh, p.splits, eh)));
    if (gw) DH_TRY((product<false, false, TOK_K, GP, P>(op, p.dw, *gw, p.wsplits, ew)));
    return DH_OK;
}

// P parts of H and W, GP of G.
template <typename T, int P, int GP, typename OT>
int backward(const Head& h, const Grads& d, void* ws, size_t ws_bytes) {
    const Plan p = make_plan(h.dtype, d.type, h.N, h.V, h.D, h.target ? 0 : h.teacher.K, h.W, h.ldw);
    Work w = lay_out(p, ws);
    const int rows = piece_rows(p, h.N, h.V, h.D, ws_bytes);
    const bool one = h.V <= rows;   // a single piece
    const long long hplane = (long long)h.N * p.Dp, wplane = (long long)rows * p.Dp;
    uint16_t* G = (uint16_t*)w.piece;
    const long long gplane = (long long)h.N * rows;
    float* wacc = (float*)(G + GP * gplane);
    uint16_t* staged = (uint16_t*)(wacc + (p.wsplits > 1 ? p.wsplits * wplane : 0));
    Pack a{};
    a.lse_in = d.lse;
    a.dloss = d.dloss;
    if (d.dH && !d.acc_dH) {
        a.dH = d.dH;
        a.lddh = d.lddh;
        a.dh_f32 = d.type == DH_F32;
    }
    const int scan = h.V < 16 * SCAN ? (h.V + 15) / 16 : SCAN;
    DH_TRY((prepare_rows<T, P>(h, w, a, scan)));
    if (!h.target && by_sums(h.V, h.teacher.K)) {
        teacher_sums<<<long_grid(h.N), 1024, 0, stream()>>>(w.rows.cnt, w.rows.row, h.teacher, h.V, w.q);
        DH_TRY(check_launch(h.op));
    }
    const int groups = (h.N + PACK - 1) / PACK;
    if (h.N > MANY) {
        scales<<<1, 1024, 0, stream()>>>(w.exps, groups, scan);
        DH_TRY(check_launch(h.op));
    }
    const Grad<OT> to_dH{(OT*)d.dH, d.lddh, d.acc_dH, w.rows.row, w.exps.E, w.rows.rest, 1};
    for (int v0 = 0;; v0 += rows) {
        const int R = h.V - v0 < rows ? h.V - v0 : rows;
        const bool last = h.V - v0 <= rows;
        const int tables = (R + 3) / 4;
        stage_scaled<T, P><<<tables + (v0 == 0 ? (h.N + 3) / 4 : 0), 256, 0, stream()>>>(
            (const T*)h.W, h.ldw, v0, R, h.D, staged, p.Dp, wplane, w.exps, groups, scan, v0 > 0 || h.N > MANY, tables,
            w.rows, (const T*)h.H, h.ldh, w.Xp, hplane);
        DH_TRY(check_launch(h.op));
        const Prod g{w.Hp, staged, p.Dp, p.Dp, hplane, wplane, h.N, R, p.Dp, 0, w.rows.cnt};
        if (h.target) {
            DH_TRY((product<true, true, TOK_M, P, P>(
                h.op, p.g, g, 1,
                EpiG<GP, true>{h.c, w.rows.lse, w.rows.w, w.rows.target, w.rows.hexp, w.exps.E, v0, G, rows, gplane})));
        } else {
            DH_TRY((product<true, true, TOK_M, P, P>(
                h.op, p.g, g, 1,
                EpiG<GP, false>{h.c, w.rows.lse, w.rows.w, nullptr, w.rows.hexp, w.exps.E, v0, G, rows, gplane})));
            auto entries = by_sums(h.V, h.teacher.K) ? teacher_entries<GP, true> : teacher_entries<GP, false>;
            entries<<<long_grid(h.N), 256, 0, stream()>>>(w.rows, h.teacher, h.V, v0, R, w.q, w.z, G, rows, gplane);
            DH_TRY(check_launch(h.op));
        }
        const Prod gh{G, staged, rows, p.Dp, gplane, wplane, h.N, h.D, R, 0, w.rows.cnt};
        const Prod gw{G, w.Xp, rows, p.Dp, gplane, hplane, R, h.D, h.N, 0, w.rows.cnt};
        const Prod *ph = d.dH ? &gh : nullptr, *pw = d.dW ? &gw : nullptr;
        const Grad<OT> to_dW{d.dW ? (OT*)d.dW + (size_t)v0 * d.lddw : nullptr, d.lddw, d.acc_dW, nullptr, w.exps.X,
                             w.exps.wtop, 0};
        // Straight to the gradient, or as sums that the last launch adds.
        const bool direct_h = one && p.splits == 1, direct_w = p.wsplits == 1;
        const EpiAcc sum_h{w.acc, p.Dp, v0 == 0, hplane}, sum_w{wacc, p.Dp, 1, wplane};
        const EpiOut<OT> out_h{to_dH}, out_w{to_dW};
        if (direct_h && direct_w) DH_TRY((gradients<P, GP>(h.op, p, ph, out_h, pw, out_w)));
        else if (direct_h) DH_TRY((gradients<P, GP>(h.op, p, ph, out_h, pw, sum_w)));
        else if (direct_w) DH_TRY((gradients<P, GP>(h.op, p, ph, sum_h, pw, out_w)));
        else DH_TRY((gradients<P, GP>(h.op, p, ph, sum_h, pw, sum_w)));
        Finish<OT> fh{to_dH, w.acc, h.N, p.Dp, p.splits, hplane, w.rows.cnt, 0};
        Finish<OT> fw{to_dW, wacc, R, p.Dp, p.wsplits, wplane, nullptr, 0};
        auto finish_groups = [&](long long n) { return (n * ((h.D + 3) / 4) + 255) / 256; };
        if (ph && last && !direct_h) fh.groups = finish_groups(h.N);
        if (pw && !direct_w) fw.groups = finish_groups(R);
        if (fh.groups + fw.groups > 0) {
            finish<OT><<<long_grid(fh.groups + fw.groups), 256, 0, stream()>>>(fh, fw, h.D);
            DH_TRY(check_launch(h.op));
        }
        if (last) return DH_OK;
    }
}

Few few_args(const Head& h) {
    Few f{};
    f.targets = {h.target, h.teacher, h.V};
    f.N = h.N;
    f.D = h.D;
    f.H = h.H;
    f.ldh = h.ldh;
    f.W = h.W;
    f.ldw = h.ldw;
    f.c = h.c;
    f.wscale = h.wscale;
    f.factor = h.factor;
    return f;
}

// The rows that count, where a teacher tells.
int few_rows(const Head& h, Few& f, const FewPlan& p, void* ws) {
    if (h.target) return DH_OK;
    f.keep = (uint32_t*)((char*)ws + p.keep);
    few_mark<<<1, 1024, 0, stream()>>>(f);
    return check_launch(h.op);
}

template <typename T>
int few_forward(const Head& h, float* loss, float* lse, void* ws) {
    const FewPlan p = few_plan(h.dtype, h.dtype, h.N, h.V, h.D, 0, 0);
    Few f = few_args(h);
    DH_TRY(few_rows(h, f, p, ws));
    f.part = (float2*)ws;
    f.loss = loss;
    f.lse_out = lse;
    auto lse_parts = p.rows == 64 ? few_lse<T, 4, 4, 1> : p.waves == 4 ? few_lse<T, 4, 1, 1> : few_lse<T, 16, 1, 1>;
    f.ldpart = FEW;
    if constexpr (sizeof(T) == 4)
        if (h.N > FEW) {
            lse_parts = p.rows == 32 ? few_lse<T, 4, 2, 2> : p.waves == 4 ? few_lse<T, 4, 1, 2> : few_lse<T, 16, 1, 2>;
            f.ldpart = 2 * FEW;
        }
    lse_parts<<<p.blocks, 64 * p.waves, 0, stream()>>>(f);
    DH_TRY(check_launch(h.op));
    few_loss<T><<<h.N, 1024, 0, stream()>>>(f, p.blocks);
    return check_launch(h.op);
}

template <typename T, typename OT>
int few_backward(const Head& h, const Grads& d, void* ws) {
    const FewPlan p = few_plan(h.dtype, d.type, h.N, h.V, h.D, h.target ? 0 : h.teacher.K, 1);
    Few f = few_args(h);
    DH_TRY(few_rows(h, f, p, ws));
    f.G = (float*)ws;
    f.acc = (float*)((char*)ws + p.acc);
    f.lse = d.lse;
    f.dloss = d.dloss;
    f.Dp = p.Dp;
    f.splits = p.splits;
    f.rows_per_split = p.rows_per_split;
    f.hslabs = p.hslabs;
    f.hblocks = d.dH ? p.hslabs * p.splits : 0;
    f.wslabs = p.wslabs;
    f.wrows = p.wrows;
    f.wlanes = p.wlanes;
    auto g = p.rows == 64 ? few_g<T, 4, 4> : p.waves == 4 ? few_g<T, 4, 1> : few_g<T, 16, 1>;
    g<<<p.blocks, 64 * p.waves, 0, stream()>>>(f);
    DH_TRY(check_launch(h.op));
    if (!h.target && h.teacher.K > 0) {
        if (by_sums(h.V, h.teacher.K)) {
            f.sums = (const float*)((char*)ws + p.sums);
            teacher_sums<<<long_grid(h.N), 1024, 0, stream()>>>(nullptr, nullptr, h.teacher, h.V, (float*)f.sums);
            DH_TRY(check_launch(h.op));
        }
        few_teacher<<<h.N, 256, 0, stream()>>>(f);
        DH_TRY(check_launch(h.op));
    }
    const Grad<OT> dW{(OT*)d.dW, d.lddw, d.acc_dW, nullptr, nullptr, nullptr, 0};
    const int wblocks = d.dW ? (h.V + p.wrows - 1) / p.wrows * p.wslabs : 0;
    auto grads = h.N <= 4 ? few_grads<T, OT, 4> : h.N <= 8 ? few_grads<T, OT, 8> : few_grads<T, OT, 16>;
    grads<<<f.hblocks + wblocks, 256, 0, stream()>>>(f, f.G, dW);
    DH_TRY(check_launch(h.op));
    if (!d.dH) return DH_OK;
    few_finish<OT><<<dim3((h.D + 63) / 64, h.N), 1024, 0, stream()>>>(
        f, Grad<OT>{(OT*)d.dH, d.lddh, d.acc_dH, nullptr, nullptr, nullptr, 0});
    return check_launch(h.op);
}

int run_forward(const Head& h, float* loss, float* lse, void* ws, size_t ws_bytes) {
    const int K = h.target ? 0 : h.teacher.K;
    DH_TRY(check_head(h, K, ws, ws_bytes, 0));
    if (h.N > 0 && (!loss || (!h.target && K > 0 && (!h.teacher.id || !h.teacher.logit))))
        return set_error(DH_ERR_INVALID, "%s: null pointer", h.op);
    DH_TRY(ensure_init());
    if (h.N == 0) return DH_OK;
    if (is_few(h.dtype, h.N, h.V, 0))
        return h.dtype == DH_F32 ? few_forward<float>(h, loss, lse, ws) : few_forward<uint16_t>(h, loss, lse, ws);
    return h.dtype == DH_F32 ? forward<float, 2>(h, loss, lse, ws, ws_bytes)
                             : forward<uint16_t, BF>(h, loss, lse, ws, ws_bytes);
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
    if (is_few(h.dtype, h.N, h.V, 1)) {
        if (h.dtype == DH_F32) return few_backward<float, float>(h, d, ws);
        return d.type == DH_F32 ? few_backward<uint16_t, float>(h, d, ws)
                                : few_backward<uint16_t, uint16_t>(h, d, ws);
    }
    if (h.dtype == DH_F32) return backward<float, 2, 2, float>(h, d, ws, ws_bytes);
    return d.type == DH_F32 ? backward<uint16_t, 1, 2, float>(h, d, ws, ws_bytes)
                            : backward<uint16_t, 1, 1, uint16_t>(h, d, ws, ws_bytes);
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

int dh_linear_loss_plan(int dtype, int grad_type, int N, int V, int D, int K, size_t ws_bytes, int* plan) {
    if ((dtype != DH_F32 && dtype != DH_BF16) || (grad_type != DH_F32 && grad_type != dtype))
        return set_error(DH_ERR_INVALID, "dh_linear_loss_plan: dtype must be fp32 or bf16, grad_type fp32 or dtype");
    if (N < 1 || V < 1 || D < 1 || K < 0 || N > MOST_ROWS || V > 0x7FFFFE00 || D > 1 << 20)
        return set_error(DH_ERR_INVALID, "dh_linear_loss_plan: shape N=%d V=%d D=%d K=%d", N, V, D, K);
    if (!plan) return set_error(DH_ERR_INVALID, "dh_linear_loss_plan: null pointer");
    std::fill(plan, plan + 8, 0);
    if (!is_few(dtype, N, V, 0)) {
        const Plan p = make_plan(dtype, -1, N, V, D, K, nullptr, 1);
        plan[0] = side(p.lse);
        plan[6] = ws_bytes < least_ws(dtype, N, V, D, K, 0) ? 0 : piece_rows(p, N, V, D, ws_bytes);
    }
    if (!is_few(dtype, N, V, 1)) {
        const Plan p = make_plan(dtype, grad_type, N, V, D, K, nullptr, 1);
        plan[1] = side(p.g);
        plan[2] = side(p.dh);
        plan[3] = side(p.dw);
        plan[4] = p.splits;
        plan[5] = p.wsplits;
        plan[7] = ws_bytes < least_ws(dtype, N, V, D, K, 1) ? 0 : piece_rows(p, N, V, D, ws_bytes);
    }
    return DH_OK;
}

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
