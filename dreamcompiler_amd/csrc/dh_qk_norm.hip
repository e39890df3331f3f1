// dh_qk_norm.hip -- RMS norm of every head's query and key and the rotation by position, in one
// pass, and its gradient.
//
//   r = (mean x^2 + eps)^(-1/2)      y = x r g      out = y with the pairs (i, j) of its first R
//   values turned by the position's angles: out[i] = y[i] c - y[j] s, out[j] = y[j] c + y[i] s
//
//   dy = dout turned back     dg = sum of dy x r     dx = r (dy g - x r mean(dy g x r))
//
// Nothing passes from forward to backward: r is recomputed from x.  All of it is bound by HBM:
// the forward reads and writes each value once, the gradient reads x and dout and writes dx.  Sums
// are held in fp32, results are rounded once.  No floating-point atomics: dg goes through fp32
// partials that are added in a fixed order.
//
// Measured, where a copy of 1 GiB moves 5.14 TB/s: 16384 tokens of 32 + 8 heads of 128 bf16 take 73 us forward (4.7 TB/s);
// 32768 of 16 + 16 heads with fp32 dout 98 us forward (5.5: the last-level cache holds part) and 220 gradient (5.0), 5 of it
// the partials; 3999 of 12 + 3 heads of 80 fp32 10 and 14; one token 3, a launch.
#include <cmath>

#include "dh_common.hpp"

namespace dh {
namespace {

constexpr int QK_MOST_D = 1024;

__device__ inline float up(float x) { return x; }
__device__ inline float up(uint16_t x) { return bf16_bits_to_f32(x); }
template <typename T> __device__ inline T down(float x);
template <> __device__ inline float down<float>(float x) { return x; }
template <> __device__ inline uint16_t down<uint16_t>(float x) {
    return __builtin_bit_cast(uint16_t, (__bf16)x);
}

// Rows of one tensor: sequence b, token t, head h at p + b s0 + t s1 + h s2.
template <typename T>
struct Rows {
    T* p;
    long long s0, s1, s2;
    __device__ T* at(int b, int t, int h) const { return p + b * s0 + t * s1 + h * s2; }
};

struct Shape {
    int B, S, H[2], D, R, P;
    bool pairs;
    float eps, by_d;   // 1 / D
    const int* pos;
    const float* table;
};

// Token n's position: below 0 if it is padding.
__device__ inline int position(const Shape& s, int b, int t) {
    const int p = s.pos ? s.pos[(long long)b * s.S + t] : t;
    return (s.pos || s.R > 0) && (unsigned)p >= (unsigned)s.P ? -1 : p;
}

// Units of work for waves: blocks of heads of a token, those of queries first; a unit is `each` of them.
struct Units {
    int nq, n, each;      // blocks of queries, of all
    FastDiv per, S;       // units of a token, tokens of a sequence
    uint32_t units;
};

// 1 / sqrt(mean + eps) to 2^-22: the sum's own rounding is up to 2^-20.
__device__ inline float norm_of(float sum, const Shape& s) {
    return __builtin_amdgcn_rsqf(fmaf(sum, s.by_d, s.eps));
}

// ---- any rows ------------------------------------------------------------------------------------
// A wave per row, J values a lane, 64 apart: any D, strides and alignment.  What value e = 64 j + lane turns
// with: its partner's place, cosine and sine (signed so that the forward is y[e] c + y[partner] sn).
template <int J>
struct TurnAny {
    uint32_t R, half, other[J];
    bool pairs;
    float c[J], sn[J];
    __device__ explicit TurnAny(const Shape& s) : R(s.R), half(s.R >> 1), pairs(s.pairs) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const uint32_t e = 64 * j + (threadIdx.x & 63);
            other[j] = e >= R ? min(e, (uint32_t)s.D - 1) : pairs ? e ^ 1 : e < half ? e + half : e - half;
        }
    }
    __device__ void load(const float* __restrict__ row) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const uint32_t e = 64 * j + (threadIdx.x & 63), i = pairs ? e >> 1 : e < half ? e : e - half;
            const bool second = pairs ? e & 1 : e >= half;
            c[j] = 1.f, sn[j] = 0.f;
            if (e < R) c[j] = row[i], sn[j] = second ? row[half + i] : -row[half + i];
        }
    }
};
// The lane's weights, and its partners'.
template <int J>
struct WeightsAny {
    float w[J], wo[J];
    __device__ WeightsAny(const float* __restrict__ g, const Shape& s, const TurnAny<J>& turn) {
#pragma unroll
        for (int j = 0; j < J; ++j) {
            w[j] = g ? g[(uint32_t)min(64 * j + (int)(threadIdx.x & 63), s.D - 1)] : 1.f;
            wo[j] = g ? g[turn.other[j]] : 1.f;
        }
    }
};

// A rows of a wave are in flight: one at a time took 2 to 3 times as long (6592 tokens of 40 heads of 100 bf16 with
// R = 100 in halves, forward and gradient: 300 us with one, 145 with four, 100 with eight; of 6 heads: 54, 28, 31).
template <typename T, int J, int A>
__global__ void __launch_bounds__(256) qk_fwd(Shape s, Units u, Rows<const T> q, Rows<const T> k,
                                              const float* __restrict__ gq, const float* __restrict__ gk,
                                              Rows<T> qo, Rows<T> ko) {
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    TurnAny<J> turn(s);
    const WeightsAny<J> wq(gq, s, turn), wk(gk, s, turn);
    auto block = [&](const Rows<const T>& x, const Rows<T>& o, const WeightsAny<J>& w, int H, int b, int t, int h0, bool there) {
        float v[A][J], vo[A][J];
#pragma unroll
        for (int a = 0; a < A; ++a) {   // without a condition each, so that they are on their way together
            const T* p = x.at(b, t, min(h0 + a, H - 1));
#pragma unroll
            for (int j = 0; j < J; ++j) v[a][j] = up(p[(uint32_t)min(64 * j + lane, s.D - 1)]), vo[a][j] = up(p[turn.other[j]]);
        }
        wave_fence();   // o may be x
#pragma unroll
        for (int a = 0; a < A; ++a) {
            if (h0 + a >= H) break;
            float sum = 0.f;
#pragma unroll
            for (int j = 0; j < J; ++j) sum += 64 * j + lane < s.D ? v[a][j] * v[a][j] : 0.f;
            const float inv = norm_of(wave_reduce(sum, OpSum()), s);
            T* p = o.at(b, t, h0 + a);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const int e = 64 * j + lane;
                float y = v[a][j] * inv * w.w[j];
                if (e < s.R) y = y * turn.c[j] + vo[a][j] * inv * w.wo[j] * turn.sn[j];
                if (e < s.D) p[e] = down<T>(there ? y : 0.f);   // padding: whatever the rest holds
            }
        }
    };
    for (uint32_t i = 4 * blockIdx.x + wave; i < u.units; i += 4 * gridDim.x) {
        const uint32_t n = fdiv(i, u.per);
        const int b = fdiv(n, u.S), t = n - b * s.S, j0 = (i - n * u.per.d) * u.each, j1 = min(j0 + u.each, u.n);
        const int p = position(s, b, t);
        turn.load(s.table + (long long)max(p, 0) * s.R);
        for (int j = j0; j < j1; ++j) {
            if (j < u.nq) block(q, qo, wq, s.H[0], b, t, j * A, p >= 0);
            else block(k, ko, wk, s.H[1], b, t, (j - u.nq) * A, p >= 0);
        }
    }
}

// The gradient: a work-group leaves its sums of dgq and dgk in rows blockIdx.x and gridDim.x + blockIdx.x of part.
template <typename T, typename GT, typename OT, int J, int A>
__global__ void __launch_bounds__(256) qk_bwd(Shape s, Units u, Rows<const T> q, Rows<const T> k,
                                              const float* __restrict__ gq, const float* __restrict__ gk,
                                              Rows<const GT> dqo, Rows<const GT> dko, Rows<OT> dq, Rows<OT> dk,
                                              float* __restrict__ part) {
    __shared__ float red[4][64 * J];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    TurnAny<J> turn(s);
    const WeightsAny<J> wq(gq, s, turn), wk(gk, s, turn);
    float acc[2][J] = {};
    auto block = [&](const Rows<const T>& x, const Rows<const GT>& d, const Rows<OT>& o, const WeightsAny<J>& w,
                     float (&acc)[J], int H, int b, int t, int h0, bool there) {
        float v[A][J], dy[A][J], other[A][J];
#pragma unroll
        for (int a = 0; a < A; ++a) {
            const int h = min(h0 + a, H - 1);
            const T* p = x.at(b, t, h);
            const GT* r = d.at(b, t, h);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const uint32_t e = min(64 * j + lane, s.D - 1);
                v[a][j] = up(p[e]), dy[a][j] = up(r[e]), other[a][j] = up(r[turn.other[j]]);
            }
        }
        wave_fence();   // o may be x or d
#pragma unroll
        for (int a = 0; a < A; ++a) {
            if (h0 + a >= H) break;
            float sum = 0.f, dot = 0.f;
#pragma unroll
            for (int j = 0; j < J; ++j) {
                const bool in = there && 64 * j + lane < s.D;   // a row of padding: whatever the rest holds
                v[a][j] = in ? v[a][j] : 0.f;
                if (64 * j + lane < s.R) dy[a][j] = dy[a][j] * turn.c[j] - other[a][j] * turn.sn[j];
                dy[a][j] = in ? dy[a][j] : 0.f;
                sum += v[a][j] * v[a][j];
            }
            const float inv = norm_of(wave_reduce(sum, OpSum()), s);
#pragma unroll
            for (int j = 0; j < J; ++j) {
                v[a][j] *= inv;
                acc[j] += dy[a][j] * v[a][j];
                dy[a][j] *= 64 * j + lane < s.D ? w.w[j] : 0.f;
                dot += dy[a][j] * v[a][j];
            }
            const float mean = wave_reduce(dot, OpSum()) * s.by_d;
            OT* p = o.at(b, t, h0 + a);
#pragma unroll
            for (int j = 0; j < J; ++j)
                if (64 * j + lane < s.D) p[64 * j + lane] = down<OT>(there ? inv * (dy[a][j] - v[a][j] * mean) : 0.f);
        }
    };
    for (uint32_t i = 4 * blockIdx.x + wave; i < u.units; i += 4 * gridDim.x) {
        const uint32_t n = fdiv(i, u.per);
        const int b = fdiv(n, u.S), t = n - b * s.S, j0 = (i - n * u.per.d) * u.each, j1 = min(j0 + u.each, u.n);
        const int p = position(s, b, t);
        turn.load(s.table + (long long)max(p, 0) * s.R);
        for (int j = j0; j < j1; ++j) {
            if (j < u.nq) block(q, dqo, dq, wq, acc[0], s.H[0], b, t, j * A, p >= 0);
            else block(k, dko, dk, wk, acc[1], s.H[1], b, t, (j - u.nq) * A, p >= 0);
        }
    }
#pragma unroll
    for (int side = 0; side < 2; ++side) {
        if (side) __syncthreads();
#pragma unroll
        for (int j = 0; j < J; ++j) red[wave][64 * j + lane] = acc[side][j];
        __syncthreads();
        for (int e = threadIdx.x; e < s.D; e += 256)
            part[((long long)side * gridDim.x + blockIdx.x) * s.D + e] = red[0][e] + red[1][e] + red[2][e] + red[3][e];
    }
}

// ---- rows in pieces ------------------------------------------------------------------------------
// (Both forms, where rows fit either, 6592 tokens bf16, forward and gradient, pieces first: 16 + 16 heads of 64 40 and 64 us,
// 8 + 2 of 256 49 and 58, 32 + 8 of 100 96 and 100, 2 + 1 of 128 19 and 24; 32 + 8 of 128 forward 30 and 40.)
// Where rows begin with whole pieces of V values (16 or 8 bytes) and the values that turn together lie
// in whole pieces too, a row is L lanes of a piece each, and a wave takes 64 / L heads of a token at
// once: their rows usually lie side by side, and the token's cosines and sines are read once for all
// heads.  HEADS heads make a unit: all of a token's where there are many tokens.
template <typename T, int V>
__device__ inline void load_piece(const T* p, float (&v)[V]) {
    typedef T vec __attribute__((ext_vector_type(V), aligned(V * sizeof(T) < 16 ? V * sizeof(T) : 16)));
    const vec x = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = up(x[e]);
}
template <typename T, int V>
__device__ inline void store_piece(T* p, const float (&v)[V]) {
    typedef T vec __attribute__((ext_vector_type(V), aligned(V * sizeof(T) < 16 ? V * sizeof(T) : 16)));
    vec x;
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = down<T>(v[e]);
    *reinterpret_cast<vec*>(p) = x;
}

// The sum over each L lanes, in all of them.
template <int L>
__device__ inline float group_sum(float v) {
    if (L > 1) v += dpp_quad_xor1(v);
    if (L > 2) v += dpp_quad_xor2(v);
    if (L > 4) v += dpp_half_mirror(v);
    if (L > 8) v += dpp_row_mirror(v);
    float lo, hi;
    if (L > 16) {
        halves16(v, lo, hi);
        v = lo + hi;
    }
    if (L > 32) {
        halves32(v, lo, hi);
        v = lo + hi;
    }
    return v;
}

// What a lane's piece turns with: y -> y c + partner sn, the partners in another lane's piece (halves) or
// in this one (pairs).
template <int V>
struct Turn {
    float c[V], sn[V];
    int from;   // the lane that has the partners
    bool turns;
    __device__ void find(const Shape& s, int piece) {
        const int half = s.R / (2 * V), lane = threadIdx.x & 63;
        turns = piece * V < s.R;
        from = !turns || s.pairs ? lane : piece < half ? lane + half : lane - half;
    }
    __device__ void load(const Shape& s, const float* __restrict__ row, int piece) {
#pragma unroll
        for (int e = 0; e < V; ++e) c[e] = 1.f, sn[e] = 0.f;
        if (!turns) return;
        const int half = s.R >> 1;
        if (s.pairs) {
            typedef float vec __attribute__((ext_vector_type(V / 2), aligned(4)));
            const vec a = *reinterpret_cast<const vec*>(row + piece * (V / 2));
            const vec b = *reinterpret_cast<const vec*>(row + half + piece * (V / 2));
#pragma unroll
            for (int e = 0; e < V; ++e) {
                c[e] = a[e / 2];
                sn[e] = e & 1 ? b[e / 2] : -b[e / 2];
            }
        } else {
            const bool second = piece * V >= half;
            const int i = piece * V - (second ? half : 0);
            typedef float vec __attribute__((ext_vector_type(V), aligned(4)));
            const vec a = *reinterpret_cast<const vec*>(row + i), b = *reinterpret_cast<const vec*>(row + half + i);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                c[e] = a[e];
                sn[e] = second ? b[e] : -b[e];
            }
        }
    }
    // y turned; by the angle's negative with back = -1.
    __device__ void apply(const Shape& s, float (&y)[V], float back) const {
        float other[V];
        if (s.pairs) {
#pragma unroll
            for (int e = 0; e < V; ++e) other[e] = y[e ^ 1];
        } else {
#pragma unroll
            for (int e = 0; e < V; ++e) other[e] = __shfl(y[e], from);
        }
#pragma unroll
        for (int e = 0; e < V; ++e) y[e] = y[e] * c[e] + other[e] * (sn[e] * back);
    }
};

// Rows of a lane in flight: more of them leave room for fewer waves (twice as many: 1 to 4% slower at every size).  Stores
// stay ordinary: past the last-level cache they save 8% here, but flash attention, which reads these rows next, loses more
// (both together 644 us, 652 so).
template <int V> constexpr int ahead() { return 8 / V; }

template <int V>
__device__ inline void load_weights(const float* __restrict__ g, int piece, bool in, float (&w)[V]) {
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = 1.f;
    typedef float vec __attribute__((ext_vector_type(V), aligned(4)));
    if (!g || !in) return;
    const vec x = *reinterpret_cast<const vec*>(g + piece * V);
#pragma unroll
    for (int e = 0; e < V; ++e) w[e] = x[e];
}

// A wave's tokens at once: where a token has fewer heads than the wave has places for rows, the places of a
// power of two `heads` of each side belong to a token, and a unit is as many tokens as that leaves.
struct Many {
    int heads, tokens;
    long long n;   // tokens of the call
};

template <typename T, int V, int L, bool MANY>
__global__ void __launch_bounds__(256) qk_fwd_pieces(Shape s, Units u, Many m, Rows<const T> q, Rows<const T> k,
                                                     const float* __restrict__ gq, const float* __restrict__ gk,
                                                     Rows<T> qo, Rows<T> ko) {
    constexpr int G = 64 / L, AHEAD = MANY ? 1 : ahead<V>();
    const int lane = threadIdx.x & 63, piece = lane & (L - 1), sub = lane / L;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool in = piece * V < s.D;
    float wq[V], wk[V];
    load_weights<V>(gq, piece, in, wq);
    load_weights<V>(gk, piece, in, wk);
    Turn<V> turn;
    turn.find(s, piece);
    auto block = [&](const Rows<const T>& x, const Rows<T>& o, const float (&w)[V], int H, int b, int t, int h0, bool there) {
        const int hs = MANY ? 0 : sub;   // the lane's head is h0 + hs; h0 is one for the wave unless MANY
        const T* xp = x.at(b, t, h0) + (hs * x.s2 + piece * V);
        T* op = o.at(b, t, h0) + (hs * o.s2 + piece * V);
        float v[AHEAD][V];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[a][e] = 0.f;
            if (h0 + a * G + hs < H && in && there) load_piece<T, V>(xp + a * G * x.s2, v[a]);
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (!MANY && h0 + a * G >= H) break;
            float sum = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) sum += v[a][e] * v[a][e];
            const float inv = norm_of(group_sum<L>(sum), s);
#pragma unroll
            for (int e = 0; e < V; ++e) v[a][e] *= inv * w[e];
            turn.apply(s, v[a], 1.f);
#pragma unroll
            for (int e = 0; e < V; ++e) v[a][e] = there ? v[a][e] : 0.f;   // whatever the table and the weights hold
            if (h0 + a * G + hs < H && in) store_piece<T, V>(op + a * G * o.s2, v[a]);
        }
    };
    for (uint32_t i = 4 * blockIdx.x + wave; i < u.units; i += 4 * gridDim.x) {
        if constexpr (MANY) {   // one lane's token is not another's
            const uint32_t n = i * m.tokens + sub / m.heads;
            const bool any = n < m.n;
            const int b = any ? fdiv(n, u.S) : 0, t = any ? n - b * s.S : 0, p = any ? position(s, b, t) : -1;
            turn.load(s, s.table + (long long)max(p, 0) * s.R, piece);
            const int h = sub & (m.heads - 1);
            if (s.H[0] > 0) block(q, qo, wq, any ? s.H[0] : 0, b, t, h, p >= 0);
            if (s.H[1] > 0) block(k, ko, wk, any ? s.H[1] : 0, b, t, h, p >= 0);
            continue;
        }
        const uint32_t n = fdiv(i, u.per);
        const int b = fdiv(n, u.S), t = n - b * s.S, j0 = (i - n * u.per.d) * u.each, j1 = min(j0 + u.each, u.n);
        const int p = position(s, b, t);
        turn.load(s, s.table + (long long)max(p, 0) * s.R, piece);
        for (int j = j0; j < j1; ++j) {
            if (j < u.nq) block(q, qo, wq, s.H[0], b, t, j * AHEAD * G, p >= 0);
            else block(k, ko, wk, s.H[1], b, t, (j - u.nq) * AHEAD * G, p >= 0);
        }
    }
}

// The gradient: a work-group leaves its sums of dgq and dgk in rows blockIdx.x and gridDim.x + blockIdx.x of part.
template <typename T, typename GT, typename OT, int V, int L, bool MANY>
__global__ void __launch_bounds__(256) qk_bwd_pieces(Shape s, Units u, Many m, Rows<const T> q, Rows<const T> k,
                                                     const float* __restrict__ gq, const float* __restrict__ gk,
                                                     Rows<const GT> dqo, Rows<const GT> dko, Rows<OT> dq, Rows<OT> dk,
                                                     float* __restrict__ part) {
    constexpr int G = 64 / L, AHEAD = MANY ? 1 : ahead<V>();
    __shared__ float red[4 * G][2][L * V];
    const int lane = threadIdx.x & 63, piece = lane & (L - 1), sub = lane / L;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool in = piece * V < s.D;
    float wq[V], wk[V], aq[V] = {}, ak[V] = {};
    load_weights<V>(gq, piece, in, wq);
    load_weights<V>(gk, piece, in, wk);
    Turn<V> turn;
    turn.find(s, piece);
    auto block = [&](const Rows<const T>& x, const Rows<const GT>& dy, const Rows<OT>& o, const float (&w)[V],
                     float (&acc)[V], int H, int b, int t, int h0, bool there) {
        const int hs = MANY ? 0 : sub;
        const T* xp = x.at(b, t, h0) + (hs * x.s2 + piece * V);
        const GT* dp = dy.at(b, t, h0) + (hs * dy.s2 + piece * V);
        OT* op = o.at(b, t, h0) + (hs * o.s2 + piece * V);
        float v[AHEAD][V], d[AHEAD][V];
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
#pragma unroll
            for (int e = 0; e < V; ++e) v[a][e] = d[a][e] = 0.f;
            if (h0 + a * G + hs < H && in && there) {
                load_piece<T, V>(xp + a * G * x.s2, v[a]);
                load_piece<GT, V>(dp + a * G * dy.s2, d[a]);
            }
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            if (!MANY && h0 + a * G >= H) break;
            float sum = 0.f, dot = 0.f;
#pragma unroll
            for (int e = 0; e < V; ++e) sum += v[a][e] * v[a][e];
            const float inv = norm_of(group_sum<L>(sum), s);
            turn.apply(s, d[a], -1.f);
#pragma unroll
            for (int e = 0; e < V; ++e) {
                v[a][e] *= inv;
                d[a][e] = there ? d[a][e] : 0.f;
                acc[e] += d[a][e] * v[a][e];
                d[a][e] *= w[e];
                dot += d[a][e] * v[a][e];
            }
            const float mean = group_sum<L>(dot) * s.by_d;
#pragma unroll
            for (int e = 0; e < V; ++e) d[a][e] = there ? inv * (d[a][e] - v[a][e] * mean) : 0.f;
            if (h0 + a * G + hs < H && in) store_piece<OT, V>(op + a * G * o.s2, d[a]);
        }
    };
    for (uint32_t i = 4 * blockIdx.x + wave; i < u.units; i += 4 * gridDim.x) {
        if constexpr (MANY) {   // one lane's token is not another's
            const uint32_t n = i * m.tokens + sub / m.heads;
            const bool any = n < m.n;
            const int b = any ? fdiv(n, u.S) : 0, t = any ? n - b * s.S : 0, p = any ? position(s, b, t) : -1;
            turn.load(s, s.table + (long long)max(p, 0) * s.R, piece);
            const int h = sub & (m.heads - 1);
            if (s.H[0] > 0) block(q, dqo, dq, wq, aq, any ? s.H[0] : 0, b, t, h, p >= 0);
            if (s.H[1] > 0) block(k, dko, dk, wk, ak, any ? s.H[1] : 0, b, t, h, p >= 0);
            continue;
        }
        const uint32_t n = fdiv(i, u.per);
        const int b = fdiv(n, u.S), t = n - b * s.S, j0 = (i - n * u.per.d) * u.each, j1 = min(j0 + u.each, u.n);
        const int p = position(s, b, t);
        turn.load(s, s.table + (long long)max(p, 0) * s.R, piece);
        for (int j = j0; j < j1; ++j) {
            if (j < u.nq) block(q, dqo, dq, wq, aq, s.H[0], b, t, j * AHEAD * G, p >= 0);
            else block(k, dko, dk, wk, ak, s.H[1], b, t, (j - u.nq) * AHEAD * G, p >= 0);
        }
    }
#pragma unroll
    for (int e = 0; e < V; ++e) {
        red[wave * G + sub][0][piece * V + e] = aq[e];
        red[wave * G + sub][1][piece * V + e] = ak[e];
    }
    __syncthreads();
    for (int i = threadIdx.x; i < 2 * s.D; i += 256) {
        const int side = i >= s.D, e = side ? i - s.D : i;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < 4 * G; ++j) sum += red[j][side][e];
        part[((long long)side * gridDim.x + blockIdx.x) * s.D + e] = sum;
    }
}

// dg (+)= the sum of its n partials a side: a work-group per 16 columns, 64 partials at a time, in order.
__global__ void __launch_bounds__(1024) qk_join(const float* __restrict__ part, int D, int n,
                                                float* __restrict__ dgq, float* __restrict__ dgk, int acc) {
    __shared__ float red[64][17];
    const int side = blockIdx.y, col = threadIdx.x & 15, r = threadIdx.x >> 4, e = blockIdx.x * 16 + col;
    float* out = side ? dgk : dgq;
    if (!out) return;
    float sum = 0.f;
    if (e < D) {
        const float* p = part + (long long)side * n * D + e;
#pragma unroll 8
        for (int i = r; i < n; i += 64) sum += p[(long long)i * D];
    }
    red[r][col] = sum;
    __syncthreads();
    if (r > 0 || e >= D) return;
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 64; ++i) sum += red[i][col];
    out[e] = acc ? out[e] + sum : sum;
}

// One thread per angle.
__global__ void __launch_bounds__(256) rope_table_kernel(int P, int half, double step, float* __restrict__ out) {
    const long long n = (long long)P * half, stride = (long long)gridDim.x * 256;
    for (long long i = (long long)blockIdx.x * 256 + threadIdx.x; i < n; i += stride) {
        const long long p = i / half;
        const int k = (int)(i - p * half);
        double sn, c;
        sincos((double)p * exp(k * step), &sn, &c);
        out[p * 2 * half + k] = (float)c;
        out[p * 2 * half + half + k] = (float)sn;
    }
}

// ---- host --------------------------------------------------------------------------------------
// Whether rows of D values at the strides st lie within 2^46 elements, and apart where they are
// written.
int check_rows(const char* op, const char* name, const long long* st, int B, int S, int H, int D, bool out) {
    if (!st) return set_error(DH_ERR_INVALID, "%s: null strides of %s", op, name);
    const long long n[3] = {B, S, H};
    if (n[0] == 0 || n[1] == 0 || n[2] == 0) return DH_OK;   // no rows
    int order[3] = {0, 1, 2};
    for (int i = 0; i < 3; ++i)
        for (int j = i + 1; j < 3; ++j)
            if (st[order[j]] < st[order[i]]) { const int x = order[i]; order[i] = order[j]; order[j] = x; }
    long long extent = D;
    for (int i = 0; i < 3; ++i) {
        const long long s = st[order[i]], m = n[order[i]];
        if (m <= 1) continue;
        if (s < 0 || s > (1ll << 46) / m || (out && s < extent))
            return set_error(DH_ERR_INVALID, "%s: strides (%lld, %lld, %lld) of %s", op, st[0], st[1], st[2], name);
        extent += s * (m - 1);
    }
    return DH_OK;
}

int check_qk(const char* op, int dtype, int B, int S, int Hq, int Hk, int D, int R, float eps, const void* table,
             int P, Shape& s, const int* pos, int pairs) {
    if (dtype != DH_F32 && dtype != DH_BF16) return set_error(DH_ERR_INVALID, "%s: dtype must be fp32 or bf16", op);
    if (B < 0 || S < 0 || Hq < 0 || Hk < 0 || Hq > 65536 || Hk > 65536 || D < 1 || D > QK_MOST_D ||
        (long long)B * S > 0x7FF00000)
        return set_error(DH_ERR_INVALID, "%s: shape B=%d S=%d Hq=%d Hk=%d D=%d", op, B, S, Hq, Hk, D);
    if (R < 0 || R > D || (R & 1)) return set_error(DH_ERR_INVALID, "%s: R=%d must be even and at most D", op, R);
    if (!(eps >= 1.17549435e-38f) || !(eps - eps == 0.f))
        return set_error(DH_ERR_INVALID, "%s: eps must be finite and at least 2^-126", op);
    if ((R > 0 && !table) || ((R > 0 || pos) && P < 1) || (R > 0 && !pos && S > P))
        return set_error(DH_ERR_INVALID, "%s: no table of %d positions (P=%d)", op, pos ? 1 : S, P);
    s = Shape{B, S, {Hq, Hk}, D, R, P, pairs != 0, eps, 1.f / D, pos, (const float*)table};
    return DH_OK;
}

template <typename T>
Rows<T> rows_of(const void* p, const long long* st) {
    return {(T*)p, st[0], st[1], st[2]};
}

// Values of a piece for rows of these tensors: 8 or 4 where every row begins with whole pieces of up to
// 16 bytes (`size`: of the smallest type) and pieces turn together, else 1: the form for any rows.
struct Piece {
    int V;
    const Shape& s;
    Piece(const Shape& s, int size) : V(16 / size), s(s) {
        while (V > 1 && !fits()) V = V == 8 ? 4 : 1;
    }
    bool fits() const {
        return s.D % V == 0 && s.D <= 64 * V && s.R % V == 0 && (s.pairs || s.R % (2 * V) == 0);
    }
    void rows(int H, const void* p, const long long* st, int size) {
        const int n[3] = {s.B, s.S, H};
        long long bits = 0;
        for (int i = 0; i < 3; ++i) bits |= n[i] > 1 ? st[i] : 0;
        while (V > 1 && H > 0 && (bits % V != 0 || (uintptr_t)p % (V * size < 16 ? V * size : 16) != 0 || !fits()))
            V = V == 8 ? 4 : 1;
    }
    int lanes() const {
        int L = 4;   // a row of 32 bf16
        while (L * V < s.D) L *= 2;
        return L;
    }
};
// Blocks of a unit: all of a token's where that gives each of the GPU's 8192 waves a unit, else down to one, and as
// many for each unit of a token (6592 tokens of ten blocks, forward and gradient: 104 us with nine and one, 88 with five).
// Units and tokens stay below 2^31, as FastDiv needs: there are at most 2^31 - 2^20 tokens.
Units units_of(const Shape& s, int heads) {
    const long long n = (long long)s.B * s.S;
    const int nq = (s.H[0] + heads - 1) / heads, nk = (s.H[1] + heads - 1) / heads, blocks = nq + nk;
    int each = (int)(n >= 8192 ? blocks : (n * blocks + 8191) / 8192);
    const int per = (blocks + each - 1) / each;
    each = (blocks + per - 1) / per;
    return Units{nq, blocks, each, make_fastdiv(per), make_fastdiv(s.S), (uint32_t)(n * per)};
}

// Places for `heads` heads of a side where a wave has twice as many or more, and their tokens; else 0.
Many many_of(const Shape& s, int places) {
    int heads = 1;
    while (heads < s.H[0] || heads < s.H[1]) heads *= 2;
    return Many{2 * heads <= places ? heads : 0, 2 * heads <= places ? places / heads : 0, (long long)s.B * s.S};
}
unsigned groups_of(uint32_t units, uint32_t most) {
    const uint32_t groups = (units + 3) / 4;
    return groups < most ? groups : most;
}
// Work-groups of the gradient: enough to fill the GPU (four a CU), few enough that their partials, 1 MB at D = 128, are
// a small part of the work.
constexpr int QK_GROUPS = 1024, FWD_GROUPS = 1 << 20;

struct Call {
    const void *Q, *K, *dQo, *dKo;
    const long long *sq, *sk, *sdqo, *sdko;
    const float *gq, *gk;
    void *Qo, *Ko;   // dQ, dK of the gradient
    const long long *sqo, *sko;
    float *dgq, *dgk, *part;
    int acc;
};

template <typename T, int V, int L>
int launch_fwd_pieces(const Shape& s, const Call& c) {
    Units u = units_of(s, ahead<V>() * 64 / L);
    const Many m = many_of(s, 64 / L);
    auto run = qk_fwd_pieces<T, V, L, false>;
    if constexpr (L < 64)
        if (m.heads) u.units = (uint32_t)((m.n + m.tokens - 1) / m.tokens), run = qk_fwd_pieces<T, V, L, true>;
    run<<<groups_of(u.units, FWD_GROUPS), 256, 0, stream()>>>(s, u, m, rows_of<const T>(c.Q, c.sq), rows_of<const T>(c.K, c.sk),
                                                              c.gq, c.gk, rows_of<T>(c.Qo, c.sqo), rows_of<T>(c.Ko, c.sko));
    return check_launch("dh_qk_norm_rope_fwd");
}
template <typename T, int J, int A>
int launch_fwd(const Shape& s, const Call& c) {
    const Units u = units_of(s, A);
    qk_fwd<T, J, A><<<groups_of(u.units, FWD_GROUPS), 256, 0, stream()>>>(s, u, rows_of<const T>(c.Q, c.sq),
                                                                       rows_of<const T>(c.K, c.sk), c.gq, c.gk,
                                                                       rows_of<T>(c.Qo, c.sqo), rows_of<T>(c.Ko, c.sko));
    return check_launch("dh_qk_norm_rope_fwd");
}

int join(const Shape& s, const Call& c, int n) {
    DH_TRY(check_launch("dh_qk_norm_rope_bwd"));
    if (!c.dgq && !c.dgk) return DH_OK;
    qk_join<<<dim3((s.D + 15) / 16, 2), 1024, 0, stream()>>>(c.part, s.D, n, c.dgq, c.dgk, c.acc);
    return check_launch("dh_qk_norm_rope_bwd");
}
template <typename T, typename GT, typename OT, int V, int L>
int launch_bwd_pieces(const Shape& s, const Call& c) {
    Units u = units_of(s, ahead<V>() * 64 / L);
    const Many m = many_of(s, 64 / L);
    auto run = qk_bwd_pieces<T, GT, OT, V, L, false>;
    if constexpr (L < 64)
        if (m.heads) u.units = (uint32_t)((m.n + m.tokens - 1) / m.tokens), run = qk_bwd_pieces<T, GT, OT, V, L, true>;
    const unsigned grid = groups_of(u.units, QK_GROUPS);
    run<<<grid, 256, 0, stream()>>>(s, u, m, rows_of<const T>(c.Q, c.sq), rows_of<const T>(c.K, c.sk), c.gq, c.gk,
                                    rows_of<const GT>(c.dQo, c.sdqo), rows_of<const GT>(c.dKo, c.sdko),
                                    rows_of<OT>(c.Qo, c.sqo), rows_of<OT>(c.Ko, c.sko), c.part);
    return join(s, c, grid);
}
template <typename T, typename GT, typename OT, int J, int A>
int launch_bwd(const Shape& s, const Call& c) {
    const Units u = units_of(s, A);
    const unsigned grid = groups_of(u.units, QK_GROUPS);
    qk_bwd<T, GT, OT, J, A><<<grid, 256, 0, stream()>>>(s, u, rows_of<const T>(c.Q, c.sq), rows_of<const T>(c.K, c.sk), c.gq, c.gk,
                                                     rows_of<const GT>(c.dQo, c.sdqo), rows_of<const GT>(c.dKo, c.sdko),
                                                     rows_of<OT>(c.Qo, c.sqo), rows_of<OT>(c.Ko, c.sko), c.part);
    return join(s, c, grid);
}

template <typename T, int V>
int fwd_by_lanes(int L, const Shape& s, const Call& c) {
    return L == 4    ? launch_fwd_pieces<T, V, 4>(s, c)
           : L == 8  ? launch_fwd_pieces<T, V, 8>(s, c)
           : L == 16 ? launch_fwd_pieces<T, V, 16>(s, c)
           : L == 32 ? launch_fwd_pieces<T, V, 32>(s, c)
                     : launch_fwd_pieces<T, V, 64>(s, c);
}
// With few heads most of eight rows would be loads for nothing: the figures are at the kernels.
bool few_heads(const Shape& s) { return s.H[0] <= 4 && s.H[1] <= 4; }
template <typename T>
int fwd_of(const Piece& p, const Shape& s, const Call& c) {
    if (p.V == 1)
        return s.D > 512   ? launch_fwd<T, 16, 2>(s, c)
               : s.D > 256 ? launch_fwd<T, 8, 4>(s, c)
               : s.D > 128 ? launch_fwd<T, 4, 4>(s, c)
               : few_heads(s) ? launch_fwd<T, 2, 4>(s, c) : launch_fwd<T, 2, 8>(s, c);
    if constexpr (sizeof(T) == 2)
        if (p.V == 8) return fwd_by_lanes<T, 8>(p.lanes(), s, c);
    return fwd_by_lanes<T, 4>(p.lanes(), s, c);
}
template <typename T, typename GT, typename OT, int V>
int bwd_by_lanes(int L, const Shape& s, const Call& c) {
    return L == 4    ? launch_bwd_pieces<T, GT, OT, V, 4>(s, c)
           : L == 8  ? launch_bwd_pieces<T, GT, OT, V, 8>(s, c)
           : L == 16 ? launch_bwd_pieces<T, GT, OT, V, 16>(s, c)
           : L == 32 ? launch_bwd_pieces<T, GT, OT, V, 32>(s, c)
                     : launch_bwd_pieces<T, GT, OT, V, 64>(s, c);
}
template <typename T, typename GT, typename OT>
int bwd_of(const Piece& p, const Shape& s, const Call& c) {
    if (p.V == 1)
        return s.D > 512   ? launch_bwd<T, GT, OT, 16, 1>(s, c)
               : s.D > 256 ? launch_bwd<T, GT, OT, 8, 4>(s, c)
               : s.D > 128 ? launch_bwd<T, GT, OT, 4, 4>(s, c)
               : few_heads(s) ? launch_bwd<T, GT, OT, 2, 4>(s, c) : launch_bwd<T, GT, OT, 2, 8>(s, c);
    if constexpr (sizeof(T) == 2)
        if (p.V == 8) return bwd_by_lanes<T, GT, OT, 8>(p.lanes(), s, c);
    return bwd_by_lanes<T, GT, OT, 4>(p.lanes(), s, c);
}

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" {

int dh_rope_table(int P, int R, double base, float* table) {
    if (P < 0 || R < 0 || (R & 1) || R > QK_MOST_D)
        return set_error(DH_ERR_INVALID, "dh_rope_table: shape P=%d R=%d", P, R);
    if (!(base > 0.0) || !(base - base == 0.0))
        return set_error(DH_ERR_INVALID, "dh_rope_table: base must be finite and > 0");
    if (P > 0 && R > 0 && !table) return set_error(DH_ERR_INVALID, "dh_rope_table: null pointer");
    DH_TRY(ensure_init());
    if (P == 0 || R == 0) return DH_OK;
    const long long groups = ((long long)P * (R / 2) + 255) / 256;
    rope_table_kernel<<<(unsigned)(groups < 65536 ? groups : 65536), 256, 0, stream()>>>(
        P, R / 2, -2.0 / R * std::log(base), table);
    return check_launch("dh_rope_table");
}

int dh_qk_norm_rope_fwd(int dtype, int B, int S, int Hq, int Hk, int D, int R, int pairs, float eps, const int* pos,
                        const float* table, int P, const void* Q, const long long* sq, const void* K,
                        const long long* sk, const float* gq, const float* gk, void* Qo, const long long* sqo,
                        void* Ko, const long long* sko) {
    const char* op = "dh_qk_norm_rope_fwd";
    Shape s;
    DH_TRY(check_qk(op, dtype, B, S, Hq, Hk, D, R, eps, table, P, s, pos, pairs));
    const long long none[3] = {0, 0, 0};
    if (Hq > 0) {
        DH_TRY(check_rows(op, "Q", sq, B, S, Hq, D, false));
        DH_TRY(check_rows(op, "Qo", sqo, B, S, Hq, D, true));
    }
    if (Hk > 0) {
        DH_TRY(check_rows(op, "K", sk, B, S, Hk, D, false));
        DH_TRY(check_rows(op, "Ko", sko, B, S, Hk, D, true));
    }
    const bool any = (long long)B * S > 0;
    if (any && ((Hq > 0 && (!Q || !Qo)) || (Hk > 0 && (!K || !Ko))))
        return set_error(DH_ERR_INVALID, "%s: null pointer", op);
    DH_TRY(ensure_init());
    if (!any || Hq + Hk == 0) return DH_OK;
    if (Hq == 0) sq = sqo = none;
    if (Hk == 0) sk = sko = none;
    const int size = dtype == DH_F32 ? 4 : 2;
    Piece p(s, size);
    p.rows(Hq, Q, sq, size), p.rows(Hk, K, sk, size), p.rows(Hq, Qo, sqo, size), p.rows(Hk, Ko, sko, size);
    const Call c{Q, K, nullptr, nullptr, sq, sk, none, none, gq, gk, Qo, Ko, sqo, sko, nullptr, nullptr, nullptr, 0};
    return dtype == DH_F32 ? fwd_of<float>(p, s, c) : fwd_of<uint16_t>(p, s, c);
}

size_t dh_qk_norm_rope_bwd_workspace(int D) {
    return D < 1 || D > QK_MOST_D ? 0 : (size_t)2 * QK_GROUPS * D * 4;
}

int dh_qk_norm_rope_bwd(int dtype, int B, int S, int Hq, int Hk, int D, int R, int pairs, float eps, const int* pos,
                        const float* table, int P, const void* Q, const long long* sq, const void* K,
                        const long long* sk, const float* gq, const float* gk, int dout_type, const void* dQo,
                        const long long* sdqo, const void* dKo, const long long* sdko, int grad_type, void* dQ,
                        const long long* sdq, void* dK, const long long* sdk, float* dgq, float* dgk, int accumulate,
                        void* ws, size_t ws_bytes) {
    const char* op = "dh_qk_norm_rope_bwd";
    Shape s;
    DH_TRY(check_qk(op, dtype, B, S, Hq, Hk, D, R, eps, table, P, s, pos, pairs));
    if ((dout_type != DH_F32 && dout_type != dtype) || (grad_type != DH_F32 && grad_type != dtype))
        return set_error(DH_ERR_INVALID, "%s: dout_type and grad_type must be fp32 or the inputs' type", op);
    const long long none[3] = {0, 0, 0};
    if (Hq > 0) {
        DH_TRY(check_rows(op, "Q", sq, B, S, Hq, D, false));
        DH_TRY(check_rows(op, "dQo", sdqo, B, S, Hq, D, false));
        DH_TRY(check_rows(op, "dQ", sdq, B, S, Hq, D, true));
    }
    if (Hk > 0) {
        DH_TRY(check_rows(op, "K", sk, B, S, Hk, D, false));
        DH_TRY(check_rows(op, "dKo", sdko, B, S, Hk, D, false));
        DH_TRY(check_rows(op, "dK", sdk, B, S, Hk, D, true));
    }
    const bool any = (long long)B * S > 0;
    if (any && ((Hq > 0 && (!Q || !dQo || !dQ)) || (Hk > 0 && (!K || !dKo || !dK))))
        return set_error(DH_ERR_INVALID, "%s: null pointer", op);
    if (dgq && dgk && dgq < dgk + D && dgk < dgq + D)
        return set_error(DH_ERR_INVALID, "%s: dgq and dgk must not overlap", op);
    const size_t need = dh_qk_norm_rope_bwd_workspace(D);
    if (!ws) return set_error(DH_ERR_INVALID, "%s: null pointer", op);
    if ((uintptr_t)ws & 15) return set_error(DH_ERR_INVALID, "%s: workspace not 16-byte aligned", op);
    if (ws_bytes < need)
        return set_error(DH_ERR_INVALID, "%s: workspace of %zu bytes, %zu needed", op, ws_bytes, need);
    DH_TRY(ensure_init());
    if (Hq == 0) sq = sdqo = sdq = none;
    if (Hk == 0) sk = sdko = sdk = none;
    if (!any || Hq + Hk == 0) {   // no row: sums of nothing
        if (accumulate || (!dgq && !dgk)) return DH_OK;
        qk_join<<<dim3((D + 15) / 16, 2), 1024, 0, stream()>>>((float*)ws, D, 0, dgq, dgk, 0);
        return check_launch(op);
    }
    const bool gw = dout_type == DH_F32, ow = grad_type == DH_F32;
    const int size = dtype == DH_F32 ? 4 : 2, gsize = gw ? 4 : 2, osize = ow ? 4 : 2;
    Piece p(s, size);
    p.rows(Hq, Q, sq, size), p.rows(Hk, K, sk, size), p.rows(Hq, dQo, sdqo, gsize), p.rows(Hk, dKo, sdko, gsize);
    p.rows(Hq, dQ, sdq, osize), p.rows(Hk, dK, sdk, osize);
    const Call c{Q, K, dQo, dKo, sq, sk, sdqo, sdko, gq, gk, dQ, dK, sdq, sdk, dgq, dgk, (float*)ws, accumulate};
    if (dtype == DH_F32) return bwd_of<float, float, float>(p, s, c);
    if (gw) return ow ? bwd_of<uint16_t, float, float>(p, s, c) : bwd_of<uint16_t, float, uint16_t>(p, s, c);
    return ow ? bwd_of<uint16_t, uint16_t, float>(p, s, c) : bwd_of<uint16_t, uint16_t, uint16_t>(p, s, c);
}

}  // extern "C"
