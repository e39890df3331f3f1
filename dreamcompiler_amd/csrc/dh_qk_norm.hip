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
    float eps;
    const int* pos;
    const float* table;
};

// Token n's position: below 0 if it is padding.
__device__ inline int position(const Shape& s, int b, int t) {
    const int p = s.pos ? s.pos[(long long)b * s.S + t] : t;
    return (s.pos || s.R > 0) && (unsigned)p >= (unsigned)s.P ? -1 : p;
}

// What value e of a row turns with: its partner, cosine and sine (signed so that the forward
// is y[e] c + y[partner] s).  Values past R turn with nothing.
__device__ inline int turn(const Shape& s, const float* __restrict__ row, int e, float& c, float& sn) {
    c = 1.f, sn = 0.f;
    if (e >= s.R) return e;
    const int half = s.R >> 1;
    const int i = s.pairs ? e >> 1 : e < half ? e : e - half;
    const bool second = s.pairs ? e & 1 : e >= half;
    c = row[i];
    sn = second ? row[half + i] : -row[half + i];
    if (s.pairs) return e ^ 1;
    return second ? e - half : e + half;
}

// A wave per row, 64 values at a time: any D, strides and alignment.
template <typename T, int J>
__global__ void __launch_bounds__(256) qk_fwd(Shape s, Rows<const T> q, Rows<const T> k,
                                              const float* __restrict__ gq, const float* __restrict__ gk,
                                              Rows<T> qo, Rows<T> ko) {
    const int lane = threadIdx.x & 63, heads = s.H[0] + s.H[1];
    const long long rows = (long long)s.B * s.S * heads, waves = (long long)gridDim.x * 4;
    for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += waves) {
        const long long n = r / heads;
        int h = (int)(r - n * heads);
        const int b = (int)(n / s.S), t = (int)(n - (long long)b * s.S);
        const bool key = h >= s.H[0];
        if (key) h -= s.H[0];
        const T* x = key ? k.at(b, t, h) : q.at(b, t, h);
        T* o = key ? ko.at(b, t, h) : qo.at(b, t, h);
        const float* g = key ? gk : gq;
        const int p = position(s, b, t);
        if (p < 0) {
            for (int e = lane; e < s.D; e += 64) o[e] = down<T>(0.f);
            continue;
        }
        const float* row = s.table + (long long)p * s.R;
        float v[J], sum = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int e = 64 * j + lane;
            v[j] = e < s.D ? up(x[e]) : 0.f;
            sum += v[j] * v[j];
        }
        const float inv = 1.f / sqrtf(wave_reduce(sum, OpSum()) / s.D + s.eps);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int e = 64 * j + lane;
            if (e >= s.D) continue;
            float c, sn;
            const int other = turn(s, row, e, c, sn);
            const float y = v[j] * inv * (g ? g[e] : 1.f);
            v[j] = other == e ? y : y * c + up(x[other]) * inv * (g ? g[other] : 1.f) * sn;
        }
        wave_fence();   // o may be x
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (64 * j + lane < s.D) o[64 * j + lane] = down<T>(v[j]);
    }
}

// The gradient: work-groups [0, gridq) take rows of queries, the others of keys; each leaves its sum
// of dg in part (one row of D a work-group).
template <typename T, typename GT, typename OT, int J>
__global__ void __launch_bounds__(256) qk_bwd(Shape s, int gridq, Rows<const T> q, Rows<const T> k,
                                              const float* __restrict__ gq, const float* __restrict__ gk,
                                              Rows<const GT> dqo, Rows<const GT> dko, Rows<OT> dq,
                                              Rows<OT> dk, float* __restrict__ part) {
    __shared__ float red[3][64 * J];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const bool key = (int)blockIdx.x >= gridq;
    const int H = s.H[key], group = key ? blockIdx.x - gridq : blockIdx.x;
    const long long rows = (long long)s.B * s.S * H, waves = 4LL * (key ? gridDim.x - gridq : gridq);
    const float* g = key ? gk : gq;
    float acc[J] = {};
    for (long long r = 4LL * group + w; r < rows; r += waves) {
        const long long n = r / H;
        const int h = (int)(r - n * H);
        const int b = (int)(n / s.S), t = (int)(n - (long long)b * s.S);
        const T* x = key ? k.at(b, t, h) : q.at(b, t, h);
        const GT* d = key ? dko.at(b, t, h) : dqo.at(b, t, h);
        OT* o = key ? dk.at(b, t, h) : dq.at(b, t, h);
        const int p = position(s, b, t);
        if (p < 0) {
            for (int e = lane; e < s.D; e += 64) o[e] = down<OT>(0.f);
            continue;
        }
        const float* row = s.table + (long long)p * s.R;
        float v[J], dy[J], sum = 0.f, dot = 0.f;
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int e = 64 * j + lane;
            v[j] = e < s.D ? up(x[e]) : 0.f;
            dy[j] = 0.f;
            if (e < s.D) {
                float c, sn;
                const int other = turn(s, row, e, c, sn);
                dy[j] = up(d[e]);
                if (other != e) dy[j] = dy[j] * c - up(d[other]) * sn;
            }
            sum += v[j] * v[j];
        }
        const float inv = 1.f / sqrtf(wave_reduce(sum, OpSum()) / s.D + s.eps);
#pragma unroll
        for (int j = 0; j < J; ++j) {
            const int e = 64 * j + lane;
            v[j] *= inv;
            acc[j] += dy[j] * v[j];
            dy[j] *= g && e < s.D ? g[e] : 1.f;
            dot += dy[j] * v[j];
        }
        const float mean = wave_reduce(dot, OpSum()) / s.D;
        wave_fence();   // o may be x or d
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (64 * j + lane < s.D) o[64 * j + lane] = down<OT>(inv * (dy[j] - v[j] * mean));
    }
    if (w > 0)
#pragma unroll
        for (int j = 0; j < J; ++j) red[w - 1][64 * j + lane] = acc[j];
    __syncthreads();
    if (w > 0) return;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int e = 64 * j + lane;
        for (int i = 0; i < 3; ++i) acc[j] += red[i][e];
        if (e < s.D) part[(long long)blockIdx.x * s.D + e] = acc[j];
    }
}

// ---- rows in pieces ------------------------------------------------------------------------------
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

struct Units {
    int heads, per;   // heads of a unit, units of a token
    long long n;
};

template <typename T, int V, int L>
__global__ void __launch_bounds__(256) qk_fwd_pieces(Shape s, Units u, Rows<const T> q, Rows<const T> k,
                                                     const float* __restrict__ gq, const float* __restrict__ gk,
                                                     Rows<T> qo, Rows<T> ko) {
    constexpr int G = 64 / L, AHEAD = 4;
    const int lane = threadIdx.x & 63, piece = lane & (L - 1), sub = lane / L;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), heads = s.H[0] + s.H[1];
    const bool in = piece * V < s.D;
    float wq[V], wk[V];
#pragma unroll
    for (int e = 0; e < V; ++e) {
        wq[e] = gq && in ? gq[piece * V + e] : 1.f;
        wk[e] = gk && in ? gk[piece * V + e] : 1.f;
    }
    Turn<V> turn;
    turn.find(s, piece);
    for (long long i = 4LL * blockIdx.x + wave; i < u.n; i += 4LL * gridDim.x) {
        const long long n = i / u.per;
        const int h0 = (int)(i - n * u.per) * u.heads, h1 = min(h0 + u.heads, heads);
        const int b = (int)(n / s.S), t = (int)(n - (long long)b * s.S);
        const int p = position(s, b, t);
        turn.load(s, s.table + (long long)max(p, 0) * s.R, piece);
        for (int h = h0 + sub; h - sub < h1; h += AHEAD * G) {
            float x[AHEAD][V];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int hh = h + a * G;
                const bool key = hh >= s.H[0];
#pragma unroll
                for (int e = 0; e < V; ++e) x[a][e] = 0.f;
                if (hh < h1 && in)
                    load_piece<T, V>((key ? k.at(b, t, hh - s.H[0]) : q.at(b, t, hh)) + piece * V, x[a]);
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int hh = h + a * G;
                const bool key = hh >= s.H[0];
                if (hh - sub >= h1) break;
                float sum = 0.f;
#pragma unroll
                for (int e = 0; e < V; ++e) sum += x[a][e] * x[a][e];
                const float inv = 1.f / sqrtf(group_sum<L>(sum) / s.D + s.eps);
#pragma unroll
                for (int e = 0; e < V; ++e) x[a][e] *= inv * (key ? wk[e] : wq[e]);
                turn.apply(s, x[a], 1.f);
                if (p < 0)
#pragma unroll
                    for (int e = 0; e < V; ++e) x[a][e] = 0.f;
                if (hh < h1 && in)
                    store_piece<T, V>((key ? ko.at(b, t, hh - s.H[0]) : qo.at(b, t, hh)) + piece * V, x[a]);
            }
        }
    }
}

// The gradient: a work-group leaves its sums of dgq and dgk in rows blockIdx.x and gridDim.x + blockIdx.x of part.
template <typename T, typename GT, typename OT, int V, int L>
__global__ void __launch_bounds__(256) qk_bwd_pieces(Shape s, Units u, Rows<const T> q, Rows<const T> k,
                                                     const float* __restrict__ gq, const float* __restrict__ gk,
                                                     Rows<const GT> dqo, Rows<const GT> dko, Rows<OT> dq, Rows<OT> dk,
                                                     float* __restrict__ part) {
    constexpr int G = 64 / L, AHEAD = 2;
    __shared__ float red[4 * G][2][L * V];
    const int lane = threadIdx.x & 63, piece = lane & (L - 1), sub = lane / L;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), heads = s.H[0] + s.H[1];
    const bool in = piece * V < s.D;
    float wq[V], wk[V], aq[V] = {}, ak[V] = {};
#pragma unroll
    for (int e = 0; e < V; ++e) {
        wq[e] = gq && in ? gq[piece * V + e] : 1.f;
        wk[e] = gk && in ? gk[piece * V + e] : 1.f;
    }
    Turn<V> turn;
    turn.find(s, piece);
    for (long long i = 4LL * blockIdx.x + wave; i < u.n; i += 4LL * gridDim.x) {
        const long long n = i / u.per;
        const int h0 = (int)(i - n * u.per) * u.heads, h1 = min(h0 + u.heads, heads);
        const int b = (int)(n / s.S), t = (int)(n - (long long)b * s.S);
        const int p = position(s, b, t);
        turn.load(s, s.table + (long long)max(p, 0) * s.R, piece);
        for (int h = h0 + sub; h - sub < h1; h += AHEAD * G) {
            float x[AHEAD][V], d[AHEAD][V];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int hh = h + a * G;
                const bool key = hh >= s.H[0];
#pragma unroll
                for (int e = 0; e < V; ++e) x[a][e] = d[a][e] = 0.f;
                if (hh < h1 && in && p >= 0) {
                    load_piece<T, V>((key ? k.at(b, t, hh - s.H[0]) : q.at(b, t, hh)) + piece * V, x[a]);
                    load_piece<GT, V>((key ? dko.at(b, t, hh - s.H[0]) : dqo.at(b, t, hh)) + piece * V, d[a]);
                }
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int hh = h + a * G;
                const bool key = hh >= s.H[0];
                if (hh - sub >= h1) break;
                float sum = 0.f, dot = 0.f;
#pragma unroll
                for (int e = 0; e < V; ++e) sum += x[a][e] * x[a][e];
                const float inv = 1.f / sqrtf(group_sum<L>(sum) / s.D + s.eps);
                turn.apply(s, d[a], -1.f);
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    x[a][e] *= inv;
                    const float w = d[a][e] * x[a][e];
                    aq[e] += key ? 0.f : w;
                    ak[e] += key ? w : 0.f;
                    d[a][e] *= key ? wk[e] : wq[e];
                    dot += d[a][e] * x[a][e];
                }
                const float mean = group_sum<L>(dot) / s.D;
#pragma unroll
                for (int e = 0; e < V; ++e) d[a][e] = inv * (d[a][e] - x[a][e] * mean);
                if (hh < h1 && in)
                    store_piece<OT, V>((key ? dk.at(b, t, hh - s.H[0]) : dq.at(b, t, hh)) + piece * V, d[a]);
            }
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

// dg (+)= the sum of its partials: 16 waves take every 16th, in order.
__global__ void __launch_bounds__(1024) qk_join(const float* __restrict__ part, int D, int gridq, int grid,
                                                float* __restrict__ dgq, float* __restrict__ dgk, int acc) {
    __shared__ float red[16][64];
    const bool key = blockIdx.y;
    float* out = key ? dgk : dgq;
    if (!out) return;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, e = blockIdx.x * 64 + lane;
    float sum = 0.f;
    if (e < D) {
        const int end = key ? grid : gridq;
#pragma unroll 8
        for (int i = (key ? gridq : 0) + w; i < end; i += 16) sum += part[(long long)i * D + e];
    }
    red[w][lane] = sum;
    __syncthreads();
    if (w > 0 || e >= D) return;
    sum = 0.f;
#pragma unroll
    for (int i = 0; i < 16; ++i) sum += red[i][lane];
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
    if (!(eps > 0.f) || !(eps - eps == 0.f)) return set_error(DH_ERR_INVALID, "%s: eps must be finite and > 0", op);
    if ((R > 0 && !table) || ((R > 0 || pos) && P < 1) || (R > 0 && !pos && S > P))
        return set_error(DH_ERR_INVALID, "%s: no table of %d positions (P=%d)", op, pos ? 1 : S, P);
    s = Shape{B, S, {Hq, Hk}, D, R, P, pairs != 0, eps, pos, (const float*)table};
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
// Heads of a unit: all of a token's where that gives each of the GPU's 8192 waves a unit, else as few as
// the wave takes at once.
Units units_of(const Shape& s, int at_once) {
    const long long n = (long long)s.B * s.S;
    const int heads = s.H[0] + s.H[1];
    int per = (heads + at_once - 1) / at_once;
    int each = (int)(n >= 8192 ? per : (n * per + 8191) / 8192);
    if (each < 1) each = 1;
    const int unit = each * at_once;
    per = (heads + unit - 1) / unit;
    return Units{unit, per, n * per};
}

template <typename T, int V, int L>
int launch_fwd_pieces(const Shape& s, const void* Q, const long long* sq, const void* K, const long long* sk,
                      const float* gq, const float* gk, void* Qo, const long long* sqo, void* Ko,
                      const long long* sko) {
    const Units u = units_of(s, 64 / L);
    const long long groups = (u.n + 3) / 4, most = 1 << 20;
    qk_fwd_pieces<T, V, L><<<(unsigned)(groups < most ? groups : most), 256, 0, stream()>>>(
        s, u, rows_of<const T>(Q, sq), rows_of<const T>(K, sk), gq, gk, rows_of<T>(Qo, sqo), rows_of<T>(Ko, sko));
    return check_launch("dh_qk_norm_rope_fwd");
}

template <typename T, int J>
int launch_fwd(const Shape& s, const void* Q, const long long* sq, const void* K, const long long* sk, const float* gq,
               const float* gk, void* Qo, const long long* sqo, void* Ko, const long long* sko) {
    const long long rows = (long long)s.B * s.S * (s.H[0] + s.H[1]), most = num_cus() * 32LL;
    const long long groups = (rows + 3) / 4;
    qk_fwd<T, J><<<(unsigned)(groups < most ? groups : most), 256, 0, stream()>>>(
        s, rows_of<const T>(Q, sq), rows_of<const T>(K, sk), gq, gk, rows_of<T>(Qo, sqo), rows_of<T>(Ko, sko));
    return check_launch("dh_qk_norm_rope_fwd");
}

// Work-groups of the gradient for queries and keys: enough to fill the GPU, few enough that their
// partials are a small part of the work.
constexpr int QK_GROUPS = 2048;
void bwd_groups(const Shape& s, int& gridq, int& gridk) {
    const long long n = (long long)s.B * s.S;
    auto groups = [&](int H) {
        const long long g = (n * H + 3) / 4, most = (long long)QK_GROUPS * H / (s.H[0] + s.H[1]) + 1;
        return (int)(g < most ? g : most);
    };
    gridq = s.H[0] ? groups(s.H[0]) : 0;
    gridk = s.H[1] ? groups(s.H[1]) : 0;
}

template <typename T, typename GT, typename OT, int V, int L>
int launch_bwd_pieces(const Shape& s, const void* Q, const long long* sq, const void* K, const long long* sk,
                      const float* gq, const float* gk, const void* dQo, const long long* sdqo, const void* dKo,
                      const long long* sdko, void* dQ, const long long* sdq, void* dK, const long long* sdk,
                      float* dgq, float* dgk, int acc, float* part) {
    const Units u = units_of(s, 64 / L);
    const long long groups = (u.n + 3) / 4, most = QK_GROUPS / 2;
    const int grid = (int)(groups < most ? groups : most);
    qk_bwd_pieces<T, GT, OT, V, L><<<grid, 256, 0, stream()>>>(
        s, u, rows_of<const T>(Q, sq), rows_of<const T>(K, sk), gq, gk, rows_of<const GT>(dQo, sdqo),
        rows_of<const GT>(dKo, sdko), rows_of<OT>(dQ, sdq), rows_of<OT>(dK, sdk), part);
    DH_TRY(check_launch("dh_qk_norm_rope_bwd"));
    if (!dgq && !dgk) return DH_OK;
    qk_join<<<dim3((s.D + 63) / 64, 2), 1024, 0, stream()>>>(part, s.D, grid, 2 * grid, dgq, dgk, acc);
    return check_launch("dh_qk_norm_rope_bwd");
}

template <typename T, typename GT, typename OT, int J>
int launch_bwd(const Shape& s, const void* Q, const long long* sq, const void* K, const long long* sk, const float* gq,
               const float* gk, const void* dQo, const long long* sdqo, const void* dKo, const long long* sdko,
               void* dQ, const long long* sdq, void* dK, const long long* sdk, float* dgq, float* dgk, int acc,
               float* part) {
    int gridq, gridk;
    bwd_groups(s, gridq, gridk);
    qk_bwd<T, GT, OT, J><<<gridq + gridk, 256, 0, stream()>>>(
        s, gridq, rows_of<const T>(Q, sq), rows_of<const T>(K, sk), gq, gk, rows_of<const GT>(dQo, sdqo),
        rows_of<const GT>(dKo, sdko), rows_of<OT>(dQ, sdq), rows_of<OT>(dK, sdk), part);
    DH_TRY(check_launch("dh_qk_norm_rope_bwd"));
    if (!dgq && !dgk) return DH_OK;
    qk_join<<<dim3((s.D + 63) / 64, 2), 1024, 0, stream()>>>(part, s.D, gridq, gridq + gridk, dgq, dgk, acc);
    return check_launch("dh_qk_norm_rope_bwd");
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
    const bool small = D <= 256;
    const int size = dtype == DH_F32 ? 4 : 2;
    Piece p(s, size);
    p.rows(Hq, Q, sq, size), p.rows(Hk, K, sk, size), p.rows(Hq, Qo, sqo, size), p.rows(Hk, Ko, sko, size);
    if (p.V > 1) {
        const int L = p.lanes();
#define DH_QK(T, V)                                                                                \
    (L == 4 ? launch_fwd_pieces<T, V, 4> : L == 8 ? launch_fwd_pieces<T, V, 8> : L == 16 ? launch_fwd_pieces<T, V, 16>                   \
     : L == 32 ? launch_fwd_pieces<T, V, 32> : launch_fwd_pieces<T, V, 64>)
        auto pieces = dtype == DH_F32 ? DH_QK(float, 4) : p.V == 8 ? DH_QK(uint16_t, 8) : DH_QK(uint16_t, 4);
#undef DH_QK
        return pieces(s, Q, sq, K, sk, gq, gk, Qo, sqo, Ko, sko);
    }
    auto run = dtype == DH_F32 ? small ? launch_fwd<float, 4> : launch_fwd<float, 16>
                               : small ? launch_fwd<uint16_t, 4> : launch_fwd<uint16_t, 16>;
    return run(s, Q, sq, K, sk, gq, gk, Qo, sqo, Ko, sko);
}

size_t dh_qk_norm_rope_bwd_workspace(int D) {
    return D < 1 || D > QK_MOST_D ? 0 : (size_t)(QK_GROUPS + 2) * D * 4;
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
        qk_join<<<dim3((D + 63) / 64, 2), 1024, 0, stream()>>>((float*)ws, D, 0, 0, dgq, dgk, 0);
        return check_launch(op);
    }
    const bool small = D <= 256;
    const bool gw = dout_type == DH_F32, ow = grad_type == DH_F32;
    const int size = dtype == DH_F32 ? 4 : 2, gsize = gw ? 4 : 2, osize = ow ? 4 : 2;
    Piece p(s, size);
    p.rows(Hq, Q, sq, size), p.rows(Hk, K, sk, size), p.rows(Hq, dQo, sdqo, gsize), p.rows(Hk, dKo, sdko, gsize);
    p.rows(Hq, dQ, sdq, osize), p.rows(Hk, dK, sdk, osize);
    if (p.V > 1) {
        const int L = p.lanes();
#define DH_QL(T, GT, OT, V)                                                                                \
    (L == 4 ? launch_bwd_pieces<T, GT, OT, V, 4> : L == 8 ? launch_bwd_pieces<T, GT, OT, V, 8> : L == 16 ? launch_bwd_pieces<T, GT, OT, V, 16>           \
     : L == 32 ? launch_bwd_pieces<T, GT, OT, V, 32> : launch_bwd_pieces<T, GT, OT, V, 64>)
#define DH_QK(GT, OT) (p.V == 8 ? DH_QL(uint16_t, GT, OT, 8) : DH_QL(uint16_t, GT, OT, 4))
        auto pieces = dtype == DH_F32 ? DH_QL(float, float, float, 4)
                      : gw ? ow ? DH_QK(float, float) : DH_QK(float, uint16_t)
                           : ow ? DH_QK(uint16_t, float) : DH_QK(uint16_t, uint16_t);
#undef DH_QK
#undef DH_QL
        return pieces(s, Q, sq, K, sk, gq, gk, dQo, sdqo, dKo, sdko, dQ, sdq, dK, sdk, dgq, dgk, accumulate,
                      (float*)ws);
    }
#define DH_QK(T, GT, OT) (small ? launch_bwd<T, GT, OT, 4> : launch_bwd<T, GT, OT, 16>)
    auto run = dtype == DH_F32 ? DH_QK(float, float, float)
               : gw ? ow ? DH_QK(uint16_t, float, float) : DH_QK(uint16_t, float, uint16_t)
                    : ow ? DH_QK(uint16_t, uint16_t, float) : DH_QK(uint16_t, uint16_t, uint16_t);
#undef DH_QK
    return run(s, Q, sq, K, sk, gq, gk, dQo, sdqo, dKo, sdko, dQ, sdq, dK, sdk, dgq, dgk, accumulate, (float*)ws);
}

}  // extern "C"
