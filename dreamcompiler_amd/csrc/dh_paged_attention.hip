// dh_paged_attention.hip -- attention of one new token of each sequence over a paged cache.
//
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t - m),  lse = m + log sum_t p_t
//
// over the tokens t of the sequence (its last `window` ones).  One pass over keys and values with the
// running maximum m and sum; a sequence's tokens are split into chunks, whose o, m and sum meet in a
// second launch.  Bound by HBM: each key and value is read once.
#include "dh_paged.hpp"

namespace dh {
namespace {

template <typename T> __device__ inline T down(float x);
template <> __device__ inline float down<float>(float x) { return x; }
template <> __device__ inline uint16_t down<uint16_t>(float x) {
    return __builtin_bit_cast(uint16_t, (__bf16)x);
}

struct Strides {
    long long seq, head;
};
struct Work {
    int B, Hq, G, groups, window, max_len, chunk, splits;
    float scale;
    const int* len;
    float* part;    // splits x B x Hq rows of D: a chunk's o before its division
    float2* stat;   // as many: its m (in units of log 2) and sum
    // The tokens that count, and where the first chunk begins: chunks begin with whole tiles.
    __device__ void span(int b, int& from, int& to, int& start) const {
        to = min(max(len[b], 0), max_len);
        from = window > 0 ? max(to - window, 0) : 0;
        start = from & ~31;
    }
    __device__ int chunks(int to, int start) const { return to > start ? (to - start + chunk - 1) / chunk : 0; }
};

constexpr float LOG2E = 1.44269504088896340736f, LN2 = 0.69314718055994530942f;

typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));

__device__ inline uint32_t pk_bf16(float a, float b) {
    return __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{a, b}, bf16x2));
}
__device__ inline f32x4 mfma(u32x4 a, u32x4 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0, 0,
                                                   0);
}
__device__ inline f32x4 mfma(float a, float b, f32x4 c) { return __builtin_amdgcn_mfma_f32_16x16x4f32(a, b, c, 0, 0, 0); }

// Four 8-bit values of a word as bf16 (exact: seven bits of an integer, four of an e4m3 float).
template <typename CT> __device__ inline u32x2 words_bf16(uint32_t w);
template <> __device__ inline u32x2 words_bf16<int8_t>(uint32_t w) {
    return u32x2{pk_bf16((float)(int8_t)w, (float)(int8_t)(w >> 8)),
                 pk_bf16((float)(int8_t)(w >> 16), (float)(int8_t)(w >> 24))};
}
template <> __device__ inline u32x2 words_bf16<uint8_t>(uint32_t w) {
    return u32x2{__builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, false)),
                 __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(w, 1.f, true))};
}

// N words at any element's alignment.
template <int N> struct Words;
template <> struct Words<1> { typedef uint32_t type; };
template <> struct Words<2> { typedef u32x2 type; };
template <> struct Words<4> { typedef u32x4 type; };

// x (8 values) in P parts of bf16 that add up to it: 8 bits each.
template <int P>
__device__ inline void split8(const float (&x)[8], u32x4 (&out)[P]) {
    float r[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) r[e] = x[e];
#pragma unroll
    for (int q = 0; q < P; ++q)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint32_t w = pk_bf16(r[2 * e], r[2 * e + 1]);
            out[q][e] = w;
            if (q + 1 < P) {
                r[2 * e] -= __builtin_bit_cast(float, w << 16);
                r[2 * e + 1] -= __builtin_bit_cast(float, w & 0xFFFF0000u);
            }
        }
}

// ---- a chunk -----------------------------------------------------------------------------------
// A work-group of 4 waves takes a chunk of a sequence's tokens for 16 RT query heads of one cache head;
// its waves take every fourth tile of TILE tokens, each with its own maximum, sum and o, which
// meet in LDS.  Keys and values go from memory into registers, with no LDS between, as both products
// take them as they lie:
//   scores  keys x queries: lane l holds 16 bytes of key l % 16 (an A operand; the order of d inside a
//           product is free, and the query has the same).  The result leaves lane l with head l % 16
//           and tokens 4 (l / 16) + r of each 16
//   o       values^T x weights: those tokens are the weights' k in that lane, as they are.  Lane l
//           loads the values of the same tokens at columns W (l % 16) .. + W - 1, so that a row is one
//           piece of memory for 16 lanes; column j of each is row l % 16 of the j-th product, 16-bit
//           pairs of two tokens put together by a permutation of bytes
// so statistics, weights and o of a head stay in its lanes.  8-bit values are widened to bf16, exactly;
// their scales go into the scores and the weights.
//
// Precision: fp32 caches take the fp32 matrix instructions.  Else a fp32 query is three parts of bf16 (24
// bits) and a weight two (16 bits; a bf16 result has 8) or, where the model is fp32, three.
template <typename T, typename CT, int DP>
struct Form {
    static constexpr bool wide = sizeof(CT) == 4, narrow = sizeof(CT) == 1;
    static constexpr int SUBS = wide ? 1 : 2, TILE = 16 * SUBS;   // 16 tokens each
    static constexpr int E = 16 / sizeof(CT);                     // values of 16 bytes
    static constexpr int KSTEPS = DP / (4 * E);                   // 16-byte pieces of a lane's part of a key
    static constexpr int QP = wide ? 1 : sizeof(T) == 4 ? 3 : 1, PP = sizeof(T) == 4 ? 3 : 2;
    // Columns of a lane: W = 8 in 128 of them or 4 in 64.
    static constexpr int W0 = wide || DP % 128 ? 4 : 8;
    static constexpr int SEGS = wide ? DP / 64 : (DP + 64) / 128;
    static constexpr int width(int seg) { return wide || 128 * seg + 64 == DP ? 4 : 8; }
    static constexpr int column(int seg) { return (wide ? 64 : 128) * seg; }
};

template <typename T, typename CT, int DP, bool FULL, int RT>
__global__ void __launch_bounds__(256) paged_chunk(Paged c, Work w, const T* __restrict__ Q, Strides sq,
                                                   T* __restrict__ O, Strides so, float* __restrict__ lse) {
    typedef Form<T, CT, DP> F;
    constexpr int SUBS = F::SUBS, KSTEPS = F::KSTEPS, E = F::E, LD = DP + 4;
    constexpr bool wide = F::wide, narrow = F::narrow;
    __shared__ float ol[4][16][LD];
    __shared__ float2 ml[4][16 * RT];
    const int D = FULL ? DP : c.D;
    const int lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int split = blockIdx.x, b = blockIdx.z;
    const int hk = blockIdx.y / w.groups, first = (blockIdx.y - hk * w.groups) * 16 * RT;   // head of the group
    int from, to, start;
    w.span(b, from, to, start);
    const int n_chunks = w.chunks(to, start);
    if (split >= max(n_chunks, 1)) return;
    const int c0 = start + split * w.chunk, c1 = min(c0 + w.chunk, to);

    // The chunk's pages, one a lane (at most 1024 tokens of at least 16 a page).
    const int page0 = c0 >> c.shift;
    int ids = -1;
    if (c0 < c1 && page0 + lane <= (c1 - 1) >> c.shift) ids = c.page_of(b, (page0 + lane) << c.shift);

    // Queries: the values of d that the lane has of a key.
    u32x4 qf[RT][F::QP][wide ? 1 : DP / 32];
    float qw[RT][wide ? DP / 4 : 1];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const int h = first + 16 * rt + l;
        const T* q = Q + b * sq.seq + (long long)(hk * w.G + min(h, w.G - 1)) * sq.head;
        constexpr int N = wide ? 4 : 8;
#pragma unroll
        for (int i = 0; i < DP / (4 * N); ++i) {
            // piece of N values: of 16-byte piece i (fp32, bf16), or a half of piece i / 2
            const int d = narrow ? 16 * (4 * (i / 2) + g) + 8 * (i % 2) : N * (4 * i + g);
            float x[N] = {};
            if (h < w.G && d < D) {
                typedef T vec __attribute__((ext_vector_type(N), aligned(sizeof(T))));
                const vec v = *reinterpret_cast<const vec*>(q + d);
#pragma unroll
                for (int e = 0; e < N; ++e) x[e] = paged_up(v[e]);
            }
            if constexpr (wide) {
#pragma unroll
                for (int e = 0; e < N; ++e) qw[rt][N * i + e] = x[e];
            } else {
                u32x4 parts[F::QP];
                split8<F::QP>(x, parts);
#pragma unroll
                for (int p = 0; p < F::QP; ++p) qf[rt][p][i] = parts[p];
            }
        }
    }

    f32x4 o[RT][DP / 16];
    float m[RT], sum[RT];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        m[rt] = -INFINITY, sum[rt] = 0.f;
#pragma unroll
        for (int j = 0; j < DP / 16; ++j) o[rt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    }
    const float unit = w.scale * LOG2E;
    const int row_bytes = D * (int)sizeof(CT);
    // In bytes from the first token of 16: the lane's part of a key, and of values in each segment.
    const uint32_t k_off = l * row_bytes + 16 * g;
    uint32_t v_off[F::SEGS];
#pragma unroll
    for (int s = 0; s < F::SEGS; ++s) {
        const int col = F::column(s) + F::width(s) * l;
        v_off[s] = 4 * g * row_bytes + (FULL || col < D ? col : 0) * (int)sizeof(CT);
    }

    for (int base = c0 + F::TILE * wave; base < c1; base += 4 * F::TILE) {
        u32x4 kr[SUBS][KSTEPS];
        uint32_t vr[SUBS][4][DP / 16 * sizeof(CT) / 4];
        f32x4 ks[SUBS], vs[SUBS];
        bool there[SUBS], whole = base >= from && base + F::TILE <= to;
#pragma unroll
        for (int s = 0; s < SUBS; ++s) {
            const int t = base + 16 * s;
            int id = -1;
            if (t < c1) id = __builtin_amdgcn_readlane(ids, (t >> c.shift) - page0);
            there[s] = id >= 0;
            whole = whole && there[s];
            const long long row = there[s] ? c.row(id, hk, t & ((1 << c.shift) - 1)) : 0;
            const char* kp = (const char*)c.K + row * row_bytes;
            const char* vp = (const char*)c.V + row * row_bytes;
#pragma unroll
            for (int i = 0; i < KSTEPS; ++i) {
                uint32_t at = k_off + 64 * i;
                if (!FULL && E * (4 * i + g) >= D) at = l * row_bytes;
                kr[s][i] = *reinterpret_cast<const u32x4*>(kp + at);
            }
            if constexpr (narrow) {
                ks[s] = *reinterpret_cast<const f32x4*>(c.Ks + row + 4 * g);
                vs[s] = *reinterpret_cast<const f32x4*>(c.Vs + row + 4 * g);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                int at = 0;
#pragma unroll
                for (int sg = 0; sg < F::SEGS; ++sg) {
                    constexpr int bytes = sizeof(CT);
                    const char* p = vp + (v_off[sg] + i * row_bytes);
                    if (F::width(sg) * bytes == 16) {
                        const u32x4 x = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
                        for (int e = 0; e < 4; ++e) vr[s][i][at + e] = x[e];
                        at += 4;
                    } else if (F::width(sg) * bytes == 8) {
                        const u32x2 x = *reinterpret_cast<const u32x2*>(p);
                        vr[s][i][at] = x[0], vr[s][i][at + 1] = x[1];
                        at += 2;
                    } else {
                        vr[s][i][at++] = *reinterpret_cast<const uint32_t*>(p);
                    }
                }
            }
        }

        // Scores, in units of log 2.
        float z[RT][SUBS][4];
#pragma unroll
        for (int s = 0; s < SUBS; ++s) {
            f32x4 acc[RT];
#pragma unroll
            for (int rt = 0; rt < RT; ++rt) acc[rt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int i = 0; i < KSTEPS; ++i) {
                u32x4 x = kr[s][i];
                if (!FULL && E * (4 * i + g) >= D) x = u32x4{0, 0, 0, 0};
                if constexpr (wide) {
#pragma unroll
                    for (int e = 0; e < 4; ++e)
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
                            acc[rt] = mfma(__builtin_bit_cast(float, (uint32_t)x[e]), qw[rt][4 * i + e], acc[rt]);
                } else if constexpr (narrow) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const u32x2 a = words_bf16<CT>(x[2 * half]), bb = words_bf16<CT>(x[2 * half + 1]);
                        const u32x4 k = {a[0], a[1], bb[0], bb[1]};
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                            for (int p = 0; p < F::QP; ++p) acc[rt] = mfma(k, qf[rt][p][2 * i + half], acc[rt]);
                    }
                } else {
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) acc[rt] = mfma(x, qf[rt][0][i], acc[rt]);
                }
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float f = unit;
                    if constexpr (narrow) f *= ks[s][r];
                    z[rt][s][r] = acc[rt][r] * f;
                }
        }
        if (!whole) {   // tokens that do not count: no score, no value, whatever lies there
#pragma unroll
            for (int s = 0; s < SUBS; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int t = base + 16 * s + 4 * g + r;
                    const bool in = there[s] && t >= from && t < to;
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) z[rt][s][r] = in ? z[rt][s][r] : -INFINITY;
#pragma unroll
                    for (int e = 0; e < (int)(DP / 16 * sizeof(CT) / 4); ++e) vr[s][r][e] = in ? vr[s][r][e] : 0;
                    if constexpr (narrow) vs[s][r] = in ? vs[s][r] : 0.f;
                }
        }

        // Weights.  The maximum only moves where it would by more than 2^8, which a weight may then be.
        u32x4 pf[RT][wide ? 1 : F::PP];
        float pw[RT][4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt) {
            float top = -INFINITY, lo, hi;
#pragma unroll
            for (int s = 0; s < SUBS; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) top = fmaxf(top, z[rt][s][r]);
            halves16(top, lo, hi);
            top = fmaxf(lo, hi);
            halves32(top, lo, hi);
            top = fmaxf(lo, hi);
            if (__any(top > m[rt] + 8.f)) {
                const float next = fmaxf(m[rt], top);
                const float f = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m[rt] - next);
                m[rt] = next;
                sum[rt] *= f;
#pragma unroll
                for (int j = 0; j < DP / 16; ++j) o[rt][j] *= f;
            }
            const float off = m[rt] == -INFINITY ? 0.f : m[rt];
            float p[8];
#pragma unroll
            for (int s = 0; s < SUBS; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = __builtin_amdgcn_exp2f(z[rt][s][r] - off);
                    sum[rt] += x;
                    if constexpr (narrow) x *= vs[s][r];
                    p[4 * s + r] = x;
                }
            if constexpr (wide) {
#pragma unroll
                for (int r = 0; r < 4; ++r) pw[rt][r] = p[r];
            } else {
                split8<F::PP>(p, pf[rt]);
            }
        }

        // o += weights x values
        if constexpr (wide) {
#pragma unroll
            for (int j = 0; j < DP / 16; ++j)
#pragma unroll
                for (int r = 0; r < 4; ++r)
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
                        o[rt][j] = mfma(__builtin_bit_cast(float, vr[0][r][j]), pw[rt][r], o[rt][j]);
        } else {
#pragma unroll
            for (int jj = 0; jj < DP / 32; ++jj) {   // two columns: a word of bf16
                uint32_t x[8];
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    if constexpr (narrow) x[i] = words_bf16<CT>(vr[i / 4][i % 4][jj / 2])[jj % 2];
                    else x[i] = vr[i / 4][i % 4][jj];
                }
#pragma unroll
                for (int odd = 0; odd < 2; ++odd) {
                    u32x4 a;
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        a[i] = odd ? pack_hi16(x[2 * i], x[2 * i + 1]) : pack_lo16(x[2 * i], x[2 * i + 1]);
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                        for (int p = 0; p < F::PP; ++p)
                            o[rt][2 * jj + odd] = mfma(a, pf[rt][p], o[rt][2 * jj + odd]);
                }
            }
        }
    }

    // The waves' sums meet: o[..][j][r] is column W (4 g + r) + j of its segment.
    const bool last = n_chunks <= 1;
    const long long heads = (long long)w.B * w.Hq;
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        float s = sum[rt], lo, hi;
        halves16(s, lo, hi);
        s = lo + hi;
        halves32(s, lo, hi);
        s = lo + hi;
        if (g == 0) ml[wave][16 * rt + l] = float2{m[rt], s};
        if (rt > 0) __syncthreads();
        int j = 0;
#pragma unroll
        for (int sg = 0; sg < F::SEGS; ++sg) {
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int e = 0; e < F::width(sg); e += 4) {
                    const f32x4 x = {o[rt][j + e][r], o[rt][j + e + 1][r], o[rt][j + e + 2][r], o[rt][j + e + 3][r]};
                    *reinterpret_cast<f32x4*>(&ol[wave][l][F::column(sg) + F::width(sg) * (4 * g + r) + e]) = x;
                }
            j += F::width(sg);
        }
        __syncthreads();
        for (int i = threadIdx.x; i < 16 * DP / 4; i += 256) {
            const int hl = i / (DP / 4), d = 4 * (i % (DP / 4)), h = first + 16 * rt + hl;
            if (h >= w.G || d >= D) continue;
            float top = -INFINITY, total = 0.f;
#pragma unroll
            for (int x = 0; x < 4; ++x) top = fmaxf(top, ml[x][16 * rt + hl].x);
            const float off = top == -INFINITY ? 0.f : top;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const float2 st = ml[x][16 * rt + hl];
                const float f = __builtin_amdgcn_exp2f(st.x - off);
                total += st.y * f;
                v += *reinterpret_cast<const f32x4*>(&ol[x][hl][d]) * f;
            }
            const int hq = hk * w.G + h;
            if (last) {
                const float f = total == 0.f ? 0.f : 1.f / total;
                T* out = O + b * so.seq + (long long)hq * so.head + d;
#pragma unroll
                for (int e = 0; e < 4; ++e) out[e] = down<T>(v[e] * f);
                if (lse && d == 0) lse[(long long)b * w.Hq + hq] = total == 0.f ? -INFINITY : top * LN2 + logf(total);
            } else {
                const long long at = split * heads + (long long)b * w.Hq + hq;
                *reinterpret_cast<f32x4*>(w.part + at * D + d) = v;
                if (d == 0) w.stat[at] = float2{top, total};
            }
        }
    }
}

// ---- the chunks of a sequence -------------------------------------------------------------------
// A work-group per head: its waves take every fourth chunk, in order, and meet in LDS.
template <typename T>
__global__ void __launch_bounds__(256) paged_join(Work w, int D, T* __restrict__ O, Strides so,
                                                  float* __restrict__ lse) {
    __shared__ float red[4][PAGED_MOST_D];
    __shared__ float2 stats[4];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, h = blockIdx.x, b = blockIdx.y;
    int from, to, start;
    w.span(b, from, to, start);
    const int n = w.chunks(to, start);
    if (n <= 1) return;   // its one chunk wrote the result
    const long long step = (long long)w.B * w.Hq, at = (long long)b * w.Hq + h;
    float m = -INFINITY, sum = 0.f;
    for (int i = lane; i < n; i += 64) m = fmaxf(m, w.stat[i * step + at].x);
    m = wave_reduce(m, OpMax());
    const float off = m == -INFINITY ? 0.f : m;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int i = wave; i < n; i += 4) {
        const float2 s = w.stat[i * step + at];
        const float f = __builtin_amdgcn_exp2f(s.x - off);
        sum += s.y * f;
        if (4 * lane < D) o += *reinterpret_cast<const f32x4*>(w.part + (i * step + at) * D + 4 * lane) * f;
    }
    *reinterpret_cast<f32x4*>(&red[wave][4 * lane]) = o;
    if (lane == 0) stats[wave] = float2{m, sum};
    __syncthreads();
    sum = stats[0].y + stats[1].y + stats[2].y + stats[3].y;
    const int d = threadIdx.x;
    if (d < D) {
        const float x = red[0][d] + red[1][d] + red[2][d] + red[3][d];
        O[b * so.seq + h * so.head + d] = down<T>(sum == 0.f ? 0.f : x / sum);
    }
    if (lse && d == 0) lse[at] = sum == 0.f ? -INFINITY : m * LN2 + logf(sum);
}

// ---- host --------------------------------------------------------------------------------------
// Work-groups of all sequences at their longest: several for every place on the GPU, so that what is left
// when the short sequences are done evens out.
constexpr int WORK_GROUPS = 2048;
constexpr int LEAST = 128, MOST = 1024;   // tokens of a chunk: a tile for each wave, a page for each lane

// Tokens of a chunk and the most chunks of a sequence.
void plan(int B, int Hk, int max_len, int window, int& chunk, int& splits) {
    // a window that begins inside a tile sees up to 31 tokens before it
    const long long seen = window > 0 && window < max_len - 31 ? window + 31LL : max_len;
    const long long want = ((long long)B * Hk * seen + WORK_GROUPS - 1) / WORK_GROUPS;
    chunk = (int)(want > MOST ? MOST : want < LEAST ? LEAST : (want + LEAST - 1) / LEAST * LEAST);
    splits = seen > chunk ? (int)((seen + chunk - 1) / chunk) : 1;
}
// At least as many for every window.
long long most_splits(int B, int Hk, int max_len) {
    const long long a = ((long long)max_len + LEAST - 1) / LEAST, b = WORK_GROUPS / ((long long)B * Hk) + 1,
                    c = ((long long)max_len + MOST - 1) / MOST;
    return a < b ? a : b > c ? b : c;
}
size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

template <typename T, typename CT, int DP, bool FULL, int RT>
int launch_form(const Paged& c, Work w, const void* Q, Strides sq, void* O, Strides so, float* lse) {
    w.groups = (w.G + 16 * RT - 1) / (16 * RT);
    paged_chunk<T, CT, DP, FULL, RT><<<dim3(w.splits, c.Hk * w.groups, w.B), 256, 0, stream()>>>(
        c, w, (const T*)Q, sq, (T*)O, so, lse);
    DH_TRY(check_launch("dh_paged_attention"));
    if (w.splits == 1) return DH_OK;
    paged_join<T><<<dim3(w.Hq, w.B), 256, 0, stream()>>>(w, c.D, (T*)O, so, lse);
    return check_launch("dh_paged_attention");
}

template <typename T, typename CT>
int launch(const Paged& c, const Work& w, const void* Q, Strides sq, void* O, Strides so, float* lse) {
    const bool two = w.G > 16;
#define DH_FORM(DP) (c.D == DP ? launch_form<T, CT, DP, true, 1> : launch_form<T, CT, DP, false, 1>)
    auto run = c.D <= 64 ? DH_FORM(64) : c.D <= 128 ? DH_FORM(128) : c.D <= 192 ? DH_FORM(192) : DH_FORM(256);
    if (two && c.D == 64) run = launch_form<T, CT, 64, true, 2>;
    if (two && c.D == 128) run = launch_form<T, CT, 128, true, 2>;
#undef DH_FORM
    return run(c, w, Q, sq, O, so, lse);
}

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" {

size_t dh_paged_attention_workspace(int cache_type, int B, int Hq, int Hk, int D, int max_len) {
    if (B < 1 || Hq < 1 || Hk < 1 || D < 1 || max_len < 1) return 0;
    const long long splits = most_splits(B, Hk, max_len);
    if (splits == 1) return 0;
    const size_t rows = (size_t)splits * B * Hq;
    return up256(rows * D * 4) + rows * 8;
}

int dh_paged_attention(int dtype, int cache_type, int B, int Hq, int Hk, int D, float scale, int window,
                       const void* Q, const long long* sq, const int* len, int max_len, int pages, int page,
                       const int* table, int ld_table, const void* Kc, const void* Vc, const float* Ks,
                       const float* Vs, void* O, const long long* so, float* lse, void* ws, size_t ws_bytes) {
    const char* op = "dh_paged_attention";
    Paged c;
    DH_TRY(check_paged(op, dtype, cache_type, B, Hk, D, pages, page, table, ld_table, Kc, Vc, Ks, Vs, c));
    if (Hq < 1 || Hq > 65535 || Hq % Hk) return set_error(DH_ERR_INVALID, "%s: Hq=%d of Hk=%d", op, Hq, Hk);
    if (!(scale > 0.f) || !(scale - scale == 0.f))
        return set_error(DH_ERR_INVALID, "%s: scale must be finite and > 0", op);
    if (window < 0 || max_len < 0 || max_len > 0x7FF00000 || (long long)max_len > (long long)ld_table * page)
        return set_error(DH_ERR_INVALID, "%s: window=%d, max_len=%d (the table has %lld)", op, window, max_len,
                         (long long)ld_table * page);
    DH_TRY(check_strides(op, "Q", sq, B, Hq, D, false));
    DH_TRY(check_strides(op, "O", so, B, Hq, D, true));
    const size_t need = dh_paged_attention_workspace(cache_type, B, Hq, Hk, D, max_len);
    if (B > 0 && (!Q || !len || !O || (need > 0 && !ws))) return set_error(DH_ERR_INVALID, "%s: null pointer", op);
    if (need > 0 && ((uintptr_t)ws & 15)) return set_error(DH_ERR_INVALID, "%s: workspace not 16-byte aligned", op);
    if (ws_bytes < need)
        return set_error(DH_ERR_INVALID, "%s: workspace of %zu bytes, %zu needed", op, ws_bytes, need);
    DH_TRY(ensure_init());
    if (B == 0) return DH_OK;
    Work w{B, Hq, Hq / Hk, 1, window, max_len, 0, 0, scale, len, nullptr, nullptr};
    plan(B, Hk, max_len, window, w.chunk, w.splits);
    w.part = (float*)ws;
    w.stat = (float2*)((char*)ws + up256((size_t)w.splits * B * Hq * D * 4));
    auto run = dtype == DH_F32 ? cache_type == DH_F32 ? launch<float, float>
                                 : cache_type == DH_I8 ? launch<float, int8_t> : launch<float, uint8_t>
                               : cache_type == DH_BF16 ? launch<uint16_t, uint16_t>
                                 : cache_type == DH_I8 ? launch<uint16_t, int8_t> : launch<uint16_t, uint8_t>;
    return run(c, w, Q, Strides{sq[0], sq[1]}, O, Strides{so[0], so[1]}, lse);
}

}  // extern "C"
