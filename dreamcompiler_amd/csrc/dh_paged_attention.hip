// dh_paged_attention.hip -- attention of one new token of each sequence over a paged cache.
//
//   o = sum_t p_t v_t / sum_t p_t,  p_t = exp(scale q . k_t - m),  lse = m + log sum_t p_t
//
// over the tokens t of the sequence (its last `window` ones).  One pass over keys and values with the
// running maximum m and sum; a sequence's tokens are split into chunks, whose o, m and sum meet in a
// second launch.  Bound by HBM: each key and value is read once.
//
// Measured, D = 128 and 8 cache heads, where a copy of 1 GiB moves 5.14 TB/s: 64 sequences of 1024 to 8192 tokens bf16 with
// 32 query heads 227 us (5.4 TB/s), 128 of e4m3 with 64 query heads 248 (5.1), one of 131072 bf16 102 (5.3), 33 of up to 2047
// fp32 (D = 64, 12 heads, the last 1000 tokens) 36 (4.7).  One of 512 tokens and 16 heads: 8.1, a launch that waits for
// length, pages and two tiles a wave, on 16 CUs: a CU takes about 22 bytes a clock from memory, whatever it asks for.
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
    int B, Hq, G, window, max_len, chunk, splits;
    float scale;
    FastDiv by_groups, by_heads;   // groups of 16 RT query heads of a cache head, cache heads
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

// x (8 values) in P parts of bf16 that add up to it: 8 bits each.  An infinity, where x may be one (INF), is its first
// part alone: what is left of it would be NaN.
template <int P, bool INF = false>
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
                const float lo = __builtin_bit_cast(float, w << 16), hi = __builtin_bit_cast(float, w & 0xFFFF0000u);
                r[2 * e] = INF && fabsf(lo) == INFINITY ? 0.f : r[2 * e] - lo;
                r[2 * e + 1] = INF && fabsf(hi) == INFINITY ? 0.f : r[2 * e + 1] - hi;
            }
        }
}

// ---- a chunk -----------------------------------------------------------------------------------
// A work-group of 4 or 8 waves takes a chunk of a sequence's tokens for 16 RT query heads of one cache head;
// its waves take the tiles of TILE tokens in turn, each with its own maximum, sum and o, which
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
// bits) and a weight two or, where the model is fp32, three.  Two are 16 bits, for a result of 8: a result is off by up to 2^-16
// of the largest |v| before its rounding.  Three would move 0.1% of the results over the border of a rounding and cost
// 0.5% at the copy's rate, but 5 to 14% where many query heads or short heads make the instructions count (32 sequences up to
// 4096 tokens e4m3, 160 heads on 8 of 64: 30.6 and 34.7 us).
//
// DP is D itself for the usual head sizes (FULL), else the next multiple of 64, whose columns past D are
// clamped and zeroed.
template <typename T, typename CT, int DP>
struct Form {
    static constexpr bool wide = sizeof(CT) == 4, narrow = sizeof(CT) == 1;
    static constexpr int SIZE = sizeof(CT);
    static constexpr int SUBS = wide ? 1 : 2, TILE = 16 * SUBS;   // 16 tokens each
    static constexpr int E = 16 / SIZE;                           // values of 16 bytes
    static constexpr int KSTEPS = (DP + 4 * E - 1) / (4 * E);     // 16-byte pieces of a lane's part of a key
    static constexpr int QP = wide ? 1 : sizeof(T) == 4 ? 3 : 1, PP = sizeof(T) == 4 ? 3 : 2;
    static constexpr int QN = wide ? 4 : 8, QI = narrow ? 2 * KSTEPS : KSTEPS;        // the same of a query, by operands
    // Values of a row, in segments of 16 W columns: W = 8 (4 in fp32: 16 bytes) as often as it goes, then 4, 2, 1.
    static constexpr int width_at(int column) {
        const int left = (DP - column) / 16;
        return left >= 8 && !wide ? 8 : left >= 4 ? 4 : left >= 2 ? 2 : 1;
    }
    static constexpr int column(int seg) {
        int c = 0;
        for (int i = 0; i < seg; ++i) c += 16 * width_at(c);
        return c;
    }
    static constexpr int width(int seg) { return width_at(column(seg)); }
    static constexpr int segments() {
        int n = 0;
        while (column(n) < DP) ++n;
        return n;
    }
    static constexpr int SEGS = segments();
    static constexpr int words(int seg) { return (width(seg) * SIZE + 3) / 4; }   // registers of a token's part
    static constexpr int word(int seg) {
        int n = 0;
        for (int i = 0; i < seg; ++i) n += words(i);
        return n;
    }
    static constexpr int WORDS = word(SEGS);
};

// What a lane loads of a tile.
template <typename F>
struct Tile {
    u32x4 kr[F::SUBS][F::KSTEPS];
    uint32_t vr[F::SUBS][4][F::WORDS];
    f32x4 ks[F::SUBS], vs[F::SUBS];   // scales of tokens 4 g .. 4 g + 3 of each 16
    bool there[F::SUBS], whole;       // whether there is a page, and whether all tokens count
};

template <typename T, typename CT, int DP, bool FULL, int RT, int WAVES>
__global__ void __launch_bounds__(64 * WAVES) paged_chunk(Paged c, Work w, const T* __restrict__ Q, Strides sq,
                                                   T* __restrict__ O, Strides so, float* __restrict__ lse) {
    typedef Form<T, CT, DP> F;
    constexpr int SUBS = F::SUBS, KSTEPS = F::KSTEPS, E = F::E, LD = DP + 4;
    constexpr bool wide = F::wide, narrow = F::narrow;
    // Queries that would take too many registers wait in LDS, where the waves' sums meet afterwards.
    constexpr int QN = F::QN, QI = F::QI, Q_WORDS = RT * F::QP * QI * 4;
    constexpr bool Q_LDS = Q_WORDS > 32 || (!wide && Q_WORDS > 16);
    __shared__ union {
        float o[4][16][LD];
        u32x4 q[Q_LDS ? Q_WORDS / 4 : 1][64];
    } shared;
    auto& ol = shared.o;
    __shared__ float2 ml[WAVES][16 * RT];
    const int D = FULL ? DP : c.D;
    const int lane = threadIdx.x & 63, l = lane & 15, g = lane >> 4;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    // Chunks of a sequence are spread over the XCDs (work-group i runs on XCD i % 8), and so are a
    // chunk's sequences: long sequences have more chunks than short ones.  128 sequences of 1024 to 8192 tokens
    // e4m3: 318 us with chunk j of each on XCD j.
    const int split = blockIdx.y;
    uint32_t at = blockIdx.x + split % gridDim.x;
    if (at >= gridDim.x) at -= gridDim.x;
    const int pair = fdiv(at, w.by_groups), b = fdiv(pair, w.by_heads), hk = pair - b * c.Hk;
    const int first = (at - pair * w.by_groups.d) * 16 * RT;   // head of the group

    // Queries, lengths and pages are on their way together: with no window, the chunk's pages do not hang on the
    // length.  (Loads under a condition would wait for each other: 4 us of a call.)
    typedef T qvec __attribute__((ext_vector_type(wide ? 4 : 8), aligned(sizeof(T))));
    qvec qr[RT][QI];
    auto ends = [](int column) { return FULL && column <= DP; };   // all lanes' pieces up to there are columns
    auto q_column = [&](int i) {   // piece of QN values: of 16-byte piece i (fp32, bf16), or a half of piece i / 2
        return narrow ? 16 * (4 * (i / 2) + g) + 8 * (i % 2) : QN * (4 * i + g);
    };
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const T* q = Q + b * sq.seq + (long long)(hk * w.G + min(first + 16 * rt + l, w.G - 1)) * sq.head;
#pragma unroll
        for (int i = 0; i < QI; ++i)
            qr[rt][i] = *reinterpret_cast<const qvec*>(q + (q_column(i) < D ? q_column(i) : 0));
    }
    int from, to, start = 0;
    if (w.window > 0) w.span(b, from, to, start);
    const int c0 = start + split * w.chunk, page0 = c0 >> c.shift;
    // Two pages a lane (at most 2048 tokens of at least 16 a page).
    int ids[2];
#pragma unroll
    for (int i = 0; i < 2; ++i) ids[i] = c.table[(long long)b * c.ld + min(page0 + 64 * i + lane, c.ld - 1)];
    w.span(b, from, to, start);
    const int n_chunks = w.chunks(to, start);
    if (split >= max(n_chunks, 1)) return;
    const int c1 = min(c0 + w.chunk, to);
#pragma unroll
    for (int i = 0; i < 2; ++i)
        if (page0 + 64 * i + lane >= c.ld || (unsigned)ids[i] >= (unsigned)c.pages) ids[i] = -1;

    // Queries: the values of d that the lane has of a key, as words of operands.
    u32x4 qf[Q_LDS ? 1 : Q_WORDS / 4];
#pragma unroll
    for (int rt = 0; rt < RT; ++rt) {
        const bool head = first + 16 * rt + l < w.G;
#pragma unroll
        for (int i = 0; i < QI; ++i) {
            float x[QN];
#pragma unroll
            for (int e = 0; e < QN; ++e) x[e] = head && q_column(i) < D ? paged_up(qr[rt][i][e]) : 0.f;
            u32x4 parts[F::QP];
            if constexpr (wide) {
#pragma unroll
                for (int e = 0; e < QN; ++e) parts[0][e] = __builtin_bit_cast(uint32_t, x[e]);
            } else {
                split8<F::QP, true>(x, parts);
            }
#pragma unroll
            for (int p = 0; p < F::QP; ++p) {
                const int at = (rt * QI + i) * F::QP + p;
                if constexpr (!Q_LDS) qf[at] = parts[p];
                else if (wave == 0) shared.q[at][lane] = parts[p];
            }
        }
    }
    if constexpr (Q_LDS) __syncthreads();

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

    Tile<F> x;
    auto load = [&](Tile<F>& x, int base) {
        x.whole = base >= from && base + F::TILE <= to;
#pragma unroll
        for (int s = 0; s < SUBS; ++s) {
            const int t = base + 16 * s;
            int id = -1;
            if (t < c1) {
                const int i = (t >> c.shift) - page0;
                id = __builtin_amdgcn_readlane(i < 64 ? ids[0] : ids[1], i & 63);
            }
            x.there[s] = id >= 0;
            x.whole = x.whole && x.there[s];
            const long long row = x.there[s] ? c.row(id, hk, t & ((1 << c.shift) - 1)) : 0;
            const char* kp = (const char*)c.K + row * row_bytes;
            const char* vp = (const char*)c.V + row * row_bytes;
#pragma unroll
            for (int i = 0; i < KSTEPS; ++i) {
                uint32_t at = k_off + 64 * i;
                if (!ends(4 * E * (i + 1)) && E * (4 * i + g) >= D) at = l * row_bytes;
                x.kr[s][i] = *reinterpret_cast<const u32x4*>(kp + at);
            }
            if constexpr (narrow) {
                x.ks[s] = *reinterpret_cast<const f32x4*>(c.Ks + row + 4 * g);
                x.vs[s] = *reinterpret_cast<const f32x4*>(c.Vs + row + 4 * g);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int sg = 0; sg < F::SEGS; ++sg) {
                    const char* p = vp + (v_off[sg] + i * row_bytes);
                    uint32_t* to_ = x.vr[s][i] + F::word(sg);
                    const int bytes = F::width(sg) * F::SIZE;
                    if (bytes == 16) {
                        const u32x4 y = *reinterpret_cast<const u32x4*>(p);
#pragma unroll
                        for (int e = 0; e < 4; ++e) to_[e] = y[e];
                    } else if (bytes == 8) {
                        const u32x2 y = *reinterpret_cast<const u32x2*>(p);
                        to_[0] = y[0], to_[1] = y[1];
                    } else if (bytes == 4) {
                        *to_ = *reinterpret_cast<const uint32_t*>(p);
                    } else if (bytes == 2) {
                        *to_ = *reinterpret_cast<const uint16_t*>(p);
                    } else {
                        *to_ = *reinterpret_cast<const uint8_t*>(p);
                    }
                }
        }
    };
    auto compute = [&](Tile<F>& x, int base) {
        // Scores, in units of log 2.
        uint32_t q_lane = lane;
        if constexpr (Q_LDS) asm volatile("" : "+v"(q_lane));   // read for each tile, not kept
        auto query = [&](int rt, int i, int p) {
            const int at = (rt * QI + i) * F::QP + p;
            if constexpr (Q_LDS) return shared.q[at][q_lane];
            else return qf[at];
        };
        f32x4 acc[RT][SUBS];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int s = 0; s < SUBS; ++s) acc[rt][s] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int i = 0; i < QI; ++i) {
            u32x4 k[SUBS];
#pragma unroll
            for (int s = 0; s < SUBS; ++s) {
                if constexpr (narrow) {
                    const u32x4 y = x.kr[s][i / 2];
                    const u32x2 a = words_bf16<CT>(y[2 * (i % 2)]), c = words_bf16<CT>(y[2 * (i % 2) + 1]);
                    k[s] = u32x4{a[0], a[1], c[0], c[1]};
                } else {
                    k[s] = x.kr[s][i];
                }
                if (!ends(narrow ? 64 * (i / 2 + 1) : 4 * QN * (i + 1)) && q_column(i) >= D) k[s] = u32x4{0, 0, 0, 0};
            }
#pragma unroll
            for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                for (int p = 0; p < F::QP; ++p) {
                    const u32x4 qq = query(rt, i, p);
#pragma unroll
                    for (int s = 0; s < SUBS; ++s) {
                        if constexpr (wide) {
#pragma unroll
                            for (int e = 0; e < 4; ++e)
                                acc[rt][s] = mfma(__builtin_bit_cast(float, (uint32_t)k[s][e]),
                                                  __builtin_bit_cast(float, (uint32_t)qq[e]), acc[rt][s]);
                        } else {
                            acc[rt][s] = mfma(k[s], qq, acc[rt][s]);
                        }
                    }
                }
        }
        float z[RT][SUBS][4];
#pragma unroll
        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
            for (int s = 0; s < SUBS; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float f = unit;
                    if constexpr (narrow) f *= x.ks[s][r];
                    z[rt][s][r] = acc[rt][s][r] * f;
                }
        if (!x.whole) {   // tokens that do not count: no score, no value, whatever lies there
#pragma unroll
            for (int s = 0; s < SUBS; ++s)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int t = base + 16 * s + 4 * g + r;
                    const bool in = x.there[s] && t >= from && t < to;
#pragma unroll
                    for (int rt = 0; rt < RT; ++rt) z[rt][s][r] = in ? z[rt][s][r] : -INFINITY;
#pragma unroll
                    for (int e = 0; e < F::WORDS; ++e) x.vr[s][r][e] = in ? x.vr[s][r][e] : 0;
                    if constexpr (narrow) x.vs[s][r] = in ? x.vs[s][r] : 0.f;
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
                    float y = __builtin_amdgcn_exp2f(z[rt][s][r] - off);
                    sum[rt] += y;
                    if constexpr (narrow) y *= x.vs[s][r];
                    p[4 * s + r] = y;
                }
            if constexpr (wide) {
#pragma unroll
                for (int r = 0; r < 4; ++r) pw[rt][r] = p[r];
            } else {
                split8<F::PP>(p, pf[rt]);
            }
        }

        // o += weights x values
#pragma unroll
        for (int sg = 0; sg < F::SEGS; ++sg) {
            const int j0 = F::column(sg) / 16, W = F::width(sg), w0 = F::word(sg);
            if constexpr (wide) {
#pragma unroll
                for (int j = 0; j < W; ++j)
#pragma unroll
                    for (int r = 0; r < 4; ++r)
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
                            o[rt][j0 + j] = mfma(__builtin_bit_cast(float, x.vr[0][r][w0 + j]), pw[rt][r], o[rt][j0 + j]);
            } else {
#pragma unroll
                for (int jj = 0; jj < (W + 1) / 2; ++jj) {   // two columns: a word of bf16
                    uint32_t y[8];
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        if constexpr (narrow) y[i] = words_bf16<CT>(x.vr[i / 4][i % 4][w0 + jj / 2])[jj % 2];
                        else y[i] = x.vr[i / 4][i % 4][w0 + jj];
                    }
#pragma unroll
                    for (int odd = 0; odd < (W > 1 ? 2 : 1); ++odd) {
                        u32x4 a;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            a[i] = odd ? pack_hi16(y[2 * i], y[2 * i + 1]) : pack_lo16(y[2 * i], y[2 * i + 1]);
#pragma unroll
                        for (int rt = 0; rt < RT; ++rt)
#pragma unroll
                            for (int p = 0; p < F::PP; ++p)
                                o[rt][j0 + 2 * jj + odd] = mfma(a, pf[rt][p], o[rt][j0 + 2 * jj + odd]);
                    }
                }
            }
        }
    };
    for (int base = c0 + F::TILE * wave; base < c1; base += WAVES * F::TILE) {
        load(x, base);
        compute(x, base);
    }

    // The waves' sums meet, four waves at a time: o[..][j][r] is column W (4 g + r) + j of its segment.
    constexpr int PER = (16 * DP / 4 + 64 * WAVES - 1) / (64 * WAVES);   // pieces of 4 columns a thread
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
        f32x4 v[PER];
        float top[PER], total[PER];
#pragma unroll
        for (int round = 0; round < WAVES / 4; ++round) {
            if (rt + round > 0 || Q_LDS) __syncthreads();
            if (wave / 4 == round) {
#pragma unroll
                for (int sg = 0; sg < F::SEGS; ++sg) {
                    const int j0 = F::column(sg) / 16, W = F::width(sg);
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        float* to_ = &ol[wave % 4][l][F::column(sg) + W * (4 * g + r)];
                        if (W >= 4) {
#pragma unroll
                            for (int e = 0; e < W; e += 4)
                                *reinterpret_cast<f32x4*>(to_ + e) = f32x4{o[rt][j0 + e][r], o[rt][j0 + e + 1][r],
                                                                           o[rt][j0 + e + 2][r], o[rt][j0 + e + 3][r]};
                        } else {
#pragma unroll
                            for (int e = 0; e < W; ++e) to_[e] = o[rt][j0 + e][r];
                        }
                    }
                }
            }
            __syncthreads();
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int at = threadIdx.x + 64 * WAVES * i, hl = min(at / (DP / 4), 15), d = 4 * (at % (DP / 4));
                if (round == 0) {
                    top[i] = -INFINITY, total[i] = 0.f, v[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int x = 0; x < WAVES; ++x) top[i] = fmaxf(top[i], ml[x][16 * rt + hl].x);
                }
                const float off = top[i] == -INFINITY ? 0.f : top[i];
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const float2 st = ml[4 * round + x][16 * rt + hl];
                    const float f = __builtin_amdgcn_exp2f(st.x - off);
                    total[i] += st.y * f;
                    v[i] += *reinterpret_cast<const f32x4*>(&ol[x][hl][d]) * f;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int at = threadIdx.x + 64 * WAVES * i, hl = at / (DP / 4), d = 4 * (at % (DP / 4)), h = first + 16 * rt + hl;
            if (hl >= 16 || h >= w.G || d >= D) continue;
            const int hq = hk * w.G + h;
            if (last) {
                const bool none = total[i] == 0.f;   // no score: whatever the values hold
                const float f = 1.f / total[i];
                T* out = O + b * so.seq + (long long)hq * so.head + d;
#pragma unroll
                for (int e = 0; e < 4; ++e) out[e] = down<T>(none ? 0.f : v[i][e] * f);
                if (lse && d == 0) lse[(long long)b * w.Hq + hq] = none ? -INFINITY : top[i] * LN2 + logf(total[i]);
            } else {
                const long long to_ = split * heads + (long long)b * w.Hq + hq;
                *reinterpret_cast<f32x4*>(w.part + to_ * D + d) = v[i];
                if (d == 0) w.stat[to_] = float2{top[i], total[i]};
            }
        }
    }
}

// ---- the chunks of a sequence -------------------------------------------------------------------
// WAVES waves join a head's chunks (four heads a work-group of single waves): L lanes hold a row of D, so
// that 64 / L rows a wave and four times that are in flight, in a fixed order.
template <typename T, int L, int WAVES>
__global__ void __launch_bounds__(WAVES == 1 ? 256 : 64 * WAVES) paged_join(Work w, int D, T* __restrict__ O, Strides so,
                                                                           float* __restrict__ lse) {
    constexpr int ROWS = 64 / L, STEP = ROWS * WAVES, AHEAD = 4;
    __shared__ f32x4 red[WAVES == 1 ? 1 : WAVES][L];
    __shared__ float reds[WAVES == 1 ? 1 : WAVES];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, d = 4 * (lane & (L - 1)), b = blockIdx.y;
    const int h = WAVES == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
    int from, to, start;
    w.span(b, from, to, start);
    const int n = w.chunks(to, start);
    if (n <= 1 || h >= w.Hq) return;   // its one chunk wrote the result
    const long long step = (long long)w.B * w.Hq, at = (long long)b * w.Hq + h;
    const int i0 = (WAVES == 1 ? 0 : wave * ROWS) + lane / L;
    f32x4 x[AHEAD];
    float2 st[AHEAD];
    auto load = [&](int i) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            x[a] = f32x4{0.f, 0.f, 0.f, 0.f};
            st[a] = float2{-INFINITY, 0.f};
            if (i + a * STEP < n) {
                st[a] = w.stat[(i + a * STEP) * step + at];
                if (d < D) x[a] = *reinterpret_cast<const f32x4*>(w.part + ((i + a * STEP) * step + at) * D + d);
            }
        }
    };
    load(i0);
    float m = -INFINITY, sum = 0.f;
    for (int i = lane; i < n; i += 64) m = fmaxf(m, w.stat[i * step + at].x);
    m = wave_reduce(m, OpMax());
    const float off = m == -INFINITY ? 0.f : m;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    for (int i = i0;;) {
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const float f = __builtin_amdgcn_exp2f(st[a].x - off);
            sum += st[a].y * f;
            o += x[a] * f;
        }
        i += AHEAD * STEP;
        if (i - i0 >= n) break;
        load(i);
    }
#pragma unroll
    for (int x = L; x < 64; x *= 2) {
        sum += __shfl_xor(sum, x);
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] += __shfl_xor(o[e], x);
    }
    if constexpr (WAVES > 1) {
        if (lane < L) red[wave][lane] = o;
        if (lane == 0) reds[wave] = sum;
        __syncthreads();
        if (wave > 0) return;
        sum = 0.f, o = f32x4{0.f, 0.f, 0.f, 0.f};
        for (int x = 0; x < WAVES; ++x) {
            sum += reds[x];
            o += red[x][lane & (L - 1)];
        }
    }
    const bool none = sum == 0.f;   // no score: whatever the values hold
    if (lane < L && d < D) {
        const float f = 1.f / sum;
        T* out = O + b * so.seq + (long long)h * so.head + d;
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = down<T>(none ? 0.f : o[e] * f);
    }
    if (lse && lane == 0) lse[at] = none ? -INFINITY : m * LN2 + logf(sum);
}

// ---- host --------------------------------------------------------------------------------------
// How the work is split.  A chunk is a multiple of LEAST tokens (a tile for each of four waves) and at most
// MOST (the pages that a work-group's lanes hold) or CHUNK_BYTES of keys and values; a sequence has as many as make about
// WORK_GROUPS of all sequences at their longest: three a CU (two or four: up to 13% slower with few long sequences,
// the same with many).  Larger chunks leave a tail of busy work-groups while others are
// done, smaller ones wait more often for their first loads (64 sequences up to 8192 bf16, chunks of 256 /
// 512 / 1024 / 2048 tokens: 288 / 234 / 230 / 236 us; 128 of e4m3: 364 / 271 / 257 / 251).
// Joining costs a launch: what one work-group reads in the same time stays whole, FEW_BYTES of keys and values, at most
// ONE tokens.  One sequence on 1 to 32 heads, whole and split: 256 KB are 8.6 and 9.4 us in fp32 of D = 64, 9.5 and
// 10.6 of D = 128, 8.8 and 10.0 in bf16 of D = 64; 512 KB 14.5 and 10.2 in fp32 of D = 128, 13.9 and 11.0 in bf16 of
// D = 256; 1 MB (512 tokens in fp32 of D = 256) 29.8 and 15.0.  Where there are pairs of sequence and head for half the CUs
// (MANY), up to ONE tokens, 1024 and some that follow, whatever their bytes: 16 x 8 heads x 1088 tokens bf16 of D = 128
// 14.0 us whole, 14.9 split, e4m3 11.2 and 12.5 (bytes would tell better there too: bf16 of D = 256 24.9 and 21.4, fp32
// of D = 64 17.8 and 14.2, of D = 256 61 and 42).
constexpr int LEAST = 128, MOST = 2048, CHUNK_BYTES = 512 << 10, WORK_GROUPS = 768;
constexpr int FEW_BYTES = 256 << 10, ONE = 1088, MANY = 128;
constexpr int MOST_SPLITS = 65535;   // of a launch; at most 2^25 tokens in chunks of MOST are fewer

struct Plan {
    int chunk, splits;
};
int whole_tokens(long long pairs, int D, int size) {
    const int n = FEW_BYTES / (2 * D * size);
    return pairs >= MANY || n > ONE ? ONE : n;
}
int most_tokens(int D, int size) {
    const int n = CHUNK_BYTES / (2 * D * size) / LEAST * LEAST;
    return n > MOST ? MOST : n;   // D size <= 1024
}
Plan plan(long long pairs, int D, int size, int max_len, int window) {
    // a window that begins inside a tile sees up to 31 tokens before it
    const long long seen = window > 0 && window < max_len - 31 ? window + 31LL : max_len;
    if (seen <= whole_tokens(pairs, D, size)) return {(ONE + LEAST - 1) / LEAST * LEAST, 1};
    const int most = most_tokens(D, size);
    long long n = WORK_GROUPS / pairs;   // chunks of the longest sequence
    if (n < (seen + most - 1) / most) n = (seen + most - 1) / most;
    if (n > (seen + LEAST - 1) / LEAST) n = (seen + LEAST - 1) / LEAST;
    if (n > MOST_SPLITS) n = MOST_SPLITS;
    const int chunk = (int)(((seen + n - 1) / n + LEAST - 1) / LEAST * LEAST);
    return {chunk, (int)((seen + chunk - 1) / chunk)};
}
// At least as many for every window.
long long most_splits(long long pairs, int D, int size, int max_len) {
    if (max_len <= whole_tokens(pairs, D, size)) return 1;
    const int most = most_tokens(D, size);
    const long long a = ((long long)max_len + LEAST - 1) / LEAST, b = WORK_GROUPS / pairs,
                    c = ((long long)max_len + most - 1) / most, n = a < b ? a : b > c ? b : c;
    return n < MOST_SPLITS ? n : MOST_SPLITS;
}
// Waves of a work-group: eight where they have two tiles each and the registers leave room for two such
// work-groups on a CU (33 x 12 sequences fp32: 37 us with eight, 45 with four), or where there is at most one for each CU
// (5 x 8 of up to 3024 tokens, D = 192, in 480 work-groups: 22.7 with eight, 18.9 with four).  Two tiles of query
// rows have twice the sums to join: four (the same with 160 heads: 29.9 with eight, 22.1 with four; 1 x 8: 15.9, 13.7).
int waves_of(int D, int row_tiles, int chunk, long long groups) {
    return row_tiles == 1 && ((D <= 128 && chunk >= 512) || groups <= 256) ? 8 : 4;
}
int row_tiles_of(int G) { return G > 16 ? 2 : 1; }
int size_of(int cache_type) { return cache_type == DH_F32 ? 4 : cache_type == DH_BF16 ? 2 : 1; }
size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

// A wave for what it has in flight at once (8 chunks of D = 128), four or sixteen for more.
template <typename T, int L>
int join(const Work& w, int D, void* O, Strides so, float* lse) {
    const int once = 4 * 64 / L;
    if (w.splits <= once) paged_join<T, L, 1><<<dim3((w.Hq + 3) / 4, w.B), 256, 0, stream()>>>(w, D, (T*)O, so, lse);
    else if (w.splits <= 4 * once) paged_join<T, L, 4><<<dim3(w.Hq, w.B), 256, 0, stream()>>>(w, D, (T*)O, so, lse);
    else paged_join<T, L, 16><<<dim3(w.Hq, w.B), 1024, 0, stream()>>>(w, D, (T*)O, so, lse);
    return check_launch("dh_paged_attention");
}

template <typename T, typename CT, int DP, bool FULL, int RT>
int launch_form(const Paged& c, Work w, const void* Q, Strides sq, void* O, Strides so, float* lse) {
    const int groups = (w.G + 16 * RT - 1) / (16 * RT);
    w.by_groups = make_fastdiv(groups);
    const dim3 grid(w.B * c.Hk * groups, w.splits);
    const int waves = waves_of(c.D, RT, w.chunk, (long long)grid.x * grid.y);
    auto run = paged_chunk<T, CT, DP, FULL, RT, 4>;
    if constexpr (RT == 1)
        if (waves == 8) run = paged_chunk<T, CT, DP, FULL, RT, 8>;
    run<<<grid, 64 * waves, 0, stream()>>>(c, w, (const T*)Q, sq, (T*)O, so, lse);
    DH_TRY(check_launch("dh_paged_attention"));
    if (w.splits == 1) return DH_OK;
    return c.D <= 64 ? join<T, 16>(w, c.D, O, so, lse) : c.D <= 128 ? join<T, 32>(w, c.D, O, so, lse)
                                                                    : join<T, 64>(w, c.D, O, so, lse);
}

template <typename T, typename CT>
int launch(const Paged& c, const Work& w, const void* Q, Strides sq, void* O, Strides so, float* lse) {
    // Up to 32 query heads of a cache head read it once.
    auto run = [&](auto one, auto two) { return row_tiles_of(w.G) == 2 ? two(c, w, Q, sq, O, so, lse) : one(c, w, Q, sq, O, so, lse); };
#define DH_FORM(DP, FULL) run(launch_form<T, CT, DP, FULL, 1>, launch_form<T, CT, DP, FULL, 2>)
    switch (c.D) {
        case 32: return DH_FORM(32, true);
        case 64: return DH_FORM(64, true);
        case 80: return DH_FORM(80, true);
        case 96: return DH_FORM(96, true);
        case 128: return DH_FORM(128, true);
        case 192: return DH_FORM(192, true);
        case 256: return DH_FORM(256, true);
    }
    return c.D < 64 ? DH_FORM(64, false) : c.D < 128 ? DH_FORM(128, false) : c.D < 192 ? DH_FORM(192, false)
                                                                                       : DH_FORM(256, false);
#undef DH_FORM
}

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" {

size_t dh_paged_attention_workspace(int cache_type, int B, int Hq, int Hk, int D, int max_len) {
    if (B < 1 || Hq < 1 || Hk < 1 || D < 1 || D > PAGED_MOST_D || max_len < 1) return 0;
    const long long splits = most_splits((long long)B * Hk, D, size_of(cache_type), max_len);
    if (splits == 1) return 0;
    const size_t rows = (size_t)splits * B * Hq;
    return up256(rows * D * 4) + rows * 8;
}

int dh_paged_attention_plan(int cache_type, int B, int Hq, int Hk, int D, int max_len, int window, int* plan_out) {
    if (!plan_out) return set_error(DH_ERR_INVALID, "dh_paged_attention_plan: null pointer");
    if (B < 1 || Hk < 1 || Hq < 1 || Hq % Hk || D < 1 || D > PAGED_MOST_D || max_len < 0 || max_len > 1 << 25 || window < 0)
        return set_error(DH_ERR_INVALID, "dh_paged_attention_plan: shape B=%d Hq=%d Hk=%d D=%d max_len=%d window=%d", B,
                         Hq, Hk, D, max_len, window);
    const Plan p = plan((long long)B * Hk, D, size_of(cache_type), max_len, window);
    const int rt = row_tiles_of(Hq / Hk), groups = (Hq / Hk + 16 * rt - 1) / (16 * rt);
    plan_out[0] = p.chunk, plan_out[1] = p.splits;
    plan_out[2] = waves_of(D, rt, p.chunk, (long long)B * Hk * groups * p.splits), plan_out[3] = groups;
    return DH_OK;
}

int dh_paged_attention(int dtype, int cache_type, int B, int Hq, int Hk, int D, float scale, int window,
                       const void* Q, const long long* sq, const int* len, int max_len, int pages, int page,
                       const int* table, int ld_table, const void* Kc, const void* Vc, const float* Ks,
                       const float* Vs, void* O, const long long* so, float* lse, void* ws, size_t ws_bytes) {
    const char* op = "dh_paged_attention";
    Paged c;
    DH_TRY(check_paged(op, dtype, cache_type, B, Hk, D, pages, page, table, ld_table, Kc, Vc, Ks, Vs, c));
    if (Hq < 1 || Hq > 65535 || Hq % Hk) return set_error(DH_ERR_INVALID, "%s: Hq=%d of Hk=%d", op, Hq, Hk);
    if ((long long)B * Hq > 1 << 22) return set_error(DH_ERR_INVALID, "%s: shape B=%d Hq=%d", op, B, Hq);
    if (!(scale > 0.f) || !(scale - scale == 0.f))
        return set_error(DH_ERR_INVALID, "%s: scale must be finite and > 0", op);
    if (window < 0 || max_len < 0 || max_len > 1 << 25 || (long long)max_len > (long long)ld_table * page)
        return set_error(DH_ERR_INVALID, "%s: window=%d, max_len=%d (the table has %lld)", op, window, max_len,
                         (long long)ld_table * page);
    DH_TRY(check_strides(op, "Q", sq, B, Hq, D, false));
    DH_TRY(check_strides(op, "O", so, B, Hq, D, true));
    const Plan p = B > 0 ? plan((long long)B * Hk, D, size_of(cache_type), max_len, window) : Plan{LEAST, 1};
    // One chunk (a short window) leaves nothing to join, whatever the longest sequence.
    const size_t need = p.splits > 1 ? dh_paged_attention_workspace(cache_type, B, Hq, Hk, D, max_len) : 0;
    if (B > 0 && (!Q || !len || !O || (need > 0 && !ws))) return set_error(DH_ERR_INVALID, "%s: null pointer", op);
    if (need > 0 && ((uintptr_t)ws & 15)) return set_error(DH_ERR_INVALID, "%s: workspace not 16-byte aligned", op);
    if (ws_bytes < need)
        return set_error(DH_ERR_INVALID, "%s: workspace of %zu bytes, %zu needed", op, ws_bytes, need);
    DH_TRY(ensure_init());
    if (B == 0) return DH_OK;
    Work w{B, Hq, Hq / Hk, window, max_len, 0, 0, scale, {}, make_fastdiv(Hk), len, nullptr, nullptr};
    w.chunk = p.chunk, w.splits = p.splits;
    w.part = (float*)ws;
    w.stat = (float2*)((char*)ws + up256((size_t)w.splits * B * Hq * D * 4));
    auto run = dtype == DH_F32 ? cache_type == DH_F32 ? launch<float, float>
                                 : cache_type == DH_I8 ? launch<float, int8_t> : launch<float, uint8_t>
                               : cache_type == DH_BF16 ? launch<uint16_t, uint16_t>
                                 : cache_type == DH_I8 ? launch<uint16_t, int8_t> : launch<uint16_t, uint8_t>;
    return run(c, w, Q, Strides{sq[0], sq[1]}, O, Strides{so[0], so[1]}, lse);
}

}  // extern "C"
