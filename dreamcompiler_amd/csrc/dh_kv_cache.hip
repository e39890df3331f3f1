// dh_kv_cache.hip -- keys and values of new tokens into a paged cache, rounded to 8 bits where its
// type has them, and read back.
//
//   8 bits: s = max |x| / top over a row of D (top 127 for integers, 448 for e4m3), value = x / s
//   rounded to the nearest, ties to even; it stands for value * s
//
// The scale is the fp32 quotient; the values are those of the exact quotient by it (`quotient`), so
// that they do not hang on how a division rounds.  A row with an infinity or a NaN gets a NaN as its
// scale, and reads back as NaN.
//
// Bound by HBM: 32512 tokens of 8 heads of 128 bf16 into e4m3 and 80896 of them back take 149 us in turn, 4.7 TB/s, where
// a copy of 1 GiB moves 5.14 (a trace of both: 55 and 93); each by itself 51 and 104, to and from int8 47 and 104, in bf16
// 53 and 129, in fp32 107 and 252, at the copy's rate 39 and 98, 52 and 129, 104 and 258.  Few tokens are bound by the
// waits for beginnings, a length, a page and a row after each other: 64 sequences' next token 4.7 us, read back 4.1.
#include "dh_kv_split.hpp"
#include "dh_paged.hpp"

namespace dh {

int check_paged(const char* op, int dtype, int cache_type, int B, int Hk, int D, int pages, int page,
                const int* table, int ld, const void* Kc, const void* Vc, const float* Ks, const float* Vs,
                Paged& c) {
    if (dtype != DH_F32 && dtype != DH_BF16) return set_error(DH_ERR_INVALID, "%s: dtype must be fp32 or bf16", op);
    const bool scaled = cache_type == DH_I8 || cache_type == DH_F8;
    if (cache_type != dtype && !scaled)
        return set_error(DH_ERR_INVALID, "%s: cache_type must be the inputs' type, int8 or e4m3", op);
    if (B < 0 || B > 65535 || Hk < 1 || Hk > 65535 || D < 16 || D > PAGED_MOST_D || D % 16)
        return set_error(DH_ERR_INVALID, "%s: shape B=%d Hk=%d D=%d (D a multiple of 16 up to %d)", op, B, Hk, D,
                         PAGED_MOST_D);
    if (page < 16 || page > 4096 || (page & (page - 1)))
        return set_error(DH_ERR_INVALID, "%s: page=%d must be a power of two from 16 to 4096", op, page);
    if (pages < 1 || ld < 1 || (double)pages * Hk * page * D > (double)(1ll << 46))
        return set_error(DH_ERR_INVALID, "%s: pages=%d, ld_table=%d", op, pages, ld);
    if (!table || !Kc || !Vc || (scaled && (!Ks || !Vs))) return set_error(DH_ERR_INVALID, "%s: null pointer", op);
    if (((uintptr_t)Kc | (uintptr_t)Vc) & 15) return set_error(DH_ERR_INVALID, "%s: cache not 16-byte aligned", op);
    if (scaled && (((uintptr_t)Ks | (uintptr_t)Vs) & 15))
        return set_error(DH_ERR_INVALID, "%s: scales not 16-byte aligned", op);
    int shift = 0;
    while ((1 << shift) < page) ++shift;
    c = Paged{pages, shift, Hk, D, table, ld, (void*)Kc, (void*)Vc, (float*)Ks, (float*)Vs};
    return DH_OK;
}

int check_strides(const char* op, const char* name, const long long* st, long long n0, long long n1, int D,
                  bool out) {
    if (!st) return set_error(DH_ERR_INVALID, "%s: null strides of %s", op, name);
    if (n0 == 0 || n1 == 0) return DH_OK;   // no rows
    const bool swap = st[0] < st[1];   // the larger stride last
    const long long s[2] = {swap ? st[0] : st[1], swap ? st[1] : st[0]}, n[2] = {swap ? n0 : n1, swap ? n1 : n0};
    long long extent = D;
    for (int i = 0; i < 2; ++i) {
        if (n[i] <= 1) continue;
        if (s[i] < 0 || s[i] > (1ll << 46) / n[i] || (out && s[i] < extent))
            return set_error(DH_ERR_INVALID, "%s: strides (%lld, %lld) of %s", op, st[0], st[1], name);
        extent += s[i] * (n[i] - 1);
    }
    return DH_OK;
}

namespace {

template <typename T> __device__ inline T down(float x);
template <> __device__ inline float down<float>(float x) { return x; }
template <> __device__ inline uint16_t down<uint16_t>(float x) {
    return __builtin_bit_cast(uint16_t, (__bf16)x);
}

// A value from which rounding to fewer bits, nearest and ties to even, gives what it gives from the
// exact x / s (s > 0): the quotient cut off towards zero, its last bit set if anything was cut.  The
// remainder of a correctly rounded quotient is exact in fp32 unless it underflows, where |x / s| is
// far below every border.
__device__ inline float quotient(float x, float s) {
    const float y = x / s, r = fmaf(-y, s, x);
    uint32_t u = __builtin_bit_cast(uint32_t, y);
    if (r == 0.f || y == 0.f) return y;
    if ((r < 0.f) != (y < 0.f)) --u;
    return __builtin_bit_cast(float, u | 1u);
}

// What a cache's type makes of a row: its top, and the code of x / s.
template <typename CT> struct Code;
template <> struct Code<int8_t> {
    static constexpr float top = 127.f;
    __device__ static int8_t of(float x, float s) {
        return (int8_t)(int)fminf(fmaxf(rintf(quotient(x, s)), -top), top);
    }
};
template <> struct Code<uint8_t> {
    static constexpr float top = 448.f;
    __device__ static uint8_t of(float x, float s) {
        const float y = fminf(fmaxf(quotient(x, s), -top), top);
        return (uint8_t)(__builtin_amdgcn_cvt_pk_fp8_f32(y, y, 0, false) & 0xFF);
    }
};

struct Strides {
    long long token, head;
};

// The sequence that row n is of, and its token's position there: the rows of sequence b are its last
// first[b + 1] - first[b] tokens (first NULL: one each); t = -1 if it has fewer.  False for a row of
// no sequence.  A wave looks at 64 beginnings at once: two loads for up to 4096 sequences.
__device__ inline bool place(const int* __restrict__ first, const int* __restrict__ len, int B, int n, int& b,
                             int& t) {
    long long behind = 1;
    b = n;
    if (first) {
        const int lane = threadIdx.x & 63;
        int lo = 0, count = B;   // the last one at or before n is among lo .. lo + count - 1, or none
        while (count > 1) {
            const int step = (count + 63) >> 6, at = lo + lane * step;
            const uint64_t before = __ballot(lane * step < count && first[min(at, B)] <= n);
            const int k = max(__popcll(before), 1) - 1;
            lo += k * step;
            count = min(step, count - k * step);
        }
        b = __builtin_amdgcn_readfirstlane(lo);
        behind = (long long)first[b + 1] - n;
        if (first[b] > n || behind <= 0) return false;
    }
    const long long at = len[b] - behind;
    t = at < 0 ? -1 : (int)at;
    return true;
}

// ---- any rows: a wave each ---------------------------------------------------------------------
template <typename T, typename CT>
__global__ void __launch_bounds__(256) cache_write(Paged c, int B, int N, const int* __restrict__ first,
                                                   const int* __restrict__ len, const T* __restrict__ K, Strides sk,
                                                   const T* __restrict__ V, Strides sv) {
    constexpr bool scaled = sizeof(CT) == 1;
    const int lane = threadIdx.x & 63;
    const long long rows = 2LL * N * c.Hk, waves = (long long)gridDim.x * 4;
    for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += waves) {
        const int n = (int)(r / (2 * c.Hk)), i = (int)(r - 2LL * n * c.Hk);
        const bool value = i >= c.Hk;
        const int h = value ? i - c.Hk : i;
        int b, t;
        if (!place(first, len, B, n, b, t)) continue;
        const int id = c.page_of(b, t);
        if (id < 0) continue;
        const long long row = c.row(id, h, t & ((1 << c.shift) - 1));
        const T* x = value ? V + n * sv.token + h * sv.head : K + n * sk.token + h * sk.head;
        CT* o = (CT*)(value ? c.V : c.K) + row * c.D;
        float v[PAGED_MOST_D / 64];
        uint32_t most = 0;   // bits of |x|: their order is that of the values, NaN above infinity
#pragma unroll
        for (int j = 0; j < PAGED_MOST_D / 64; ++j) {
            const int e = 64 * j + lane;
            v[j] = e < c.D ? paged_up(x[e]) : 0.f;
            most = max(most, __builtin_bit_cast(uint32_t, v[j]) & 0x7FFFFFFFu);
        }
        float s = 1.f;
        if constexpr (scaled) {
            for (int m = 1; m < 64; m <<= 1) most = max(most, (uint32_t)__shfl_xor((int)most, m));
            s = most >= 0x7F800000u ? __builtin_nanf("") : __builtin_bit_cast(float, most) / Code<CT>::top;
            if (lane == 0) (value ? c.Vs : c.Ks)[row] = s;
        }
#pragma unroll
        for (int j = 0; j < PAGED_MOST_D / 64; ++j) {
            const int e = 64 * j + lane;
            if (e >= c.D) continue;
            if constexpr (scaled) {
                // Far below 1 both go up by 2^64, so that no remainder underflows.
                const float f = s < 0x1p-40f ? 0x1p64f : 1.f;
                o[e] = s > 0.f ? Code<CT>::of(v[j] * f, s * f) : CT(0);
            } else {
                o[e] = down<CT>(v[j]);
            }
        }
    }
}

template <typename T, typename CT>
__global__ void __launch_bounds__(256) cache_read(Paged c, int B, int N, const int* __restrict__ first,
                                                  const int* __restrict__ len, T* __restrict__ K, Strides sk,
                                                  T* __restrict__ V, Strides sv) {
    const int lane = threadIdx.x & 63;
    const long long rows = 2LL * N * c.Hk, waves = (long long)gridDim.x * 4;
    for (long long r = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); r < rows; r += waves) {
        const int n = (int)(r / (2 * c.Hk)), i = (int)(r - 2LL * n * c.Hk);
        const bool value = i >= c.Hk;
        const int h = value ? i - c.Hk : i;
        int b, t;
        if (!place(first, len, B, n, b, t)) continue;
        const int id = c.page_of(b, t);
        T* o = value ? V + n * sv.token + h * sv.head : K + n * sk.token + h * sk.head;
        const long long row = id < 0 ? 0 : c.row(id, h, t & ((1 << c.shift) - 1));
        const CT* x = (const CT*)(value ? c.V : c.K) + row * c.D;
        float s = 1.f;
        if constexpr (sizeof(CT) == 1)
            if (id >= 0) s = (value ? c.Vs : c.Ks)[row];
        for (int e = lane; e < c.D; e += 64) o[e] = down<T>(id < 0 ? 0.f : paged_up(x[e]) * s);
    }
}

// ---- rows that begin with 16 bytes ---------------------------------------------------------------
// A row is L lanes of P values, 16 bytes of the model's type, so a wave has 64 / L heads at once, keys and values (the
// read twice that).  A wave takes `tokens` rows of K and V, the four waves of a work-group in turn (what lies side by
// side is then read at the same time): its lanes find a token's place each, so that the waits for beginnings, lengths
// and pages are those of one token.  Where there are few tokens it takes one of the blocks of heads of one.  Where there
// are few heads (MANY) the wave has several tokens at once.  (Places found by a work-group of 16 tokens for its four
// waves, with a barrier, cost 2 to 10% more.)
struct Units : Split {
    FastDiv by_per;
};
// Rows of a wave: row t is base + (t / side) step + t % side, side = 1 << shift of them side by side.
struct Rows {
    int base, shift, side, step;
    __device__ int at(int t) const { return base + (t >> shift) * step + (t & (side - 1)); }
};
__device__ inline Rows rows_of(const Units& u, uint32_t group, int shift) {
    const int turns = u.per == 1 ? 4 : 1, side = 1 << shift, turn = group & (turns - 1);
    return Rows{(int)(group - turn) * u.tokens + turn * side, shift, side, turns * side};
}

// The lane's row, of `lane` as t: page and place in it, page -1 for one that holds nothing and -2 for a row of no
// sequence.
__device__ inline int2 find_place(const Paged& c, int B, int N, const int* __restrict__ first,
                                  const int* __restrict__ len, const Rows& rows, int tokens) {
    const int lane = threadIdx.x & 63, n = rows.at(lane);
    const bool any = lane < tokens && n < N;
    int b = n;
    long long behind = 1;
    if (first) {
        b = 0;
        if (B <= 64) {   // all beginnings at once, then each token against them
            const int v = first[min(lane, B - 1)];
            for (int i = 0; i < tokens; ++i) {
                const int k = max(__popcll(__ballot(lane < B && v <= rows.at(i))), 1) - 1;
                b = lane == i ? k : b;
            }
        } else {
            int hi = B;
            while (hi - b > 1) {
                const int mid = (b + hi) >> 1;
                if (first[mid] <= n) b = mid;
                else hi = mid;
            }
        }
        behind = any && first[b] <= n ? (long long)first[b + 1] - n : 0;
    }
    int2 at = {-2, 0};
    if (any && behind > 0) {
        const long long t = len[b] - behind;
        at = int2{t < 0 ? -1 : c.page_of(b, (int)t), (int)t & ((1 << c.shift) - 1)};
    }
    return at;
}
__device__ inline int2 lane_of(int2 at, int i) {   // i the same in all lanes
    return int2{__builtin_amdgcn_readlane(at.x, i), __builtin_amdgcn_readlane(at.y, i)};
}

typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));

// 16 bytes of a row: its values, and the bits of the largest |x| (their order is that of the values, NaN above
// infinity).
template <typename T> struct Piece;
template <> struct Piece<float> {
    static constexpr int V = 4;
    __device__ static void values(const u32x4& w, float (&v)[V]) {
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = __builtin_bit_cast(float, (uint32_t)w[e]);
    }
    __device__ static uint32_t most(const u32x4& w) {
        uint32_t m = 0;
#pragma unroll
        for (int e = 0; e < 4; ++e) m = max(m, w[e] & 0x7FFFFFFFu);
        return m;
    }
};
template <> struct Piece<uint16_t> {
    static constexpr int V = 8;
    __device__ static void values(const u32x4& w, float (&v)[V]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            v[2 * e] = __builtin_bit_cast(float, w[e] << 16);
            v[2 * e + 1] = __builtin_bit_cast(float, w[e] & 0xFFFF0000u);
        }
    }
    __device__ static uint32_t most(const u32x4& w) {
        u16x2 m = {0, 0};
#pragma unroll
        for (int e = 0; e < 4; ++e) m = __builtin_elementwise_max(m, __builtin_bit_cast(u16x2, w[e] & 0x7FFF7FFFu));
        return (uint32_t)max(m[0], m[1]) << 16;
    }
};

template <typename T, int V>
__device__ inline void load_piece(const T* p, float (&v)[V]) {
    typedef T vec __attribute__((ext_vector_type(V)));
    const vec x = *reinterpret_cast<const vec*>(p);
#pragma unroll
    for (int e = 0; e < V; ++e) v[e] = paged_up(x[e]);
}
template <typename T, int V>
__device__ inline void store_piece(T* p, const float (&v)[V]) {
    typedef T vec __attribute__((ext_vector_type(V)));
    vec x;
#pragma unroll
    for (int e = 0; e < V; ++e) x[e] = down<T>(v[e]);
    *reinterpret_cast<vec*>(p) = x;
}

// The largest of L lanes' bits, in all of them.
template <int L>
__device__ inline uint32_t group_max(uint32_t v) {
    auto step = [](uint32_t a, float b) { return max(a, __builtin_bit_cast(uint32_t, b)); };
    auto f = [](uint32_t a) { return __builtin_bit_cast(float, a); };
    if (L > 1) v = step(v, dpp_quad_xor1(f(v)));
    if (L > 2) v = step(v, dpp_quad_xor2(f(v)));
    if (L > 4) v = step(v, dpp_half_mirror(f(v)));
    if (L > 8) v = step(v, dpp_row_mirror(f(v)));
    float lo, hi;
    if (L > 16) {
        halves16(f(v), lo, hi);
        v = step(__builtin_bit_cast(uint32_t, lo), hi);
    }
    if (L > 32) {
        halves32(f(v), lo, hi);
        v = step(__builtin_bit_cast(uint32_t, lo), hi);
    }
    return v;
}

// The scale of a row whose largest |x| is m: the correctly rounded m / top, by one step from the product with
// the rounded 1 / top (Markstein, "Computation of elementary functions on the IBM RISC System/6000", 1990).
template <typename CT>
__device__ inline float scale_of(float m) {
    constexpr float top = Code<CT>::top, by = 1.f / top;
    const float s = m * by;
    return fmaf(fmaf(-s, top, m), by, s);
}

// Codes of four values y, rounded.
template <typename CT> __device__ inline uint32_t codes_of(const float (&y)[4]);
template <> __device__ inline uint32_t codes_of<int8_t>(const float (&y)[4]) {
    uint32_t c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)   // 1.5 2^23 leaves the rounded integer in the last bits
        c[e] = __builtin_bit_cast(uint32_t, y[e] + 12582912.f);
    const uint32_t a = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), b = __builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400u);
    return a | b << 16;
}
template <> __device__ inline uint32_t codes_of<uint8_t>(const float (&y)[4]) {
    const int a = __builtin_amdgcn_cvt_pk_fp8_f32(y[0], y[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(y[2], y[3], a, true);
}
// Value of byte e of a word of codes.
template <typename CT> __device__ inline float value_of(uint32_t w, int e);
template <> __device__ inline float value_of<int8_t>(uint32_t w, int e) { return (float)(int8_t)(w >> (8 * e)); }
template <> __device__ inline float value_of<uint8_t>(uint32_t w, int e) {
    return e == 0 ? __builtin_amdgcn_cvt_f32_fp8(w, 0) : e == 1 ? __builtin_amdgcn_cvt_f32_fp8(w, 1)
           : e == 2 ? __builtin_amdgcn_cvt_f32_fp8(w, 2) : __builtin_amdgcn_cvt_f32_fp8(w, 3);
}
// Scale and codes of a row from the bits of its largest |x|.  x times the reciprocal of s, less and more by 2^-21 of it, has
// the exact quotient (which the product is to 2^-22) between: where both round to one code, that is its.  Else the
// border t between the two codes decides: the sign of x - t s, which fma gives exactly, and the even code where it is
// zero.  bf16 rows often have such ties (one row of seven has some), so this path is made short: 32512 x 16 rows of
// 128 bf16 to e4m3 take 43 us without it, 50 with it, 66 with the exact quotient of every value instead.  Scales below 2^-40,
// where remainders could underflow, and rows that are not finite take the exact quotient.
template <typename CT, int V>
__device__ inline float quantise(const float (&x)[V], uint32_t most, uint32_t (&out)[V / 4]) {
    const float m = __builtin_bit_cast(float, most);
    float s = scale_of<CT>(m);
    const bool plain = (s >= 0x1p-40f && most < 0x7F800000u) || most == 0;   // zeros round to zeros
    const float rs = plain && most > 0 ? __builtin_amdgcn_rcpf(s) : 0.f;
    const float below = rs * (1.f - 0x1p-21f), above = rs * (1.f + 0x1p-21f);
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
        float lo[4], hi[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) lo[e] = x[4 * i + e] * below, hi[e] = x[4 * i + e] * above;
        out[i] = codes_of<CT>(lo);
        const uint32_t up = codes_of<CT>(hi);
        if (!__any(out[i] != up)) continue;
        uint32_t pick = 0;   // bytes of up
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float t = 0.5f * (value_of<CT>(out[i], e) + value_of<CT>(up, e));
            const float r = fmaf(-fabsf(t), s, fabsf(x[4 * i + e]));
            if (r > 0.f || (r == 0.f && (out[i] >> (8 * e) & 1))) pick |= 0xFFu << (8 * e);
        }
        out[i] = (out[i] & ~pick) | (up & pick);
    }
    if (!__any(!plain)) return s;
    const float exact = most >= 0x7F800000u ? __builtin_nanf("") : m / Code<CT>::top;
    const float f = exact < 0x1p-40f ? 0x1p64f : 1.f;   // both up by 2^64
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e)
            y[e] = exact > 0.f ? fminf(fmaxf(quotient(x[4 * i + e] * f, exact * f), -Code<CT>::top), Code<CT>::top) : 0.f;
        const uint32_t codes = codes_of<CT>(y);
        out[i] = plain ? out[i] : codes;
    }
    return plain ? s : exact;
}

template <typename T, typename CT, int L, bool MANY>
__global__ void __launch_bounds__(256) cache_write_pieces(Paged c, Units u, int B, int N, const int* __restrict__ first,
                                                          const int* __restrict__ len, const T* __restrict__ K,
                                                          Strides sk, const T* __restrict__ V, Strides sv) {
    constexpr int P = Piece<T>::V, G = 64 / L;
    constexpr bool scaled = sizeof(CT) == 1;
    const int lane = threadIdx.x & 63, piece = lane & (L - 1), sub = lane / L;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool in = piece * P < c.D;
    const uint32_t unit = 4 * blockIdx.x + wave;
    if (unit >= u.units) return;
    const uint32_t group = fdiv(unit, u.by_per);
    const Rows rows = rows_of(u, group, MANY ? __builtin_ctz(G) - u.log_heads : 0);
    const int j0 = (unit - group * u.per) * u.each, j1 = min(j0 + u.each, u.blocks);   // blocks of heads
    u32x4 x[2];
    // Head h0 of the wave (the lane's own where MANY) of token i.  Lanes without one read another's row.
    auto load = [&](int i, int h0) {
        const int h = min(MANY ? h0 : h0 + sub, c.Hk - 1), e = in ? piece * P : 0;
        const long long n = min(rows.at(min(i, u.tokens - 1)), N - 1);
        x[0] = *reinterpret_cast<const u32x4*>(K + n * sk.token + h * sk.head + e);
        x[1] = *reinterpret_cast<const u32x4*>(V + n * sv.token + h * sv.head + e);
    };
    auto store = [&](int2 at, int h0, bool any) {
        const int h = MANY ? h0 : h0 + sub;
        const bool there = any && h < c.Hk && at.x >= 0;
        const long long row = c.row(at.x, h, at.y);
#pragma unroll
        for (int side = 0; side < 2; ++side) {
            const u32x4 w = x[side];
            CT* o = (CT*)(side ? c.V : c.K) + row * c.D + piece * P;
            if constexpr (!scaled) {
                if (there && in) *reinterpret_cast<u32x4*>(o) = w;
            } else {
                uint32_t out[P / 4];
                float v[P];
                Piece<T>::values(w, v);
                const float s = quantise<CT, P>(v, group_max<L>(Piece<T>::most(w)), out);
                if (there && piece == 0) (side ? c.Vs : c.Ks)[row] = s;
                if (there && in) {
                    if constexpr (P == 8) *reinterpret_cast<u32x2*>(o) = u32x2{out[0], out[1]};
                    else *reinterpret_cast<uint32_t*>(o) = out[0];
                }
            }
        }
    };
    if constexpr (MANY) {
        const int h = sub & ((1 << u.log_heads) - 1);
        int i = first_token(sub, u.log_heads);
        load(i, h);   // on their way while the places are found
        const int2 places = find_place(c, B, N, first, len, rows, u.tokens);
        for (int i0 = 0; i0 < u.tokens; i0 += rows.side) {
            const int2 at = {__shfl(places.x, min(i, 63)), __shfl(places.y, min(i, 63))};
            store(at, h, i < u.tokens);
            i += rows.side;
            load(i, h);
        }
    } else {
        load(0, j0 * G);
        const int2 places = find_place(c, B, N, first, len, rows, u.tokens);
        for (int i = 0, j = j0; i < u.tokens && rows.at(i) < N;) {
            store(lane_of(places, i), j * G, true);
            if (++j == j1) j = j0, ++i;
            if (i < u.tokens) load(i, j * G);
        }
    }
}

// P values of a cache's type.
template <typename CT, int V>
__device__ inline void load_codes(const CT* p, float (&v)[V]) {
    if constexpr (sizeof(CT) > 1) {
        load_piece<CT, V>(p, v);
    } else {
        uint32_t w[V / 4];
        if constexpr (V == 8) {
            const u32x2 x = *reinterpret_cast<const u32x2*>(p);
            w[0] = x[0], w[1] = x[1];
        } else {
            w[0] = *reinterpret_cast<const uint32_t*>(p);
        }
#pragma unroll
        for (int i = 0; i < V / 4; ++i) {
            if constexpr (__is_same(CT, int8_t)) {
#pragma unroll
                for (int e = 0; e < 4; ++e) v[4 * i + e] = (float)(int8_t)(w[i] >> (8 * e));
            } else {
                v[4 * i] = __builtin_amdgcn_cvt_f32_fp8(w[i], 0), v[4 * i + 1] = __builtin_amdgcn_cvt_f32_fp8(w[i], 1);
                v[4 * i + 2] = __builtin_amdgcn_cvt_f32_fp8(w[i], 2), v[4 * i + 3] = __builtin_amdgcn_cvt_f32_fp8(w[i], 3);
            }
        }
    }
}

template <typename T, typename CT, int L, bool MANY>
__global__ void __launch_bounds__(256) cache_read_pieces(Paged c, Units u, int B, int N, const int* __restrict__ first,
                                                         const int* __restrict__ len, T* __restrict__ K, Strides sk,
                                                         T* __restrict__ V, Strides sv) {
    constexpr int P = Piece<T>::V, G = 64 / L, AHEAD = 2;
    constexpr bool scaled = sizeof(CT) == 1;
    const int lane = threadIdx.x & 63, piece = lane & (L - 1), sub = lane / L;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool in = piece * P < c.D;
    const uint32_t unit = 4 * blockIdx.x + wave;
    if (unit >= u.units) return;
    const uint32_t group = fdiv(unit, u.by_per);
    const Rows rows = rows_of(u, group, MANY ? __builtin_ctz(G) - u.log_heads : 0);
    const int j0 = (unit - group * u.per) * u.each, j1 = min(j0 + u.each, u.blocks);   // blocks of heads
    const int2 places = find_place(c, B, N, first, len, rows, u.tokens);
    // AHEAD heads of the lane, G apart (MANY: head h0 of AHEAD tokens, side by side).
    auto move = [&](const int2 (&at)[AHEAD], int i, int h0) {
        float x[AHEAD][2][P], s[AHEAD][2];
        const int h = MANY ? h0 : h0 + sub, e = in ? piece * P : 0;
        const long long row0 = MANY ? 0 : c.row(max(at[0].x, 0), min(h, c.Hk - 1), at[0].y);
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {   // lanes without a row read another's
            const long long row = MANY ? c.row(max(at[a].x, 0), min(h, c.Hk - 1), at[a].y)
                                       : row0 + ((long long)min(a * G, max(c.Hk - 1 - h, 0)) << c.shift);
#pragma unroll
            for (int side = 0; side < 2; ++side) {
                s[a][side] = 1.f;
                if constexpr (scaled) s[a][side] = (side ? c.Vs : c.Ks)[row];
                load_codes<CT, P>((const CT*)(side ? c.V : c.K) + row * c.D + e, x[a][side]);
            }
        }
#pragma unroll
        for (int a = 0; a < AHEAD; ++a) {
            const long long n = rows.at(MANY ? i + a * rows.side : i);
            const int ha = h + (MANY ? 0 : a * G);
            const bool there = in && at[a].x >= -1 && ha < c.Hk;
#pragma unroll
            for (int side = 0; side < 2; ++side) {
                if constexpr (scaled)
#pragma unroll
                    for (int e = 0; e < P; ++e) x[a][side][e] *= s[a][side];
                if (at[a].x < 0)
#pragma unroll
                    for (int e = 0; e < P; ++e) x[a][side][e] = 0.f;
                if (there)
                    store_piece<T, P>((side ? V + n * sv.token + ha * sv.head : K + n * sk.token + ha * sk.head) + piece * P,
                                      x[a][side]);
            }
        }
    };
    int2 at[AHEAD];
    if constexpr (MANY) {
        const int h = sub & ((1 << u.log_heads) - 1), rounds = rounds_of(u.tokens, rows.side, AHEAD);
        for (int k = 0, i = first_token(sub, u.log_heads); k < rounds; ++k, i += AHEAD * rows.side) {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int t = i + a * rows.side;
                at[a] = int2{__shfl(places.x, min(t, 63)), __shfl(places.y, min(t, 63))};
                if (t >= u.tokens) at[a].x = -2;
            }
            move(at, i, h);
        }
    } else {
        for (int i = 0; i < u.tokens && rows.at(i) < N; ++i) {
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) at[a] = lane_of(places, i);
            for (int j = j0; j < j1; ++j) move(at, i, j * AHEAD * G);
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------
int groups_of(long long rows) {
    const long long groups = (rows + 3) / 4, most = num_cus() * 32LL;
    return (int)(groups < most ? groups : most);
}

Units units_of(int N, int Hk, int places, int ahead) {
    const Split s = split_tokens(N, Hk, places, ahead);
    return Units{s, make_fastdiv(s.per)};
}
bool whole_pieces(const void* p, Strides st, int N, int Hk, int size) {
    const long long bits = (N > 1 ? st.token : 0) | (Hk > 1 ? st.head : 0);
    return ((uintptr_t)p & 15) == 0 && bits * size % 16 == 0;
}
template <typename T, typename CT>
auto by_lanes_write(int L, bool many) {
    return L == 4    ? many ? cache_write_pieces<T, CT, 4, true> : cache_write_pieces<T, CT, 4, false>
           : L == 8  ? many ? cache_write_pieces<T, CT, 8, true> : cache_write_pieces<T, CT, 8, false>
           : L == 16 ? many ? cache_write_pieces<T, CT, 16, true> : cache_write_pieces<T, CT, 16, false>
           : L == 32 ? many ? cache_write_pieces<T, CT, 32, true> : cache_write_pieces<T, CT, 32, false>
                     : cache_write_pieces<T, CT, 64, false>;
}
template <typename T, typename CT>
auto by_lanes_read(int L, bool many) {
    return L == 4    ? many ? cache_read_pieces<T, CT, 4, true> : cache_read_pieces<T, CT, 4, false>
           : L == 8  ? many ? cache_read_pieces<T, CT, 8, true> : cache_read_pieces<T, CT, 8, false>
           : L == 16 ? many ? cache_read_pieces<T, CT, 16, true> : cache_read_pieces<T, CT, 16, false>
           : L == 32 ? many ? cache_read_pieces<T, CT, 32, true> : cache_read_pieces<T, CT, 32, false>
                     : cache_read_pieces<T, CT, 64, false>;
}
template <typename T, typename CT>
int launch_write(const Paged& c, int B, int N, const int* first, const int* len, const void* K, Strides sk,
                 const void* V, Strides sv) {
    if (whole_pieces(K, sk, N, c.Hk, sizeof(T)) && whole_pieces(V, sv, N, c.Hk, sizeof(T))) {
        const int lanes = c.D / Piece<T>::V, L = lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64;
        const Units u = units_of(N, c.Hk, 64 / L, 1);
        auto run = by_lanes_write<T, CT>(L, u.many);
        run<<<(u.units + 3) / 4, 256, 0, stream()>>>(c, u, B, N, first, len, (const T*)K, sk, (const T*)V, sv);
    } else {
        cache_write<T, CT><<<groups_of(2LL * N * c.Hk), 256, 0, stream()>>>(c, B, N, first, len, (const T*)K, sk,
                                                                            (const T*)V, sv);
    }
    return check_launch("dh_kv_cache_write");
}
template <typename T, typename CT>
int launch_read(const Paged& c, int B, int N, const int* first, const int* len, void* K, Strides sk, void* V,
                Strides sv) {
    if (whole_pieces(K, sk, N, c.Hk, sizeof(T)) && whole_pieces(V, sv, N, c.Hk, sizeof(T))) {
        const int lanes = c.D / Piece<T>::V, L = lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64;
        const Units u = units_of(N, c.Hk, 64 / L, 2);
        auto run = by_lanes_read<T, CT>(L, u.many);
        run<<<(u.units + 3) / 4, 256, 0, stream()>>>(c, u, B, N, first, len, (T*)K, sk, (T*)V, sv);
    } else {
        cache_read<T, CT><<<groups_of(2LL * N * c.Hk), 256, 0, stream()>>>(c, B, N, first, len, (T*)K, sk, (T*)V, sv);
    }
    return check_launch("dh_kv_cache_read");
}

int check_tokens(const char* op, int B, int N, int Hk, int D, const int* first, const int* len, const void* K,
                 const long long* sk, const void* V, const long long* sv, bool out) {
    if (N < 0 || N > 1 << 29 || (!first && N != B))
        return set_error(DH_ERR_INVALID, "%s: N=%d tokens of B=%d sequences", op, N, B);
    DH_TRY(check_strides(op, "K", sk, N, Hk, D, out));
    DH_TRY(check_strides(op, "V", sv, N, Hk, D, out));
    if (N > 0 && B > 0 && (!len || !K || !V)) return set_error(DH_ERR_INVALID, "%s: null pointer", op);
    return DH_OK;
}

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" {

int dh_kv_cache_write(int dtype, int cache_type, int B, int N, int Hk, int D, const void* K, const long long* sk,
                      const void* V, const long long* sv, const int* first, const int* len, int pages, int page,
                      const int* table, int ld_table, void* Kc, void* Vc, float* Ks, float* Vs) {
    const char* op = "dh_kv_cache_write";
    Paged c;
    DH_TRY(check_paged(op, dtype, cache_type, B, Hk, D, pages, page, table, ld_table, Kc, Vc, Ks, Vs, c));
    DH_TRY(check_tokens(op, B, N, Hk, D, first, len, K, sk, V, sv, false));
    DH_TRY(ensure_init());
    if (N == 0 || B == 0) return DH_OK;
    auto run = dtype == DH_F32 ? cache_type == DH_F32 ? launch_write<float, float>
                                 : cache_type == DH_I8 ? launch_write<float, int8_t> : launch_write<float, uint8_t>
                               : cache_type == DH_BF16 ? launch_write<uint16_t, uint16_t>
                                 : cache_type == DH_I8 ? launch_write<uint16_t, int8_t>
                                                       : launch_write<uint16_t, uint8_t>;
    return run(c, B, N, first, len, K, Strides{sk[0], sk[1]}, V, Strides{sv[0], sv[1]});
}

int dh_kv_cache_read(int dtype, int cache_type, int B, int N, int Hk, int D, void* K, const long long* sk, void* V,
                     const long long* sv, const int* first, const int* len, int pages, int page, const int* table,
                     int ld_table, const void* Kc, const void* Vc, const float* Ks, const float* Vs) {
    const char* op = "dh_kv_cache_read";
    Paged c;
    DH_TRY(check_paged(op, dtype, cache_type, B, Hk, D, pages, page, table, ld_table, Kc, Vc, Ks, Vs, c));
    DH_TRY(check_tokens(op, B, N, Hk, D, first, len, K, sk, V, sv, true));
    DH_TRY(ensure_init());
    if (N == 0 || B == 0) return DH_OK;
    auto run = dtype == DH_F32 ? cache_type == DH_F32 ? launch_read<float, float>
                                 : cache_type == DH_I8 ? launch_read<float, int8_t> : launch_read<float, uint8_t>
                               : cache_type == DH_BF16 ? launch_read<uint16_t, uint16_t>
                                 : cache_type == DH_I8 ? launch_read<uint16_t, int8_t>
                                                       : launch_read<uint16_t, uint8_t>;
    return run(c, B, N, first, len, K, Strides{sk[0], sk[1]}, V, Strides{sv[0], sv[1]});
}

}  // extern "C"
