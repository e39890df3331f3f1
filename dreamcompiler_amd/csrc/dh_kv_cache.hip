// dh_kv_cache.hip -- keys and values of new tokens into a paged cache, rounded to 8 bits where its
// type has them, and read back.
//
//   8 bits: s = max |x| / top over a row of D (top 127 for integers, 448 for e4m3), value = x / s
//   rounded to the nearest, ties to even; it stands for value * s
//
// The scale is the fp32 quotient; the values are those of the exact quotient by it (`quotient`), so
// that they do not hang on how a division rounds.  A row with an infinity or a NaN gets a NaN as its
// scale, and reads back as NaN.  Bound by HBM.
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
// A row is L lanes of V values, 16 bytes of the model's type; a wave takes 64 / L of a token's 2 Hk rows (keys
// of all heads, then values) at once, `rows` of them in all: a token's whole where there are many tokens.
struct Units {
    int rows, per;   // of a unit, units of a token
    long long n;
};

template <typename T> struct Piece;
template <> struct Piece<float> { static constexpr int V = 4; };
template <> struct Piece<uint16_t> { static constexpr int V = 8; };

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

// Codes of four values x / s.  A quotient's neighbours 2^-22 of it below and above x (1 / s) have the exact one
// between them: where both round to one code, that is its; else (3 of 10^5 values) the wave takes the
// exact quotient's.
template <typename CT> __device__ inline uint32_t codes_of(const float (&y)[4]);
template <> __device__ inline uint32_t codes_of<int8_t>(const float (&y)[4]) {
    uint32_t c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e)   // 1.5 2^23 leaves the rounded integer in the last bits
        c[e] = __builtin_bit_cast(uint32_t, fminf(fmaxf(y[e], -127.f), 127.f) + 12582912.f);
    const uint32_t a = __builtin_amdgcn_perm(c[1], c[0], 0x0c0c0400u), b = __builtin_amdgcn_perm(c[3], c[2], 0x0c0c0400u);
    return a | b << 16;
}
template <> __device__ inline uint32_t codes_of<uint8_t>(const float (&y)[4]) {
    float v[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) v[e] = fminf(fmaxf(y[e], -448.f), 448.f);
    const int a = __builtin_amdgcn_cvt_pk_fp8_f32(v[0], v[1], 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(v[2], v[3], a, true);
}
template <typename CT, int V>
__device__ inline void codes(const float (&x)[V], float s, float rs, uint32_t (&out)[V / 4]) {
    bool unsure = false;
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
        float lo[4], hi[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const float y = x[4 * i + e] * rs;
            lo[e] = y * (1.f - 0x1p-22f);
            hi[e] = y * (1.f + 0x1p-22f);
        }
        out[i] = codes_of<CT>(lo);
        unsure |= out[i] != codes_of<CT>(hi);
    }
    if (!__any(unsure)) return;
#pragma unroll
    for (int i = 0; i < V / 4; ++i) {
        float y[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) y[e] = quotient(x[4 * i + e], s);
        out[i] = codes_of<CT>(y);
    }
}

template <typename T, typename CT, int L>
__global__ void __launch_bounds__(256) cache_write_pieces(Paged c, Units u, int B, const int* __restrict__ first,
                                                          const int* __restrict__ len, const T* __restrict__ K,
                                                          Strides sk, const T* __restrict__ V, Strides sv) {
    constexpr int P = Piece<T>::V, G = 64 / L, AHEAD = 4;
    constexpr bool scaled = sizeof(CT) == 1;
    const int lane = threadIdx.x & 63, piece = lane & (L - 1), sub = lane / L;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool in = piece * P < c.D;
    for (long long i = 4LL * blockIdx.x + wave; i < u.n; i += 4LL * gridDim.x) {
        const int n = (int)(i / u.per), r0 = (int)(i - (long long)n * u.per) * u.rows, r1 = min(r0 + u.rows, 2 * c.Hk);
        int id = -1, at = 0;
        for (int r = r0; r < r1; r += AHEAD * G) {
            float x[AHEAD][P];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int k = r + a * G + sub, h = k < c.Hk ? k : k - c.Hk;
#pragma unroll
                for (int e = 0; e < P; ++e) x[a][e] = 0.f;
                if (k < r1 && in)
                    load_piece<T, P>((k < c.Hk ? K + n * sk.token + h * sk.head : V + n * sv.token + h * sv.head) + piece * P,
                                     x[a]);
            }
            if (r == r0) {   // the rows are on their way meanwhile
                int b, t;
                if (!place(first, len, B, n, b, t)) break;
                id = c.page_of(b, t);
                at = t & ((1 << c.shift) - 1);
            }
            if (id < 0) break;
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int k = r + a * G + sub, h = k < c.Hk ? k : k - c.Hk;
                if (r + a * G >= r1) break;
                const long long row = c.row(id, h, at);
                CT* o = (CT*)(k < c.Hk ? c.K : c.V) + row * c.D + piece * P;
                if constexpr (!scaled) {
                    if (k < r1 && in) store_piece<CT, P>(o, x[a]);
                } else {
                    uint32_t most = 0, out[P / 4];
#pragma unroll
                    for (int e = 0; e < P; ++e) most = max(most, __builtin_bit_cast(uint32_t, x[a][e]) & 0x7FFFFFFFu);
                    most = group_max<L>(most);
                    const float s = most >= 0x7F800000u ? __builtin_nanf("")
                                                        : __builtin_bit_cast(float, most) / Code<CT>::top;
                    if (k < r1 && piece == 0) (k < c.Hk ? c.Ks : c.Vs)[row] = s;
                    const float f = s < 0x1p-40f ? 0x1p64f : 1.f, sf = s > 0.f ? s * f : 1.f;
#pragma unroll
                    for (int e = 0; e < P; ++e) x[a][e] = s > 0.f ? x[a][e] * f : 0.f;
                    codes<CT, P>(x[a], sf, 1.f / sf, out);
                    if (k < r1 && in) {
                        if constexpr (P == 8) *reinterpret_cast<u32x2*>(o) = u32x2{out[0], out[1]};
                        else *reinterpret_cast<uint32_t*>(o) = out[0];
                    }
                }
            }
        }
    }
}

// V values of a cache's type.
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

template <typename T, typename CT, int L>
__global__ void __launch_bounds__(256) cache_read_pieces(Paged c, Units u, int B, const int* __restrict__ first,
                                                         const int* __restrict__ len, T* __restrict__ K, Strides sk,
                                                         T* __restrict__ V, Strides sv) {
    constexpr int P = Piece<T>::V, G = 64 / L, AHEAD = 4;
    constexpr bool scaled = sizeof(CT) == 1;
    const int lane = threadIdx.x & 63, piece = lane & (L - 1), sub = lane / L;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const bool in = piece * P < c.D;
    for (long long i = 4LL * blockIdx.x + wave; i < u.n; i += 4LL * gridDim.x) {
        const int n = (int)(i / u.per), r0 = (int)(i - (long long)n * u.per) * u.rows, r1 = min(r0 + u.rows, 2 * c.Hk);
        int b, t;
        if (!place(first, len, B, n, b, t)) continue;
        const int id = c.page_of(b, t), at = t & ((1 << c.shift) - 1);
        for (int r = r0; r < r1; r += AHEAD * G) {
            float x[AHEAD][P], s[AHEAD];
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int k = r + a * G + sub, h = k < c.Hk ? k : k - c.Hk;
                s[a] = 1.f;
#pragma unroll
                for (int e = 0; e < P; ++e) x[a][e] = 0.f;
                if (k < r1 && in && id >= 0) {
                    const long long row = c.row(id, h, at);
                    if constexpr (scaled) s[a] = (k < c.Hk ? c.Ks : c.Vs)[row];
                    load_codes<CT, P>((const CT*)(k < c.Hk ? c.K : c.V) + row * c.D + piece * P, x[a]);
                }
            }
#pragma unroll
            for (int a = 0; a < AHEAD; ++a) {
                const int k = r + a * G + sub, h = k < c.Hk ? k : k - c.Hk;
                if (k >= r1 || !in) continue;
                if constexpr (scaled)
#pragma unroll
                    for (int e = 0; e < P; ++e) x[a][e] *= s[a];
                store_piece<T, P>((k < c.Hk ? K + n * sk.token + h * sk.head : V + n * sv.token + h * sv.head) + piece * P,
                                  x[a]);
            }
        }
    }
}

// ---- host ----------------------------------------------------------------------------------------
int groups_of(long long rows) {
    const long long groups = (rows + 3) / 4, most = num_cus() * 32LL;
    return (int)(groups < most ? groups : most);
}

// Rows of a unit: all of a token's where that gives each of the GPU's 8192 waves a unit, else as few
// as the wave takes at once.
Units units_of(int N, int rows, int at_once) {
    int per = (rows + at_once - 1) / at_once, each = (int)(N >= 8192 ? per : ((long long)N * per + 8191) / 8192);
    if (each < 1) each = 1;
    per = (per + each - 1) / each;
    return Units{each * at_once, per, (long long)N * per};
}
bool whole_pieces(const void* p, Strides st, int N, int Hk, int size) {
    const long long bits = (N > 1 ? st.token : 0) | (Hk > 1 ? st.head : 0);
    return ((uintptr_t)p & 15) == 0 && bits * size % 16 == 0;
}
int piece_groups(const Units& u) {
    const long long groups = (u.n + 3) / 4;
    return (int)(groups < 1 << 20 ? groups : 1 << 20);
}

template <typename T, typename CT>
int launch_write(const Paged& c, int B, int N, const int* first, const int* len, const void* K, Strides sk,
                 const void* V, Strides sv) {
    if (whole_pieces(K, sk, N, c.Hk, sizeof(T)) && whole_pieces(V, sv, N, c.Hk, sizeof(T))) {
        const int lanes = c.D / Piece<T>::V, L = lanes <= 4 ? 4 : lanes <= 8 ? 8 : lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64;
        const Units u = units_of(N, 2 * c.Hk, 64 / L);
        auto run = L == 4 ? cache_write_pieces<T, CT, 4> : L == 8 ? cache_write_pieces<T, CT, 8>
                   : L == 16 ? cache_write_pieces<T, CT, 16> : L == 32 ? cache_write_pieces<T, CT, 32>
                                                                       : cache_write_pieces<T, CT, 64>;
        run<<<piece_groups(u), 256, 0, stream()>>>(c, u, B, first, len, (const T*)K, sk, (const T*)V, sv);
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
        const Units u = units_of(N, 2 * c.Hk, 64 / L);
        auto run = L == 4 ? cache_read_pieces<T, CT, 4> : L == 8 ? cache_read_pieces<T, CT, 8>
                   : L == 16 ? cache_read_pieces<T, CT, 16> : L == 32 ? cache_read_pieces<T, CT, 32>
                                                                      : cache_read_pieces<T, CT, 64>;
        run<<<piece_groups(u), 256, 0, stream()>>>(c, u, B, first, len, (T*)K, sk, (T*)V, sv);
    } else {
        cache_read<T, CT><<<groups_of(2LL * N * c.Hk), 256, 0, stream()>>>(c, B, N, first, len, (T*)K, sk, (T*)V, sv);
    }
    return check_launch("dh_kv_cache_read");
}

int check_tokens(const char* op, int B, int N, int Hk, int D, const int* first, const int* len, const void* K,
                 const long long* sk, const void* V, const long long* sv, bool out) {
    if (N < 0 || N > 0x7FF00000 || (!first && N != B))
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
