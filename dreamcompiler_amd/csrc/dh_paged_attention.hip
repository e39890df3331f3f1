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
    int Hq, G, window, max_len, chunk, splits;
    float scale;
    const int* len;
    float* part;    // splits x B x Hq rows of D: a chunk's o before its division
    float2* stat;   // as many: its m and sum
    __device__ void span(int b, int& from, int& to) const {
        to = min(max(len[b], 0), max_len);
        from = window > 0 ? max(to - window, 0) : 0;
    }
};

// A wave per chunk of a head.
template <typename T, typename CT>
__global__ void __launch_bounds__(64) paged_chunk(Paged c, Work w, const T* __restrict__ Q, Strides sq,
                                                  T* __restrict__ O, Strides so, float* __restrict__ lse) {
    constexpr int J = PAGED_MOST_D / 64;
    const int lane = threadIdx.x, split = blockIdx.x, h = blockIdx.y, b = blockIdx.z, hk = h / w.G;
    int from, to;
    w.span(b, from, to);
    const int t0 = from + split * w.chunk, t1 = min(t0 + w.chunk, to);
    float q[J], o[J] = {}, m = -INFINITY, sum = 0.f;
#pragma unroll
    for (int j = 0; j < J; ++j) {
        const int e = 64 * j + lane;
        q[j] = e < c.D ? paged_up(Q[b * sq.seq + h * sq.head + e]) * w.scale : 0.f;
    }
    for (int t = t0; t < t1; ++t) {
        const int id = c.page_of(b, t);
        if (id < 0) continue;
        const long long row = c.row(id, hk, t & ((1 << c.shift) - 1));
        const CT* k = (const CT*)c.K + row * c.D;
        const CT* v = (const CT*)c.V + row * c.D;
        float z = 0.f, ks = 1.f, vs = 1.f;
        if constexpr (sizeof(CT) == 1) ks = c.Ks[row], vs = c.Vs[row];
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (64 * j + lane < c.D) z += q[j] * paged_up(k[64 * j + lane]);
        z = wave_reduce(z, OpSum()) * ks;
        const float most = fmaxf(m, z), base = most == -INFINITY ? 0.f : most;
        const float old = __expf(m - base), p = __expf(z - base);
        sum = sum * old + p;
#pragma unroll
        for (int j = 0; j < J; ++j)
            if (64 * j + lane < c.D) o[j] = o[j] * old + p * vs * paged_up(v[64 * j + lane]);
        m = most;
    }
    if (w.splits == 1) {
        for (int j = 0; j < J; ++j)
            if (64 * j + lane < c.D)
                O[b * so.seq + h * so.head + 64 * j + lane] = down<T>(sum == 0.f ? 0.f : o[j] / sum);
        if (lse && lane == 0) lse[(long long)b * w.Hq + h] = sum == 0.f ? -INFINITY : m + logf(sum);
        return;
    }
    const long long at = ((long long)split * gridDim.z + b) * w.Hq + h;
    for (int j = 0; j < J; ++j)
        if (64 * j + lane < c.D) w.part[at * c.D + 64 * j + lane] = o[j];
    if (lane == 0) w.stat[at] = float2{m, sum};
}

// A wave per head joins its chunks in order.
template <typename T>
__global__ void __launch_bounds__(64) paged_join(Work w, int D, T* __restrict__ O, Strides so,
                                                 float* __restrict__ lse) {
    const int lane = threadIdx.x, h = blockIdx.x, b = blockIdx.y;
    int from, to;
    w.span(b, from, to);
    const int n = min(w.splits, (to - from + w.chunk - 1) / w.chunk);
    const long long step = (long long)gridDim.y * w.Hq, at = (long long)b * w.Hq + h;
    float m = -INFINITY, sum = 0.f;
    for (int i = 0; i < n; ++i) m = fmaxf(m, w.stat[i * step + at].x);
    const float base = m == -INFINITY ? 0.f : m;
    float o[PAGED_MOST_D / 64] = {};
    for (int i = 0; i < n; ++i) {
        const float2 s = w.stat[i * step + at];
        const float f = __expf(s.x - base);
        sum += s.y * f;
        for (int j = 0; j < PAGED_MOST_D / 64; ++j)
            if (64 * j + lane < D) o[j] += f * w.part[(i * step + at) * D + 64 * j + lane];
    }
    for (int j = 0; j < PAGED_MOST_D / 64; ++j)
        if (64 * j + lane < D) O[b * so.seq + h * so.head + 64 * j + lane] = down<T>(sum == 0.f ? 0.f : o[j] / sum);
    if (lse && lane == 0) lse[at] = sum == 0.f ? -INFINITY : m + logf(sum);
}

// Tokens of a chunk and the most chunks of a sequence.
void plan(int B, int Hq, int max_len, int& chunk, int& splits) {
    const long long rows = (long long)B * Hq;
    chunk = 256;
    while (rows * ((max_len + (long long)chunk - 1) / chunk) > 65536 && chunk < max_len) chunk *= 2;
    splits = max_len > chunk ? (max_len + chunk - 1) / chunk : 1;
}
size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

template <typename T, typename CT>
int launch(const Paged& c, const Work& w, int B, const void* Q, Strides sq, void* O, Strides so, float* lse) {
    paged_chunk<T, CT><<<dim3(w.splits, w.Hq, B), 64, 0, stream()>>>(c, w, (const T*)Q, sq, (T*)O, so, lse);
    DH_TRY(check_launch("dh_paged_attention"));
    if (w.splits == 1) return DH_OK;
    paged_join<T><<<dim3(w.Hq, B), 64, 0, stream()>>>(w, c.D, (T*)O, so, lse);
    return check_launch("dh_paged_attention");
}

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" {

size_t dh_paged_attention_workspace(int cache_type, int B, int Hq, int Hk, int D, int max_len) {
    if (B < 1 || Hq < 1 || Hk < 1 || D < 1 || max_len < 1) return 0;
    int chunk, splits;
    plan(B, Hq, max_len, chunk, splits);
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
    if (window < 0 || max_len < 0 || (long long)max_len > (long long)ld_table * page)
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
    Work w{Hq, Hq / Hk, window, max_len, 0, 0, scale, len, nullptr, nullptr};
    plan(B, Hq, max_len, w.chunk, w.splits);
    w.part = (float*)ws;
    w.stat = (float2*)((char*)ws + up256((size_t)w.splits * B * Hq * D * 4));
    auto run = dtype == DH_F32 ? cache_type == DH_F32 ? launch<float, float>
                                 : cache_type == DH_I8 ? launch<float, int8_t> : launch<float, uint8_t>
                               : cache_type == DH_BF16 ? launch<uint16_t, uint16_t>
                                 : cache_type == DH_I8 ? launch<uint16_t, int8_t> : launch<uint16_t, uint8_t>;
    return run(c, w, B, Q, Strides{sq[0], sq[1]}, O, Strides{so[0], so[1]}, lse);
}

}  // extern "C"
