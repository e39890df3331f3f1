// dh_embedding.hip -- embedding lookup with scaling, and its gradient by sorted tokens.
//
//   Y[n] = s W[id[n]]          dW[v] (+)= s * sum of dY[n] over id[n] = v
//
// An id outside 0 .. V-1 is padding: a zero row of Y, no gradient.  Both are HBM-bound: the
// lookup reads N rows and writes N rows, the gradient reads N rows of dY and writes every row
// of dW (the rows that have tokens, when it accumulates).
//
// The gradient sorts the tokens by id (stable, so a table row's tokens stay in order), then adds
// each run of equal ids in token order: no floating-point atomics, reruns are bit-identical.
//   sort     LSD radix, digits of at most 9 bits (2 passes up to 262143 rows), in LDS for one
//            work-group's worth of tokens, else a histogram and a scatter launch per pass
//   sum      a wave adds EMB_CHUNK sorted tokens of a 64-lane slab of columns; runs that end
//            inside the chunk go to dW, those that cross its ends to fp32 partials
//   join     partials of a run that crosses chunks, added in order by its first chunk's group
#include "dh_common.hpp"

namespace dh {
namespace {

constexpr int EMB_TILE = 8192;     // tokens one work-group sorts
constexpr int EMB_CHUNK = 16;      // sorted tokens added by one wave
constexpr int EMB_BITS = 9, EMB_BINS = 1 << EMB_BITS;

// ---- rows as 16-byte chunks at element alignment ---------------------------------------------
template <typename T> struct RowType;
template <> struct RowType<float> {
    static constexpr int E = 4;                       // elements per chunk
    typedef float vec __attribute__((ext_vector_type(4), aligned(4)));
    __device__ static float up(float x) { return x; }
    __device__ static float down(float x) { return x; }
};
template <> struct RowType<uint16_t> {
    static constexpr int E = 8;
    typedef uint16_t vec __attribute__((ext_vector_type(8), aligned(2)));
    __device__ static float up(uint16_t x) { return bf16_bits_to_f32(x); }
    // One rounding to nearest even of the fp32 value: the type of the result holds no more.
    __device__ static uint16_t down(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
};

// Columns c .. c + E - 1 of a row of D values, zero past its end.
template <typename T, int E>
__device__ inline void load_cols(const T* __restrict__ p, int c, int D, float (&v)[E]) {
    static_assert(E % RowType<T>::E == 0, "whole chunks");
    constexpr int R = RowType<T>::E;
#pragma unroll
    for (int q = 0; q < E / R; ++q) {
        if (c + R * (q + 1) <= D) {
            const auto x = *reinterpret_cast<const typename RowType<T>::vec*>(p + c + R * q);
#pragma unroll
            for (int e = 0; e < R; ++e) v[R * q + e] = RowType<T>::up(x[e]);
        } else {
#pragma unroll
            for (int e = 0; e < R; ++e)
                v[R * q + e] = c + R * q + e < D ? RowType<T>::up(p[c + R * q + e]) : 0.f;
        }
    }
}
template <typename T, int E>
__device__ inline void store_cols(T* __restrict__ p, int c, int D, const float (&v)[E]) {
    constexpr int R = RowType<T>::E;
#pragma unroll
    for (int q = 0; q < E / R; ++q) {
        if (c + R * (q + 1) <= D) {
            typename RowType<T>::vec x;
#pragma unroll
            for (int e = 0; e < R; ++e) x[e] = RowType<T>::down(v[R * q + e]);
            __builtin_nontemporal_store(x, reinterpret_cast<typename RowType<T>::vec*>(p + c + R * q));
        } else {
#pragma unroll
            for (int e = 0; e < R; ++e)
                if (c + R * q + e < D) p[c + R * q + e] = RowType<T>::down(v[R * q + e]);
        }
    }
}

// ---- lookup ------------------------------------------------------------------------------------
// A wave per row and slab of 64 chunks of 8 columns, four rows of one slab in flight.
template <typename T>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(const int* __restrict__ ids, int N, int V,
                                                            int D, float scale,
                                                            const T* __restrict__ W, int ldw,
                                                            T* __restrict__ Y, int ldy) {
    constexpr int E = RowType<T>::E;
    const int lane = threadIdx.x & 63;
    const int c = (blockIdx.y * 64 + lane) * E;
    if (c >= D) return;
    const long long wave = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    const long long waves = (long long)gridDim.x * 4;
    for (long long n = wave; n < N; n += waves) {
        const int id = ids[n];
        float v[E];
        if ((unsigned)id < (unsigned)V) {
            load_cols<T, E>(W + (size_t)id * ldw, c, D, v);
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] *= scale;
        } else {
#pragma unroll
            for (int e = 0; e < E; ++e) v[e] = 0.f;
        }
        store_cols<T, E>(Y + (size_t)n * ldy, c, D, v);
    }
}

// ---- sort --------------------------------------------------------------------------------------
// Stable ranks of a tile's digits: the tile's items sit wave by wave, row by row (item j of lane
// l in wave w is w * 64 * ITEMS + 64 j + l), so their order is the order of (w, j, l).  Lanes with
// the same digit find each other by ballots; cnt[w][d] counts the wave's earlier ones.  Returns
// each item's rank among the tile's items of its digit; base[d] = first place of digit d in the
// tile, total[d] the digit's items.  Items past the tile's end have digit -1.
template <int ITEMS>
__device__ inline void tile_ranks(const int (&digit)[ITEMS], int bits, uint16_t (*cnt)[EMB_BINS],
                                  int* base, int (&rank)[ITEMS]) {
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int bins = 1 << bits;
    for (int i = threadIdx.x; i < 16 * EMB_BINS; i += 1024) (&cnt[0][0])[i] = 0;
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        uint64_t peers = __ballot(digit[j] >= 0);
        for (int b = 0; b < bits; ++b) {
            const uint64_t set = __ballot((digit[j] >> b) & 1);
            peers &= (digit[j] >> b) & 1 ? set : ~set;
        }
        if (digit[j] >= 0) {
            const int before = __popcll(peers & ((1ull << lane) - 1));
            const int c = cnt[w][digit[j]];
            rank[j] = c + before;
            // the wave's lanes have read the count before its first peer raises it
            __builtin_amdgcn_wave_barrier();
            if (before == 0) cnt[w][digit[j]] = (uint16_t)(c + __popcll(peers));
        }
        __builtin_amdgcn_wave_barrier();
    }
    __syncthreads();
    // Per digit: exclusive counts over the waves, then exclusive over the digits (512 threads).
    int total = 0;
    if ((int)threadIdx.x < bins) {
        for (int x = 0; x < 16; ++x) {
            const int c = cnt[x][threadIdx.x];
            cnt[x][threadIdx.x] = (uint16_t)total;
            total += c;
        }
    }
    if (threadIdx.x < EMB_BINS) base[threadIdx.x] = total;
    __syncthreads();
    if (w == 0) {   // 8 digits per lane of one wave
        int s[8], sum = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            s[e] = sum;
            sum += base[8 * lane + e];
        }
        int inc = sum;
        for (int m = 1; m < 64; m <<= 1) {
            const int o = __shfl_up(inc, m, 64);
            if (lane >= m) inc += o;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) base[8 * lane + e] = s[e] + inc - sum;
    }
    __syncthreads();
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
        if (digit[j] >= 0) rank[j] += cnt[w][digit[j]];
}

__device__ inline int key_of(int id, int V) { return (unsigned)id < (unsigned)V ? id : V; }

// All passes of at most EMB_TILE tokens in one work-group: (key, position) pairs go through LDS
// between passes.  Also marks the table rows that have a token.  Latency-bound.
__global__ void __launch_bounds__(1024) sort_small(const int* __restrict__ ids, int N, int V,
                                                   int passes, int bits, int* __restrict__ key_out,
                                                   int* __restrict__ pos_out,
                                                   uint8_t* __restrict__ present) {
    constexpr int ITEMS = EMB_TILE / 1024;
    __shared__ int skey[EMB_TILE];
    __shared__ uint16_t spos[EMB_TILE];
    __shared__ uint16_t cnt[16][EMB_BINS];
    __shared__ int base[EMB_BINS];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    if (present)
        for (int v = threadIdx.x; v < (V + 3) / 4; v += 1024)
            reinterpret_cast<uint32_t*>(present)[v] = 0u;
    int key[ITEMS], pos[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        const int i = w * 64 * ITEMS + 64 * j + lane;
        key[j] = i < N ? key_of(ids[i], V) : -1;
        pos[j] = i;
    }
    for (int p = 0; p < passes; ++p) {
        int digit[ITEMS], rank[ITEMS];
#pragma unroll
        for (int j = 0; j < ITEMS; ++j)
            digit[j] = key[j] < 0 ? -1 : (key[j] >> (p * bits)) & ((1 << bits) - 1);
        tile_ranks<ITEMS>(digit, bits, cnt, base, rank);
#pragma unroll
        for (int j = 0; j < ITEMS; ++j)
            if (key[j] >= 0) {
                const int to = base[digit[j]] + rank[j];
                skey[to] = key[j];
                spos[to] = (uint16_t)pos[j];
            }
        __syncthreads();
#pragma unroll
        for (int j = 0; j < ITEMS; ++j) {
            const int i = w * 64 * ITEMS + 64 * j + lane;
            if (i < N) {
                key[j] = skey[i];
                pos[j] = spos[i];
            }
        }
        __syncthreads();
    }
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        const int i = w * 64 * ITEMS + 64 * j + lane;
        if (i >= N) continue;
        key_out[i] = key[j];
        pos_out[i] = pos[j];
        if (present && key[j] < V) present[key[j]] = 1;
    }
}

// One pass over more tokens, first launch: the digit counts of every tile.  hist[tile][digit].
__global__ void __launch_bounds__(1024) sort_hist(const int* __restrict__ in, int raw, int N, int V,
                                                  int shift, int bits, int* __restrict__ hist,
                                                  uint8_t* __restrict__ clear) {
    __shared__ int h[EMB_BINS];
    if (threadIdx.x < EMB_BINS) h[threadIdx.x] = 0;
    if (clear)
        for (long long v = (long long)blockIdx.x * 1024 + threadIdx.x; v < (V + 3) / 4;
             v += (long long)gridDim.x * 1024)
            reinterpret_cast<uint32_t*>(clear)[v] = 0u;
    __syncthreads();
    for (int j = 0; j < EMB_TILE / 1024; ++j) {
        const long long i = (long long)blockIdx.x * EMB_TILE + 1024 * j + threadIdx.x;
        if (i < N) {
            const int k = raw ? key_of(in[i], V) : in[i];
            atomicAdd(&h[(k >> shift) & ((1 << bits) - 1)], 1);
        }
    }
    __syncthreads();
    if (threadIdx.x < EMB_BINS) hist[(size_t)blockIdx.x * EMB_BINS + threadIdx.x] = h[threadIdx.x];
}

// Second launch: every tile to its place.  A digit's tokens of this tile follow all tokens of
// lower digits and this digit's tokens of earlier tiles.
__global__ void __launch_bounds__(1024) sort_scatter(const int* __restrict__ key_in, int raw,
                                                     const int* __restrict__ pos_in, int N, int V,
                                                     int shift, int bits,
                                                     const int* __restrict__ hist,
                                                     int* __restrict__ key_out,
                                                     int* __restrict__ pos_out,
                                                     uint8_t* __restrict__ present) {
    constexpr int ITEMS = EMB_TILE / 1024;
    __shared__ uint16_t cnt[16][EMB_BINS];
    __shared__ int base[EMB_BINS];
    __shared__ int first[EMB_BINS];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    // All tiles' counts of a digit, and those of the tiles before this one: two threads per digit.
    {
        const int d = threadIdx.x & (EMB_BINS - 1), half = threadIdx.x / EMB_BINS;
        int all = 0;
        const int t0 = half == 0 ? 0 : (int)blockIdx.x, t1 = half == 0 ? (int)blockIdx.x : (int)gridDim.x;
        for (int t = t0; t < t1; ++t) all += hist[(size_t)t * EMB_BINS + d];
        if (half == 0) first[d] = all;
        __syncthreads();
        if (half == 1) base[d] = all + first[d];
        __syncthreads();
        if (w == 0) {   // exclusive sum over the digits, 8 per lane
            int s[8], sum = 0;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                s[e] = sum;
                sum += base[8 * lane + e];
            }
            int inc = sum;
            for (int m = 1; m < 64; m <<= 1) {
                const int o = __shfl_up(inc, m, 64);
                if (lane >= m) inc += o;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) first[8 * lane + e] += s[e] + inc - sum;
        }
        __syncthreads();
    }
    int key[ITEMS], pos[ITEMS], digit[ITEMS], rank[ITEMS];
#pragma unroll
    for (int j = 0; j < ITEMS; ++j) {
        const long long i = (long long)blockIdx.x * EMB_TILE + w * 64 * ITEMS + 64 * j + lane;
        key[j] = i < N ? (raw ? key_of(key_in[i], V) : key_in[i]) : -1;
        pos[j] = i < N ? (raw ? (int)i : pos_in[i]) : 0;
        digit[j] = i < N ? (key[j] >> shift) & ((1 << bits) - 1) : -1;
    }
    tile_ranks<ITEMS>(digit, bits, cnt, base, rank);
#pragma unroll
    for (int j = 0; j < ITEMS; ++j)
        if (digit[j] >= 0) {
            const int to = first[digit[j]] + rank[j];
            key_out[to] = key[j];
            pos_out[to] = pos[j];
            if (present && key[j] < V) present[key[j]] = 1;
        }
}

// ---- sums --------------------------------------------------------------------------------------
template <typename OT, int E>
__device__ inline void put_row(OT* __restrict__ row, int c, int D, float scale, int acc,
                               const float (&sum)[E]) {
    float v[E];
#pragma unroll
    for (int e = 0; e < E; ++e) v[e] = sum[e] * scale;
    if (acc) {
        float o[E];
        load_cols<OT, E>(row, c, D, o);
#pragma unroll
        for (int e = 0; e < E; ++e) v[e] += o[e];
    }
    store_cols<OT, E>(row, c, D, v);
}

// Work-groups [0, chunk_groups): a wave per chunk of EMB_CHUNK sorted tokens and slab
// (blockIdx.y) of 512 columns (8 per lane), rows fetched four at a time.  part[chunk][0] is the
// sum of the run that came in from the chunk before, part[chunk][1] that of the run that goes on
// behind it; a run that does both is in part[chunk][0].  The other work-groups (none when
// accumulating) write zeros to the table rows without a token.
template <typename T, typename OT>
__global__ void __launch_bounds__(256) embedding_sum(const int* __restrict__ key,
                                                     const int* __restrict__ pos, int N, int V, int D,
                                                     float scale, const T* __restrict__ dY, int ldy,
                                                     OT* __restrict__ dW, int ldw, int acc,
                                                     float* __restrict__ part, int ldp,
                                                     int chunk_groups,
                                                     const uint8_t* __restrict__ present) {
    constexpr int E = 8, FLY = 4;
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int c = (blockIdx.y * 64 + lane) * E;
    if ((int)blockIdx.x >= chunk_groups) {
        if (c >= D) return;
        const float zero[E] = {};
        const int waves = 4 * (gridDim.x - chunk_groups);
        for (int v = 4 * (blockIdx.x - chunk_groups) + w; v < V; v += waves)
            if (!present[v]) store_cols<OT, E>(dW + (size_t)v * ldw, c, D, zero);
        return;
    }
    const long long chunk = (long long)blockIdx.x * 4 + w;
    const long long i0 = chunk * EMB_CHUNK;
    if (i0 >= N || c >= D) return;
    const int n = (int)(N - i0 < EMB_CHUNK ? N - i0 : EMB_CHUNK);
    int cur = key[i0];
    bool carried = i0 > 0 && key[i0 - 1] == cur;   // the run began in an earlier chunk
    float sum[E] = {};
    for (int j0 = 0; j0 < n; j0 += FLY) {
        float x[FLY][E];
        int k[FLY];
#pragma unroll
        for (int f = 0; f < FLY; ++f) {
            const int j = j0 + f < n ? j0 + f : n - 1;   // past the end: the last token again, unused
            k[f] = key[i0 + j];
            const int p = k[f] < V ? pos[i0 + j] : 0;
            load_cols<T, E>(dY + (size_t)p * ldy, c, D, x[f]);
        }
#pragma unroll
        for (int f = 0; f < FLY; ++f) {
            if (j0 + f >= n || k[f] >= V) break;
            if (k[f] != cur) {
                if (carried) store_cols<float, E>(part + (size_t)(2 * chunk) * ldp, c, D, sum);
                else put_row<OT, E>(dW + (size_t)cur * ldw, c, D, scale, acc, sum);
                carried = false;
                cur = k[f];
#pragma unroll
                for (int e = 0; e < E; ++e) sum[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] += x[f][e];
        }
    }
    if (cur >= V) return;   // padding, sorted behind every row
    const bool goes_on = i0 + n < N && key[i0 + n] == cur;
    if (carried) store_cols<float, E>(part + (size_t)(2 * chunk) * ldp, c, D, sum);
    else if (goes_on) store_cols<float, E>(part + (size_t)(2 * chunk + 1) * ldp, c, D, sum);
    else put_row<OT, E>(dW + (size_t)cur * ldw, c, D, scale, acc, sum);
}

// A work-group of 4 waves per chunk and slab of 512 columns: if a run begins in the chunk and
// goes on behind it, adds its partials -- the waves take every fourth chunk of the run, and their
// sums meet in LDS in wave order.
template <typename OT>
__global__ void __launch_bounds__(256) embedding_join(const int* __restrict__ key, int N, int V, int D,
                                                      float scale, OT* __restrict__ dW, int ldw,
                                                      int acc, const float* __restrict__ part,
                                                      int ldp, int chunks) {
    constexpr int E = 8;
    __shared__ float red[3][64][E + 1];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int c = (blockIdx.y * 64 + lane) * E;
    const long long chunk = blockIdx.x;
    const long long i1 = (chunk + 1) * EMB_CHUNK;
    if (i1 >= N) return;
    const int k = key[i1 - 1];
    if (k >= V || key[i1] != k) return;                            // no run goes on
    const long long i0 = chunk * EMB_CHUNK;
    if (i0 > 0 && key[i0] == k && key[i0 - 1] == k) return;          // it began earlier
    float sum[E] = {};
    if (w == 0 && c < D) load_cols<float, E>(part + (size_t)(2 * chunk + 1) * ldp, c, D, sum);
    for (long long t = chunk + 1 + w; t < chunks && key[t * EMB_CHUNK] == k; t += 4) {
        float x[E];
        if (c < D) {
            load_cols<float, E>(part + (size_t)(2 * t) * ldp, c, D, x);
#pragma unroll
            for (int e = 0; e < E; ++e) sum[e] += x[e];
        }
    }
    if (w > 0)
#pragma unroll
        for (int e = 0; e < E; ++e) red[w - 1][lane][e] = sum[e];
    __syncthreads();
    if (w != 0 || c >= D) return;
    for (int x = 0; x < 3; ++x)
#pragma unroll
        for (int e = 0; e < E; ++e) sum[e] += red[x][lane][e];
    put_row<OT, E>(dW + (size_t)k * ldw, c, D, scale, acc, sum);
}

// ---- host --------------------------------------------------------------------------------------
struct EmbWs {
    size_t key[2], pos[2], hist, present, part, total;
    int ldp, chunks, tiles;
};
size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

EmbWs emb_ws(int N, int V, int D) {
    EmbWs w{};
    w.tiles = (int)(((long long)N + EMB_TILE - 1) / EMB_TILE);
    w.chunks = (int)(((long long)N + EMB_CHUNK - 1) / EMB_CHUNK);
    w.ldp = (int)(((long long)D + 3) / 4 * 4);
    size_t at = 0;
    for (int i = 0; i < 2; ++i) {
        w.key[i] = at, at += up256((size_t)N * 4);
        w.pos[i] = at, at += up256((size_t)N * 4);
    }
    w.hist = at, at += up256((size_t)w.tiles * EMB_BINS * 4);
    w.present = at, at += up256((size_t)V + 4);
    w.part = at, at += up256((size_t)w.chunks * 2 * w.ldp * 4);
    w.total = at;
    return w;
}

int check_emb(const char* op, int dtype, int N, int V, int D, float scale) {
    if (dtype != DH_F32 && dtype != DH_BF16)
        return set_error(DH_ERR_INVALID, "%s: dtype must be fp32 or bf16", op);
    if (N < 0 || V < 1 || D < 1 || V == 0x7FFFFFFF || D > 1 << 24)
        return set_error(DH_ERR_INVALID, "%s: shape N=%d V=%d D=%d", op, N, V, D);
    if (!(scale - scale == 0.f)) return set_error(DH_ERR_INVALID, "%s: scale must be finite", op);
    return DH_OK;
}

template <typename T, typename OT>
int emb_bwd(int N, int V, int D, float scale, const int* ids, const T* dY, int ldy, OT* dW, int ldw,
            int acc, char* ws) {
    const EmbWs o = emb_ws(N, V, D);
    auto I = [&](size_t at) { return reinterpret_cast<int*>(ws + at); };
    float* part = reinterpret_cast<float*>(ws + o.part);
    uint8_t* present = acc ? nullptr : reinterpret_cast<uint8_t*>(ws + o.present);
    int total_bits = 1;
    while ((1ll << total_bits) <= V) ++total_bits;   // keys 0 .. V
    const int passes = (total_bits + EMB_BITS - 1) / EMB_BITS;
    const int bits = (total_bits + passes - 1) / passes;
    int last = 0;
    if (N <= EMB_TILE) {
        sort_small<<<1, 1024, 0, stream()>>>(ids, N, V, passes, bits, I(o.key[0]), I(o.pos[0]), present);
        DH_TRY(check_launch("dh_embedding_bwd"));
    } else {
        const int* kin = ids;
        const int* pin = nullptr;
        for (int p = 0; p < passes; ++p) {
            last = p & 1;
            sort_hist<<<o.tiles, 1024, 0, stream()>>>(kin, p == 0, N, V, p * bits, bits, I(o.hist),
                                                      p == 0 ? present : nullptr);
            DH_TRY(check_launch("dh_embedding_bwd"));
            sort_scatter<<<o.tiles, 1024, 0, stream()>>>(kin, p == 0, pin, N, V, p * bits, bits,
                                                         I(o.hist), I(o.key[last]), I(o.pos[last]),
                                                         p == passes - 1 ? present : nullptr);
            DH_TRY(check_launch("dh_embedding_bwd"));
            kin = I(o.key[last]);
            pin = I(o.pos[last]);
        }
    }
    const int slabs = (int)(((long long)D + 511) / 512);
    const int chunk_groups = (o.chunks + 3) / 4;
    const int zero_groups = acc ? 0 : (int)((V + 15LL) / 16 < 2048 ? (V + 15LL) / 16 : 2048);
    embedding_sum<T, OT><<<dim3(chunk_groups + zero_groups, slabs), 256, 0, stream()>>>(
        I(o.key[last]), I(o.pos[last]), N, V, D, scale, dY, ldy, dW, ldw, acc, part, o.ldp, chunk_groups,
        present);
    DH_TRY(check_launch("dh_embedding_bwd"));
    if (o.chunks > 1) {
        embedding_join<OT><<<dim3(o.chunks, slabs), 256, 0, stream()>>>(
            I(o.key[last]), N, V, D, scale, dW, ldw, acc, part, o.ldp, o.chunks);
        DH_TRY(check_launch("dh_embedding_bwd"));
    }
    return DH_OK;
}

template <typename OT>
__global__ void __launch_bounds__(256) zero_rows(OT* __restrict__ p, int V, int D, int ld) {
    const int lane = threadIdx.x & 63;
    const int c = (blockIdx.y * 64 + lane) * 8;
    if (c >= D) return;
    const float zero[8] = {};
    for (long long v = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); v < V; v += (long long)gridDim.x * 4)
        store_cols<OT, 8>(p + (size_t)v * ld, c, D, zero);
}

template <typename OT>
int zero_table(OT* p, int V, int D, int ld) {
    const int slabs = (int)(((long long)D + 511) / 512);
    zero_rows<OT><<<dim3((int)((V + 15LL) / 16 < 4096 ? (V + 15LL) / 16 : 4096), slabs), 256, 0,
                    stream()>>>(p, V, D, ld);
    return check_launch("dh_embedding_bwd");
}

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" {

int dh_embedding_fwd(int dtype, int N, int V, int D, float scale, const int* ids, const void* W,
                     int ldw, void* Y, int ldy) {
    DH_TRY(check_emb("dh_embedding_fwd", dtype, N, V, D, scale));
    if (ldw < D || ldy < D)
        return set_error(DH_ERR_INVALID, "dh_embedding_fwd: leading dimension below D");
    if (N > 0 && (!ids || !W || !Y)) return set_error(DH_ERR_INVALID, "dh_embedding_fwd: null pointer");
    DH_TRY(ensure_init());
    if (N == 0) return DH_OK;
    const int E = dtype == DH_F32 ? 4 : 8;
    const int slabs = (int)(((long long)D + 64 * E - 1) / (64 * E));
    const long long groups = (N + 3LL) / 4;
    const dim3 grid((int)(groups < 65536 ? groups : 65536), slabs);
    if (dtype == DH_F32)
        embedding_fwd_kernel<float><<<grid, 256, 0, stream()>>>(ids, N, V, D, scale, (const float*)W, ldw,
                                                                (float*)Y, ldy);
    else
        embedding_fwd_kernel<uint16_t><<<grid, 256, 0, stream()>>>(
            ids, N, V, D, scale, (const uint16_t*)W, ldw, (uint16_t*)Y, ldy);
    return check_launch("dh_embedding_fwd");
}

size_t dh_embedding_bwd_workspace(int N, int V, int D) {
    return N < 0 || V < 1 || D < 1 ? 0 : emb_ws(N, V, D).total;
}

int dh_embedding_bwd(int dtype, int N, int V, int D, float scale, const int* ids, const void* dY,
                     int lddy, void* dW, int lddw, int grad_type, int accumulate, void* ws,
                     size_t ws_bytes) {
    DH_TRY(check_emb("dh_embedding_bwd", dtype, N, V, D, scale));
    if (grad_type != DH_F32 && grad_type != dtype)
        return set_error(DH_ERR_INVALID, "dh_embedding_bwd: grad_type must be fp32 or the inputs' type");
    if (lddy < D || lddw < D)
        return set_error(DH_ERR_INVALID, "dh_embedding_bwd: leading dimension below D");
    if (!dW || (N > 0 && (!ids || !dY || !ws)))
        return set_error(DH_ERR_INVALID, "dh_embedding_bwd: null pointer");
    if (N > 0 && ((uintptr_t)ws & 15))
        return set_error(DH_ERR_INVALID, "dh_embedding_bwd: workspace not 16-byte aligned");
    if (N > 0 && ws_bytes < emb_ws(N, V, D).total)
        return set_error(DH_ERR_INVALID, "dh_embedding_bwd: workspace of %zu bytes, %zu needed", ws_bytes,
                         emb_ws(N, V, D).total);
    DH_TRY(ensure_init());
    if (N == 0) {
        if (accumulate) return DH_OK;
        return grad_type == DH_F32 ? zero_table((float*)dW, V, D, lddw)
                                   : zero_table((uint16_t*)dW, V, D, lddw);
    }
    if (dtype == DH_F32)
        return emb_bwd(N, V, D, scale, ids, (const float*)dY, lddy, (float*)dW, lddw, accumulate, (char*)ws);
    if (grad_type == DH_F32)
        return emb_bwd(N, V, D, scale, ids, (const uint16_t*)dY, lddy, (float*)dW, lddw, accumulate, (char*)ws);
    return emb_bwd(N, V, D, scale, ids, (const uint16_t*)dY, lddy, (uint16_t*)dW, lddw, accumulate, (char*)ws);
}

}  // extern "C"
