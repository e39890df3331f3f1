// dh_embedding.hip -- embedding lookup with scaling, and its gradient by sorted tokens.
//
//   Y[n] = s W[id[n]]          dW[v] (+)= s * sum of dY[n] over id[n] = v
//
// An id outside 0 .. V-1 is padding: a zero row of Y, no gradient.  Both are HBM-bound: the
// lookup reads N rows and writes N rows, the gradient reads N rows of dY and writes every row
// of dW (the rows that have tokens, when it accumulates).
//
// No floating-point atomics: a table row's tokens are added in token order, reruns are
// bit-identical.  Up to EMB_DIRECT tokens one launch does it all: every work-group looks through all
// ids for those it needs.  Beyond that the tokens are sorted by id (stable), and each run of equal
// ids is added:
//   sort     LSD radix, digits of at most 9 bits (2 passes up to 262143 rows): up to EMB_TILE tokens
//            in the LDS of one work-group, while the others clear the rows without a token; else a
//            histogram and a scatter launch per pass
//   sum      a wave adds EMB_CHUNK sorted tokens of a slab of 512 columns; runs that end inside the
//            chunk go to dW, those that cross its ends to fp32 partials
//   join     partials of a run that crosses chunks, added in order by its first chunk's group
#include "dh_common.hpp"

namespace dh {
namespace {

// Tokens that are not sorted: forward and gradient of 300 / 1000 / 2048 x 50001 x 1024 bf16 take 19 / 22 / 29 us
// so and 33 / 34 / 36 sorted, of 2048 x 500 x 1024 fp32 15 and 23.
constexpr int EMB_DIRECT = 2048;
// Tokens one work-group sorts: 8192 ids below 50001 in 26 us, the cleared rows beside; the launches per
// pass that more tokens take cost 20 us for each of the two passes.
constexpr int EMB_TILE = 8192;
constexpr int EMB_CHUNK = 16;      // sorted tokens added by one wave
constexpr int EMB_BITS = 9, EMB_BINS = 1 << EMB_BITS;

// ---- rows in chunks of 4 or 8 values at element alignment ---------------------------------------
template <typename T, int R> struct Chunk;
template <int R> struct Chunk<float, R> {
    typedef float vec __attribute__((ext_vector_type(R), aligned(4)));
    __device__ static float up(float x) { return x; }
    __device__ static float down(float x) { return x; }
};
template <int R> struct Chunk<uint16_t, R> {
    typedef uint16_t vec __attribute__((ext_vector_type(R), aligned(2)));
    __device__ static float up(uint16_t x) { return bf16_bits_to_f32(x); }
    // One rounding to nearest even of the fp32 value: the type of the result holds no more.
    __device__ static uint16_t down(float x) { return __builtin_bit_cast(uint16_t, (__bf16)x); }
};

// A wave's slab of 512 columns: 8 values per lane in chunks of R, chunk q of lane l at column
// 64 R q + R l of it, so an access of the wave is one piece of 64 R values.  R = 8 where all is
// bf16, else 4 (16 bytes of fp32).
template <int R>
__device__ inline int slab_col(int c0, int q) { return c0 + 64 * R * q + R * (threadIdx.x & 63); }

// Columns c .. c + R - 1 of a row of D values, zero past its end.
template <typename T, int R>
__device__ inline void load_chunk(const T* __restrict__ p, int c, int D, float* v) {
    if (c + R <= D) {
        const auto x = *reinterpret_cast<const typename Chunk<T, R>::vec*>(p + c);
#pragma unroll
        for (int e = 0; e < R; ++e) v[e] = Chunk<T, R>::up(x[e]);
    } else {
#pragma unroll
        for (int e = 0; e < R; ++e) v[e] = c + e < D ? Chunk<T, R>::up(p[c + e]) : 0.f;
    }
}
// Streamed past the caches (which leaves them to what is read) where the rows begin with 128-byte
// lines: a streamed piece of a line costs a whole one.  Same box, us, streamed / not: gradient of
// 8192 x 50001 x 1024 bf16 45 / 56, of 6 x 62528 x 3312 bf16 (rows begin inside a line) 100 / 82.
template <typename T, int R>
__device__ inline void store_chunk(T* __restrict__ p, int c, int D, const float* v, bool stream) {
    if (c + R <= D) {
        typedef typename Chunk<T, R>::vec vec;
        vec x;
#pragma unroll
        for (int e = 0; e < R; ++e) x[e] = Chunk<T, R>::down(v[e]);
        if (stream) __builtin_nontemporal_store(x, reinterpret_cast<vec*>(p + c));
        else *reinterpret_cast<vec*>(p + c) = x;
    } else {
#pragma unroll
        for (int e = 0; e < R; ++e)
            if (c + e < D) p[c + e] = Chunk<T, R>::down(v[e]);
    }
}
template <typename T, int R>
__device__ inline void load_slab(const T* __restrict__ p, int c0, int D, float (&v)[8]) {
#pragma unroll
    for (int q = 0; q < 8 / R; ++q) load_chunk<T, R>(p, slab_col<R>(c0, q), D, v + R * q);
}
template <typename T, int R>
__device__ inline void store_slab(T* __restrict__ p, int c0, int D, const float (&v)[8], bool stream) {
#pragma unroll
    for (int q = 0; q < 8 / R; ++q) store_chunk<T, R>(p, slab_col<R>(c0, q), D, v + R * q, stream);
}
inline bool whole_lines(const void* p, int ld, size_t size) {
    return ((uintptr_t)p & 127) == 0 && (ld * size) % 128 == 0;
}

// ---- lookup ------------------------------------------------------------------------------------
// A wave per row and slab of 512 columns.  65536 x 2048 fp32: 174 us, 3.1 TB/s written and as much read
// (partly from cache, as tokens repeat).
template <typename T, int R>
__global__ void __launch_bounds__(256) embedding_fwd_kernel(const int* __restrict__ ids, int N, int V,
                                                            int D, float scale,
                                                            const T* __restrict__ W, int ldw,
                                                            T* __restrict__ Y, int ldy, bool stream) {
    const int c0 = blockIdx.y * 512;
    const long long waves = (long long)gridDim.x * 4;
    for (long long n = (long long)blockIdx.x * 4 + (threadIdx.x >> 6); n < N; n += waves) {
        const int id = ids[n];
        float v[8] = {};
        if ((unsigned)id < (unsigned)V) {
            load_slab<T, R>(W + (size_t)id * ldw, c0, D, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] *= scale;
        }
        store_slab<T, R>(Y + (size_t)n * ldy, c0, D, v, stream);
    }
}

// ---- gradient, shared ----------------------------------------------------------------------------
// Where table rows go: dW (+)= scale sum, rounded once.
template <typename OT, int R>
struct Out {
    OT* dW;
    int ldw, V, D;
    float scale;
    int acc;
    bool stream;
    __device__ void put(int row, int c0, const float (&sum)[8]) const {
        OT* p = dW + (size_t)row * ldw;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = sum[e] * scale;
        if (acc) {
            float o[8];
            load_slab<OT, R>(p, c0, D, o);
#pragma unroll
            for (int e = 0; e < 8; ++e) v[e] += o[e];
        }
        store_slab<OT, R>(p, c0, D, v, stream);
    }
    // Zeros in rows v0 .. v0 + rows - 1 that are not marked, by a work-group: its threads walk
    // over the rows' 16-byte pieces side by side.
    __device__ void clear(int v0, int rows, const uint8_t* mark) const {
        constexpr int Z = 16 / sizeof(OT);
        const float zero[Z] = {};
        const int per = (D + Z - 1) / Z;
        int r = threadIdx.x / per, c = threadIdx.x % per;
        const int dr = blockDim.x / per, dc = blockDim.x % per;
        while (r < rows) {
            if (!mark[r]) store_chunk<OT, Z>(dW + (size_t)(v0 + r) * ldw, Z * c, D, zero, stream);
            r += dr;
            c += dc;
            if (c >= per) {
                c -= per;
                ++r;
            }
        }
    }
};

// Zeros in n values side by side, by a work-group: whole 128-byte lines, and what lies before and
// behind them value by value.
template <typename OT>
__device__ inline void clear_flat(OT* p, long long n) {
    const uintptr_t a = (uintptr_t)p, b = a + n * sizeof(OT);
    const uintptr_t a1 = (a + 127) & ~(uintptr_t)127, b1 = b & ~(uintptr_t)127;
    if (a1 >= b1) {
        for (long long i = threadIdx.x; i < n; i += blockDim.x) p[i] = OT(0);
        return;
    }
    for (OT* x = p + threadIdx.x; (uintptr_t)x < a1; x += blockDim.x) *x = OT(0);
    for (OT* x = (OT*)b1 + threadIdx.x; (uintptr_t)x < b; x += blockDim.x) *x = OT(0);
    for (f32x4* x = (f32x4*)a1 + threadIdx.x; (uintptr_t)x < b1; x += blockDim.x)
        *x = f32x4{0.f, 0.f, 0.f, 0.f};
}

constexpr int CLEAR_ROWS = 1024;   // most table rows that one work-group clears

// Clears the rows v0 .. v0 + rows - 1 that no token has, by looking through all N ids.  FLAT: where none has
// one and the rows follow each other without gaps but do not begin with lines, they are written as one range
// (us, row by row / so: 100 x 100000 x 1001 fp32 89 / 79, 6 x 62528 x 3312 bf16 87 / 79, 15 x 101300 x 3504 fp32
// 264 / 262; with thousands of tokens few groups have none).
template <bool FLAT, typename OT, int R>
__device__ inline void clear_absent(const Out<OT, R>& out, const int* __restrict__ ids, int N, int v0,
                                    int rows, uint8_t* mark) {
    rows = min(rows, out.V - v0);
    for (int r = threadIdx.x; r < rows; r += blockDim.x) mark[r] = 0;
    __syncthreads();
    int found = 0;
    for (int n = threadIdx.x; n < N; n += blockDim.x) {
        const int id = ids[n];
        if (id >= v0 && id < v0 + rows) mark[id - v0] = 1, found = 1;
    }
    if (FLAT && out.ldw == out.D && !out.stream) {
        if (!__syncthreads_or(found)) {
            clear_flat(out.dW + (size_t)v0 * out.ldw, (long long)rows * out.D);
            return;
        }
    } else {
        __syncthreads();
    }
    out.clear(v0, rows, mark);
}

// ---- gradient of few tokens ------------------------------------------------------------------------
// Work-groups [0, N): token n's group finds the tokens of its id, each of its 8 waves in an eighth of
// the ids; if n is the first of them it adds their rows of dY, each wave its own, four in flight,
// and the waves' sums meet in LDS in wave order.  The other work-groups (none when accumulating)
// clear `rows` table rows each.
constexpr int DIRECT_WAVES = 8;
template <typename T, typename OT, int R>
__global__ void __launch_bounds__(64 * DIRECT_WAVES) embedding_direct(const int* __restrict__ ids, int N,
                                                                      const T* __restrict__ dY, int ldy,
                                                                      Out<OT, R> out, int rows) {
    constexpr int W = DIRECT_WAVES;
    __shared__ uint16_t list[W][EMB_DIRECT / W];
    __shared__ float red[W - 1][8][64];
    __shared__ int first[W], count[W];
    const int lane = threadIdx.x & 63;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = blockIdx.x;
    if (n >= N) {
        if (blockIdx.y == 0)
            clear_absent<true>(out, ids, N, (n - N) * rows, rows, reinterpret_cast<uint8_t*>(red));
        return;
    }
    const int id = ids[n];
    if ((unsigned)id >= (unsigned)out.V) return;
    const int part = (N + W - 1) / W, end = min(N, (w + 1) * part);
    int mine = 0, at = N;
    for (int i0 = w * part; i0 < end; i0 += 256) {
        int x[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const int i = i0 + 64 * j + lane;
            x[j] = i < end ? ids[i] : -1;
        }
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            const uint64_t mask = __ballot(x[j] == id);
            if (!mask) continue;
            if (mine == 0) at = i0 + 64 * j + __ffsll((unsigned long long)mask) - 1;
            if (x[j] == id) list[w][mine + __popcll(mask & ((1ull << lane) - 1))] = (uint16_t)(i0 + 64 * j + lane);
            mine += __popcll(mask);
        }
    }
    if (lane == 0) {
        first[w] = at;
        count[w] = mine;
    }
    __syncthreads();
    int waves = 0;   // that have some
    for (int x = 0; x < W; ++x) {
        if (first[x] < n) return;   // an earlier token's group does it
        waves += count[x] > 0;
    }
    for (int c0 = 512 * blockIdx.y; c0 < out.D; c0 += 512 * gridDim.y) {
        float sum[8] = {};
        for (int j = 0; j < mine; j += 4) {
            float x[4][8];
#pragma unroll
            for (int f = 0; f < 4; ++f)   // past the end: the last one again, unused
                load_slab<T, R>(dY + (size_t)list[w][min(j + f, mine - 1)] * ldy, c0, out.D, x[f]);
#pragma unroll
            for (int f = 0; f < 4; ++f)
                if (j + f < mine)
#pragma unroll
                    for (int e = 0; e < 8; ++e) sum[e] += x[f][e];
        }
        if (waves == 1) {   // the same in all waves
            if (mine > 0) out.put(id, c0, sum);
            continue;
        }
        __syncthreads();   // red[] of the slab before has been read
        if (w > 0)
#pragma unroll
            for (int e = 0; e < 8; ++e) red[w - 1][e][lane] = sum[e];
        __syncthreads();
        if (w == 0) {
            for (int x = 0; x < W - 1; ++x)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] += red[x][e][lane];
            out.put(id, c0, sum);
        }
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
            wave_fence();
            if (before == 0) cnt[w][digit[j]] = (uint16_t)(c + __popcll(peers));
        }
        wave_fence();
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

// All passes of at most EMB_TILE tokens in the first work-group: (key, position) pairs go through
// LDS between passes.  Latency-bound, so the other work-groups (none when accumulating) clear
// `rows` table rows each at the same time.
template <typename OT, int R>
__global__ void __launch_bounds__(1024) sort_small(const int* __restrict__ ids, int N, int V,
                                                   int passes, int bits, int* __restrict__ key_out,
                                                   int* __restrict__ pos_out, Out<OT, R> out, int rows) {
    constexpr int ITEMS = EMB_TILE / 1024;
    __shared__ int skey[EMB_TILE];
    __shared__ uint16_t spos[EMB_TILE];
    __shared__ uint16_t cnt[16][EMB_BINS];
    __shared__ int base[EMB_BINS];
    if (blockIdx.x > 0) {
        clear_absent<false>(out, ids, N, (blockIdx.x - 1) * rows, rows, reinterpret_cast<uint8_t*>(skey));
        return;
    }
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
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
// Partial sums of a slab as its wave holds them: lane l's 8 values in two pieces of 16 bytes.
__device__ inline void store_part(float* p, const float (&v)[8]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int q = 0; q < 2; ++q)
        reinterpret_cast<f32x4*>(p)[64 * q + lane] = f32x4{v[4 * q], v[4 * q + 1], v[4 * q + 2], v[4 * q + 3]};
}
__device__ inline void load_part(const float* p, float (&v)[8]) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const f32x4 x = reinterpret_cast<const f32x4*>(p)[64 * q + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e) v[4 * q + e] = x[e];
    }
}

// Work-groups [0, chunk_groups): a wave per chunk of EMB_CHUNK sorted tokens and slab (blockIdx.y)
// of 512 columns, rows fetched four at a time.  part[chunk][0] is the sum of the run that came in
// from the chunk before, part[chunk][1] that of the run that goes on behind it; a run that does
// both is in part[chunk][0].  The other work-groups (with `present`) clear `rows` table rows each.
// 65536 x 131072 x 2048 fp32: 398 us for 0.54 GB read and 1.07 GB written, 4.1 TB/s (a copy: 4.8).
template <typename T, typename OT, int R>
__global__ void __launch_bounds__(256) embedding_sum(const int* __restrict__ key,
                                                     const int* __restrict__ pos, int N,
                                                     const T* __restrict__ dY, int ldy,
                                                     Out<OT, R> out, float* __restrict__ part, int ldp,
                                                     int chunk_groups,
                                                     const uint8_t* __restrict__ present, int rows) {
    constexpr int FLY = 4;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int V = out.V, D = out.D, c0 = blockIdx.y * 512;
    if ((int)blockIdx.x >= chunk_groups) {
        // the slabs' copies of a group share its rows
        const int share = (rows + gridDim.y - 1) / gridDim.y;
        const long long v0 = (long long)(blockIdx.x - chunk_groups) * rows + blockIdx.y * share;
        const int end = min((int)blockIdx.y * share + share, rows) - (int)blockIdx.y * share;
        if (v0 < V && end > 0) out.clear((int)v0, min((long long)end, V - v0), present + v0);
        return;
    }
    const long long chunk = (long long)blockIdx.x * 4 + w;
    const long long i0 = chunk * EMB_CHUNK;
    if (i0 >= N) return;
    const int n = (int)(N - i0 < EMB_CHUNK ? N - i0 : EMB_CHUNK);
    int cur = key[i0];
    bool carried = i0 > 0 && key[i0 - 1] == cur;   // the run began in an earlier chunk
    float sum[8] = {};
    for (int j0 = 0; j0 < n; j0 += FLY) {
        float x[FLY][8];
        int k[FLY];
#pragma unroll
        for (int f = 0; f < FLY; ++f) {
            const int j = j0 + f < n ? j0 + f : n - 1;   // past the end: the last token again, unused
            k[f] = key[i0 + j];
            const int p = k[f] < V ? pos[i0 + j] : 0;
            load_slab<T, R>(dY + (size_t)p * ldy, c0, D, x[f]);
        }
#pragma unroll
        for (int f = 0; f < FLY; ++f) {
            if (j0 + f >= n || k[f] >= V) break;
            if (k[f] != cur) {
                if (carried) store_part(part + (size_t)(2 * chunk) * ldp + c0, sum);
                else out.put(cur, c0, sum);
                carried = false;
                cur = k[f];
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] = 0.f;
            }
#pragma unroll
            for (int e = 0; e < 8; ++e) sum[e] += x[f][e];
        }
    }
    if (cur >= V) return;   // padding, sorted behind every row
    const bool goes_on = i0 + n < N && key[i0 + n] == cur;
    if (carried) store_part(part + (size_t)(2 * chunk) * ldp + c0, sum);
    else if (goes_on) store_part(part + (size_t)(2 * chunk + 1) * ldp + c0, sum);
    else out.put(cur, c0, sum);
}

// A work-group of 4 waves per chunk and slab of 512 columns: if a run begins in the chunk and
// goes on behind it, adds its partials -- the waves take every fourth chunk of the run, four in
// flight, and their sums meet in LDS in wave order.
template <typename OT, int R>
__global__ void __launch_bounds__(256) embedding_join(const int* __restrict__ key, int N, Out<OT, R> out,
                                                      const float* __restrict__ part, int ldp,
                                                      int chunks) {
    __shared__ float red[3][8][64];
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6;
    const int c0 = blockIdx.y * 512;
    const long long chunk = blockIdx.x;
    const long long i1 = (chunk + 1) * EMB_CHUNK;
    if (i1 >= N) return;
    const int k = key[i1 - 1];
    if (k >= out.V || key[i1] != k) return;                        // no run goes on
    const long long i0 = chunk * EMB_CHUNK;
    if (i0 > 0 && key[i0] == k && key[i0 - 1] == k) return;          // it began earlier
    // chunks behind this one that begin with the run, 64 looked at at a time
    int more = 0;
    for (;;) {
        const long long t = chunk + 1 + more + lane;
        const uint64_t same = __ballot(t < chunks && key[t * EMB_CHUNK] == k);
        if (same != ~0ull) {
            more += __ffsll((unsigned long long)~same) - 1;
            break;
        }
        more += 64;
    }
    float sum[8] = {};
    if (w == 0) load_part(part + (size_t)(2 * chunk + 1) * ldp + c0, sum);
    for (int j0 = w; j0 < more; j0 += 16) {
        float x[4][8];
#pragma unroll
        for (int f = 0; f < 4; ++f) {   // past the end: the first one again, unused
            const int j = j0 + 4 * f < more ? j0 + 4 * f : j0;
            load_part(part + (size_t)(2 * (chunk + 1 + j)) * ldp + c0, x[f]);
        }
#pragma unroll
        for (int f = 0; f < 4; ++f)
            if (j0 + 4 * f < more)
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] += x[f][e];
    }
    if (w > 0)
#pragma unroll
        for (int e = 0; e < 8; ++e) red[w - 1][e][lane] = sum[e];
    __syncthreads();
    if (w != 0) return;
    for (int x = 0; x < 3; ++x)
#pragma unroll
        for (int e = 0; e < 8; ++e) sum[e] += red[x][e][lane];
    out.put(k, c0, sum);
}

// ---- host --------------------------------------------------------------------------------------
struct EmbWs {
    size_t key[2], pos[2], hist, present, part, total;
    int ldp, chunks, tiles;
};
size_t up256(size_t x) { return (x + 255) & ~(size_t)255; }

EmbWs emb_ws(int N, int V, int D) {
    EmbWs w{};
    if (N <= EMB_DIRECT) return w;   // no workspace
    w.tiles = (int)(((long long)N + EMB_TILE - 1) / EMB_TILE);
    w.chunks = (int)(((long long)N + EMB_CHUNK - 1) / EMB_CHUNK);
    w.ldp = (D + 511) / 512 * 512;
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

// The most tokens of a gradient: embedding_join has 256 threads per EMB_CHUNK of them, and a launch
// less than 2^32.
constexpr int EMB_MOST = EMB_CHUNK * ((1 << 24) - 1);

int check_emb(const char* op, int dtype, int N, int V, int D, float scale, int most) {
    if (dtype != DH_F32 && dtype != DH_BF16)
        return set_error(DH_ERR_INVALID, "%s: dtype must be fp32 or bf16", op);
    // 2^20 below the ends of int, which the strides of the kernels' loops stay under
    if (N < 0 || V < 1 || D < 1 || N > most || V > 0x7FF00000 || D > 1 << 24)
        return set_error(DH_ERR_INVALID, "%s: shape N=%d V=%d D=%d", op, N, V, D);
    if (!(scale - scale == 0.f)) return set_error(DH_ERR_INVALID, "%s: scale must be finite", op);
    return DH_OK;
}

template <typename T, typename OT>
int emb_bwd(int N, int V, int D, float scale, const int* ids, const void* dY_, int ldy, void* dW, int ldw,
            int acc, char* ws) {
    constexpr int R = sizeof(T) == 2 && sizeof(OT) == 2 ? 8 : 4;
    const T* dY = (const T*)dY_;
    const Out<OT, R> out{(OT*)dW, ldw, V, D, scale, acc, whole_lines(dW, ldw, sizeof(OT))};
    const int slabs = (D + 511) / 512;
    // Clearing: about 2048 work-groups, each of at least 16 KB.
    long long rows = (V + 2047LL) / 2048, least = (16384 + (long long)sizeof(OT) * D - 1) / ((long long)sizeof(OT) * D);
    if (rows < least) rows = least;
    if (rows > CLEAR_ROWS) rows = CLEAR_ROWS;
    const int clears = acc ? 0 : (int)((V + rows - 1) / rows);
    if (N <= EMB_DIRECT) {
        embedding_direct<T, OT, R><<<dim3(N + clears, slabs < 64 ? slabs : 64), 64 * DIRECT_WAVES, 0, stream()>>>(
            ids, N, dY, ldy, out, (int)rows);
        return check_launch("dh_embedding_bwd");
    }
    const EmbWs o = emb_ws(N, V, D);
    auto I = [&](size_t at) { return reinterpret_cast<int*>(ws + at); };
    float* part = reinterpret_cast<float*>(ws + o.part);
    uint8_t* present = acc || N <= EMB_TILE ? nullptr : reinterpret_cast<uint8_t*>(ws + o.present);
    int total_bits = 1;
    while ((1ll << total_bits) <= V) ++total_bits;   // keys 0 .. V
    const int passes = (total_bits + EMB_BITS - 1) / EMB_BITS;
    const int bits = (total_bits + passes - 1) / passes;
    int last = 0;
    if (N <= EMB_TILE) {
        sort_small<OT, R><<<1 + clears, 1024, 0, stream()>>>(ids, N, V, passes, bits, I(o.key[0]), I(o.pos[0]),
                                                             out, (int)rows);
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
    const int chunk_groups = (o.chunks + 3) / 4;
    embedding_sum<T, OT, R><<<dim3(chunk_groups + (present ? clears : 0), slabs), 256, 0, stream()>>>(
        I(o.key[last]), I(o.pos[last]), N, dY, ldy, out, part, o.ldp, chunk_groups, present, (int)rows);
    DH_TRY(check_launch("dh_embedding_bwd"));
    embedding_join<OT, R><<<dim3(o.chunks, slabs), 256, 0, stream()>>>(I(o.key[last]), N, out, part, o.ldp,
                                                                       o.chunks);
    return check_launch("dh_embedding_bwd");
}

// The gradient of no tokens.
template <typename OT>
__global__ void __launch_bounds__(256) zero_rows(Out<OT, 4> out, int rows) {
    __shared__ uint8_t mark[CLEAR_ROWS];
    clear_absent<true>(out, (const int*)nullptr, 0, blockIdx.x * rows, rows, mark);
}
template <typename OT>
int zero_table(void* p, int V, int D, int ld) {
    const int rows = V < 4096 * 64 ? 64 : CLEAR_ROWS;
    zero_rows<OT><<<(unsigned)(((long long)V + rows - 1) / rows), 256, 0, stream()>>>(
        Out<OT, 4>{(OT*)p, ld, V, D, 0.f, 0, whole_lines(p, ld, sizeof(OT))}, rows);
    return check_launch("dh_embedding_bwd");
}

}  // namespace
}  // namespace dh

using namespace dh;

extern "C" {

int dh_embedding_fwd(int dtype, int N, int V, int D, float scale, const int* ids, const void* W,
                     int ldw, void* Y, int ldy) {
    DH_TRY(check_emb("dh_embedding_fwd", dtype, N, V, D, scale, 0x7FF00000));
    if (ldw < D || ldy < D)
        return set_error(DH_ERR_INVALID, "dh_embedding_fwd: leading dimension below D");
    if (N > 0 && (!ids || !W || !Y)) return set_error(DH_ERR_INVALID, "dh_embedding_fwd: null pointer");
    DH_TRY(ensure_init());
    if (N == 0) return DH_OK;
    const long long groups = (N + 3LL) / 4;
    const dim3 grid((int)(groups < 65536 ? groups : 65536), (D + 511) / 512);
    if (dtype == DH_F32)
        embedding_fwd_kernel<float, 4><<<grid, 256, 0, stream()>>>(ids, N, V, D, scale, (const float*)W, ldw,
                                                                   (float*)Y, ldy, whole_lines(Y, ldy, 4));
    else
        embedding_fwd_kernel<uint16_t, 8><<<grid, 256, 0, stream()>>>(
            ids, N, V, D, scale, (const uint16_t*)W, ldw, (uint16_t*)Y, ldy, whole_lines(Y, ldy, 2));
    return check_launch("dh_embedding_fwd");
}

size_t dh_embedding_bwd_workspace(int N, int V, int D) {
    return N < 0 || V < 1 || D < 1 ? 0 : emb_ws(N, V, D).total;
}

int dh_embedding_bwd(int dtype, int N, int V, int D, float scale, const int* ids, const void* dY,
                     int lddy, void* dW, int lddw, int grad_type, int accumulate, void* ws,
                     size_t ws_bytes) {
    DH_TRY(check_emb("dh_embedding_bwd", dtype, N, V, D, scale, EMB_MOST));
    if (grad_type != DH_F32 && grad_type != dtype)
        return set_error(DH_ERR_INVALID, "dh_embedding_bwd: grad_type must be fp32 or the inputs' type");
    if (lddy < D || lddw < D)
        return set_error(DH_ERR_INVALID, "dh_embedding_bwd: leading dimension below D");
    const size_t need = emb_ws(N, V, D).total;
    if (!dW || (N > 0 && (!ids || !dY)) || (need > 0 && !ws))
        return set_error(DH_ERR_INVALID, "dh_embedding_bwd: null pointer");
    if (need > 0 && ((uintptr_t)ws & 15))
        return set_error(DH_ERR_INVALID, "dh_embedding_bwd: workspace not 16-byte aligned");
    if (ws_bytes < need)
        return set_error(DH_ERR_INVALID, "dh_embedding_bwd: workspace of %zu bytes, %zu needed", ws_bytes, need);
    DH_TRY(ensure_init());
    if (N == 0) {
        if (accumulate) return DH_OK;
        return grad_type == DH_F32 ? zero_table<float>(dW, V, D, lddw) : zero_table<uint16_t>(dW, V, D, lddw);
    }
    auto run = dtype == DH_F32 ? emb_bwd<float, float>
               : grad_type == DH_F32 ? emb_bwd<uint16_t, float> : emb_bwd<uint16_t, uint16_t>;
    return run(N, V, D, scale, ids, dY, lddy, dW, lddw, accumulate, (char*)ws);
}

}  // extern "C"
