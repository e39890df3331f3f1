// dh_gemm_bf16.hpp -- operand tiles of the bf16 matrix-core kernels: global -> LDS by direct DMA,
// LDS -> MFMA fragments, and the steps of their main loops.  Used by dh_gemm_bf16.hip and
// dh_vocab.hip.
#pragma once

#include "dh_common.hpp"

namespace dh {
namespace {

// ---------------------------------------------------------------------------------
// Fast path for tile-aligned shapes (M, N multiples of 256, K of 32, leading dims of 8,
// 16-byte aligned operands): both operands travel global -> LDS by direct-to-LDS DMA
// (buffer_load_dwordx4 ... lds: lane l's 16 bytes land at base + 16 l), so no registers or
// LDS-write instructions are spent on staging.  LDS tiles keep the global orientation:
//   k-contiguous operand  : [256 rows][32 k],  16-byte chunk c of row r at position
//                           c ^ (r / 4 % 4)  -> MFMA fragment = one ds_read_b128
//   mn-contiguous operand : [32 k][256 cols], chunk c of row k at c ^ 4 (k % 4)
//                           -> MFMA fragment = two ds_read_b64_tr_b16
// ds_read_b64_tr_b16 semantics (measured on gfx950): in each 16-lane group, lane i names
// a row R_i of 4 consecutive 16-bit values; lane j receives R_{j/4 + 4e}[j % 4] for
// e = 0..3.  Pointing lane i at [kb + i/4][nb + 4 (i % 4)] therefore hands lane j the 4
// values [kb .. kb + 3][nb + j], the MFMA operand layout.  The LDS serves 64 banks of
// 4 bytes (16 lanes of a b128 read, 32 lanes of a b64 read per pass); both swizzles make
// the fragment reads conflict free under that model.  A ring of four LDS stages (128 KB);
// fragments of the next k-step are read while the matrix cores run the current one.
// ---------------------------------------------------------------------------------

template <bool KCONTIG, int WAVES, int T = 256>
struct FastOperand {
    // One 32-k stage of a T-wide operand tile (T = 256 or 128) is T / 16 DMA blocks of 1 KB;
    // wave w issues blocks PER*w .. PER*w + PER-1.  Per-lane element offsets at k0 = 0 and
    // the per-stage step.
    static constexpr int NBLK = T / 16;
    static constexpr int PER = NBLK / WAVES;
    static constexpr int KPB = 512 / T;    // k rows of an mn-contiguous tile per DMA block
    static constexpr int CPR = T / 8;      // 16-byte chunks in one of those rows
    static constexpr int CPR_LOG = T == 256 ? 5 : 4;
    static_assert(T == 256 || T == 128, "tile widths");
    uint32_t off[PER];     // byte offsets from the operand base at stage 0
    uint32_t step;         // bytes per stage
    uint32_t bytes;        // operand extent (rows x ld x 2 < 2^32, checked by the host)

    __device__ void init(int ld, int rows, int t0, int wave, int lane) {
#pragma unroll
        for (int t = 0; t < PER; ++t) {
            const int b = PER * wave + t;
            if (KCONTIG) {                     // block b = rows 16b .. 16b+15 of [t][32 k]
                const int row = 16 * b + (lane >> 2);
                const int c = (lane & 3) ^ ((lane >> 4) & 3);   // = p ^ ((row >> 2) & 3)
                off[t] = 2u * ((uint32_t)(t0 + row) * ld + 8 * c);
            } else {                           // block b = k rows KPB b .. of [32 k][T]
                const int k = KPB * b + (lane >> CPR_LOG);
                const int c = (lane & (CPR - 1)) ^ (4 * (k & 3));
                off[t] = 2u * ((uint32_t)k * ld + t0 + 8 * c);
            }
        }
        step = KCONTIG ? 64u : 64u * (uint32_t)ld;
        bytes = 2u * (uint32_t)rows * (uint32_t)ld;
    }
    // Buffer-resource DMA: the per-lane offsets stay in VGPRs for the whole loop and the
    // stage advance is a scalar offset, so an issue costs no vector instructions.
    __device__ void issue(const uint16_t* __restrict__ g, int kt, uint16_t* lds, int wave) const {
        const uint32_t soff = __builtin_amdgcn_readfirstlane((uint32_t)kt * step);
        const uint32_t base = __builtin_amdgcn_readfirstlane(lds_addr(lds) + 1024u * PER * wave);
        const u32x4 rs = make_rsrc(g, bytes);
#pragma unroll
        for (int t = 0; t < PER; ++t) lds_dma16_buf_so(off[t], rs, soff, base + 1024u * t);
    }
    // MFMA operand for tile rows/cols o .. o+31, k-step kk (16 k) of the stage.
    __device__ static bf16x8 frag(const uint16_t* lds, int o, int kk, int lane) {
        const int h = lane >> 5;
        if (KCONTIG) {                         // [256][32]: chunk c of row r at c ^ (r/4 % 4)
            const int row = o + (lane & 31);
            const int p = (2 * kk + h) ^ ((row >> 2) & 3);
            return *reinterpret_cast<const bf16x8*>(lds + row * 32 + 8 * p);
        } else {                               // [32][T]: chunk c of row k at c ^ 4 (k % 4)
            const int G = (lane & 31) >> 4, i = lane & 15;
            const int n = o + 16 * G + 4 * (i & 3);
            s16x4 r[2];
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                const int k = 16 * kk + 8 * h + 4 * q + (i >> 2);
                const int p = (n >> 3) ^ (4 * (k & 3));
                r[q] = ds_read_tr(lds + k * T + 8 * p + 4 * ((n >> 2) & 1));
            }
            return __builtin_bit_cast(bf16x8, __builtin_shufflevector(r[0], r[1], 0, 1, 2, 3, 4, 5, 6, 7));
        }
    }
    // The same fragment as PARTS separate LDS instructions (one b128 read, or two
    // transposing b64 reads), so that a schedule can place each between matrix-core ops.
    static constexpr int PARTS = KCONTIG ? 1 : 2;
    __device__ static void part(const uint16_t* lds, int o, int kk, int lane, int q,
                                s16x4 (&f)[2]) {
        const int h = lane >> 5;
        if (KCONTIG) {
            const int row = o + (lane & 31);
            const int p = (2 * kk + h) ^ ((row >> 2) & 3);
            const s16x8 v = *reinterpret_cast<const s16x8*>(lds + row * 32 + 8 * p);
            f[0] = __builtin_shufflevector(v, v, 0, 1, 2, 3);
            f[1] = __builtin_shufflevector(v, v, 4, 5, 6, 7);
        } else {
            const int G = (lane & 31) >> 4, i = lane & 15;
            const int n = o + 16 * G + 4 * (i & 3);
            const int k = 16 * kk + 8 * h + 4 * q + (i >> 2);
            const int p = (n >> 3) ^ (4 * (k & 3));
            f[q] = ds_read_tr(lds + k * T + 8 * p + 4 * ((n >> 2) & 1));
        }
    }
    // DMA block t of this wave's share of a stage (see issue()).
    __device__ void issue_one(u32x4 rs, uint32_t soff, uint32_t base, int t) const {
        lds_dma16_buf_so(off[t], rs, soff, base + 1024u * t);
    }
};

// A k-contiguous operand in double stages of 64 k for the one-wave-per-SIMD schedule: the
// 32-k stages above fetch 64 bytes per row, half an L2 line (the next stage fetches the other
// half again), while a 64-k stage fetches each row's full 128-byte line once.  LDS tile
// [256 rows][64 k] = 32 KB; 16-byte chunk c of row r at position c ^ ((r >> 1) & 7): the 16
// rows of one b128 pass fall on 8 even and 8 odd rows, so the 16-byte units they read are
// all different (conflict free).  DMA block b = rows 8b .. 8b+7, 8 lanes x 16 B per row;
// 32 blocks per double stage, 32 / WAVES per wave.
template <int WAVES>
struct DeepKOperand {
    static constexpr int PER = 32 / WAVES;
    static constexpr int PARTS = 1;
    static constexpr int ELEMS = 256 * 64;   // elements of one double stage
    uint32_t off[PER];                        // byte offsets from the operand base, pair 0
    uint32_t bytes;

    __device__ void init(int ld, int rows, int t0, int wave, int lane) {
#pragma unroll
        for (int t = 0; t < PER; ++t) {
            const int row = 8 * (PER * wave + t) + (lane >> 3);
            const int c = (lane & 7) ^ ((row >> 1) & 7);
            off[t] = 2u * ((uint32_t)(t0 + row) * ld + 8 * c);
        }
        bytes = 2u * (uint32_t)rows * (uint32_t)ld;
    }
    static constexpr uint32_t STEP = 128u;    // bytes per double stage along a row
    __device__ void issue_one(u32x4 rs, uint32_t soff, uint32_t base, int t) const {
        lds_dma16_buf_so(off[t], rs, soff, base + 1024u * t);
    }
    // k-step kk (0..3, 16 k each) of the double stage for tile rows o .. o+31.
    __device__ static void part(const uint16_t* lds, int o, int kk, int lane, int,
                                s16x4 (&f)[2]) {
        const int row = o + (lane & 31);
        const int p = (2 * kk + (lane >> 5)) ^ ((row >> 1) & 7);
        const s16x8 v = *reinterpret_cast<const s16x8*>(lds + row * 64 + 8 * p);
        f[0] = __builtin_shufflevector(v, v, 0, 1, 2, 3);
        f[1] = __builtin_shufflevector(v, v, 4, 5, 6, 7);
    }
};

constexpr int FAST_TILE = 256 * 32;   // elements of one operand stage (32 k)
constexpr int FAST_NSTAGE = 4;        // LDS ring: 4 x (A + B) x 16 KB = 128 KB

// Fragments of one 16-k step for the wave's FM x FN block of 32 x 32 MFMA tiles (the stage's
// B tile BOFF elements after its A tile).
template <typename OA, typename OB, int FM, int FN, int BOFF = FAST_TILE>
__device__ inline void load_frags(const uint16_t* st, int kk, int wm, int wn, int lane,
                                  bf16x8 (&fa)[FM], bf16x8 (&fb)[FN]) {
#pragma unroll
    for (int x = 0; x < FM; ++x) fa[x] = OA::frag(st, wm + 32 * x, kk, lane);
#pragma unroll
    for (int x = 0; x < FN; ++x) fb[x] = OB::frag(st + BOFF, wn + 32 * x, kk, lane);
}

template <int FM, int FN>
__device__ inline void mfma_block(const bf16x8 (&fa)[FM], const bf16x8 (&fb)[FN],
                                  f32x16 (&acc)[FM][FN]) {
#pragma unroll
    for (int a = 0; a < FM; ++a)
#pragma unroll
        for (int b = 0; b < FN; ++b)
            acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[a], fb[b], acc[a][b], 0, 0, 0);
}

__device__ inline bf16x8 cat8(const s16x4 (&f)[2]) {
    return __builtin_bit_cast(bf16x8, __builtin_shufflevector(f[0], f[1], 0, 1, 2, 3, 4, 5, 6, 7));
}

// One 16-k step of a one-wave-per-SIMD schedule: the FM x FN matrix-core ops on the
// current fragments (ca, cb), with the LDS reads of the next fragments (na, nb, from stage
// `nst`, k-step nkk) and, when DMA, this wave's 2 x PER DMA blocks of a later stage placed
// one per op.  A single wave per SIMD issues at most one instruction every few cycles, so
// grouped reads or DMA issues would leave the matrix core idle; spread out, each hides
// under the op before it.
template <typename OA, typename OB, int FM, int FN, bool DMA>
__device__ inline void step_interleaved(const s16x4 (&ca)[FM][2], const s16x4 (&cb)[FN][2],
                                        f32x16 (&acc)[FM][FN], const uint16_t* nst, int nkk,
                                        int wm, int wn, int lane, s16x4 (&na)[FM][2],
                                        s16x4 (&nb)[FN][2], const OA& oa, const OB& ob,
                                        u32x4 rsa, u32x4 rsb, uint32_t soa, uint32_t sob,
                                        uint32_t basea, uint32_t baseb) {
    constexpr int NRA = FM * OA::PARTS, NR = NRA + FN * OB::PARTS;
    constexpr int NDMA = DMA ? OA::PER + OB::PER : 0;
    static_assert(NR <= FM * FN && NDMA <= FM * FN, "schedule slots");
#pragma unroll
    for (int i = 0; i < FM * FN; ++i) {
        const int a = i / FN, b = i % FN;
        acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(cat8(ca[a]), cat8(cb[b]), acc[a][b],
                                                            0, 0, 0);
        if (i < NRA) {
            OA::part(nst, wm + 32 * (i / OA::PARTS), nkk, lane, i % OA::PARTS, na[i / OA::PARTS]);
        } else if (i < NR) {
            const int j = i - NRA;
            OB::part(nst + FAST_TILE, wn + 32 * (j / OB::PARTS), nkk, lane, j % OB::PARTS,
                     nb[j / OB::PARTS]);
        }
        // DMA blocks go after the later ops, once the reads are under way.
        const int d = i - (FM * FN - NDMA);
        if (d >= 0) {
            if (d < OA::PER) oa.issue_one(rsa, soa, basea, d);
            else ob.issue_one(rsb, sob, baseb, d - OA::PER);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// As step_interleaved, with the two operands' next fragments in separate LDS stages (A of
// the deep ring, B of the 32-k ring) and NDB B blocks then NDA A blocks of DMA.
template <typename OA, typename OB, int FM, int FN, int NDA, int NDB>
__device__ inline void step_deep(const s16x4 (&ca)[FM][2], const s16x4 (&cb)[FN][2],
                                 f32x16 (&acc)[FM][FN], const uint16_t* la, int kka,
                                 const uint16_t* lb, int kkb, int wm, int wn, int lane,
                                 s16x4 (&na)[FM][2], s16x4 (&nb)[FN][2], const OA& oa,
                                 const OB& ob, u32x4 rsa, u32x4 rsb, uint32_t soa, uint32_t sob,
                                 uint32_t basea, uint32_t baseb) {
    constexpr int NRA = FM * OA::PARTS, NR = NRA + FN * OB::PARTS;
    constexpr int ND = NDA + NDB;
    static_assert(NR <= FM * FN && ND <= FM * FN, "schedule slots");
#pragma unroll
    for (int i = 0; i < FM * FN; ++i) {
        const int a = i / FN, b = i % FN;
        acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(cat8(ca[a]), cat8(cb[b]), acc[a][b],
                                                            0, 0, 0);
        if (i < NRA) {
            OA::part(la, wm + 32 * (i / OA::PARTS), kka, lane, i % OA::PARTS, na[i / OA::PARTS]);
        } else if (i < NR) {
            const int j = i - NRA;
            OB::part(lb, wn + 32 * (j / OB::PARTS), kkb, lane, j % OB::PARTS, nb[j / OB::PARTS]);
        }
        const int d = i - (FM * FN - ND);
        if (d >= 0) {
            if (d < NDB) ob.issue_one(rsb, sob, baseb, d);
            else oa.issue_one(rsa, soa, basea, d - NDB);
        }
        __builtin_amdgcn_sched_barrier(0);
    }
}

// Wait until at most n of this wave's DMA stages (2 * PER loads each) are in flight.
template <int PER2>
__device__ inline void wait_dma_stages(int n) {
    if (PER2 == 8) {
        if (n >= 2) asm volatile("s_waitcnt vmcnt(16)" ::: "memory");
        else if (n == 1) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    } else {
        if (n >= 2) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
        else if (n == 1) asm volatile("s_waitcnt vmcnt(4)" ::: "memory");
        else asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    }
}

}  // namespace
}  // namespace dh
