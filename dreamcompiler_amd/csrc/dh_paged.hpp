// dh_paged.hpp -- the paged key-value cache: where a sequence's tokens lie, what its 8-bit values
// stand for, and the checks that its operators share.
//
// Keys and values are pages x Hk x page x D each, of the cache's type; 8-bit types have a scale for
// every row of D, pages x Hk x page.  Sequence b's token t is in page table[b ld + t / page], at place
// t % page.  A table entry outside 0 .. pages - 1 holds nothing.
#pragma once

#include "dh_common.hpp"

namespace dh {

constexpr int PAGED_MOST_D = 256;

struct Paged {
    int pages, shift, Hk, D;   // page = 1 << shift
    const int* table;
    int ld;
    void *K, *V;
    float *Ks, *Vs;

    // Page of token t of sequence b, or -1.
    __device__ int page_of(int b, int t) const {
        const int i = t >> shift;
        if (t < 0 || i >= ld) return -1;
        const int id = table[(long long)b * ld + i];
        return (unsigned)id < (unsigned)pages ? id : -1;
    }
    // Row of D values (and of its scale) of place `at` of a page, head h.
    __device__ long long row(int id, int h, int at) const {
        return ((((long long)id * Hk + h) << shift) + at);
    }
};

__device__ inline float paged_up(float x) { return x; }
__device__ inline float paged_up(uint16_t x) { return bf16_bits_to_f32(x); }
__device__ inline float paged_up(int8_t x) { return (float)x; }
__device__ inline float paged_up(uint8_t x) { return __builtin_amdgcn_cvt_f32_fp8(x, 0); }

// Checks of a cache and its table; fills c.  `op` names the call.
int check_paged(const char* op, int dtype, int cache_type, int B, int Hk, int D, int pages, int page,
                const int* d_table, int ld_table, const void* d_Kc, const void* d_Vc, const float* d_Ks,
                const float* d_Vs, Paged& c);
// Whether n0 x n1 rows of D values at the strides st lie within 2^46 elements, and apart where they
// are written.
int check_strides(const char* op, const char* name, const long long* st, long long n0, long long n1, int D,
                  bool out);

}  // namespace dh
