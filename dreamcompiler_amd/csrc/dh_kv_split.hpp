// dh_kv_split.hpp -- how the cache's reads and writes are split over waves.  Plain C++, so that it can be
// checked without a GPU.
#pragma once
#include <cstdint>

namespace dh {

// A wave has `places` rows of a side at once, `ahead` times.  Where there are fewer heads than half of that (many), a
// power of two of places, 2^log_heads, belong to a token and the wave has several tokens at once; else it takes
// `each` of a token's `blocks` of heads, and `per` waves take the same tokens.
struct Split {
    int tokens, log_heads, blocks, each, per;
    uint32_t units;   // waves
    bool many;
};

constexpr int MOST_TOKENS = 64;

// Tokens of a wave: as many as leave each of 24576 waves some (three times what the GPU holds, for the tail's sake);
// blocks of heads, where there are fewer tokens, likewise.
constexpr Split split_tokens(int N, int Hk, int places, int ahead) {
    int log_heads = 0, tokens = N / 24576;
    while (1 << log_heads < Hk) ++log_heads;
    const bool many = 2 << log_heads <= places;
    const int side = many ? places >> log_heads : 1;
    tokens = (tokens + side - 1) / side * side;
    tokens = tokens < side ? side : tokens > MOST_TOKENS ? MOST_TOKENS : tokens;
    const int blocks = many ? 1 : (Hk + places * ahead - 1) / (places * ahead);
    long long groups = ((long long)N + tokens - 1) / tokens;
    int each = (int)((groups * blocks + 24575) / 24576);
    if (each > blocks) each = blocks;
    const int per = (blocks + each - 1) / each;
    each = (blocks + per - 1) / per;   // as many for each
    if (per == 1) groups = (groups + 3) / 4 * 4;   // four waves in turn
    return Split{tokens, log_heads, blocks, each, per, (uint32_t)groups * per, many};
}

// Where many: the place `sub` has head sub % 2^log_heads of the tokens first_token + side k, k < ahead rounds.  The
// rounds are the wave's, not the lane's: its lanes read each other's places.
constexpr int first_token(int sub, int log_heads) { return sub >> log_heads; }
constexpr int rounds_of(int tokens, int side, int ahead) { return (tokens + ahead * side - 1) / (ahead * side); }

}  // namespace dh
