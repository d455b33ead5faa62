// Limits of the list of tiles that attention over a paged cache deals to its resident CTAs. Host arithmetic only.
#pragma once
#include <stdint.h>

// Parts of one q head that a join takes: seven of each of its 256 threads. A unit has a part of every warp of the CTAs that touch it, at most of all of them: 444 CTAs
// of four warps leave 1776.
constexpr uint32_t PAGED_PARTS_MOST = 1792;

// CTAs that share a list: as many as are resident, but no more than a join takes the parts of. Only devices of 150 SMs or more have fewer at work for it.
inline uint32_t paged_list_ctas(uint32_t sms, uint32_t per_sm, uint32_t warps) {
    const uint32_t resident = sms * per_sm, most = PAGED_PARTS_MOST / warps;
    return resident < most ? resident : most;
}

// Whether no CTA's equal run of a list of `rows` rows, `units` units a row and `tiles` tiles a unit passes 32 bits, in which its tiles are counted. rows <= 256,
// units <= 65535 and tiles <= 2^27 (2^30 entries by 8), so that the list itself and its product with the CTAs fit 64.
inline bool paged_list_fits(uint32_t rows, uint64_t units, uint32_t tiles, uint32_t ctas) { return rows * units * tiles / 0xffffffffu < ctas; }
