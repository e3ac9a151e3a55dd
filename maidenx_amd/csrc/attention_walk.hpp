// What the attention kernels count and address with whole numbers, for device and host alike (a host test walks through it):
// which wave brings which part of a tile, and the ring of places that tiles pass through.
#pragma once
#include <cstdint>

#if defined(__HIPCC__)
#include <hip/hip_runtime.h>
#define ATTN_HD __host__ __device__ __forceinline__
#else
#define ATTN_HD inline
#endif

namespace mxh {

// A tile of ROWS rows of PITCH bytes comes in wave instructions of 1 KB, shared out among GROUP waves.  Every wave issues the same
// number, N: it counts them to know what has come, so none may issue fewer.  Where a tile has fewer instructions than there are
// waves, two waves bring the same bytes to the same place; each waits for its own.
template <int ROWS, int PITCH, int GROUP>
struct AttnShare {
    static constexpr int PIECES = PITCH / 16;                  // of a row in LDS
    static constexpr int CALLS = ROWS * PITCH / 1024;
    static constexpr int N = (CALLS + GROUP - 1) / GROUP;
    static_assert(CALLS > 0 && (CALLS % GROUP == 0 || GROUP % CALLS == 0), "every wave issues N loads");
    static_assert(PIECES <= 64, "an instruction brings whole rows: a lane of it has the first piece of one, which is always there");
    ATTN_HD static int call_of(int u, int wave) { return CALLS < GROUP ? wave % CALLS : u * GROUP + wave; }
    ATTN_HD static int row_of(int u, int wave, int lane) { return (call_of(u, wave) * 64 + lane) / PIECES; }
};

// The tiles of a walk pass through a ring of `stages` (2 to 4) places in LDS: the place of a tile that is done with takes the next
// one behind those on their way.  A wave has issued PER loads for each, which come back in order: it waits until only those of the
// later tiles are out, then meets the others.
struct AttnRing {
    int stages, at = 0, to = 0, ahead = 0, left = 0;         // ahead: fetched and not done with; left: not fetched
    ATTN_HD explicit AttnRing(int stages_) : stages(stages_) {}
    template <class Fetch>
    ATTN_HD void begin(int total, Fetch&& fetch) {           // fetch(place)
        left = total;
        while (ahead < stages && left > 0) put(fetch);
    }
    template <class Fetch>
    ATTN_HD void put(Fetch&& fetch) {
        fetch(to);
        --left;
        ++ahead;
        to = to + 1 == stages ? 0 : to + 1;
    }
    template <class Fetch>
    ATTN_HD void refill(Fetch&& fetch) {                     // the place of the tile before
        if (left > 0 && ahead < stages) put(fetch);
    }
    ATTN_HD int later() const { return ahead - 1; }          // tiles behind the one at `at` that are on their way
    ATTN_HD void done() {
        --ahead;
        at = at + 1 == stages ? 0 : at + 1;
    }
};

// ---- sequences ------------------------------------------------------------------------------------------------------------
// The largest offset up to `row` (lo), the smallest above it (hi): one offset at a time, or by halves among many.
ATTN_HD void attn_take_offset(int off, int row, int& lo, int& hi, bool& above) {
    const bool upto = off <= row;
    lo = upto && off > lo ? off : lo;
    hi = !upto && off < hi ? off : hi;
    above |= !upto;
}
ATTN_HD void attn_search(const int32_t* offsets, int sequences, int row, int& lo, int& hi, bool& above) {
    int upto = 0, b = sequences + 1;           // offsets[0 .. upto) <= row < offsets[b ..)
    while (upto < b) {
        const int m = (upto + b) >> 1;
        if (offsets[m] <= row) upto = m + 1;
        else b = m;
    }
    if (upto > 0) lo = offsets[upto - 1];
    if (upto <= sequences) { above = true; hi = offsets[upto]; }
    if (hi <= row) hi = row + 1;
}
// The sequence [first, last) of a row, from what was found; false if none holds it.  Whatever the offsets: first <= row < last <= tokens.
ATTN_HD bool attn_bounds(int row, int tokens, int lo, int hi, bool above, int& first, int& last) {
    first = lo < 0 ? 0 : lo > row ? row : lo;
    last = hi > tokens ? tokens : hi;
    return row < tokens && lo >= 0 && above;
}

// What a wave has to know of its 32 rows, and a block of all its rows: the other axis from lo to hi; [inner, top) is what every row
// sees.  Rows see keys [first, row], keys are seen by queries [key, last): where offsets ascend, both ends ascend from row to row,
// and the first and the last row say it all.
struct AttnSpan {
    int lo = 0x7fffffff, hi = 0, inner = 0, top = 0x7fffffff;         // no rows
    ATTN_HD AttnSpan() {}
    ATTN_HD AttnSpan(int from_first, int upto_first, int from_last, int upto_last) : lo(from_first), hi(upto_last), inner(from_last), top(upto_first) {}
    ATTN_HD void put(int* s) const { s[0] = hi > lo ? lo : 0x7fffffff; s[1] = hi; s[2] = inner; s[3] = top; }
    ATTN_HD void join(const int* s) {
        lo = s[0] < lo ? s[0] : lo;
        hi = s[1] > hi ? s[1] : hi;
        inner = s[2] > inner ? s[2] : inner;
        top = s[3] < top ? s[3] : top;
    }
    // Offsets that do not ascend, among many sequences, may let the first row see further than the last: a walk ends at hi all the
    // same, for every tile is fetched up to there.
    ATTN_HD void close() { top = top < hi ? top : hi; }
};

// The tiles of a block's walk over [begin, end): first those that every row of the block sees whole, [clean, dirty) in steps of
// STEP, then the rest, in front of them and behind.
template <int STEP>
struct AttnWalk {
    int begin, clean, dirty, nclean, nfront, total;
    ATTN_HD AttnWalk(int begin_, int end, int from, int upto) : begin(begin_) {
        clean = from > begin ? begin + (from - begin + STEP - 1) / STEP * STEP : begin;
        nclean = upto > clean ? (upto - clean) / STEP : 0;
        if (nclean == 0) clean = begin;
        dirty = clean + nclean * STEP;
        nfront = (clean - begin) / STEP;
        total = nclean + nfront + (end > dirty ? (end - dirty + STEP - 1) / STEP : 0);
    }
    // (sums of selected values: a choice between members would keep the whole struct in memory)
    ATTN_HD int at(int n) const {
        return clean + n * STEP + (n >= nclean ? begin - dirty : 0) + (n >= nclean + nfront ? dirty - clean : 0);
    }
};

// A walk in rounds: in each, KG groups of waves take a tile of their own (every KG-th), all clean or none.  A group that is left without one in the
// last round fetches one that it does not need: every wave counts the same loads.
template <class Walk, int KG>
struct AttnRounds {
    const Walk& walk;
    int group, clean, total;
    ATTN_HD AttnRounds(const Walk& walk_, int group_)
        : walk(walk_), group(group_), clean((walk_.nclean + KG - 1) / KG), total(clean + (walk_.total - walk_.nclean + KG - 1) / KG) {}
    ATTN_HD int tile(int round) const { return round * KG + group + (round >= clean ? walk.nclean - clean * KG : 0); }
    ATTN_HD int nearest(int round) const {
        const int n = tile(round), last = walk.nclean - 1 + (round >= clean ? walk.total - walk.nclean : 0);
        return n < last ? n : last;
    }
};

}  // namespace mxh
