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

}  // namespace mxh
