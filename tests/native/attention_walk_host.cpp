// The whole-number part of the attention kernels (maidenx_amd/csrc/attention_walk.hpp) on the host: which wave brings what of a
// tile, and whether a tile has come when the ring says so.
#include <cstring>
#include <deque>
#include <vector>

#include "../../maidenx_amd/csrc/attention_walk.hpp"

using namespace mxh;

namespace {

// what a wave has issued and not waited for, in order: the number of the tile
struct Wave {
    std::deque<int> out;
    void wait(int left) { while ((int)out.size() > left) out.pop_front(); }
};

template <int ROWS, int PITCH, int GROUP>
struct Walked {
    using Share = AttnShare<ROWS, PITCH, GROUP>;
    // every 16-byte place of the tile is filled, from the row that lies there, and every wave issues N instructions with a lane that
    // has something to bring (the first piece of a row is always there); what goes wrong, counted
    static int shares() {
        std::vector<int> filled(Share::CALLS, 0);
        int wrong = 0;
        for (int wave = 0; wave < GROUP; ++wave)
            for (int u = 0; u < Share::N; ++u) {
                const int call = Share::call_of(u, wave);
                if (call < 0 || call >= Share::CALLS) { ++wrong; continue; }
                ++filled[call];
                for (int lane = 0; lane < 64; ++lane) {
                    const int row = Share::row_of(u, wave, lane);
                    wrong += row < 0 || row >= ROWS || row != (call * 64 + lane) * 16 / PITCH;
                }
            }
        for (int n : filled) wrong += n == 0;
        return wrong;
    }
    // `total` tiles of two operands through a ring; an operand that is not direct goes through registers, after which nothing is
    // out; `own` loads of every wave besides.  How often a wave goes on while a load of its tile is still out.
    static int waits(int stages, int total, bool direct_a, bool direct_b, int own) {
        const int per = 2 * Share::N + own;
        std::vector<Wave> waves(GROUP);
        AttnRing ring(stages);
        int next = 0, early = 0;
        std::vector<int> in_place(stages, -1);
        auto fetch = [&](int place) {
            for (int w = 0; w < GROUP; ++w) {
                for (bool direct : {direct_a, direct_b}) {
                    for (int u = 0; direct && u < Share::N; ++u)
                        if (Share::row_of(u, w, 0) < ROWS) waves[w].out.push_back(next);
                    if (!direct) waves[w].wait(0);
                }
                for (int x = 0; x < own; ++x) waves[w].out.push_back(next);
            }
            in_place[place] = next++;
        };
        ring.begin(total, fetch);
        for (int tile = 0; tile < total; ++tile) {
            const int later = ring.later();
            for (Wave& w : waves) {
                w.wait((later < 3 ? later : 3) * per);
                for (int t : w.out) early += t <= tile;
            }
            early += in_place[ring.at] != tile;
            ring.refill(fetch);
            ring.done();
        }
        return early + ring.left;
    }
};

template <class F>
int each(F&& f) {
    int wrong = 0;
    wrong += f(Walked<32, 64, 4>{}) + f(Walked<32, 128, 4>{}) + f(Walked<32, 256, 4>{}) + f(Walked<32, 512, 4>{});
    wrong += f(Walked<64, 64, 4>{}) + f(Walked<64, 128, 4>{}) + f(Walked<64, 256, 4>{});
    wrong += f(Walked<32, 128, 2>{}) + f(Walked<32, 256, 2>{}) + f(Walked<64, 64, 2>{}) + f(Walked<64, 128, 2>{});
    return wrong;
}

// ---- the walks that offsets make ------------------------------------------------------------------------------------------
bool sequence(const int32_t* offsets, int sequences, int tokens, int row, int& first, int& last) {
    int lo = -1, hi = tokens;
    bool above = false;
    if (sequences < 64)
        for (int e = 0; e <= sequences; ++e) attn_take_offset(offsets[e], row, lo, hi, above);
    else
        attn_search(offsets, sequences, row, lo, hi, above);
    return attn_bounds(row, tokens, lo, hi, above, first, last);
}

// Every block of WAVES waves of 32 rows: the tiles of its walk, of STEP tokens, must begin in front of the token up to which they are
// fetched, clean ones lie whole in front of it, and nothing lie outside the tokens.  Where offsets ascend, also: the tiles hold every
// token that a row sees, once, and every row sees the clean ones whole.  `keys`: rows are queries and see keys.
template <int WAVES, int STEP, int KG>
int walked(const int32_t* offsets, int sequences, int tokens, bool keys, bool ascending) {
    int wrong = 0;
    for (int block = 0; block < tokens; block += 32 * WAVES) {
        AttnSpan all;
        std::vector<int> from(32 * WAVES, 0), upto(32 * WAVES, 0);
        for (int w = 0; w < WAVES; ++w) {
            int a = -1, b = -1;
            for (int r = 32 * w; r < 32 * w + 32; ++r) {
                int first, last;
                if (!sequence(offsets, sequences, tokens, block + r, first, last)) continue;
                from[r] = keys ? first : block + r;
                upto[r] = keys ? block + r + 1 : last;
                wrong += from[r] < 0 || from[r] >= upto[r] || upto[r] > tokens;
                if (a < 0) a = r;
                b = r;
            }
            const AttnSpan own = a < 0 ? AttnSpan() : AttnSpan(from[a], upto[a], from[b], upto[b]);
            int s[4];
            own.put(s);
            all.join(s);
        }
        all.close();
        if (keys && all.hi <= all.lo) continue;
        const AttnWalk<STEP> walk(all.lo, all.hi > all.lo ? all.hi : all.lo, all.inner, all.top);
        std::vector<int> held(tokens + STEP, 0);
        for (int n = 0; n < walk.total; ++n) {
            const int t = walk.at(n);
            wrong += t < 0 || t >= all.hi || all.hi > tokens || (n < walk.nclean && t + STEP > all.hi);
            if (t < 0 || t >= tokens) continue;
            for (int x = t; x < t + STEP; ++x) ++held[x];
            if (ascending && n < walk.nclean)
                for (int r = 0; r < 32 * WAVES; ++r) wrong += upto[r] > 0 && (t < from[r] || t + STEP > upto[r]);
        }
        if (ascending)
            for (int r = 0; r < 32 * WAVES; ++r)
                for (int x = from[r]; x < upto[r]; ++x) wrong += held[x] != 1;
        for (int group = 0; group < KG; ++group) {
            const AttnRounds<AttnWalk<STEP>, KG> rounds(walk, group);
            for (int r = 0; r < rounds.total; ++r) wrong += rounds.nearest(r) < 0 || rounds.nearest(r) >= walk.total;
        }
    }
    return wrong;
}

}  // namespace

extern "C" {
int walk_offsets(const int32_t* offsets, int sequences, int tokens, int ascending) {
    return walked<4, 64, 1>(offsets, sequences, tokens, true, ascending != 0) + walked<4, 32, 2>(offsets, sequences, tokens, true, ascending != 0) +
           walked<2, 64, 4>(offsets, sequences, tokens, true, ascending != 0) + walked<2, 32, 4>(offsets, sequences, tokens, true, ascending != 0) +
           walked<4, 32, 1>(offsets, sequences, tokens, false, ascending != 0);
}
int walk_shares() { return each([](auto w) { return w.shares(); }); }
int walk_waits(int stages, int total, int direct_a, int direct_b, int own) {
    return each([&](auto w) { return w.waits(stages, total, direct_a != 0, direct_b != 0, own); });
}
}
