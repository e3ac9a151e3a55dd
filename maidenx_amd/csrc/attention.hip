// Attention for f32 tensors, and the bucket borders of the relative position bias (see attention.hpp).
#include "attention.hpp"

namespace mxh {

// a whole number of 32-bit limbs, least first; the largest here is 4096^128 = 2^1536
struct Whole {
    static constexpr int MOST = (12 * ATTN_MAX_BUCKETS / 2 + 31) / 32 + 1;
    static_assert(ATTN_MAX_DISTANCE <= 4096, "12 bits a factor");
    uint32_t limb[MOST] = {1};
    int size = 1;
    void multiply(uint32_t x) {
        uint64_t carry = 0;
        for (int i = 0; i < size; ++i) {
            carry += (uint64_t)limb[i] * x;
            limb[i] = (uint32_t)carry;
            carry >>= 32;
        }
        if (carry && size < MOST) limb[size++] = (uint32_t)carry;
    }
    bool below(const Whole& b) const {
        if (size != b.size) return size < b.size;
        for (int i = size; i-- > 0;)
            if (limb[i] != b.limb[i]) return limb[i] < b.limb[i];
        return false;
    }
};

// Bucket E + m begins at the least whole n with (n / E)^M >= (X / E)^m, that is n^M >= X^m E^(M - m) (E = buckets / 2,
// M = buckets - E, X = max_distance).  The logarithms of the definition are whole numbers exactly there, where floating
// point falls on either side: the estimate is corrected with whole numbers.
bool attn_borders(int buckets, int max_distance, uint16_t* borders) {
    static int known_buckets = 0, known_distance = 0;            // (under the library's lock)
    static uint16_t known[ATTN_MAX_BUCKETS / 2];
    const int E = buckets / 2, M = buckets - E;
    if (known_buckets != buckets || known_distance != max_distance) {
        for (int m = 1; m < M; ++m) {
            Whole right;
            for (int i = 0; i < m; ++i) right.multiply((uint32_t)max_distance);
            for (int i = m; i < M; ++i) right.multiply((uint32_t)E);
            auto reaches = [&](int n) {
                Whole left;
                for (int i = 0; i < M; ++i) left.multiply((uint32_t)n);
                return !left.below(right);
            };
            int n = (int)std::floor((double)E * std::pow((double)max_distance / E, (double)m / M));
            while (n > 1 && reaches(n - 1)) --n;
            while (!reaches(n)) ++n;
            known[m - 1] = (uint16_t)n;
        }
        known_buckets = buckets;
        known_distance = max_distance;
    }
    std::memcpy(borders, known, (size_t)(M - 1) * sizeof(uint16_t));
    return true;
}

}  // namespace mxh
using namespace mxh;

MXH_ATTENTION(float, f32)
