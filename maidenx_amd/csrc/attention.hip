// Attention for f32 tensors, and the bucket borders of the relative position bias (see attention.hpp).
#include <vector>

#include "attention.hpp"

namespace mxh {

// x^n as whole numbers of 32-bit limbs, least first
typedef std::vector<uint32_t> Whole;
static void multiply(Whole& w, uint32_t x) {
    uint64_t carry = 0;
    for (uint32_t& limb : w) {
        carry += (uint64_t)limb * x;
        limb = (uint32_t)carry;
        carry >>= 32;
    }
    if (carry) w.push_back((uint32_t)carry);
}
static bool less(const Whole& a, const Whole& b) {
    if (a.size() != b.size()) return a.size() < b.size();
    for (size_t i = a.size(); i-- > 0;)
        if (a[i] != b[i]) return a[i] < b[i];
    return false;
}

// Bucket E + m begins at the least whole n with (n / E)^M >= (X / E)^m, that is n^M >= X^m E^(M - m) (E = buckets / 2,
// M = buckets - E, X = max_distance).  The logarithms of the definition are whole numbers exactly there, where floating
// point falls on either side: the estimate is corrected with whole numbers.
bool attn_borders(int buckets, int max_distance, uint16_t* borders) {
    static int known_buckets = 0, known_distance = 0;            // (under the library's lock)
    static uint16_t known[ATTN_MAX_BUCKETS / 2];
    const int E = buckets / 2, M = buckets - E;
    if (known_buckets != buckets || known_distance != max_distance) {
        for (int m = 1; m < M; ++m) {
            Whole right{1};
            for (int i = 0; i < m; ++i) multiply(right, (uint32_t)max_distance);
            for (int i = m; i < M; ++i) multiply(right, (uint32_t)E);
            auto reaches = [&](int n) {
                Whole left{1};
                for (int i = 0; i < M; ++i) multiply(left, (uint32_t)n);
                return !less(left, right);
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
