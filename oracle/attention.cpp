// TEST INFRASTRUCTURE ONLY — causal attention over packed sequences with grouped heads and a bucketed relative position
// bias, from its formulas in f64, pair by pair (no counterpart in the reference).  Argument lists of hip_attention_<t> and
// hip_attention_backward_<t>; results are rounded to the tensors' type once.  Rows outside every sequence are not written.
#include <algorithm>

#include "common.hpp"

using namespace orc;

namespace {

inline double value(float x) { return x; }
template <class C> inline double value(half_t<C> x) { return x.to_f32(); }
inline void put(float& x, double v) { x = (float)v; }
template <class C> inline void put(half_t<C>& x, double v) { x = half_t<C>::from_f32((float)v); }

// bucket of a distance: E = buckets / 2 distances have one each, the rest share theirs by their logarithm.  The quotient of the
// logarithms is a whole number exactly where a bucket begins; 1e-12 keeps those on the right side of the floor.
int bucket_of(long n, int buckets, int max_distance) {
    const int E = buckets / 2;
    if (n < E) return (int)n;
    const long double q = std::log((long double)n / E) / std::log((long double)max_distance / E) * (buckets - E);
    return std::min(buckets - 1, E + (int)std::floor(q + 1e-12L));
}

template <class T>
struct Call {
    size_t tokens, heads, kv, dim, sequences, buckets, distance;
    const size_t *qs, *ks, *vs;
    const T *q, *k, *v, *table;
    double scale;
    Call(const size_t* md, const T* q_, const T* k_, const T* v_, const T* table_, float scale_)
        : tokens(md[0]), heads(md[1]), kv(md[2]), dim(md[3]), sequences(md[4]), buckets(md[5]), distance(md[6]), qs(md + 7), ks(md + 10), vs(md + 13),
          q(q_ + md[16]), k(k_ + md[17]), v(v_ + md[18]), table(table_), scale(scale_) {}
    double Q(size_t t, size_t h, size_t d) const { return value(q[t * qs[0] + h * qs[1] + d * qs[2]]); }
    double K(size_t t, size_t h, size_t d) const { return value(k[t * ks[0] + h * ks[1] + d * ks[2]]); }
    double V(size_t t, size_t h, size_t d) const { return value(v[t * vs[0] + h * vs[1] + d * vs[2]]); }
    // scores of query i from the first key of its sequence on
    void scores(size_t first, size_t i, size_t h, std::vector<double>& s) const {
        s.resize(i - first + 1);
        for (size_t j = first; j <= i; ++j) {
            double x = 0;
            for (size_t d = 0; d < dim; ++d) x += Q(i, h, d) * K(j, h / (heads / kv), d);
            s[j - first] = scale * x + (table ? value(table[bucket_of((long)(i - j), (int)buckets, (int)distance) * heads + h]) : 0.0);
        }
    }
    // exp(S - lse); a row of nothing but -inf is all zeros
    double softmax(std::vector<double>& s) const {
        double top = -INFINITY, sum = 0;
        for (double x : s) top = x > top || std::isnan(x) ? x : top;
        if (top == -INFINITY) { for (double& x : s) x = 0; return -INFINITY; }
        for (double& x : s) sum += x = std::exp(x - top);
        for (double& x : s) x /= sum;
        return top + std::log(sum);
    }
};

template <class T>
void forward(const size_t* md, const int32_t* offsets, const T* q, const T* k, const T* v, const T* table, float scale, T* out, float* lse) {
    const Call<T> c(md, q, k, v, table, scale);
#pragma omp parallel for schedule(static)
    for (size_t h = 0; h < c.heads; ++h) {
        std::vector<double> p;
        for (size_t s = 0; s < c.sequences; ++s)
            for (size_t i = offsets[s]; i < (size_t)offsets[s + 1]; ++i) {
                c.scores(offsets[s], i, h, p);
                lse[h * c.tokens + i] = (float)c.softmax(p);
                for (size_t d = 0; d < c.dim; ++d) {
                    double x = 0;
                    for (size_t j = 0; j < p.size(); ++j) x += p[j] * c.V(offsets[s] + j, h / (c.heads / c.kv), d);
                    put(out[(i * c.heads + h) * c.dim + d], x);
                }
            }
    }
}

// (o and lse are formed again in f64: the gradients are those of the exact forward pass)
template <class T>
void backward(const size_t* md, const int32_t* offsets, const T* q, const T* k, const T* v, const T* table, float scale, const T*, const float*, const T* go,
              T* gq, T* gk, T* gv, T* gt) {
    const Call<T> c(md, q, k, v, table, scale);
    const size_t group = c.heads / c.kv;
    std::vector<double> gtable(table ? c.buckets * c.heads : 0, 0.0);
#pragma omp parallel for schedule(static)
    for (size_t g = 0; g < c.kv; ++g) {
        std::vector<double> p, dk(c.tokens * c.dim, 0.0), dv(c.tokens * c.dim, 0.0), dp, dq(c.dim);
        for (size_t h = g * group; h < (g + 1) * group; ++h)
            for (size_t s = 0; s < c.sequences; ++s)
                for (size_t i = offsets[s]; i < (size_t)offsets[s + 1]; ++i) {
                    const size_t first = offsets[s];
                    c.scores(first, i, h, p);
                    c.softmax(p);
                    dp.assign(p.size(), 0.0);
                    double delta = 0;
                    for (size_t j = 0; j < p.size(); ++j) {
                        for (size_t d = 0; d < c.dim; ++d) {
                            const double o = value(go[(i * c.heads + h) * c.dim + d]);
                            dp[j] += o * c.V(first + j, g, d);
                            dv[(first + j) * c.dim + d] += p[j] * o;
                        }
                        delta += p[j] * dp[j];
                    }
                    std::fill(dq.begin(), dq.end(), 0.0);
                    for (size_t j = 0; j < p.size(); ++j) {
                        const double ds = p[j] == 0 ? 0 : p[j] * (dp[j] - delta);
                        for (size_t d = 0; d < c.dim; ++d) {
                            dq[d] += ds * c.K(first + j, g, d);
                            dk[(first + j) * c.dim + d] += ds * c.Q(i, h, d);
                        }
                        if (table) gtable[bucket_of((long)(i - first - j), (int)c.buckets, (int)c.distance) * c.heads + h] += ds;
                    }
                    if (gq) for (size_t d = 0; d < c.dim; ++d) put(gq[(i * c.heads + h) * c.dim + d], c.scale * dq[d]);
                }
        for (size_t s = 0; s < c.sequences; ++s)
            for (size_t j = offsets[s]; j < (size_t)offsets[s + 1]; ++j)
                for (size_t d = 0; d < c.dim; ++d) {
                    if (gk) put(gk[(j * c.kv + g) * c.dim + d], c.scale * dk[j * c.dim + d]);
                    if (gv) put(gv[(j * c.kv + g) * c.dim + d], dv[j * c.dim + d]);
                }
    }
    if (gt) for (size_t n = 0; n < gtable.size(); ++n) put(gt[n], gtable[n]);
}

}  // namespace

#define ORC_ATTENTION(T, S)                                                                                                            \
    extern "C" void oracle_attention_##S(const size_t* md, const int32_t* offsets, const T* q, const T* k, const T* v, const T* bias, \
                                         float scale, T* out, float* lse) {                                                           \
        forward<T>(md, offsets, q, k, v, bias, scale, out, lse);                                                                       \
    }                                                                                                                                  \
    extern "C" void oracle_attention_backward_##S(const size_t* md, const int32_t* offsets, const T* q, const T* k, const T* v,       \
                                                  const T* bias, float scale, const T* out, const float* lse, const T* go, T* gq,     \
                                                  T* gk, T* gv, T* gbias) {                                                           \
        backward<T>(md, offsets, q, k, v, bias, scale, out, lse, go, gq, gk, gv, gbias);                                               \
    }
ORC_ATTENTION(float, f32)
ORC_ATTENTION(bf16, bf16)
ORC_ATTENTION(f16, f16)
