// TEST INFRASTRUCTURE ONLY — the clipped policy loss with a KL term and its gradient, from their formulas in f64 (no counterpart
// in the reference).  Argument lists of hip_policy_loss_<t>_<i>, hip_policy_loss_backward_.. and hip_policy_loss_step_..
#include <algorithm>

#include "common.hpp"

using namespace orc;

namespace {

inline double value(float x) { return x; }
template <class C> inline double value(half_t<C> x) { return x.to_f32(); }
inline void put(float& x, double v) { x = (float)v; }
template <class C> inline void put(half_t<C>& x, double v) { x = half_t<C>::from_f32((float)v); }

template <class T, class I>
struct Call {
    size_t rows, vocab, row, elem;
    const T* x;
    const I* target;
    const float *old_logp, *ref_logp, *advantage, *weight;
    double least, most, beta;
    Call(const size_t* md, const I* target_, const T* logits, const float* o, const float* r, const float* a, const float* w, float low, float high, float kl)
        : rows(md[0]), vocab(md[1]), row(md[2]), elem(md[3]), x(logits + md[4]), target(target_), old_logp(o), ref_logp(r), advantage(a), weight(w),
          least(1.0 - low), most(1.0 + high), beta(kl) {}
    bool counts(size_t t) const { return weight[t] != 0 && target[t] >= 0 && (size_t)target[t] < vocab; }
    double X(size_t t, size_t v) const { return value(x[t * row + v * elem]); }
    double log_sum(size_t t) const {
        double top = -INFINITY, sum = 0;
        for (size_t v = 0; v < vocab; ++v) top = X(t, v) > top || std::isnan(X(t, v)) ? X(t, v) : top;
        for (size_t v = 0; v < vocab; ++v) sum += std::exp(X(t, v) - top);
        return top + std::log(sum);
    }
    // the row's term, and its derivative with respect to lp
    double term(size_t t, double lp, double& g) const {
        const double r = std::exp(lp - old_logp[t]), a = advantage[t], plain = r * a, clipped = std::min(std::max(r, least), most) * a;
        double x = -std::min(plain, clipped);
        g = plain <= clipped ? -plain : 0;
        if (beta != 0) {
            const double away = ref_logp[t] - lp;
            x += beta * (std::exp(away) - away - 1);
            g += beta * (1 - std::exp(away));
        }
        g *= weight[t];
        return x * weight[t];
    }
    void forward(float* loss, float* logp, float* lse) const {
        double sum = 0, g;
        for (size_t t = 0; t < rows; ++t) {
            const double s = counts(t) ? log_sum(t) : 0, lp = counts(t) ? X(t, (size_t)target[t]) - s : 0;
            logp[t] = (float)lp;
            lse[t] = (float)s;
            if (counts(t)) sum += term(t, lp, g);
        }
        loss[0] = (float)sum;
    }
    // (the sums are formed again in f64)
    void gradient(const float* grad_loss, T* grad) const {
        for (size_t t = 0; t < rows; ++t) {
            double s = 0, g = 0;
            if (counts(t)) {
                s = log_sum(t);
                term(t, X(t, (size_t)target[t]) - s, g);
            }
            g *= grad_loss ? grad_loss[0] : 1.0;
            for (size_t v = 0; v < vocab; ++v) put(grad[t * vocab + v], g == 0 ? 0 : g * ((v == (size_t)target[t]) - std::exp(X(t, v) - s)));
        }
    }
};

}  // namespace

#define ORC_POLICY_ARGS(T, I) const size_t *md, const I *target, const T *logits, const float *old_logp, const float *ref_logp, const float *advantage, const float *weight, float low, float high, float kl
#define ORC_POLICY(T, S, I, IS)                                                                                                        \
    extern "C" void oracle_policy_loss_##S##_##IS(ORC_POLICY_ARGS(T, I), float* loss, float* logp, float* lse) {                       \
        Call<T, I>(md, target, logits, old_logp, ref_logp, advantage, weight, low, high, kl).forward(loss, logp, lse);                 \
    }                                                                                                                                  \
    extern "C" void oracle_policy_loss_backward_##S##_##IS(ORC_POLICY_ARGS(T, I), const float*, const float*, const float* grad_loss, T* grad) { \
        Call<T, I>(md, target, logits, old_logp, ref_logp, advantage, weight, low, high, kl).gradient(grad_loss, grad);                \
    }                                                                                                                                  \
    extern "C" void oracle_policy_loss_step_##S##_##IS(ORC_POLICY_ARGS(T, I), const float* grad_loss, float* loss, float* logp, float* lse, T* grad) { \
        const Call<T, I> c(md, target, logits, old_logp, ref_logp, advantage, weight, low, high, kl);                                  \
        c.forward(loss, logp, lse);                                                                                                    \
        c.gradient(grad_loss, grad);                                                                                                   \
    }
#define ORC_POLICY_BOTH(T, S) ORC_POLICY(T, S, int32_t, i32) ORC_POLICY(T, S, int64_t, i64)
ORC_POLICY_BOTH(float, f32)
ORC_POLICY_BOTH(bf16, bf16)
ORC_POLICY_BOTH(f16, f16)
