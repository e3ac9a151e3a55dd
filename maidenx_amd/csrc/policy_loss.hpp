// Clipped policy loss with a KL term over logits [rows, vocabulary], and its gradient.
//
//   lse = ln sum_v exp x_v;  lp = x_target - lse;  r = exp(lp - old);  c = min(max(r, 1 - low), 1 + high)
//   term = weight * (-min(r A, c A) + beta (exp(ref - lp) - (ref - lp) - 1));  loss = sum of the terms
//   g = weight * (-[r A <= c A] r A + beta (1 - exp(ref - lp)))                          d loss / d lp
//   d loss / d x_v = grad_loss * g * ([v == target] - exp(x_v - lse))
//
// Rows of weight zero (prompt tokens) are not read.  Bound by memory: a forward pass reads the logits once; forward and gradient
// together hold a row in one block's registers between the two, so that it is read once and written once.
// Sums are f32 in a fixed order (the loss itself is added in f64); the gradient is rounded to the logits' type once.
#pragma once
#include <cmath>
#include <cstring>
#include <type_traits>

#include "mxh.hpp"

namespace mxh {

constexpr float POLICY_LOG2E = 1.4426950408889634f, POLICY_LN2 = 0.6931471805599453f;
constexpr int POLICY_SUM_THREADS = 1024;
typedef uint32_t policy_piece __attribute__((ext_vector_type(4)));

template <class E> struct PolicyType;
template <> struct PolicyType<float> {
    static constexpr int N = 4;       // elements in 16 bytes
    __device__ static float get(float x) { return x; }
    __device__ static float put(float x) { return x; }
};
template <> struct PolicyType<bf16_t> {
    static constexpr int N = 8;
    __device__ static float get(bf16_t x) { return bf2f(x); }
    __device__ static bf16_t put(float x) { return f2bf(x); }
};
template <> struct PolicyType<f16_t> {
    static constexpr int N = 8;
    __device__ static float get(f16_t x) { return h2f(x); }
    __device__ static f16_t put(float x) { return f2h(x); }
};

template <class E, class I>
struct PolicyArgs {
    const E* logits;
    int64_t row, elem;                // strides
    const I* target;
    const float *old_logp, *ref_logp, *advantage, *weight, *grad_loss;
    float least, most, beta;          // 1 - low, 1 + high
    int32_t rows, vocab, row0;        // row0: of a launch's first block
    float *loss, *logp, *lse, *terms;
    E* grad;
    int* flag;
};

// ---- a row in 16-byte pieces ---------------------------------------------------------------------------------------------
// Piece p of a row are its elements p N - lead .. p N - lead + N - 1, lead being what keeps the pieces on 16-byte boundaries:
// a row of an odd vocabulary starts anywhere.  Pieces that are not whole are moved element by element.
template <class E>
__device__ inline int policy_lead(const E* row) { return (int)(((uintptr_t)row & 15) / sizeof(E)); }

template <class E>
__device__ inline void policy_load(const E* row, int64_t elem, int vocab, int lead, int piece, bool whole_pieces, float (&x)[PolicyType<E>::N]) {
    constexpr int N = PolicyType<E>::N;
    const int v0 = piece * N - lead;
    if (whole_pieces && v0 >= 0 && v0 + N <= vocab) {
        const policy_piece p = *(const policy_piece*)(row + v0);
        E y[N];
        __builtin_memcpy(y, &p, 16);
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = PolicyType<E>::get(y[e]);
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e) x[e] = v0 + e >= 0 && v0 + e < vocab ? PolicyType<E>::get(row[(int64_t)(v0 + e) * elem]) : -INFINITY;
    }
}
// the same, kept in its storage form (elements outside the row: undefined)
template <class E>
__device__ inline policy_piece policy_fetch(const E* row, int vocab, int lead, int piece) {
    constexpr int N = PolicyType<E>::N;
    const int v0 = piece * N - lead;
    if (v0 >= 0 && v0 + N <= vocab) return *(const policy_piece*)(row + v0);
    E y[N];
#pragma unroll
    for (int e = 0; e < N; ++e) {
        y[e] = PolicyType<E>::put(-INFINITY);
        if (v0 + e >= 0 && v0 + e < vocab) y[e] = row[v0 + e];
    }
    policy_piece p;
    __builtin_memcpy(&p, y, 16);
    return p;
}
template <class E>
__device__ inline void policy_store(E* row, int vocab, int lead, int piece, bool whole_pieces, const float (&x)[PolicyType<E>::N]) {
    constexpr int N = PolicyType<E>::N;
    const int v0 = piece * N - lead;
    E y[N];
#pragma unroll
    for (int e = 0; e < N; ++e) y[e] = PolicyType<E>::put(x[e]);
    if (whole_pieces && v0 >= 0 && v0 + N <= vocab) {
        policy_piece p;
        __builtin_memcpy(&p, y, 16);
        *(policy_piece*)(row + v0) = p;
    } else {
#pragma unroll
        for (int e = 0; e < N; ++e)
            if (v0 + e >= 0 && v0 + e < vocab) row[v0 + e] = y[e];
    }
}

// running (base, sum) of a row: the sum of exp(x - base).  The difference is taken before it is brought to units of log2: logits near
// the type's limits have no such units.
struct PolicySum {
    float base, sum;
};
// An instruction less for each logit: exp(x - base) as 2^(x log2(e) - base log2(e)), where base is small enough for its product's rounding
// to be nothing beside the tensors' own (16 bits; 256 log2(e) 2^-24 = 2^-15).  bf16, 8192 rows of 50001: 329 us with
// the choice, 395 where every logit is subtracted from; 2048 rows of 32000 are the same, 50.
template <class E>
__device__ inline bool policy_near(float base) { return sizeof(E) == 2 && __builtin_fabsf(base) <= 256.0f; }
__device__ inline float policy_exp(float x) { return __builtin_amdgcn_exp2f(x * POLICY_LOG2E); }
__device__ inline PolicySum policy_join(PolicySum a, PolicySum b) {
    const float base = fmaxf(a.base, b.base);
    if (base == -INFINITY) return {base, a.sum + b.sum};     // (nothing yet: sums are zero, or NaN)
    return {base, a.sum * policy_exp(a.base - base) + b.sum * policy_exp(b.base - base)};
}
template <int N>
__device__ inline void policy_take(PolicySum& s, const float (&x)[N]) {
    float top = x[0];
#pragma unroll
    for (int e = 1; e < N; ++e) top = fmaxf(top, x[e]);
    if (top > s.base) {
        s.sum *= policy_exp(s.base - top);
        s.base = top;
    }
    const float base = s.base == -INFINITY ? 0.0f : s.base;
#pragma unroll
    for (int e = 0; e < N; ++e) s.sum += policy_exp(x[e] - base);
}
__device__ inline PolicySum policy_join_wave(PolicySum s) {
#pragma unroll
    for (int d = 1; d < WAVE; d <<= 1) s = policy_join(s, PolicySum{__shfl_xor(s.base, d, WAVE), __shfl_xor(s.sum, d, WAVE)});
    return s;
}
template <int THREADS>
__device__ inline PolicySum policy_join_block(PolicySum s, PolicySum* shared) {
    s = policy_join_wave(s);
    if (threadIdx.x % WAVE == 0) shared[threadIdx.x / WAVE] = s;
    __syncthreads();
    s = shared[0];
#pragma unroll
    for (int w = 1; w < THREADS / WAVE; ++w) s = policy_join(s, shared[w]);
    return s;
}

// lp = x_target - lse.  What follows subtracts it from numbers near to it and sums terms that cancel: the subtraction of the two
// is made in f64, and the logarithm of the sum gets the digits that f32 drops from a product of its own with what it stands for.
__device__ inline double policy_logp(float x, PolicySum s, float log_sum) {
    const float base = s.base == -INFINITY ? 0.0f : s.base;
    const float missing = __builtin_isinf(log_sum) ? 0.0f : __builtin_fmaf(s.sum, __builtin_amdgcn_exp2f(-log_sum), -1.0f) * POLICY_LOG2E;
    return (double)x - (double)base - ((double)log_sum + (double)missing) * 0.6931471805599453;
}

// ---- a row's term of the loss and its gradient with respect to lp -----------------------------------------------------------
struct PolicyToken {
    float term, g;
};
template <class E, class I>
__device__ inline PolicyToken policy_token(const PolicyArgs<E, I>& a, int row, double logp) {
    const float w = a.weight[row], adv = a.advantage[row];
    const float ratio = expf((float)(logp - (double)a.old_logp[row]));
    const float clipped = fminf(fmaxf(ratio, a.least), a.most) * adv, plain = ratio * adv;
    PolicyToken t;
    t.term = -(plain <= clipped || plain != plain ? plain : clipped);
    t.g = plain <= clipped ? -plain : plain != plain ? plain : 0.0f;
    if (a.beta != 0.0f) {
        const float away = (float)((double)a.ref_logp[row] - logp), grown = expm1f(away);
        t.term += a.beta * (grown - away);
        t.g -= a.beta * grown;
    }
    t.term *= w;
    t.g *= w;
    return t;
}
// the target of a row that counts; -1 for one that does not (weight zero, or a target outside the vocabulary: reported)
template <class E, class I>
__device__ inline int policy_target(const PolicyArgs<E, I>& a, int row, bool report) {
    if (a.weight[row] == 0.0f) return -1;
    const int64_t t = (int64_t)a.target[row];
    if (t >= 0 && t < a.vocab) return (int)t;
    if (report) *a.flag = 1;
    return -1;
}
template <class E, class I>
__device__ inline void policy_write(const PolicyArgs<E, I>& a, int row, float logp, float lse, float term) {
    a.logp[row] = logp;
    a.lse[row] = lse;
    a.terms[row] = term;
}

// ---- one block a row -------------------------------------------------------------------------------------------------------
// K pieces of a thread stay in registers between the sums and the gradient; K = 0: rows that do not fit, or whose elements are not
// neighbours, are read again (from the caches, as a block's row is what its CU read last).
// Loss and gradient, bf16: 2048 rows of 32000 (six in ten count) 50 us in a row of calls = 4.2 TB/s, 8192 rows of 50001 329 us = 4.7 TB/s, where a large
// copy reaches 4.7; loss alone, f32, 3000 rows of 32000 (seven in ten) 50 us = 5.3 TB/s.
template <class E, class I, int THREADS, int K, bool STEP>
__global__ __launch_bounds__(THREADS) void policy_row_kernel(const PolicyArgs<E, I> a) {
    using T = PolicyType<E>;
    constexpr int N = T::N;
    __shared__ PolicySum shared[THREADS / WAVE];
    const int row = a.row0 + blockIdx.x, tid = threadIdx.x;
    const E* const x = a.logits + (int64_t)row * a.row;
    const int target = policy_target(a, row, tid == 0);
    const int lead = K || a.elem == 1 ? policy_lead(x) : 0, pieces = (lead + a.vocab + N - 1) / N;
    E* const y = STEP ? a.grad + (int64_t)row * a.vocab : nullptr;
    const bool aligned = STEP && policy_lead(y) == lead && (K || a.elem == 1);
    float scale = 0.0f, base = 0.0f, log_sum = 0.0f;
    policy_piece held[K ? K : 1];
    if (target >= 0) {
        PolicySum s{-INFINITY, 0.0f};
        if constexpr (K > 0) {
#pragma unroll
            for (int u = 0; u < K; ++u)
                if (tid + u * THREADS < pieces) held[u] = policy_fetch(x, a.vocab, lead, tid + u * THREADS);
            float top = -INFINITY;
#pragma unroll
            for (int u = 0; u < K; ++u) {
                if (tid + u * THREADS < pieces) {
                    E z[N];
                    __builtin_memcpy(z, &held[u], 16);
#pragma unroll
                    for (int e = 0; e < N; ++e) top = fmaxf(top, T::get(z[e]));
                }
            }
            s.base = top;
            const float from = s.base == -INFINITY ? 0.0f : s.base;
            auto add = [&](auto exponential) {
#pragma unroll
                for (int u = 0; u < K; ++u) {
                    if (tid + u * THREADS < pieces) {
                        E z[N];
                        __builtin_memcpy(z, &held[u], 16);
#pragma unroll
                        for (int e = 0; e < N; ++e) s.sum += exponential(T::get(z[e]));
                    }
                }
            };
            if (policy_near<E>(from)) {
                const float from2 = from * POLICY_LOG2E;
                add([&](float z) { return __builtin_amdgcn_exp2f(__builtin_fmaf(z, POLICY_LOG2E, -from2)); });
                s.sum *= __builtin_amdgcn_exp2f(-__builtin_fmaf(from, POLICY_LOG2E, -from2));      // what the product's rounding left in every term
            } else {
                add([&](float z) { return policy_exp(z - from); });
            }
        } else {
            for (int p = tid; p < pieces; p += THREADS) {
                float z[N];
                policy_load(x, a.elem, a.vocab, lead, p, a.elem == 1, z);
                policy_take(s, z);
            }
        }
        s = policy_join_block<THREADS>(s, shared);
        base = s.base == -INFINITY ? 0.0f : s.base;
        log_sum = __builtin_amdgcn_logf(s.sum);
        if (tid == 0 || STEP) {
            const double logp = policy_logp(T::get(x[(int64_t)target * a.elem]), s, log_sum);
            const PolicyToken t = policy_token(a, row, logp);
            if (tid == 0) policy_write(a, row, (float)logp, __builtin_fmaf(log_sum, POLICY_LN2, base), t.term);
            scale = STEP ? t.g * (a.grad_loss ? a.grad_loss[0] : 1.0f) : 0.0f;
        }
    } else if (tid == 0) {
        policy_write(a, row, 0.0f, 0.0f, 0.0f);
    }
    if constexpr (STEP) {
        const int out_lead = policy_lead(y), out_pieces = (out_lead + a.vocab + N - 1) / N;
        if (scale == 0.0f) {          // (a row that does not count, or whose ratio is clipped: nothing to read again)
            const float zero[N] = {};
            for (int p = tid; p < out_pieces; p += THREADS) policy_store(y, a.vocab, out_lead, p, true, zero);
            return;
        }
        const float lse2 = __builtin_fmaf(base, POLICY_LOG2E, log_sum);
        auto finish = [&](auto near, float (&z)[N], int p) {
            const int v0 = p * N - lead;
#pragma unroll
            for (int e = 0; e < N; ++e) {
                const float share = near ? __builtin_fmaf(z[e], POLICY_LOG2E, -lse2) : __builtin_fmaf(z[e] - base, POLICY_LOG2E, -log_sum);
                z[e] = scale * ((v0 + e == target ? 1.0f : 0.0f) - __builtin_amdgcn_exp2f(share));
            }
            policy_store(y, a.vocab, lead, p, aligned, z);
        };
        auto all = [&](auto near) {
            if constexpr (K > 0) {
#pragma unroll
                for (int u = 0; u < K; ++u) {
                    if (tid + u * THREADS < pieces) {
                        E h[N];
                        float z[N];
                        __builtin_memcpy(h, &held[u], 16);
#pragma unroll
                        for (int e = 0; e < N; ++e) z[e] = T::get(h[e]);
                        finish(near, z, tid + u * THREADS);
                    }
                }
            } else {
                for (int p = tid; p < pieces; p += THREADS) {
                    float z[N];
                    policy_load(x, a.elem, a.vocab, lead, p, a.elem == 1, z);
                    finish(near, z, p);
                }
            }
        };
        if (policy_near<E>(base)) all(std::true_type{});
        else all(std::false_type{});
    }
}

// ---- a few long rows: several blocks a row -----------------------------------------------------------------------------------
// f16, 16 rows of 128000: 5 us, and 3 us to join them.
constexpr int POLICY_PART_THREADS = 256;
constexpr int POLICY_MAX_PARTS = 64;
template <class E, class I>
__global__ __launch_bounds__(POLICY_PART_THREADS) void policy_part_kernel(const PolicyArgs<E, I> a, PolicySum* parts, int per) {
    constexpr int N = PolicyType<E>::N;
    __shared__ PolicySum shared[POLICY_PART_THREADS / WAVE];
    const int row = blockIdx.y;
    if (policy_target(a, row, false) < 0) return;
    const E* const x = a.logits + (int64_t)row * a.row;
    const int lead = a.elem == 1 ? policy_lead(x) : 0, pieces = (lead + a.vocab + N - 1) / N;
    const int from = blockIdx.x * per, upto = from + per < pieces ? from + per : pieces;
    PolicySum s{-INFINITY, 0.0f};
    for (int p = from + threadIdx.x; p < upto; p += POLICY_PART_THREADS) {
        float z[N];
        policy_load(x, a.elem, a.vocab, lead, p, a.elem == 1, z);
        policy_take(s, z);
    }
    s = policy_join_block<POLICY_PART_THREADS>(s, shared);
    if (threadIdx.x == 0) parts[(int64_t)row * gridDim.x + blockIdx.x] = s;
}
// one block: a wave joins the parts of a row, then the terms are summed
template <class E, class I>
__global__ __launch_bounds__(POLICY_SUM_THREADS) void policy_join_kernel(const PolicyArgs<E, I> a, const PolicySum* parts, int nparts) {
    const int lane = threadIdx.x % WAVE, wave = threadIdx.x / WAVE;
    __shared__ double shared[POLICY_SUM_THREADS / WAVE];
    double sum = 0.0;
    for (int row = wave; row < a.rows; row += POLICY_SUM_THREADS / WAVE) {
        const int target = policy_target(a, row, lane == 0);
        float logp = 0.0f, lse = 0.0f, term = 0.0f;
        if (target >= 0) {
            PolicySum s = policy_join_wave(lane < nparts ? parts[(int64_t)row * nparts + lane] : PolicySum{-INFINITY, 0.0f});
            const float base = s.base == -INFINITY ? 0.0f : s.base, log_sum = __builtin_amdgcn_logf(s.sum);
            lse = __builtin_fmaf(log_sum, POLICY_LN2, base);
            const double lp = policy_logp(PolicyType<E>::get(a.logits[(int64_t)row * a.row + (int64_t)target * a.elem]), s, log_sum);
            logp = (float)lp;
            term = policy_token(a, row, lp).term;
        }
        if (lane == 0) {
            a.logp[row] = logp;
            a.lse[row] = lse;
        }
        sum += (double)term;
    }
    if (lane == 0) shared[wave] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = 0.0;
        for (int w = 0; w < POLICY_SUM_THREADS / WAVE; ++w) total += shared[w];
        a.loss[0] = (float)total;
    }
}
// the gradient from lp and lse
template <class E, class I>
__global__ __launch_bounds__(POLICY_PART_THREADS) void policy_grad_kernel(const PolicyArgs<E, I> a, int per) {
    constexpr int N = PolicyType<E>::N;
    const int row = a.row0 + blockIdx.y;
    const int target = policy_target(a, row, blockIdx.x == 0 && threadIdx.x == 0);
    const E* const x = a.logits + (int64_t)row * a.row;
    E* const y = a.grad + (int64_t)row * a.vocab;
    const int lead = policy_lead(y), pieces = (lead + a.vocab + N - 1) / N;
    const bool aligned = a.elem == 1 && policy_lead(x) == lead;
    const int from = blockIdx.x * per, upto = from + per < pieces ? from + per : pieces;
    const float scale = target >= 0 ? policy_token(a, row, a.logp[row]).g * (a.grad_loss ? a.grad_loss[0] : 1.0f) : 0.0f;
    // x - lse = (x - x_target) + lp: whichever of lse and lp is the smaller has lost less to its rounding
    const float lse = a.lse[row], lp = a.logp[row];
    const bool by_target = target >= 0 && __builtin_fabsf(lp) <= __builtin_fabsf(lse);
    const float base = by_target ? PolicyType<E>::get(x[(int64_t)target * a.elem]) : lse, rest = by_target ? lp * POLICY_LOG2E : 0.0f;
    for (int p = from + threadIdx.x; p < upto; p += POLICY_PART_THREADS) {
        float z[N] = {};
        if (scale != 0.0f) {
            policy_load(x, a.elem, a.vocab, lead, p, aligned, z);
            const int v0 = p * N - lead;
#pragma unroll
            for (int e = 0; e < N; ++e) z[e] = scale * ((v0 + e == target ? 1.0f : 0.0f) - __builtin_amdgcn_exp2f(__builtin_fmaf(z[e] - base, POLICY_LOG2E, rest)));
        }
        policy_store(y, a.vocab, lead, p, true, z);
    }
}

// ---- host ----------------------------------------------------------------------------------------------------------------
// policy_loss.hip: loss[0] = the sum of n terms, in a fixed order in f64
void policy_sum(const float* terms, int n, float* loss);

template <class E, class I>
inline bool policy_arguments(PolicyArgs<E, I>& a, const size_t* md, const I* target, const E* logits, const float* old_logp, const float* ref_logp,
                             const float* advantage, const float* weight, float low, float high, float beta, const E* grad) {
    const bool some = !md || md[0] != 0;        // (tensors of no rows have no address)
    if (!md || (some && (!target || !logits || !old_logp || !advantage || !weight))) { set_status(ERR_INVALID, "policy_loss: null argument"); return false; }
    if (some && !ref_logp && beta != 0.0f) { set_status(ERR_INVALID, "policy_loss: the KL term needs ref_logp"); return false; }
    if (!(low >= 0.0f) || !(high >= 0.0f)) { set_status(ERR_INVALID, "policy_loss: the clip range is not negative"); return false; }
    if (md[1] == 0) { set_status(ERR_INVALID, "policy_loss: an empty vocabulary"); return false; }
    if (md[0] >= (1ull << 31) - 1024 || md[1] >= (1ull << 31) - 1024) { set_status(ERR_TOO_LARGE, "policy_loss: too many rows or logits"); return false; }
    std::memset((void*)&a, 0, sizeof(a));
    a.logits = logits + md[4];
    a.row = (int64_t)md[2];
    a.elem = md[1] == 1 ? 1 : (int64_t)md[3];
    a.target = target;
    a.old_logp = old_logp;
    a.ref_logp = ref_logp;
    a.advantage = advantage;
    a.weight = weight;
    a.least = 1.0f - low;
    a.most = 1.0f + high;
    a.beta = beta;
    a.rows = (int32_t)md[0];
    a.vocab = (int32_t)md[1];
    if (a.rows == 0) return true;
    if (grad) {      // a row's threads write while others still read its target
        const int64_t ends[2] = {(int64_t)(a.rows - 1) * a.row, (int64_t)(a.vocab - 1) * a.elem};
        const E *lo = a.logits, *hi = a.logits + 1;
        for (int64_t end : ends) (end < 0 ? lo : hi) += end;
        if (grad < hi && lo < grad + (size_t)a.rows * a.vocab) { set_status(ERR_INVALID, "policy_loss: grad_logits overlaps the logits"); return false; }
    }
    a.flag = index_flag();
    return a.flag != nullptr;
}
// pieces of a row, whatever its alignment
template <class E, class I>
inline int policy_pieces(const PolicyArgs<E, I>& a) { return (a.vocab + 2 * (PolicyType<E>::N - 1)) / PolicyType<E>::N; }

// a launch takes less than 2^32 threads, and 65535 blocks along the second axis
template <class E, class I, class F>
inline void policy_by_rows(const PolicyArgs<E, I>& a, int most, F&& launch) {
    PolicyArgs<E, I> b = a;
    for (int64_t row0 = 0; row0 < a.rows; row0 += most) {
        b.row0 = (int32_t)row0;
        launch(b, (unsigned)(a.rows - row0 < most ? a.rows - row0 : most));
    }
}

template <class E, class I>
inline void policy_grad_launch(const PolicyArgs<E, I>& a) {
    // four pieces a thread, or less where rows are few
    const int pieces = policy_pieces(a);
    int per = 4 * POLICY_PART_THREADS;
    while (per > POLICY_PART_THREADS && (int64_t)cdiv(pieces, per) * a.rows < 512) per /= 2;
    const unsigned blocks = cdiv((size_t)pieces, (size_t)per);
    policy_by_rows(a, 65535, [&](const PolicyArgs<E, I>& b, unsigned n) {
        hipLaunchKernelGGL((policy_grad_kernel<E, I>), dim3(blocks, n), dim3(POLICY_PART_THREADS), 0, stream(), b, per);
        MXH_LAUNCH_CHECK("policy_loss (gradient)");
    });
}

template <class E, class I, int THREADS, int K>
inline void policy_row_launch(const PolicyArgs<E, I>& a) {
    policy_by_rows(a, 1 << 21, [&](const PolicyArgs<E, I>& b, unsigned n) {
        if (a.grad) hipLaunchKernelGGL((policy_row_kernel<E, I, THREADS, K, true>), dim3(n), dim3(THREADS), 0, stream(), b);
        else hipLaunchKernelGGL((policy_row_kernel<E, I, THREADS, K, false>), dim3(n), dim3(THREADS), 0, stream(), b);
        MXH_LAUNCH_CHECK("policy_loss");
    });
}

// loss, logp and lse, and the gradient where one is wanted
template <class E, class I>
inline void policy_entry(const size_t* md, const I* target, const E* logits, const float* old_logp, const float* ref_logp, const float* advantage,
                         const float* weight, float low, float high, float beta, const float* grad_loss, float* loss, float* logp, float* lse, E* grad, bool step) {
    PolicyArgs<E, I> a;
    const bool some = !md || md[0] != 0;
    if (!loss || (some && (!logp || !lse || (step && !grad)))) { set_status(ERR_INVALID, "policy_loss: null output"); return; }
    if (!policy_arguments(a, md, target, logits, old_logp, ref_logp, advantage, weight, low, high, beta, step ? grad : nullptr)) return;
    a.grad_loss = grad_loss;
    a.loss = loss;
    a.logp = logp;
    a.lse = lse;
    a.grad = step ? grad : nullptr;
    if (a.rows == 0) { policy_sum(nullptr, 0, loss); return; }
    const int pieces = policy_pieces(a);
    if (a.rows < 256 && pieces >= 4 * POLICY_PART_THREADS) {
        int per = POLICY_PART_THREADS;
        while (cdiv((size_t)pieces, (size_t)per) > (unsigned)POLICY_MAX_PARTS || (int64_t)cdiv((size_t)pieces, (size_t)per) * a.rows > 2048) per *= 2;
        const unsigned nparts = cdiv((size_t)pieces, (size_t)per);
        PolicySum* parts = (PolicySum*)scratch((size_t)a.rows * nparts * sizeof(PolicySum));
        if (!parts) return;
        hipLaunchKernelGGL((policy_part_kernel<E, I>), dim3(nparts, (unsigned)a.rows), dim3(POLICY_PART_THREADS), 0, stream(), a, parts, per);
        MXH_LAUNCH_CHECK("policy_loss (parts)");
        hipLaunchKernelGGL((policy_join_kernel<E, I>), dim3(1), dim3(POLICY_SUM_THREADS), 0, stream(), a, parts, (int)nparts);
        MXH_LAUNCH_CHECK("policy_loss (join)");
        if (step) policy_grad_launch(a);
        return;
    }
    a.terms = (float*)scratch((size_t)a.rows * sizeof(float));
    if (!a.terms) return;
    if (a.elem != 1) policy_row_launch<E, I, 256, 0>(a);
    else if (pieces <= 256 * 2) policy_row_launch<E, I, 256, 2>(a);
    else if (pieces <= 512 * 4) policy_row_launch<E, I, 512, 4>(a);
    else if (pieces <= 1024 * 4) policy_row_launch<E, I, 1024, 4>(a);
    else if (pieces <= 1024 * 8) policy_row_launch<E, I, 1024, 8>(a);
    else policy_row_launch<E, I, 1024, 0>(a);
    policy_sum(a.terms, a.rows, loss);
}

template <class E, class I>
inline void policy_backward_entry(const size_t* md, const I* target, const E* logits, const float* old_logp, const float* ref_logp, const float* advantage,
                                  const float* weight, float low, float high, float beta, const float* logp, const float* lse, const float* grad_loss, E* grad) {
    PolicyArgs<E, I> a;
    if ((!logp || !lse || !grad) && !(md && md[0] == 0)) { set_status(ERR_INVALID, "policy_loss_backward: null argument"); return; }
    if (!policy_arguments(a, md, target, logits, old_logp, ref_logp, advantage, weight, low, high, beta, grad)) return;
    if (a.rows == 0) return;
    a.grad_loss = grad_loss;
    a.logp = (float*)logp;
    a.lse = (float*)lse;
    a.grad = grad;
    policy_grad_launch(a);
}

#define MXH_POLICY_LOSS(E, S, I, IS)                                                                                                                  \
    extern "C" void hip_policy_loss_##S##_##IS(const size_t* metadata, const I* target, const E* logits, const float* old_logp, const float* ref_logp, \
                                               const float* advantage, const float* weight, float clip_low, float clip_high, float kl_weight,         \
                                               float* loss, float* logp, float* lse) { MXH_API;                                                       \
        ::mxh::policy_entry<E, I>(metadata, target, logits, old_logp, ref_logp, advantage, weight, clip_low, clip_high, kl_weight, nullptr, loss,     \
                                  logp, lse, nullptr, false);                                                                                         \
    }                                                                                                                                                 \
    extern "C" void hip_policy_loss_backward_##S##_##IS(const size_t* metadata, const I* target, const E* logits, const float* old_logp,              \
                                                        const float* ref_logp, const float* advantage, const float* weight, float clip_low,           \
                                                        float clip_high, float kl_weight, const float* logp, const float* lse,                        \
                                                        const float* grad_loss, E* grad_logits) { MXH_API;                                            \
        ::mxh::policy_backward_entry<E, I>(metadata, target, logits, old_logp, ref_logp, advantage, weight, clip_low, clip_high, kl_weight, logp,     \
                                           lse, grad_loss, grad_logits);                                                                              \
    }                                                                                                                                                 \
    extern "C" void hip_policy_loss_step_##S##_##IS(const size_t* metadata, const I* target, const E* logits, const float* old_logp,                  \
                                                    const float* ref_logp, const float* advantage, const float* weight, float clip_low,               \
                                                    float clip_high, float kl_weight, const float* grad_loss, float* loss, float* logp, float* lse,   \
                                                    E* grad_logits) { MXH_API;                                                                        \
        ::mxh::policy_entry<E, I>(metadata, target, logits, old_logp, ref_logp, advantage, weight, clip_low, clip_high, kl_weight, grad_loss, loss,   \
                                  logp, lse, grad_logits, true);                                                                                      \
    }
#define MXH_POLICY_LOSS_BOTH(E, S) MXH_POLICY_LOSS(E, S, int32_t, i32) MXH_POLICY_LOSS(E, S, int64_t, i64)

}  // namespace mxh
