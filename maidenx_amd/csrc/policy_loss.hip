// The clipped policy loss for f32 logits, and the sum of its terms (see policy_loss.hpp).
#include "policy_loss.hpp"

namespace mxh {

__global__ __launch_bounds__(POLICY_SUM_THREADS) void policy_sum_kernel(const float* __restrict__ terms, int n, float* __restrict__ loss) {
    __shared__ double shared[POLICY_SUM_THREADS / WAVE];
    double sum = 0.0;
    for (int64_t i = threadIdx.x; i < n; i += POLICY_SUM_THREADS) sum += (double)terms[i];
#pragma unroll
    for (int d = 32; d > 0; d >>= 1) sum += __shfl_xor(sum, d, WAVE);
    if (threadIdx.x % WAVE == 0) shared[threadIdx.x / WAVE] = sum;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = 0.0;
        for (int w = 0; w < POLICY_SUM_THREADS / WAVE; ++w) total += shared[w];
        loss[0] = (float)total;
    }
}
void policy_sum(const float* terms, int n, float* loss) {
    hipLaunchKernelGGL(policy_sum_kernel, dim3(1), dim3(POLICY_SUM_THREADS), 0, stream(), terms, n, loss);
    MXH_LAUNCH_CHECK("policy_loss (sum)");
}

}  // namespace mxh
using namespace mxh;

MXH_POLICY_LOSS_BOTH(float, f32)
