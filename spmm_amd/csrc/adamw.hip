// adamw.hip -- C ABI of the AdamW step (include/tca_train.h).
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <utility>
#include <vector>

#include "../../include/tca_train.h"
#include "adamw_kernel.hpp"
#include "common.hpp"
#include "train_launch.hpp"

namespace tca {
namespace {

// Arrays of more than this are streamed past the caches (256 MB behind the L2s).
// Where one state is stepped over and over with nothing between, that pays only from
// 384 MB on (fp32 parameters, 16 bytes each in all arrays: 8M 35 us cached, 41
// streamed; 16M 67 and 83; 24M 129 and 128; 134M 693 and 617; 8-bit states 381 and
// 305).  In a training program other passes go through the caches between two steps,
// and then it pays at each of these sizes: with a copy of 256 MB between, copy and
// step of 8M take 154 us cached, 150 streamed, of 16M 199 and 193, of 48M 364 and 356;
// with the gradients written before the step and the parameters read after it as well
// 170 and 166, 222 and 219, 484 and 460.  Half of what the caches hold is the bound.
constexpr int64_t kAdamStreamBytes = 128ll << 20;

template <typename T, bool kStream>
void launch_adam(const AdamArgs& a, int blocks, bool bits8, hipStream_t s) {
    if (bits8) hipLaunchKernelGGL((adamw_8bit_kernel<T, kStream>), dim3(blocks), dim3(kAdamThreads), 0, s, a);
    else hipLaunchKernelGGL((adamw_kernel<T, kStream>), dim3(blocks), dim3(kAdamThreads), 0, s, a);
}

template <typename T>
void launch_adam(const AdamArgs& a, int blocks, bool bits8, bool stream, hipStream_t s) {
    if (stream) launch_adam<T, true>(a, blocks, bits8, s);
    else launch_adam<T, false>(a, blocks, bits8, s);
}

constexpr int64_t kAdamBlocks = 0xffffffffll / kAdamThreads;  // of a launch: 2^32 - 1 lanes

int check_tensor(const char* name, const tca_adamw_tensor& t, int k, bool master, bool bits8, int32_t dtype) {
    if (t.n < 0) return fail(TCA_ERR_INVALID, "%s: tensor %d has %lld elements", name, k, (long long)t.n);
    if (t.n == 0) return TCA_OK;
    if (!t.param || !t.grad || !t.m || !t.v || (master && !t.master) || (bits8 && (!t.m_scale || !t.v_scale)))
        return fail(TCA_ERR_INVALID, "%s: NULL device pointer in tensor %d", name, k);
    if (misaligned(t.param, dtype) || misaligned(t.grad, dtype) || misaligned(t.master, TCA_F32) ||
        misaligned(t.m, TCA_F32) || misaligned(t.v, TCA_F32) || misaligned(t.m_scale, TCA_F32) ||
        misaligned(t.v_scale, TCA_F32))
        return fail(TCA_ERR_INVALID, "%s: tensor %d: pointers need their element's alignment, codes 4 bytes", name, k);
    if (t.n > kAdamBlocks * kAdamThreads * kAdamVec)
        return fail(TCA_ERR_UNSUPPORTED, "%s: tensor %d has %lld elements (at most %lld)", name, k, (long long)t.n,
                    (long long)(kAdamBlocks * kAdamThreads * kAdamVec));
    return TCA_OK;
}

// Two tensors on the same values: the workgroups of a launch would race on them.
int check_apart(const char* name, const tca_adamw_tensor* tensors, int count, int32_t dtype) {
    if (count < 2) return TCA_OK;
    return api_guard(name, [&] {
        std::vector<std::pair<uintptr_t, uintptr_t>> spans;  // [first, past the last) byte
        spans.reserve(count);
        for (int k = 0; k < count; ++k) {
            if (tensors[k].n == 0) continue;
            const uintptr_t first = reinterpret_cast<uintptr_t>(tensors[k].param);
            spans.emplace_back(first, first + static_cast<uintptr_t>(tensors[k].n) * dtype_size(dtype));
        }
        std::sort(spans.begin(), spans.end());
        for (size_t k = 1; k < spans.size(); ++k)
            if (spans[k].first < spans[k - 1].second)
                return fail(TCA_ERR_INVALID, "%s: two tensors' parameters share memory", name);
        return static_cast<int>(TCA_OK);
    });
}

// Both entry points: step counts of the host (d_steps NULL) or of the device.
int adam_step(const char* name, const tca_adamw_tensor* tensors, int64_t* const* d_steps, int32_t count,
              int32_t param_dtype, int32_t state_bits, int64_t step, double lr, double beta1, double beta2, double eps,
              double weight_decay, float2* d_factors, void* stream) {
    if (count < 0 || (count > 0 && !tensors)) return fail(TCA_ERR_INVALID, "%s: no tensors", name);
    if (!dtype_ok(param_dtype)) return fail(TCA_ERR_INVALID, "%s: unknown value type", name);
    if (state_bits != 32 && state_bits != 8)
        return fail(TCA_ERR_INVALID, "%s: state_bits %d (32 or 8)", name, state_bits);
    if (step < 1) return fail(TCA_ERR_INVALID, "%s: step %lld (the first is 1)", name, (long long)step);
    if (!(lr >= 0.0) || !(beta1 >= 0.0 && beta1 < 1.0) || !(beta2 >= 0.0 && beta2 < 1.0) || !(weight_decay >= 0.0))
        return fail(TCA_ERR_INVALID, "%s: lr %g, betas %g, %g, weight decay %g", name, lr, beta1, beta2, weight_decay);
    if (!(eps >= 0.0) || (state_bits == 8 && !(eps > 0.0)))
        return fail(TCA_ERR_INVALID, "%s: eps %g (above 0 for states in 8 bits)", name, eps);
    const bool bits8 = state_bits == 8, master = param_dtype != TCA_F32;
    for (int k = 0; k < count; ++k)
        if (const int st = check_tensor(name, tensors[k], k, master, bits8, param_dtype)) return st;
    if (const int st = check_apart(name, tensors, count, param_dtype)) return st;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    AdamArgs a;
    a.keep = static_cast<float>(1.0 - lr * weight_decay);
    a.rate = static_cast<float>(lr / (1.0 - std::pow(beta1, static_cast<double>(step))));
    a.correct = static_cast<float>(1.0 / std::sqrt(1.0 - std::pow(beta2, static_cast<double>(step))));
    a.eps = static_cast<float>(eps);
    a.b1 = static_cast<float>(beta1);
    a.c1 = static_cast<float>(1.0 - beta1);
    a.b2 = static_cast<float>(beta2);
    a.c2 = static_cast<float>(1.0 - beta2);
    const int64_t per_block = static_cast<int64_t>(kAdamThreads) * kAdamVec;
    int64_t values = 0;
    for (int k = 0; k < count; ++k) values += tensors[k].n;
    // bytes of a value in all its arrays
    const int64_t each = 2 * static_cast<int64_t>(dtype_size(param_dtype)) + (master ? 4 : 0) + (bits8 ? 2 : 8);
    const bool past = values > kAdamStreamBytes / each;
    for (int k = 0; k < count;) {
        AdamCounts counts;
        a.count = counts.count = 0;
        a.start[0] = 0;
        a.factors = counts.factors = d_steps ? d_factors + k : nullptr;
        int64_t blocks = 0;
        // an empty tensor takes no workgroup, but a place where steps are counted
        for (; k < count && a.count < kAdamTensors; ++k) {
            if (tensors[k].n == 0 && !d_steps) continue;
            const int64_t more = (tensors[k].n + per_block - 1) / per_block;
            if (blocks + more > kAdamBlocks) break;
            if (d_steps) counts.step[counts.count++] = d_steps[k];
            a.t[a.count++] = tensors[k];
            blocks += more;
            a.start[a.count] = static_cast<int>(blocks);
        }
        if (counts.count) {
            counts.lr = lr;
            counts.b1 = beta1;
            counts.b2 = beta2;
            hipLaunchKernelGGL(adamw_count_kernel, dim3(1), dim3(64), 0, s, counts);
            if (const int st = launched()) return st;
        }
        if (blocks == 0) continue;
        if (param_dtype == TCA_F16) launch_adam<_Float16>(a, static_cast<int>(blocks), bits8, past, s);
        else if (param_dtype == TCA_BF16) launch_adam<bf16_t>(a, static_cast<int>(blocks), bits8, past, s);
        else launch_adam<float>(a, static_cast<int>(blocks), bits8, past, s);
        if (const int st = launched()) return st;
    }
    return TCA_OK;
}

}  // namespace
}  // namespace tca

using namespace tca;

extern "C" {

int tca_adamw_step(const tca_adamw_tensor* tensors, int32_t count, int32_t param_dtype, int32_t state_bits,
                   int64_t step, double lr, double beta1, double beta2, double eps, double weight_decay,
                   void* stream) {
    return adam_step("tca_adamw_step", tensors, nullptr, count, param_dtype, state_bits, step, lr, beta1, beta2, eps,
                     weight_decay, nullptr, stream);
}

int tca_adamw_step_device(const tca_adamw_tensor* tensors, int64_t* const* d_steps, int32_t count, int32_t param_dtype,
                          int32_t state_bits, double lr, double beta1, double beta2, double eps, double weight_decay,
                          float* d_factors, void* stream) {
    const char* name = "tca_adamw_step_device";
    if (count > 0 && (!d_steps || !d_factors)) return fail(TCA_ERR_INVALID, "%s: NULL pointer", name);
    if (reinterpret_cast<uintptr_t>(d_factors) % 8) return fail(TCA_ERR_INVALID, "%s: factors need 8-byte alignment", name);
    for (int k = 0; k < count; ++k)
        if (!d_steps[k] || reinterpret_cast<uintptr_t>(d_steps[k]) % 8)
            return fail(TCA_ERR_INVALID, "%s: step count %d is NULL or not aligned to 8 bytes", name, k);
    return adam_step(name, tensors, d_steps, count, param_dtype, state_bits, 1, lr, beta1, beta2, eps, weight_decay,
                     reinterpret_cast<float2*>(d_factors), stream);
}

}  // extern "C"
