// cross_entropy.hip -- C ABI of the softmax cross entropy (include/tca_train.h).
#include <hip/hip_runtime.h>

#include "../../include/tca_train.h"
#include "common.hpp"
#include "cross_entropy_kernel.hpp"
#include "train_launch.hpp"

namespace tca {
namespace {

// Workgroups of a launch: enough to fill the chip several times over (2.4M rows of
// 47 fp32 logits, backward: 118 us, 132 with 2048), and the parts that a join adds.
constexpr int kLossBlocks = 8192;
// Rows up to which each wavefront of narrow rows counts those with a label itself
// (1000 rows 5.6 us, 6.8 in two launches; 2000 rows 6.8 and 7.2).
constexpr int64_t kLossOwnCount = 2048;

// One launch; the number of workgroups.  Rows at a time (R) and rows per chunk only
// grow where every unit has that many.
template <typename T, int kMode, int E, int G, int V, int R, bool kStream>
int go_rows(const CrossEntropyArgs& a, hipStream_t s) {
    constexpr int kTurn = (G < 64 ? 64 / G : 1) * R;         // rows a unit takes at once
    constexpr int kUnits = G > 64 ? 1 : 4;                   // units of a workgroup
    const int64_t each = static_cast<int64_t>(kLossBlocks) * kUnits * kTurn;
    const int turns = static_cast<int>(std::min<int64_t>((a.rows + each - 1) / each, 64 / kTurn));
    const int chunk = turns * kTurn;
    const int64_t per_block = static_cast<int64_t>(kUnits) * chunk;
    const int blocks = static_cast<int>(std::min<int64_t>((a.rows + per_block - 1) / per_block, kLossBlocks));
    hipLaunchKernelGGL((cross_entropy_kernel<T, kMode, E, G, V, R, kStream>), dim3(blocks), dim3(team_threads(G)), 0, s,
                       a, chunk);
    return blocks;
}

// Whether a pass moves more than the caches hold.
template <typename T, int kMode>
bool streamed(const CrossEntropyArgs& a) {
    const int64_t passes = kMode == kLossForward ? 1 : 2;
    return static_cast<int64_t>(a.rows) * a.n > kStreamBytes / passes / static_cast<int64_t>(sizeof(T));
}

template <typename T, int kMode, int E, int G, int V>
int go(const CrossEntropyArgs& a, hipStream_t s) {
    constexpr int R = G <= 64 && V <= 2 ? 2 : 1;
    if constexpr (G <= 64) {
        // not streamed: neighbouring rows share lines here, which streaming fetches and
        // writes for each row anew (2.4M rows of 47 fp32 logits 190 us, 329 streamed)
        if (R > 1 && a.rows >= R * row_teams(G, 2048)) return go_rows<T, kMode, E, G, V, R, false>(a, s);
        return go_rows<T, kMode, E, G, V, 1, false>(a, s);
    } else {
        return streamed<T, kMode>(a) ? go_rows<T, kMode, E, G, V, R, true>(a, s) : go_rows<T, kMode, E, G, V, R, false>(a, s);
    }
}

// V vectors per lane, of at most kMax (see launch_loss).
template <typename T, int kMode, int E, int G, int V, int kMax>
int go_from(const CrossEntropyArgs& a, int nv, hipStream_t s) {
    if constexpr (V < kMax) {
        if (nv > V * G) return go_from<T, kMode, E, G, V + 1, kMax>(a, nv, s);
    }
    return go<T, kMode, E, G, V>(a, s);
}

// The launch of a row of n classes in vectors of E: G lanes per row, V vectors
// per lane, (V - 1) G E < n <= V G E; the number of workgroups.  Two vectors per
// lane, not one, for narrow rows: half the steps of a sum and half the rows'
// overhead per value (233k rows of 41 fp32 logits 24 us with one, 20 with two).  A
// wavefront per row needs no barrier (20000 x 2500 bf16 logits 38 us, 61 with a
// workgroup of 256); beyond six vectors per lane two wavefronts share a row
// (20000 x 5000 fp16, forward: 44 us, 61 with one, 54 with four).  From 1024 vectors
// on, loss and gradient at once take eight (20000 rows of 5000, 7000 and 10000 bf16
// logits: 87, 118 and 167 us with two, 106, 113 and 155 with eight) up to sixteen
// vectors per lane, all that the registers hold (4194 x 50001: 198 us, 212 in the long
// kernel), and a single direction takes the long kernel (20000 x 10000, backward:
// 144 us, 169 with two wavefronts; forward, where two would still be ahead up to 1536
// vectors, 89 and 66).
template <typename T, int kMode>
int launch_loss(const CrossEntropyArgs& a, hipStream_t s) {
    constexpr int E = 16 / sizeof(T);
    if (a.n < E) return go<T, kMode, 1, 8, 1>(a, s);
    const int nv = (a.n - 1) / E + 1;
    if (nv <= 4) return go<T, kMode, E, 4, 1>(a, s);
    if (nv <= 8) return go<T, kMode, E, 4, 2>(a, s);
    if (nv <= 16) return go<T, kMode, E, 8, 2>(a, s);
    if (nv <= 32) return go<T, kMode, E, 16, 2>(a, s);
    if (nv <= 64) return go<T, kMode, E, 32, 2>(a, s);
    if (nv <= 384) return go_from<T, kMode, E, 64, 2, 6>(a, nv, s);
    if (nv <= 1024) return go_from<T, kMode, E, 128, 4, 8>(a, nv, s);
    if constexpr (kMode == kLossBoth) {
        if (nv <= 8192) return go_from<T, kMode, E, 512, 3, 16>(a, nv, s);
    }
    const int blocks = static_cast<int>(std::min<int64_t>(a.rows, kLossBlocks));
    if (streamed<T, kMode>(a))
        hipLaunchKernelGGL((cross_entropy_long_kernel<T, kMode, true>), dim3(blocks), dim3(kLongThreads), 0, s, a);
    else
        hipLaunchKernelGGL((cross_entropy_long_kernel<T, kMode, false>), dim3(blocks), dim3(kLongThreads), 0, s, a);
    return blocks;
}

template <int kMode>
int launch_loss_type(const CrossEntropyArgs& a, int32_t dtype, hipStream_t s) {
    if (dtype == TCA_F16) return launch_loss<_Float16, kMode>(a, s);
    if (dtype == TCA_BF16) return launch_loss<bf16_t, kMode>(a, s);
    return launch_loss<float, kMode>(a, s);
}

// Workspace: the workgroups' parts, then the counts.
size_t loss_workspace() { return kLossBlocks * sizeof(float2) + kLossParts * sizeof(int); }

int check_loss(const char* name, const void* x, int64_t rows, int32_t classes, int64_t pitch, int32_t dtype,
               const void* targets, int32_t target_bytes) {
    if (!dtype_ok(dtype)) return fail(TCA_ERR_INVALID, "%s: unknown value type", name);
    if (rows < 0 || classes < 1 || pitch < 0)
        return fail(TCA_ERR_INVALID, "%s: bad shape rows=%lld classes=%d pitch=%lld", name, (long long)rows, classes,
                    (long long)pitch);
    if (rows > 0x7fffffff || pitch > 0x7fffffff || classes > (1 << 30))
        return fail(TCA_ERR_UNSUPPORTED, "%s: more than 2^31 - 1 rows, or elements between rows, or 2^30 classes", name);
    if (target_bytes != 8 && target_bytes != 4)
        return fail(TCA_ERR_INVALID, "%s: targets are int64 or int32 (target_bytes %d)", name, target_bytes);
    if (rows > 0 && (!x || !targets)) return fail(TCA_ERR_INVALID, "%s: NULL device pointer", name);
    if (misaligned(x, dtype) || reinterpret_cast<uintptr_t>(targets) % target_bytes)
        return fail(TCA_ERR_INVALID, "%s: pointers need their element's alignment", name);
    return TCA_OK;
}

int check_workspace(const char* name, const void* p, size_t bytes) {
    if (!p || bytes < loss_workspace())
        return fail(TCA_ERR_INVALID, "%s: a workspace of %zu bytes is needed, %zu given", name, loss_workspace(),
                    p ? bytes : 0);
    if (reinterpret_cast<uintptr_t>(p) % 8) return fail(TCA_ERR_INVALID, "%s: the workspace needs 8-byte alignment", name);
    return TCA_OK;
}

CrossEntropyArgs loss_args(const void* x, int64_t rows, int32_t classes, int64_t pitch, const void* targets,
                           int32_t target_bytes, int64_t ignore_index) {
    CrossEntropyArgs a = {};
    a.x = x;
    a.targets = targets;
    a.pitch = static_cast<int>(pitch);
    a.ignore = ignore_index;
    a.rows = static_cast<int>(rows);
    a.n = classes;
    a.wide_targets = target_bytes == 8;
    return a;
}

void launch_join(const float2* parts, int n, bool mean, float* loss, float* norm, hipStream_t s) {
    hipLaunchKernelGGL(loss_join_kernel, dim3(1), dim3(kLossJoinThreads), 0, s, parts, n, mean, loss, norm);
}

}  // namespace
}  // namespace tca

using namespace tca;

extern "C" {

int tca_cross_entropy_workspace(int64_t rows, int32_t classes, size_t* bytes) {
    if (!bytes || rows < 0 || classes < 1) return fail(TCA_ERR_INVALID, "tca_cross_entropy_workspace: bad argument");
    *bytes = loss_workspace();
    return TCA_OK;
}

int tca_cross_entropy(const void* d_logits, int64_t rows, int32_t classes, int64_t pitch, int32_t dtype,
                      const void* d_targets, int32_t target_bytes, int64_t ignore_index, int32_t reduction,
                      float* d_loss, float* d_stats, float* d_norm, void* d_workspace, size_t workspace_bytes,
                      void* stream) {
    const char* name = "tca_cross_entropy";
    if (const int st = check_loss(name, d_logits, rows, classes, pitch, dtype, d_targets, target_bytes)) return st;
    if (reduction < TCA_LOSS_NONE || reduction > TCA_LOSS_MEAN) return fail(TCA_ERR_INVALID, "%s: reduction %d", name, reduction);
    if (!d_loss && (rows > 0 || reduction != TCA_LOSS_NONE)) return fail(TCA_ERR_INVALID, "%s: NULL device pointer", name);
    if (reinterpret_cast<uintptr_t>(d_loss) % 4 || reinterpret_cast<uintptr_t>(d_norm) % 4 ||
        reinterpret_cast<uintptr_t>(d_stats) % 8)
        return fail(TCA_ERR_INVALID, "%s: loss and norm need 4-byte alignment, stats 8 bytes", name);
    if (const int st = check_workspace(name, d_workspace, workspace_bytes)) return st;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    CrossEntropyArgs a = loss_args(d_logits, rows, classes, pitch, d_targets, target_bytes, ignore_index);
    const bool none = reduction == TCA_LOSS_NONE;
    a.row_loss = none ? d_loss : nullptr;
    a.stats = reinterpret_cast<float2*>(d_stats);
    a.parts = static_cast<float2*>(d_workspace);
    int blocks = 0;
    if (rows > 0) {
        blocks = launch_loss_type<kLossForward>(a, dtype, s);
        if (const int st = launched()) return st;
    }
    if (none && !d_norm) return TCA_OK;
    launch_join(a.parts, blocks, reduction == TCA_LOSS_MEAN, none ? nullptr : d_loss, d_norm, s);
    return launched();
}

int tca_cross_entropy_backward(const float* d_gloss, int64_t gloss_stride, const void* d_logits, int64_t rows,
                               int32_t classes, int64_t pitch, int32_t dtype, const void* d_targets,
                               int32_t target_bytes, int64_t ignore_index, const float* d_stats, const float* d_norm,
                               void* d_dlogits, void* stream) {
    const char* name = "tca_cross_entropy_backward";
    if (const int st = check_loss(name, d_logits, rows, classes, pitch, dtype, d_targets, target_bytes)) return st;
    if (gloss_stride < 0) return fail(TCA_ERR_INVALID, "%s: gloss_stride %lld", name, (long long)gloss_stride);
    if (rows == 0) return TCA_OK;
    if (!d_gloss || !d_stats || !d_dlogits) return fail(TCA_ERR_INVALID, "%s: NULL device pointer", name);
    if (misaligned(d_dlogits, dtype) || reinterpret_cast<uintptr_t>(d_gloss) % 4 ||
        reinterpret_cast<uintptr_t>(d_norm) % 4 || reinterpret_cast<uintptr_t>(d_stats) % 8)
        return fail(TCA_ERR_INVALID, "%s: pointers need their element's alignment, stats 8 bytes", name);
    CrossEntropyArgs a = loss_args(d_logits, rows, classes, pitch, d_targets, target_bytes, ignore_index);
    a.gloss = d_gloss;
    a.gloss_stride = gloss_stride;
    a.stats = const_cast<float2*>(reinterpret_cast<const float2*>(d_stats));
    a.norm = d_norm;
    a.dx = d_dlogits;
    launch_loss_type<kLossBackward>(a, dtype, static_cast<hipStream_t>(stream));
    return launched();
}

int tca_cross_entropy_grad(const void* d_logits, int64_t rows, int32_t classes, int64_t pitch, int32_t dtype,
                           const void* d_targets, int32_t target_bytes, int64_t ignore_index, int32_t reduction,
                           float scale, float* d_loss, void* d_dlogits, void* d_workspace, size_t workspace_bytes,
                           void* stream) {
    const char* name = "tca_cross_entropy_grad";
    if (const int st = check_loss(name, d_logits, rows, classes, pitch, dtype, d_targets, target_bytes)) return st;
    if (reduction != TCA_LOSS_SUM && reduction != TCA_LOSS_MEAN)
        return fail(TCA_ERR_INVALID, "%s: reduction %d (sum or mean)", name, reduction);
    if (!d_loss || (rows > 0 && !d_dlogits)) return fail(TCA_ERR_INVALID, "%s: NULL device pointer", name);
    if (misaligned(d_dlogits, dtype) || reinterpret_cast<uintptr_t>(d_loss) % 4)
        return fail(TCA_ERR_INVALID, "%s: pointers need their element's alignment", name);
    if (const int st = check_workspace(name, d_workspace, workspace_bytes)) return st;
    const hipStream_t s = static_cast<hipStream_t>(stream);
    CrossEntropyArgs a = loss_args(d_logits, rows, classes, pitch, d_targets, target_bytes, ignore_index);
    const bool mean = reduction == TCA_LOSS_MEAN;
    a.parts = static_cast<float2*>(d_workspace);
    a.dx = d_dlogits;
    a.scale = scale;
    int blocks = 0;
    if (rows > 0) {
        // up to 128 vectors a wavefront or less takes a row (launch_loss)
        if (mean && rows <= kLossOwnCount && classes <= 128 * 16 / static_cast<int>(dtype_size(dtype))) {
            a.own_count = true;
        } else if (mean) {
            int* counts = reinterpret_cast<int*>(a.parts + kLossBlocks);
            hipLaunchKernelGGL(loss_count_kernel, dim3(kLossParts), dim3(kLossCountThreads), 0, s, a, counts);
            if (const int st = launched()) return st;
            a.counts = counts;
        }
        blocks = launch_loss_type<kLossBoth>(a, dtype, s);
        if (const int st = launched()) return st;
    }
    launch_join(a.parts, blocks, mean, d_loss, nullptr, s);
    return launched();
}

}  // extern "C"
