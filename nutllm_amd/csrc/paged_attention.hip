// paged_attention.hip — attention of one new token a sequence over a paged
// KV cache.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "device.hpp"
#include "paged_device.hpp"
#include "runtime.hpp"

namespace nut {

namespace {

template <int TYPE> __device__ __forceinline__ float component(const char *row, uint32_t d)
{
    if constexpr (TYPE == NUT_F32)
        return reinterpret_cast<const float *>(row)[d];
    const uint32_t bits = reinterpret_cast<const uint16_t *>(row)[d];
    return TYPE == NUT_BF16 ? from_bf16(bits) : from_f16(bits);
}

// A workgroup per (sequence, query head), 256 rows at a time: a thread per
// row takes its score, then a thread per component adds the weighted values.
template <int TYPE>
__global__ __launch_bounds__(256) void attend_kernel(PagedView kv, PagedSeqs s,
                                                     const float *__restrict__ query,
                                                     size_t query_stride, uint32_t heads,
                                                     float scale,
                                                     const int *__restrict__ selected,
                                                     uint32_t top, float *__restrict__ out,
                                                     float *__restrict__ lse,
                                                     float *__restrict__ scores,
                                                     size_t score_stride)
{
    __shared__ float q[256], p[256], red[8];
    __shared__ size_t at[256];
    const uint32_t hq = blockIdx.x % heads, b = blockIdx.x / heads;
    const uint32_t h = hq / (heads / kv.kv_heads), t = threadIdx.x;
    const uint32_t n = paged_length(kv, s, b, t == 0 && hq == 0);
    if (t < kv.head_dim)
        q[t] = query[b * query_stride + size_t(hq) * kv.head_dim + t] * scale;
    const uint32_t total = selected == nullptr ? n : top * kv.page_size;
    float most = -INFINITY, sum = 0.0f, acc = 0.0f;
    for (uint32_t base = 0; base < total; base += 256) {
        __syncthreads();
        const uint32_t i = base + t;
        size_t row = kNoRow;
        if (i < total) {
            int index = int(i / kv.page_size);
            const uint32_t slot = i % kv.page_size;
            if (selected != nullptr) {
                index = selected[(size_t(b) * kv.kv_heads + h) * top + index];
                if (index < -1 || index >= int((s.max_length - 1) / kv.page_size + 1))
                    paged_flag(kv.status, kBadPage);
            }
            if (index >= 0 && uint64_t(index) * kv.page_size + slot < n)
                row = paged_row(kv, s, b, uint32_t(index), slot, h);
        }
        float score = -INFINITY;
        if (row != kNoRow) {
            score = 0.0f;
            for (uint32_t d = 0; d < kv.head_dim; d++)
                score = fmaf(q[d], component<TYPE>(kv.keys + row, d), score);
        }
        if (scores != nullptr && i < total)
            scores[(size_t(b) * heads + hq) * score_stride + i] = score;
        float top_here = wave_max(score);
        if (t % kWave == 0)
            red[t / kWave] = top_here;
        __syncthreads();
        top_here = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float now = fmaxf(most, top_here);
        const float ref = now == -INFINITY ? 0.0f : now;
        const float keep = most == -INFINITY ? 0.0f : expf(most - ref);
        p[t] = expf(score - ref);
        at[t] = row;
        const float here = wave_sum(p[t]);
        if (t % kWave == 0)
            red[4 + t / kWave] = here;
        __syncthreads();
        sum = sum * keep + red[4] + red[5] + red[6] + red[7];
        acc *= keep;
        if (t < kv.head_dim)
            for (uint32_t j = 0; j < min(256u, total - base); j++)
                if (at[j] != kNoRow)
                    acc = fmaf(p[j], component<TYPE>(kv.values + at[j], t), acc);
        most = now;
    }
    if (t < kv.head_dim)
        out[(size_t(b) * heads + hq) * kv.head_dim + t] = sum == 0.0f ? 0.0f : acc / sum;
    if (t == 0 && lse != nullptr)
        lse[size_t(b) * heads + hq] = sum == 0.0f ? -INFINITY : most + logf(sum);
}

__global__ __launch_bounds__(256) void weigh_kernel(PagedView kv, PagedSeqs s, uint32_t heads,
                                                    const float *__restrict__ scores,
                                                    const float *__restrict__ lse,
                                                    size_t score_stride, float *weights,
                                                    size_t stride, uint32_t blocks)
{
    const uint32_t c = blockIdx.x % blocks, h = blockIdx.x / blocks % kv.kv_heads;
    const uint32_t b = blockIdx.x / blocks / kv.kv_heads, i = c * 256 + threadIdx.x;
    const uint32_t group = heads / kv.kv_heads;
    if (i >= paged_length(kv, s, b, false))
        return;
    float w = 0.0f;
    for (uint32_t j = 0; j < group; j++) {
        const size_t head = size_t(b) * heads + h * group + j;
        if (lse[head] != -INFINITY)
            w += expf(scores[head * score_stride + i] - lse[head]);
    }
    weights[(size_t(b) * kv.kv_heads + h) * stride + i] += w;
}

} // namespace

AttentionPlan plan_attention(const PagedView &kv, const PagedSeqs &seqs, uint32_t heads,
                             uint32_t top, bool weighted)
{
    (void)kv, (void)top;
    AttentionPlan plan{};
    plan.stats = 0;
    plan.scores = (size_t(seqs.batch) * heads * sizeof(float) + 255) / 256 * 256;
    plan.bytes = weighted ? plan.scores + size_t(seqs.batch) * heads * seqs.max_length * 4 : 0;
    return plan;
}

void launch_paged_attention(const PagedView &kv, const PagedSeqs &seqs, const float *query,
                            size_t query_stride, uint32_t heads, float scale,
                            const int *selected, uint32_t top, const PagedHistory &history,
                            float *out, float *lse, char *workspace, hipStream_t stream)
{
    const bool weighted = history.weights != nullptr;
    const AttentionPlan plan = plan_attention(kv, seqs, heads, top, weighted);
    float *scores = weighted ? reinterpret_cast<float *>(workspace + plan.scores) : nullptr;
    if (weighted && lse == nullptr)
        lse = reinterpret_cast<float *>(workspace);
    const auto kernel = kv.type == NUT_F32   ? attend_kernel<NUT_F32>
                        : kv.type == NUT_F16 ? attend_kernel<NUT_F16>
                                             : attend_kernel<NUT_BF16>;
    hipLaunchKernelGGL(kernel, paged_grid(uint64_t(seqs.batch) * heads, 256), dim3(256), 0, stream,
                       kv, seqs, query, query_stride, heads, scale, selected, top, out, lse,
                       scores, size_t(seqs.max_length));
    check_launch("paged attention");
    if (!weighted)
        return;
    const uint32_t blocks = (seqs.max_length + 255) / 256;
    hipLaunchKernelGGL(weigh_kernel,
                       paged_grid(uint64_t(seqs.batch) * kv.kv_heads * blocks, 256), dim3(256), 0,
                       stream, kv, seqs, heads, scores, lse, size_t(seqs.max_length),
                       history.weights, history.stride, blocks);
    check_launch("paged attention");
}

} // namespace nut
