// Attention of a tree of drafted tokens over the INT8 shared-KV cache, sm_100a.  The contract is in
// include/sharedkv_c_abi.h.
//
// One thread block per (token, eight heads), a warp per head: lane l holds channels 16 l .. 16 l + 15
// of the scaled query and of the running output.  Keys are taken one by one with an FP32 online
// softmax (running maximum, sum and output in registers).  Every token fetches its own keys, so the
// kernel is bound by instruction issue and by L2, far from what the tensor cores allow.
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include "../../include/sharedkv_c_abi.h"
#include "ptx_sm100.cuh"
#include "sharedkv_internal.h"

namespace sharedkv {
namespace {

using ptx::grid_dependency_launch_dependents;
using ptx::grid_dependency_wait;

constexpr uint32_t kTreePage = 32, kTreeDraft = 64, kTreeHeads = 8, kTreeThreads = 256;

__global__ void __launch_bounds__(kTreeThreads) tree_simple_kernel(const TreeAttentionArgs p)
{
    __shared__ uint32_t live_batch;
    grid_dependency_launch_dependents();
    grid_dependency_wait();
    const uint32_t lane = threadIdx.x & 31u, head = blockIdx.y * kTreeHeads + (threadIdx.x >> 5), t = blockIdx.x;
    const int32_t *cu = reinterpret_cast<const int32_t *>(p.cuQ), *seq = reinterpret_cast<const int32_t *>(p.seqLens);
    if (threadIdx.x == 0) live_batch = 0;
    __syncthreads();
    uint32_t live = 0;
    for (uint32_t b = threadIdx.x; b < p.batch; b += kTreeThreads) if (split::request_is_live(seq[b], cu[b + 1])) live = b + 1;
    if (live) atomicMax(&live_batch, live);
    __syncthreads();
    const uint32_t live_tokens = split::live_token_count(live_batch ? cu[live_batch] : 0, p.tokens);
    __nv_bfloat16 *out = reinterpret_cast<__nv_bfloat16 *>(p.out) + ((uint64_t)t * p.heads + head) * kDim + lane * 16u;
    float *lse = p.lse ? reinterpret_cast<float *>(p.lse) + (uint64_t)t * p.heads + head : nullptr;
    if (t >= live_tokens || (int32_t)t < cu[0]) {
        reinterpret_cast<uint4 *>(out)[0] = reinterpret_cast<uint4 *>(out)[1] = make_uint4(0, 0, 0, 0);
        if (lse && lane == 0) *lse = 0.f;
        return;
    }
    uint32_t b = 0, hi = live_batch - 1;
    while (b < hi) {
        const uint32_t mid = (b + hi) >> 1;
        if (cu[mid + 1] <= (int32_t)t) b = mid + 1; else hi = mid;
    }
    const int32_t n = cu[b + 1] - cu[b];
    const int64_t prefix = (int64_t)seq[b] - n;
    uint64_t path = reinterpret_cast<const uint64_t *>(p.paths)[t];
    if (n < (int32_t)kTreeDraft) path &= (1ull << n) - 1ull;
    const int64_t c = __popcll(path);

    float q[16], sc[2][16], acc[16], m = -INFINITY, l = 0.f;
    const __nv_bfloat16 *qs = reinterpret_cast<const __nv_bfloat16 *>(p.q) + ((uint64_t)t * p.heads + head) * kDim + lane * 16u;
    for (int i = 0; i < 16; ++i) {
        q[i] = __bfloat162float(qs[i]) * p.softmaxScale;
        sc[0][i] = reinterpret_cast<const float *>(p.oriScale)[lane * 16u + i];
        sc[1][i] = reinterpret_cast<const float *>(p.cmpScale)[lane * 16u + i];
        acc[i] = 0.f;
    }
    auto attend = [&](int kind, int64_t row) {
        const uint32_t width = kind ? p.cmpTableWidth : p.oriTableWidth, pages = kind ? p.cmpPages : p.oriPages;
        if (row < 0 || row / kTreePage >= width) return;
        const int32_t page = reinterpret_cast<const int32_t *>(kind ? p.cmpTable : p.oriTable)[(uint64_t)b * width + row / kTreePage];
        if ((uint32_t)page >= pages) return;
        const uint64_t src = (kind ? p.cmp : p.ori) + (uint64_t)page * (kind ? p.cmpStride : p.oriStride) + (uint64_t)(row % kTreePage) * kDim;
        const uint4 raw = *reinterpret_cast<const uint4 *>(src + lane * 16u);
        const int8_t *codes = reinterpret_cast<const int8_t *>(&raw);
        float v[16], s = 0.f;
        for (int i = 0; i < 16; ++i) { v[i] = (float)codes[i] * sc[kind][i]; s = fmaf(q[i], v[i], s); }
        for (int d = 16; d; d >>= 1) s += __shfl_xor_sync(0xffffffffu, s, d);
        const float top = fmaxf(m, s), r = m == -INFINITY ? 0.f : expf(m - top), w = expf(s - top);
        l = fmaf(l, r, w);
        for (int i = 0; i < 16; ++i) acc[i] = fmaf(acc[i], r, w * v[i]);
        m = top;
    };
    for (int64_t r = max((int64_t)0, prefix - (int64_t)p.window + c); r < prefix; ++r) attend(0, r);
    for (uint64_t left = path; left; left &= left - 1ull) attend(0, prefix + __ffsll((long long)left) - 1);
    const int64_t whole = prefix > 0 ? prefix / p.ratio : 0;
    if (p.ratio == 128u) {
        for (int64_t r = 0; r < whole; ++r) attend(1, r);
        if (p.cmpPaths)
            for (uint64_t left = reinterpret_cast<const uint64_t *>(p.cmpPaths)[t]; left; left &= left - 1ull) attend(1, whole + __ffsll((long long)left) - 1);
    } else if (p.ratio == 4u) {
        for (uint32_t i = 0; i < p.topk; ++i) {
            const int32_t r = reinterpret_cast<const int32_t *>(p.indices)[(uint64_t)t * p.topk + i];
            if (r >= 0 && r < whole + kTreeDraft) attend(1, r);
        }
    }
    const float sink = reinterpret_cast<const float *>(p.sinks)[head], top = fmaxf(m, sink);
    const float r = m == -INFINITY ? 0.f : expf(m - top), total = l * r + (sink == -INFINITY ? 0.f : expf(sink - top));
    for (int i = 0; i < 16; ++i) out[i] = __float2bfloat16_rn(total > 0.f || total != total ? acc[i] * r / total : 0.f);
    if (lse && lane == 0) *lse = total > 0.f || total != total ? top + logf(total) : -INFINITY;
}

}  // namespace

uint64_t tree_workspace_bytes(uint32_t, uint32_t, uint32_t, uint32_t, uint32_t) { return 256; }

int tree_attention(const TreeAttentionArgs *args, cudaStream_t stream)
{
    if (args == nullptr) return SHAREDKV_EINVAL;
    TreeAttentionArgs a = *args;
    if (a.tokens == 0 || a.batch == 0) return SHAREDKV_OK;
    if (a.ratio != 1u && a.ratio != 4u && a.ratio != 128u) return SHAREDKV_EINVAL;
    if (a.heads == 0 || a.heads % kTreeHeads || a.heads > 128u || a.window == 0 || a.window > 65536u) return SHAREDKV_EINVAL;
    if (a.ratio == 1u) {
        // no compressed kind: its fields alias the original cache so that nothing in the kernel is null
        a.cmp = a.ori; a.cmpScale = a.oriScale; a.cmpTable = a.oriTable; a.cmpStride = a.oriStride;
        a.cmpTableWidth = a.oriTableWidth; a.cmpPages = a.oriPages;
    }
    if (a.ratio != 128u) a.cmpPaths = 0;
    if (a.ratio == 4u && (a.topk == 0 || a.topk > 1024u || !a.indices || a.indices % 4u)) return SHAREDKV_EINVAL;
    if (!a.q || !a.ori || !a.cmp || !a.oriScale || !a.cmpScale || !a.oriTable || !a.cmpTable || !a.paths || !a.cuQ || !a.seqLens ||
        !a.sinks || !a.out || !a.workspace)
        return SHAREDKV_EINVAL;
    if (a.q % 16u || a.out % 16u || a.ori % 16u || a.cmp % 16u || a.oriStride % 16u || a.cmpStride % 16u || a.workspace % 256u ||
        a.oriScale % 4u || a.cmpScale % 4u || a.sinks % 4u || a.lse % 4u || a.oriTable % 4u || a.cmpTable % 4u || a.cuQ % 4u ||
        a.seqLens % 4u || a.paths % 8u || a.cmpPaths % 8u)
        return SHAREDKV_EINVAL;
    if (a.oriStride < (uint64_t)kTreePage * kDim || a.cmpStride < (uint64_t)kTreePage * kDim) return SHAREDKV_EINVAL;
    if (!a.oriTableWidth || !a.cmpTableWidth || !a.oriPages || !a.cmpPages || a.oriPages >= (1u << 26) || a.cmpPages >= (1u << 26) ||
        a.oriTableWidth >= (1u << 26) || a.cmpTableWidth >= (1u << 26))
        return SHAREDKV_EINVAL;
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(a.tokens, a.heads / kTreeHeads);
    config.blockDim = dim3(kTreeThreads);
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = programmatic_launch_enabled() ? 1u : 0u;
    return (int)cudaLaunchKernelEx(&config, tree_simple_kernel, a);
}

}  // namespace sharedkv
