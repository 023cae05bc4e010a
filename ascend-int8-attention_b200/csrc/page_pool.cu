// Page pool: block table, sequence lengths and reference counts of a set of INT8 caches that share
// their page numbering, changed on the device (resize, fork), and the page and row moves that go with
// them (copy, keep).  The contract is in include/sharedkv_c_abi.h.
//
// resize and fork are planned by one cluster of sixteen thread blocks (one block for small pools), whose
// hardware barrier separates the phases: the counts of what is released and shared are updated; zeros are counted per warp chunk and the
// counts added up, which ranks the lowest-numbered free pages; if they do not suffice the count changes are
// taken back; else they are dealt out in sequence order by a prefix sum.  Counts change by integer
// atomics, whose sum does not depend on their order; every other value is written by one thread.
// The plan is a chain of dependent L2 accesses, so it is bound by latency: a fork of 512 sequences of 85 pages
// with its copies takes 126 us with one block, 28 with eight and 24 with sixteen.
// Pages are copied by a kernel of their own, over all SMs, or by the plan's blocks where that is at most
// kPlanCopyBytes (always for resize, which copies only shared, partly filled last pages).
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/sharedkv_c_abi.h"
#include "ptx_sm100.cuh"
#include "sharedkv_internal.h"

namespace sharedkv {
namespace {

using ptx::grid_dependency_launch_dependents;
using ptx::grid_dependency_wait;

constexpr uint32_t kPlanBlocks = 16, kPlanThreads = 1024, kBlockWarps = kPlanThreads / 32;
constexpr uint32_t kAloneWork = 8192;               // pages + table entries up to which one block is as fast as a cluster
constexpr uint32_t kMaxSequences = 8192;            // rows whose bookkeeping fits the plan kernel's shared memory
constexpr uint32_t kStripWords = 16384;             // table entries a fork holds in shared memory at a time
constexpr uint32_t kCopyThreads = 256;
constexpr uint64_t kPlanCopyBytes = 1u << 20;        // a second launch costs about what the plan's blocks need for this much
constexpr uint32_t kCopyUnit = 8192, kCopyLoads = kCopyUnit / 16 / kCopyThreads;      // bytes a block moves at a time, 16-byte loads per thread
constexpr uint32_t kKeepThreads = 256, kMaxKept = 64;

// workspace: word 0 sticky status, word 1 number of page copies, words 64.. chunk counts; then the
// copy list and the fresh pages
constexpr uint64_t kWsCounts = 256, kWsCopies = 256 + 4 * 1024;      // 512 counts fit twice over
__host__ __device__ constexpr uint64_t page_ws_fresh(uint32_t batch) { return kWsCopies + 8ull * batch; }
__host__ __device__ constexpr uint64_t page_ws_bytes(uint32_t batch, uint32_t width)
{
    return page_ws_fresh(batch) + 4ull * batch * ((uint64_t)width + 1ull);
}

static_assert(kWsCounts + 4 * kPlanBlocks * kBlockWarps <= kWsCopies, "a count per warp");

struct Pool {
    const uint64_t *caches;
    int32_t *table, *lens, *refs;
    uint32_t *head, *counts;
    int2 *copies;
    int32_t *fresh;
    uint32_t layers, pages, rows, batch, width;
    uint32_t copies_here;          // the plan's blocks copy the pages
};

// Barrier of the plan's blocks; orders their memory accesses too.
template <uint32_t BLOCKS>
__device__ __forceinline__ void plan_sync()
{
    if (BLOCKS == 1) __syncthreads();
    else asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}
__device__ __forceinline__ uint32_t plan_warp() { return blockIdx.x * kBlockWarps + (threadIdx.x >> 5); }

__device__ __forceinline__ uint32_t pages_of(int32_t rows, uint32_t per_page) { return rows <= 0 ? 0u : ((uint32_t)rows + per_page - 1u) / per_page; }

// Exclusive prefix of one value per sequence, in place in shared memory; returns the total.
__device__ uint32_t scan_sequences(uint32_t *v, uint32_t count, uint32_t *scratch)
{
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t per = (count + kPlanThreads - 1u) / kPlanThreads;
    const uint32_t begin = min(threadIdx.x * per, count), end = min(begin + per, count);
    uint32_t sum = 0;
    for (uint32_t i = begin; i < end; ++i) sum += v[i];
    uint32_t incl = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t n = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= (uint32_t)d) incl += n;
    }
    if (lane == 31) scratch[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        uint32_t s = scratch[lane], si = s;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t n = __shfl_up_sync(0xffffffffu, si, d);
            if (lane >= (uint32_t)d) si += n;
        }
        scratch[lane] = si - s;
        if (lane == 31) scratch[32] = si;
    }
    __syncthreads();
    uint32_t before = scratch[warp] + incl - sum;
    for (uint32_t i = begin; i < end; ++i) {
        const uint32_t x = v[i];
        v[i] = before;
        before += x;
    }
    const uint32_t total = scratch[32];
    __syncthreads();
    return total;
}

// Pages of this warp's chunk with a zero count.
__device__ uint32_t count_free(const Pool &p, uint32_t begin, uint32_t end, uint32_t lane)
{
    uint32_t n = 0;
#pragma unroll 4
    for (uint32_t i = begin + lane; i < end; i += 32u) n += __ldcg(p.refs + i) == 0;
    return __reduce_add_sync(0xffffffffu, n);
}

// Writes the free pages of the chunk to fresh[at ..], as far as `total` reaches.
__device__ void list_free(const Pool &p, uint32_t begin, uint32_t end, uint32_t at, uint32_t total, uint32_t lane)
{
    for (uint32_t base = begin; base < end && at < total; base += 32u) {
        const uint32_t i = base + lane;
        const bool is_free = i < end && __ldcg(p.refs + i) == 0;
        const uint32_t mask = __ballot_sync(0xffffffffu, is_free);
        const uint32_t slot = at + __popc(mask & ((1u << lane) - 1u));
        if (is_free && slot < total) p.fresh[slot] = (int32_t)i;
        at += __popc(mask);
    }
}

// Adds `delta` to the counts of the pages row[begin .. end - 1] (one warp, four entries of a lane in flight).
__device__ __forceinline__ void add_refs(const Pool &p, const int32_t *row, uint32_t begin, uint32_t end, int32_t delta, uint32_t lane)
{
    for (uint32_t k = begin + lane; k < end; k += 128u) {
        int32_t page[4];
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) page[i] = k + 32u * i < end ? __ldcg(row + k + 32u * i) : -1;
#pragma unroll
        for (uint32_t i = 0; i < 4; ++i) if ((uint32_t)page[i] < p.pages) atomicAdd(p.refs + page[i], delta);
    }
}

// Finds the `total` lowest free pages; false (for every thread of the cluster) when there are fewer.
template <uint32_t BLOCKS>
__device__ bool take_free(const Pool &p, uint32_t total, uint32_t *scratch)
{
    constexpr uint32_t kWarps = BLOCKS * kBlockWarps;
    const uint32_t lane = threadIdx.x & 31u, warp = plan_warp();
    const uint32_t chunk = ((p.pages + kWarps - 1u) / kWarps + 31u) & ~31u;
    const uint32_t begin = min(warp * chunk, p.pages), end = min(begin + chunk, p.pages);
    const uint32_t mine = count_free(p, begin, end, lane);
    if (lane == 0) p.counts[warp] = mine;
    plan_sync<BLOCKS>();
    uint32_t all = 0, before = 0;
#pragma unroll
    for (uint32_t i = lane; i < kWarps; i += 32u) {
        const uint32_t n = __ldcg(p.counts + i);
        all += n;
        before += i < warp ? n : 0u;
    }
    all = __reduce_add_sync(0xffffffffu, all);
    before = __reduce_add_sync(0xffffffffu, before);
    if (all >= total) list_free(p, begin, end, before, total, lane);
    plan_sync<BLOCKS>();
    return all >= total;
}

// Copies up to four rows of a page in one cache (one warp).
__device__ __forceinline__ void copy_rows(const Pool &p, uint32_t layer, int32_t source, int32_t target, uint32_t first, uint32_t count, uint32_t lane)
{
    const uint64_t base = p.caches[2u * layer], stride = p.caches[2u * layer + 1u];
    const uint4 *src = reinterpret_cast<const uint4 *>(base + (uint64_t)source * stride) + first * 32u + lane;
    uint4 *dst = reinterpret_cast<uint4 *>(base + (uint64_t)target * stride) + first * 32u + lane;
    uint4 v[4];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) if (k < count) v[k] = src[k * 32u];
#pragma unroll
    for (uint32_t k = 0; k < 4; ++k) if (k < count) dst[k * 32u] = v[k];
}

template <uint32_t BLOCKS>
__global__ void __launch_bounds__(kPlanThreads, 1) page_resize_plan(const Pool p, const int32_t *wanted)
{
    extern __shared__ uint32_t smem[];
    uint32_t *offset = smem;                       // per sequence: fresh pages needed, then where they start
    __shared__ uint32_t scratch[64];
    grid_dependency_launch_dependents();
    grid_dependency_wait();
    constexpr uint32_t kWarps = BLOCKS * kBlockWarps;
    const uint32_t lane = threadIdx.x & 31u, warp = plan_warp();
    bool bad = false;
    for (uint32_t b = threadIdx.x; b < p.batch; b += kPlanThreads)
        bad |= wanted[b] < 0 || pages_of(wanted[b], p.rows) > p.width || pages_of(p.lens[b], p.rows) > p.width;
    if (__syncthreads_or(bad)) {                              // the same in every block
        if (threadIdx.x == 0) p.head[0] = kStatusRange;
        return;
    }
    auto release = [&](int32_t delta) {
        for (uint32_t b = warp; b < p.batch; b += kWarps) {
            const uint32_t before = pages_of(p.lens[b], p.rows), after = pages_of(wanted[b], p.rows);
            add_refs(p, p.table + (uint64_t)b * p.width, after, before, delta, lane);
        }
    };
    release(-1);
    plan_sync<BLOCKS>();
    for (uint32_t b = threadIdx.x; b < p.batch; b += kPlanThreads) {
        const uint32_t before = pages_of(p.lens[b], p.rows), after = pages_of(wanted[b], p.rows);
        uint32_t need = after > before ? after - before : 0u;
        if (wanted[b] > p.lens[b] && p.lens[b] > 0 && (uint32_t)p.lens[b] % p.rows) {
            const int32_t last = p.table[(uint64_t)b * p.width + before - 1u];
            need += (uint32_t)last < p.pages && __ldcg(p.refs + last) > 1;
        }
        offset[b] = need;
    }
    __syncthreads();
    const uint32_t total = scan_sequences(offset, p.batch, scratch);
    if (!take_free<BLOCKS>(p, total, scratch)) {
        release(1);
        if (threadIdx.x == 0) p.head[0] = kStatusRange;
        return;
    }
    for (uint32_t b = warp; b < p.batch; b += kWarps) {
        const uint32_t before = pages_of(p.lens[b], p.rows), after = pages_of(wanted[b], p.rows);
        const uint32_t first = offset[b], count = (b + 1u < p.batch ? offset[b + 1u] : total) - first;
        const uint32_t grown = after > before ? after - before : 0u, split = count - grown;      // split: 1 when the last page is replaced
        int32_t *row = p.table + (uint64_t)b * p.width;
        if (split) {
            const int32_t source = row[before - 1u], page = p.fresh[first];
            __syncwarp();
            if (lane == 0) {
                row[before - 1u] = page;
                p.refs[page] = 1;
                atomicAdd(p.refs + source, -1);
            }
            for (uint32_t layer = 0; layer < p.layers; ++layer)
                for (uint32_t r = 0; r < p.rows; r += 4u) copy_rows(p, layer, source, page, r, min(p.rows - r, 4u), lane);
        }
        for (uint32_t k = lane; k < grown; k += 32u) {
            const int32_t page = p.fresh[first + split + k];
            row[before + k] = page;
            p.refs[page] = 1;
        }
        __syncwarp();
        if (lane == 0) p.lens[b] = wanted[b];
    }
}

template <uint32_t BLOCKS>
__global__ void __launch_bounds__(kPlanThreads, 1) page_fork_plan(const Pool p, const int32_t *parents)
{
    extern __shared__ uint32_t smem[];
    uint32_t *offset = smem;                                                        // per sequence: 1 when it gets a copy, then the copy's number
    int32_t *parent = reinterpret_cast<int32_t *>(smem) + p.batch;
    int32_t *len = parent + p.batch, *children = len + p.batch, *strip = children + p.batch;
    uint32_t *first = reinterpret_cast<uint32_t *>(strip);                          // lowest child; the strips follow it in time
    __shared__ uint32_t scratch[64];
    grid_dependency_launch_dependents();
    grid_dependency_wait();
    constexpr uint32_t kWarps = BLOCKS * kBlockWarps;
    const uint32_t lane = threadIdx.x & 31u, warp = plan_warp();
    bool bad = false;
    uint32_t longest = 0;
    for (uint32_t b = threadIdx.x; b < p.batch; b += kPlanThreads) {
        parent[b] = parents[b];
        len[b] = p.lens[b];
        children[b] = 0;
        first[b] = 0xffffffffu;
        bad |= parents[b] >= (int32_t)p.batch || pages_of(len[b], p.rows) > p.width;
    }
    if (threadIdx.x == 0) scratch[40] = 0;
    if (threadIdx.x == 0 && blockIdx.x == 0) p.head[1] = 0;
    if (__syncthreads_or(bad)) {
        if (threadIdx.x == 0) p.head[0] = kStatusRange;
        return;
    }
    for (uint32_t b = threadIdx.x; b < p.batch; b += kPlanThreads) {
        if (parent[b] < 0) continue;
        atomicAdd(children + parent[b], 1);
        atomicMin(first + parent[b], b);
        longest = max(longest, pages_of(len[parent[b]], p.rows));
    }
    atomicMax(scratch + 40, longest);
    __syncthreads();
    longest = scratch[40];
    for (uint32_t b = threadIdx.x; b < p.batch; b += kPlanThreads)
        offset[b] = parent[b] >= 0 && first[parent[b]] != b && len[parent[b]] > 0 && (uint32_t)len[parent[b]] % p.rows != 0;
    // full pages gain a reference per further child; a sequence without a child gives up all of its pages
    auto share = [&](int32_t sign) {
        for (uint32_t b = warp; b < p.batch; b += kWarps) {
            if (children[b] == 1) continue;
            const uint32_t live = pages_of(len[b], p.rows), full = len[b] <= 0 ? 0u : (uint32_t)len[b] / p.rows;
            add_refs(p, p.table + (uint64_t)b * p.width, 0u, children[b] ? full : live, sign * (children[b] - 1), lane);
        }
    };
    share(1);
    plan_sync<BLOCKS>();
    const uint32_t total = scan_sequences(offset, p.batch, scratch);
    if (!take_free<BLOCKS>(p, total, scratch)) {
        share(-1);
        if (threadIdx.x == 0) p.head[0] = kStatusRange;
        return;
    }
    // The table is permuted in place, a strip of columns at a time, the strips dealt to the blocks: all rows of
    // a strip are read before one is written.
    uint32_t columns = 32;
    while (columns > 1u && columns * p.batch > kStripWords) columns >>= 1;
    while (columns > 8u && columns * BLOCKS > longest) columns >>= 1;         // a strip for every block, but whole 32-byte sectors
    const uint32_t cells = columns * p.batch, shift = 31u - __clz(columns);
    for (uint32_t left = blockIdx.x * columns; left < longest; left += BLOCKS * columns) {
        for (uint32_t base = threadIdx.x; base < cells; base += 8u * kPlanThreads) {
            int32_t page[8];                                  // eight reads of a thread in flight
#pragma unroll
            for (uint32_t n = 0; n < 8; ++n) {
                const uint32_t i = base + n * kPlanThreads, b = i >> shift, k = left + (i & (columns - 1u));
                if (i < cells && k < pages_of(len[b], p.rows)) page[n] = p.table[(uint64_t)b * p.width + k];
            }
#pragma unroll
            for (uint32_t n = 0; n < 8; ++n) if (base + n * kPlanThreads < cells) strip[base + n * kPlanThreads] = page[n];
        }
        __syncthreads();
        for (uint32_t i = threadIdx.x; i < cells; i += kPlanThreads) {
            const uint32_t b = i >> shift, k = left + (i & (columns - 1u));
            const int32_t of = parent[b];
            if (of < 0) continue;
            const uint32_t live = pages_of(len[of], p.rows);
            if (k >= live) continue;
            int32_t page = strip[((uint32_t)of << shift) + (k - left)];
            const bool copied = (b + 1u < p.batch ? offset[b + 1u] : total) != offset[b];
            if (copied && k + 1u == live) {
                const int32_t source = page;
                page = p.fresh[offset[b]];
                p.refs[page] = 1;
                p.copies[atomicAdd(p.head + 1, 1u)] = make_int2(source, page);
            } else if ((uint32_t)of == b) {
                continue;
            }
            p.table[(uint64_t)b * p.width + k] = page;
        }
        __syncthreads();
    }
    if (blockIdx.x == 0)                                      // every block has had its own copy since before the first barrier
        for (uint32_t b = threadIdx.x; b < p.batch; b += kPlanThreads) p.lens[b] = parent[b] < 0 ? 0 : len[parent[b]];
    if (p.copies_here) {
        plan_sync<BLOCKS>();
        const uint32_t count = __ldcg(p.head + 1);
        const uint32_t pieces = (p.rows + 3u) / 4u;           // a warp moves four rows of one cache at a time
        for (uint32_t i = warp; i < count * p.layers * pieces; i += kWarps) {
            const uint32_t piece = i % pieces, layer = i / pieces % p.layers;
            const int2 pair = __ldcg(p.copies + i / pieces / p.layers);
            if ((uint32_t)pair.x < p.pages) copy_rows(p, layer, pair.x, pair.y, piece * 4u, min(p.rows - piece * 4u, 4u), lane);
        }
    }
}

// Page copies: unit = 8 KB of one page of one cache; thread blocks walk the units in order.  Streaming: bound by
// HBM (a page is read and written once; 700 pages in 16 caches move at 5.6 TB/s, 0.86 of a plain copy's rate; twice the
// unit with half the blocks 5.7, but 3 us more for the 160 pages in 8 caches of a fork), or by latency when there are few.
__global__ void __launch_bounds__(kCopyThreads) page_copy_kernel(const uint64_t *caches, const int2 *pairs, const uint32_t *count_word,
                                                                  uint32_t count, uint32_t layers, uint32_t pages, uint32_t page_bytes)
{
    grid_dependency_launch_dependents();
    grid_dependency_wait();
    if (count_word) count = *count_word;
    const uint32_t pieces = (page_bytes + kCopyUnit - 1u) / kCopyUnit;
    const uint64_t units = (uint64_t)count * layers * pieces;
    for (uint64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const uint32_t piece = (uint32_t)(u % pieces);
        const uint64_t rest = u / pieces;
        const uint32_t layer = (uint32_t)(rest % layers);
        const int2 pair = pairs[rest / layers];
        if ((uint32_t)pair.x >= pages || (uint32_t)pair.y >= pages) continue;
        const uint64_t base = caches[2u * layer], stride = caches[2u * layer + 1u];
        const uint4 *src = reinterpret_cast<const uint4 *>(base + (uint64_t)pair.x * stride + (uint64_t)piece * kCopyUnit);
        uint4 *dst = reinterpret_cast<uint4 *>(base + (uint64_t)pair.y * stride + (uint64_t)piece * kCopyUnit);
        const uint32_t vectors = min(kCopyUnit, page_bytes - piece * kCopyUnit) / 16u;
        uint4 v[kCopyLoads];
#pragma unroll
        for (uint32_t i = 0; i < kCopyLoads; ++i) if (threadIdx.x + i * kCopyThreads < vectors) v[i] = src[threadIdx.x + i * kCopyThreads];
#pragma unroll
        for (uint32_t i = 0; i < kCopyLoads; ++i) if (threadIdx.x + i * kCopyThreads < vectors) dst[threadIdx.x + i * kCopyThreads] = v[i];
    }
}

// A thread block takes a sequence in some of the layers: where the rows come from and go to is looked up
// once.  A warp takes kept rows w, w + 8, ...; of kKeepLayers layers at a time, every row (32 lanes x 16 bytes)
// is in registers before the block-wide barrier, and written behind it.  Bound by the latency of the look-ups for
// small trees (3 us), by HBM for many layers: 256 trees of 1 to 17 rows in 24 caches, 57 MB, take 13 us (4.4 TB/s; 40 us
// with a look-up per layer).
template <uint32_t ROUNDS>
__global__ void __launch_bounds__(kKeepThreads) page_keep_kernel(const Pool p, const int32_t *base, const int32_t *kept, uint32_t kept_width,
                                                                 uint32_t layers_per_block)
{
    constexpr uint32_t kWarps = kKeepThreads / 32, kKeepLayers = ROUNDS <= 2 ? 4 : 2;
    grid_dependency_launch_dependents();
    grid_dependency_wait();
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t groups = (p.layers + layers_per_block - 1u) / layers_per_block;
    for (uint64_t item = blockIdx.x; item < (uint64_t)p.batch * groups; item += gridDim.x) {
        const uint32_t b = (uint32_t)(item / groups), first = (uint32_t)(item % groups) * layers_per_block;
        const uint32_t last = min(first + layers_per_block, p.layers);
        const int32_t start = base[b];
        // lane r looks up round r: page and row of source and target
        int32_t from_page = -1, to_page = -1;
        uint32_t from_row = 0, to_row = 0;
        if (lane < ROUNDS) {
            const uint32_t i = lane * kWarps + warp;
            const int32_t from = i < kept_width ? kept[(uint64_t)b * kept_width + i] : -1;
            auto place = [&](int64_t row, int32_t &page, uint32_t &in_page) {
                if (row < 0 || row >= (int64_t)p.width * p.rows) return;
                page = p.table[(uint64_t)b * p.width + (uint32_t)row / p.rows];
                in_page = (uint32_t)row % p.rows;
            };
            if (from >= 0 && (uint32_t)from != i) {           // others are in their place already
                place((int64_t)start + from, from_page, from_row);
                place((int64_t)start + i, to_page, to_row);
            }
            if ((uint32_t)from_page >= p.pages || (uint32_t)to_page >= p.pages) to_page = -1;
        }
        for (uint32_t layer = first; layer < last; layer += kKeepLayers) {
            uint4 v[kKeepLayers][ROUNDS];
#pragma unroll
            for (uint32_t l = 0; l < kKeepLayers; ++l) {
                if (layer + l >= last) continue;
                const uint64_t cache = p.caches[2u * (layer + l)], stride = p.caches[2u * (layer + l) + 1u];
#pragma unroll
                for (uint32_t r = 0; r < ROUNDS; ++r) {
                    const int32_t page = __shfl_sync(0xffffffffu, from_page, r);
                    const uint32_t row = __shfl_sync(0xffffffffu, from_row, r);
                    if (__shfl_sync(0xffffffffu, to_page, r) >= 0)
                        v[l][r] = *reinterpret_cast<const uint4 *>(cache + (uint64_t)(uint32_t)page * stride + row * 512ull + lane * 16u);
                }
            }
            __syncthreads();
#pragma unroll
            for (uint32_t l = 0; l < kKeepLayers; ++l) {
                if (layer + l >= last) continue;
                const uint64_t cache = p.caches[2u * (layer + l)], stride = p.caches[2u * (layer + l) + 1u];
#pragma unroll
                for (uint32_t r = 0; r < ROUNDS; ++r) {
                    const int32_t page = __shfl_sync(0xffffffffu, to_page, r);
                    const uint32_t row = __shfl_sync(0xffffffffu, to_row, r);
                    if (page >= 0)
                        *reinterpret_cast<uint4 *>(cache + (uint64_t)(uint32_t)page * stride + row * 512ull + lane * 16u) = v[l][r];
                }
            }
        }
    }
}

template <class... Params, class... Args>
cudaError_t launch(void (*kernel)(Params...), uint32_t cluster, uint32_t blocks, uint32_t threads, uint32_t smem, cudaStream_t stream, Args... args)
{
    cudaLaunchConfig_t config = {};
    config.gridDim = dim3(blocks);
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute[2];
    config.attrs = attribute;
    config.numAttrs = 0;
    if (cluster > 1u) {
        attribute[config.numAttrs].id = cudaLaunchAttributeClusterDimension;
        attribute[config.numAttrs].val.clusterDim.x = cluster;
        attribute[config.numAttrs].val.clusterDim.y = attribute[config.numAttrs].val.clusterDim.z = 1;
        ++config.numAttrs;
    }
    if (programmatic_launch_enabled()) {
        attribute[config.numAttrs].id = cudaLaunchAttributeProgrammaticStreamSerialization;
        attribute[config.numAttrs].val.programmaticStreamSerializationAllowed = 1;
        ++config.numAttrs;
    }
    return cudaLaunchKernelEx(&config, kernel, static_cast<Params>(args)...);
}

cudaError_t launch_copies(const PagePoolArgs &a, const int2 *pairs, const uint32_t *count_word, uint32_t count, uint32_t most, int sms, cudaStream_t stream)
{
    const uint32_t page_bytes = a.pageRows * 512u;
    const uint64_t units = (uint64_t)most * a.layers * ((page_bytes + kCopyUnit - 1u) / kCopyUnit);
    const uint64_t cap = (uint64_t)sms * 8u;                    // eight 256-thread blocks fill an SM
    const uint32_t blocks = (uint32_t)(units < cap ? units : cap);
    return launch(page_copy_kernel, 1u, blocks, kCopyThreads, 0u, stream, reinterpret_cast<const uint64_t *>(a.caches), pairs, count_word, count,
                  a.layers, a.pages, page_bytes);
}

bool caches_ok(const PagePoolArgs &a)
{
    return a.caches && a.caches % 8u == 0 && a.layers && a.pages && a.pageRows && a.pages <= 0x7fffffffu && a.pageRows <= (1u << 20);
}
bool table_ok(const PagePoolArgs &a)
{
    return a.table && a.table % 4u == 0 && a.batch && a.width && (uint64_t)a.width * a.pageRows < (1ull << 31);
}

}  // namespace

int page_plan(uint32_t op, const PagePoolArgs *args, const int32_t *input, cudaStream_t stream)
{
    if (args == nullptr) return SHAREDKV_EINVAL;
    const PagePoolArgs a = *args;
    if (a.batch == 0) return SHAREDKV_OK;
    if (!caches_ok(a) || !table_ok(a) || !a.lens || !a.refs || !a.workspace || !input || a.lens % 4u || a.refs % 4u || a.workspace % 256u ||
        reinterpret_cast<uintptr_t>(input) % 4u)
        return SHAREDKV_EINVAL;
    if (a.batch > kMaxSequences || (uint64_t)a.batch * a.width > 0xffffffffull) return SHAREDKV_ERANGE;       // fresh pages are counted in 32 bits
    const int sms = device_sm_count();
    if (sms <= 0) return (int)cudaErrorInvalidDevice;
    Pool p = {};
    char *ws = reinterpret_cast<char *>(a.workspace);
    p.caches = reinterpret_cast<const uint64_t *>(a.caches);
    p.table = reinterpret_cast<int32_t *>(a.table);
    p.lens = reinterpret_cast<int32_t *>(a.lens);
    p.refs = reinterpret_cast<int32_t *>(a.refs);
    p.head = reinterpret_cast<uint32_t *>(ws);
    p.counts = reinterpret_cast<uint32_t *>(ws + kWsCounts);
    p.copies = reinterpret_cast<int2 *>(ws + kWsCopies);
    p.fresh = reinterpret_cast<int32_t *>(ws + page_ws_fresh(a.batch));
    p.layers = a.layers; p.pages = a.pages; p.rows = a.pageRows; p.batch = a.batch; p.width = a.width;
    // a fork makes fewer copies than it has sequences
    p.copies_here = (uint64_t)a.batch * a.layers * a.pageRows * 512u <= kPlanCopyBytes;
    cudaError_t e;
    // Large dynamic shared memory and clusters of more than eight blocks are opted into, once per device.
    static std::atomic<uint64_t> configured{0};
    int device = 0;
    e = cudaGetDevice(&device);
    if (e != cudaSuccess) return (int)e;
    const uint64_t bit = device >= 0 && device < kMaxDevices ? 1ull << device : 0ull;
    if (!bit || !(configured.load(std::memory_order_relaxed) & bit)) {
        constexpr int kMost = (int)(4u * (4u * kMaxSequences + kStripWords));
        e = cudaFuncSetAttribute(page_fork_plan<1>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(page_fork_plan<kPlanBlocks>, cudaFuncAttributeMaxDynamicSharedMemorySize, kMost);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(page_fork_plan<kPlanBlocks>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e == cudaSuccess) e = cudaFuncSetAttribute(page_resize_plan<kPlanBlocks>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1);
        if (e != cudaSuccess) return (int)e;
        configured.fetch_or(bit, std::memory_order_relaxed);
    }
    const bool alone = (uint64_t)a.pages + (uint64_t)a.batch * a.width <= kAloneWork;
    const uint32_t blocks = alone ? 1u : kPlanBlocks;
    if (op == 0) {
        const auto kernel = alone ? page_resize_plan<1> : page_resize_plan<kPlanBlocks>;
        return (int)launch(kernel, blocks, blocks, kPlanThreads, 4u * a.batch, stream, p, input);
    }
    const uint32_t strip = a.batch > kStripWords ? a.batch : kStripWords;
    const auto kernel = alone ? page_fork_plan<1> : page_fork_plan<kPlanBlocks>;
    e = launch(kernel, blocks, blocks, kPlanThreads, 4u * (4u * a.batch + strip), stream, p, input);
    if (e == cudaSuccess && !p.copies_here) e = launch_copies(a, p.copies, p.head + 1, 0u, a.batch, sms, stream);
    return (int)e;
}

int page_copy(const PagePoolArgs *args, const int32_t *pairs, uint32_t count, cudaStream_t stream)
{
    if (args == nullptr || !caches_ok(*args)) return SHAREDKV_EINVAL;
    if (count == 0) return SHAREDKV_OK;
    if (!pairs || reinterpret_cast<uintptr_t>(pairs) % 8u) return SHAREDKV_EINVAL;
    const int sms = device_sm_count();
    if (sms <= 0) return (int)cudaErrorInvalidDevice;
    return (int)launch_copies(*args, reinterpret_cast<const int2 *>(pairs), nullptr, count, count, sms, stream);
}

int page_keep(const PagePoolArgs *args, const int32_t *base, const int32_t *kept, uint32_t kept_width, cudaStream_t stream)
{
    if (args == nullptr) return SHAREDKV_EINVAL;
    const PagePoolArgs a = *args;
    if (a.batch == 0 || kept_width == 0) return SHAREDKV_OK;
    if (!caches_ok(a) || !table_ok(a) || !base || !kept || kept_width > kMaxKept || reinterpret_cast<uintptr_t>(base) % 4u ||
        reinterpret_cast<uintptr_t>(kept) % 4u)
        return SHAREDKV_EINVAL;
    const int sms = device_sm_count();
    if (sms <= 0) return (int)cudaErrorInvalidDevice;
    Pool p = {};
    p.caches = reinterpret_cast<const uint64_t *>(a.caches);
    p.table = reinterpret_cast<int32_t *>(a.table);
    p.layers = a.layers; p.pages = a.pages; p.rows = a.pageRows; p.batch = a.batch; p.width = a.width;
    // Layers share the look-ups; a block takes as few of them as still give every SM eight blocks.
    const uint64_t cap = (uint64_t)sms * 8u;
    uint32_t per_block = (uint32_t)(((uint64_t)a.batch * a.layers + cap - 1u) / cap);
    per_block = per_block < a.layers ? (per_block ? per_block : 1u) : a.layers;
    const uint64_t items = (uint64_t)a.batch * ((a.layers + per_block - 1u) / per_block);
    const uint32_t blocks = (uint32_t)(items < cap ? items : cap), rounds = (kept_width + 7u) / 8u;
    const auto kernel = rounds <= 1u ? page_keep_kernel<1> : rounds <= 2u ? page_keep_kernel<2> : rounds <= 4u ? page_keep_kernel<4> : page_keep_kernel<8>;
    return (int)launch(kernel, 1u, blocks, kKeepThreads, 0u, stream, p, base, kept, kept_width, per_block);
}

uint64_t page_workspace_bytes(uint32_t batch, uint32_t width) { return page_ws_bytes(batch, width); }

int page_status(const void *workspace, cudaStream_t stream)
{
    if (workspace == nullptr) return SHAREDKV_EINVAL;
    uint32_t status = 0;
    cudaError_t e = cudaMemcpyAsync(&status, workspace, sizeof(status), cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    if (e != cudaSuccess) return (int)e;
    return status == kStatusOk ? SHAREDKV_OK : SHAREDKV_ERANGE;
}

}  // namespace sharedkv
