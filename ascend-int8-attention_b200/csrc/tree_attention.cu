// Attention of a tree of drafted tokens over the INT8 shared-KV cache, sm_100a.  The contract is in
// include/sharedkv_c_abi.h.
//
// What the tokens of a tree have in common is their keys: eight query rows of 8 heads read the same 512-byte
// key rows as their neighbours in the tree.  So the unit of work is a GROUP of up to 64 query rows of
// one request (eight OCTETS; an octet is eight consecutive heads of one token), and a 128-key tile is
// fetched once per group.  A launch is two to four kernels:
//
//   tree_encode_kernel   query rows -> two INT8 code planes per cache kind, in the layout of the shared-memory
//                        operand; one block describes the groups and cuts the launch's tiles into a range per SM
//   tree_union_kernel    (ratio 4) the top-k lists of a group's tokens -> one ascending list of rows with a
//                        count per token, through a bitmap, so that rows several tokens name are fetched once
//   tree_walk_kernel     one persistent block per SM: S = K.Q^T and O = K^T.P on the INT8 tensor cores
//   tree_merge_kernel    joins the partial results of groups that several SMs worked on  (not for narrow windows)
//
// Arithmetic of the walk.  f = q * scale, alpha = max|f| / 127, f ~ alpha (q_hi + q_lo / 254); one MMA
// of 128 keys x (64 hi rows + 64 lo rows) gives both planes, and the integers are joined exactly,
// S = 254 S_hi + S_lo < 2^31, before the one conversion to FP32.  x = log2(e) s - ref with a reference
// per row that stays at or above every logit so far; weights 2^x <= 1 become codes of 32638 steps, c = 256 c_hi + c_lo
// (15 bits, c_lo signed), so O = 256 O_hi + O_lo is again one exact integer per tile, summed over tiles in
// FP32 registers.  The codes are the upper bits of 2^23 * 2^x: the denominator sums all 23 bits, exactly per tile, and
// a number from 0 to 255 that changes from key to key and tile to tile is added before the lower eight are cut off.  So a
// code errs by less than a step, by none on average, and the errors of n keys add up to some 0.41 sqrt(n) steps; keys
// that each weigh less than a step are counted as often as their weight asks for.  (Rounded to nearest, and
// steps of 2^-12, they would all be lost: with one key 10 nats above 8192 others, 10 to 31 % of the output; so it is 0.2 to 0.3 %.)
// The reference moves only when some logit exceeds it: the exact row maximum, a reduction over the 128 lanes
// that hold the keys, is needed at those tiles alone.  It then stands three powers of two above the maximum
// (kHeadroom), one at an item's last tile, and one or two less from the next tile on if the row's weight in this tile is not
// spread over many keys.  So steps
// are 2^-14 of the largest weight where one key has most of it, as the decode attention's are, and 2^-12
// where many keys share it and hide their rounding.  Always one power: 212 us for a C128 batch that takes 176 (every second
// tile moves references), always three: 174.
// Logits are not rounded before the reference is taken off, the maximum is: half a step of FP32, which kHeadroom covers up to 2^20.
// Beyond, the unit of a row's integers is a power of two, so that its logits have no rounding either.
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <atomic>

#include "../../include/sharedkv_c_abi.h"
#include "ptx_sm100.cuh"
#include "sharedkv_internal.h"

namespace sharedkv {
namespace {

using namespace ptx;

// ------------------------------------------------------------------ geometry
constexpr uint32_t kTreePage = 32, kTreeDraft = 64;
constexpr uint32_t kOctet = 8, kGroupOctets = 8, kGroupRows = kOctet * kGroupOctets;
constexpr uint32_t kCodeRows = 2 * kGroupRows;               // hi plane, then lo plane
constexpr uint32_t kTile = 128;                              // keys of a tile
constexpr uint32_t kSeg = kTile * 128;                       // one 128-channel segment of a tile (or of the query codes): 16 KB
constexpr uint32_t kRing = 8;                                // segments in flight: two tiles
constexpr uint32_t kWalkThreads = 640;
constexpr uint32_t kEncodeThreads = 256, kUnionThreads = 1024, kMergeThreads = 256;
constexpr uint32_t kWarpAccumulate = 8, kWarpIssue = 16, kWarpProduce = 18, kProducers = 2;
// Registers: launched with 96 per thread; accumulate (two warps of every SM partition) grows to hold
// 128 running sums a thread, the others shrink.  (64 / 152 / 48: C128 batch 177 us against 174.)
constexpr uint32_t kRegsLaunch = 96, kRegsSoftmax = 72, kRegsAccumulate = 144, kRegsIssue = 48;
static_assert(2 * kRegsSoftmax + 2 * kRegsAccumulate + kRegsIssue <= 5 * kRegsLaunch, "register shares exceed the launch allocation");
constexpr float kWeightSteps = 32638.f, kFine = 256.f;       // weight 1 in codes (the largest is 127 * 256 + 127), and a code in fine steps
constexpr uint32_t kCodeBias = 0x4b008000u;                  // bits of 2^23 + 128 * 256
constexpr float kNoKey = -3.402823466e38f;                   // reference of a row that has met no key: the lowest finite value
constexpr float kHeadroom = 3.f;                             // powers of two from a new maximum to the reference
constexpr uint32_t kSpread = 21;                             // bits of an eighth in fine steps: the maximum, seen from the reference
constexpr float kWideUnit = 0x1p-11f;                        // joined integers stay below 2^31
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;
constexpr uint32_t kUnionRows = 1u << 18;                    // compressed rows a union bitmap covers at a time (32 KB)
constexpr uint32_t kTreeWaitMillions = 4000;                 // cycles, ~2 s: a wait that long is a failure
// Work split, in tiles: what a group costs besides its tiles, and the shortest piece worth a partial result.
constexpr uint32_t kGroupCost = 2, kMinPiece = 3;
constexpr uint32_t kWholeTiles = 3;                          // groups of a window layer that are never split
constexpr uint32_t kCutSlots = 2048;                         // group slots whose starts the cuts search in shared memory

// shared memory of the walk (dynamic, 1024-byte aligned, all of the 227 KB)
constexpr uint32_t kSmKey = 0;
constexpr uint32_t kSmQuery = kSmKey + kRing * kSeg;         // 64 KB: four segments of 128 code rows
constexpr uint32_t kSmWeight = kSmQuery + 4 * kSeg;          // two tiles of weight codes, 128 keys x 128 bytes
constexpr uint32_t kSmAlpha = kSmWeight + 2 * kSeg;          // FP32 [2 kinds][64]
constexpr uint32_t kSmRef = kSmAlpha + 512;                  // FP32 [64], negated
constexpr uint32_t kSmTop = kSmRef + 256;                    // INT32 [2][64] row maxima of even and odd tiles, as ordered integers
constexpr uint32_t kSmFactor = kSmTop + 512;                 // FP32 [2][64] rescale factors of a tile
constexpr uint32_t kSmSum = kSmFactor + 512;                 // FP32 [3 warps][64] shares of the denominators, then [64] their inverses
constexpr uint32_t kSmSpread = kSmSum + 256;                 // between tiles of an item, in place of a share: UINT8 [64 rows][4 warps]
constexpr uint32_t kSmPath = kSmSum + 768;               // UINT64 [8] paths, UINT64 [8] compressed paths, INT32 [8] path lengths
constexpr uint32_t kSmFlags = kSmPath + 160;                 // rescale [2 tiles][2 halves], vote [2 halves][3], page masks [4], tmem base, abort
constexpr uint32_t kSmBars = kSmFlags + 64;
constexpr uint32_t kBarKeyFull = 0, kBarKeyEmpty = 8 /* per two segments */, kBarQueryFull = 12, kBarQueryEmpty = 13, kBarScoreFull = 14,
                   kBarScoreFree = 16, kBarWeightReady = 18, kBarOutFull = 20, kBarOutFree = 22, kBarSync = 24, kBarDone = 26,
                   kBarDoneFree = 27, kTreeBars = 28;
constexpr uint32_t kWalkSmem = kSmBars + 8 * kTreeBars;
static_assert(kWalkSmem <= 232448, "dynamic shared memory limit of sm_100");
static_assert(kSmPath % 8 == 0 && kSmBars % 8 == 0, "64-bit words");
constexpr uint32_t kFlagRescale = 0, kFlagVote = 4, kFlagPages = 10, kFlagTmem = 14, kFlagAbort = 15;
constexpr uint32_t kTmemAll = 512, kColScore = 0, kColOut = 256;      // two score tiles, two 128-channel blocks of O

struct Group {
    int32_t request, first_octet, octets, prefix, drafted, ori_tiles, cmp_rows, tiles;
};
static_assert(sizeof(Group) == 32, "a descriptor is two 16-byte loads");

// ------------------------------------------------------------------ workspace
// 256 bytes head (word 0 sticky status, word 1 arrivals of the union's blocks, words 2 and 3 the live tokens
// and the tokens in front of the first request), cut points,
// group descriptors and starts, query codes and alphas, union lists (ratio 4), partial results.
// A launch writes all it reads, the arrivals included: it works on whatever bytes it finds.  Only the status outlives a
// launch; it is a failure where it holds kTreeTimedOut, and nothing else.
constexpr uint32_t kTreeTimedOut = 0x7472ee01u;
struct TreeSpace {
    uint64_t cuts, groups, starts, codes, alphas, rows, counts, partials, bytes;
    uint32_t octets, slots, kinds;
    uint32_t listed;               // list entries per octet: top-k rounded up to 16-byte loads
};
__host__ __device__ inline TreeSpace tree_space(uint32_t tokens, uint32_t heads, uint32_t batch, uint32_t ratio, uint32_t topk)
{
    TreeSpace s;
    s.octets = tokens * (heads / kOctet);
    s.slots = s.octets / kGroupOctets + batch + 1u;           // see slot_of
    s.kinds = ratio == 1u ? 1u : 2u;
    auto up = [](uint64_t v) { return (v + 255ull) & ~255ull; };
    s.cuts = 256;
    s.groups = up(s.cuts + 8ull * (split::kMaxCtas + 1u));
    s.starts = up(s.groups + 32ull * s.slots);
    s.codes = up(s.starts + 4ull * (s.slots + 1u));
    s.alphas = up(s.codes + 8192ull * s.kinds * s.octets);
    s.rows = up(s.alphas + 32ull * s.kinds * s.octets);
    s.listed = (topk + 3u) & ~3u;
    const uint64_t entries = ratio == 4u ? (uint64_t)s.octets * s.listed : 0ull;
    s.counts = up(s.rows + 4ull * entries);
    s.partials = up(s.counts + 16ull * entries);
    s.bytes = s.partials + 2ull * split::kMaxCtas * (kGroupRows * (kDim + 2ull)) * 4ull;
    return s;
}
constexpr uint32_t kPartial = kGroupRows * (kDim + 2);        // FP32: output sums [64][512], denominators [64], references [64]

struct Tree {
    TreeAttentionArgs a;
    TreeSpace s;
    uint32_t grid;                 // blocks of the walk
    uint32_t splits;               // groups may be worked on by several blocks
    __device__ __forceinline__ char *at(uint64_t offset) const { return reinterpret_cast<char *>(a.workspace) + offset; }
    __device__ __forceinline__ const int32_t *cu() const { return reinterpret_cast<const int32_t *>(a.cuQ); }
    __device__ __forceinline__ const int32_t *seq() const { return reinterpret_cast<const int32_t *>(a.seqLens); }
    __device__ __forceinline__ Group *groups() const { return reinterpret_cast<Group *>(at(s.groups)); }
    __device__ __forceinline__ uint32_t *head() const { return reinterpret_cast<uint32_t *>(a.workspace); }
};

// Two FP32 values to a register pair, for the packed FMA and add.
__device__ __forceinline__ uint64_t pack2(float a, float b)
{
    uint64_t v;
    asm("mov.b64 %0, {%1, %2};" : "=l"(v) : "f"(a), "f"(b));
    return v;
}
__device__ __forceinline__ float low2(uint64_t v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float high2(uint64_t v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c)
{
    uint64_t v;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(v) : "l"(a), "l"(b), "l"(c));
    return v;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b)
{
    uint64_t v;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t v;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(v) : "l"(a), "l"(b));
    return v;
}

// Descriptor slot of the j-th group of request b.  floor(x + y) + 1 >= floor(x) + ceil(y), so requests
// do not run into each other and the slots are in request order; the ones between stay empty.
__device__ __forceinline__ uint32_t slot_of(uint32_t octets_before, uint32_t request, uint32_t j) { return octets_before / kGroupOctets + request + j; }

// Live requests (trailing ones without rows or with a negative cumulative count are padding).
__device__ uint32_t live_requests(const Tree &p, uint32_t *shared)
{
    if (threadIdx.x == 0) *shared = 0;
    __syncthreads();
    uint32_t live = 0;
    for (uint32_t b = threadIdx.x; b < p.a.batch; b += blockDim.x) if (split::request_is_live(p.seq()[b], p.cu()[b + 1])) live = b + 1;
    live = __reduce_max_sync(0xffffffffu, live);
    if (live && (threadIdx.x & 31u) == 0) atomicMax(shared, live);
    __syncthreads();
    return *shared;
}

// Rows of the union of a request's windows start at a page: the committed rows a path without a bit sees.
__device__ __forceinline__ int32_t window_page(int32_t prefix, uint32_t window)
{
    return prefix > (int32_t)window ? (prefix - (int32_t)window) / (int32_t)kTreePage : 0;
}

// ------------------------------------------------------------------ work split
// Runs in one block of the kernel in front of the walk.  The tiles of all groups, each group with
// kGroupCost units in front, are cut into p.grid ranges of equal cost; a cut that would leave a piece of fewer than
// kMinPiece tiles (a quarter of a range where that is less: with little work, tiles run side by side) moves to the group's edge.  Cut i is (slot, tile): block i walks from cut i to cut i + 1.
__device__ void cut_tiles(const Tree &p)
{
    __shared__ uint32_t sums[34], near[kCutSlots];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, warps = blockDim.x / 32u;
    uint32_t *starts = p.s.slots < kCutSlots ? near : reinterpret_cast<uint32_t *>(p.at(p.s.starts));
    const uint32_t per = (p.s.slots + blockDim.x - 1u) / blockDim.x;
    const uint32_t begin = min(threadIdx.x * per, p.s.slots), end = min(begin + per, p.s.slots);
    auto cost = [&](uint32_t slot) {
        const uint32_t tiles = (uint32_t)__ldcg(&p.groups()[slot].tiles);
        return tiles ? tiles + kGroupCost : 0u;
    };
    uint32_t sum = 0;
    uint32_t stop = 0;                                        // behind the last group: padding has slots too
    for (uint32_t i = begin; i < end; ++i) {
        const uint32_t c = cost(i);
        starts[i] = c;                                        // until the start takes its place
        sum += c;
        if (c) stop = i + 1u;
    }
    if (threadIdx.x == 0) sums[33] = 0;
    uint32_t incl = sum;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const uint32_t n = __shfl_up_sync(0xffffffffu, incl, d);
        if (lane >= (uint32_t)d) incl += n;
    }
    if (lane == 31) sums[warp] = incl;
    __syncthreads();
    if (warp == 0) {
        const uint32_t s = lane < warps ? sums[lane] : 0u;
        uint32_t si = s;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const uint32_t n = __shfl_up_sync(0xffffffffu, si, d);
            if (lane >= (uint32_t)d) si += n;
        }
        sums[lane] = si - s;
        if (lane == 31) sums[32] = si;
    }
    __syncthreads();
    uint32_t before = sums[warp] + incl - sum;
    for (uint32_t i = begin; i < end; ++i) {
        const uint32_t c = starts[i];
        starts[i] = before;
        before += c;
    }
    if (stop) atomicMax(sums + 33, stop);
    const uint32_t total = sums[32];
    if (threadIdx.x == 0) starts[p.s.slots] = total;
    __syncthreads();
    const uint32_t quota = total ? (total + p.grid - 1u) / p.grid : 1u;
    const uint32_t shortest = p.splits ? max(1u, min(quota / 4u, kMinPiece)) : 0x40000000u;
    uint2 *cuts = reinterpret_cast<uint2 *>(p.at(p.s.cuts));
    for (uint32_t i = threadIdx.x; i <= p.grid; i += blockDim.x) {
        const uint32_t position = i * quota;
        if (i == p.grid || position >= total) { cuts[i] = make_uint2(sums[33], 0); continue; }
        uint32_t lo = 0, hi = p.s.slots - 1u;                 // last slot that starts at or before the position
        while (lo < hi) {
            const uint32_t mid = (lo + hi + 1u) >> 1;
            if (starts[mid] <= position) lo = mid; else hi = mid - 1u;
        }
        const uint32_t inside = position - starts[lo], tiles = starts[lo + 1u] - starts[lo] - kGroupCost;
        const uint32_t tile = inside > kGroupCost ? inside - kGroupCost : 0u;
        cuts[i] = tile < shortest ? make_uint2(lo, 0) : tiles - tile < shortest ? make_uint2(lo + 1u, 0) : make_uint2(lo, tile);
    }
}

// One arrival per block; true in the block that arrives last, which sees what the others wrote.
__device__ bool last_block(const Tree &p, uint32_t blocks)
{
    __shared__ uint32_t mine;
    __syncthreads();
    if (threadIdx.x == 0) mine = atomic_add_acq_rel(p.head() + 1, 1u);
    __syncthreads();
    return mine + 1u == blocks;
}

// ------------------------------------------------------------------ encode
// A block takes octets in turn, a warp per head: lane l owns channels 16 l .. 16 l + 15, one 16-byte chunk of a code
// row.  Codes go out as the walk's B operand wants them: [kind][segment][plane][octet] blocks of 8 rows x
// 128 bytes, swizzled, so that a group's rows of a plane are one contiguous copy.  160 instructions a row and
// kind, packed FP32 where it can be, against 8 KB read and 8 KB per kind written an octet: 4096 octets of a
// ratio-128 layer take 22 us (4.5 TB/s, two thirds of the issue slots).
__device__ __forceinline__ void encode_row(const Tree &p, uint32_t kind, uint32_t octet, uint32_t row, const uint64_t (&q)[8], const float *sm_scale)
{
    const uint32_t lane = threadIdx.x & 31u;
    const ulonglong2 *scale = reinterpret_cast<const ulonglong2 *>(sm_scale + kind * kDim) + lane;      // [4][32 lanes]: no bank conflicts
    uint64_t f[8];
    float top = 0.f;                                          // largest |f|; a NaN stays one
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const ulonglong2 v = scale[i * 32];
        f[2 * i] = mul2(q[2 * i], v.x);
        f[2 * i + 1] = mul2(q[2 * i + 1], v.y);
    }
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(low2(f[i]))));
        asm("max.NaN.f32 %0, %0, %1;" : "+f"(top) : "f"(fabsf(high2(f[i]))));
    }
    const uint32_t bits = __reduce_max_sync(0xffffffffu, __float_as_uint(top));        // as integers a NaN is above all
    const float alpha = fmaxf(__uint_as_float(bits) * (float)(1.0 / 127), 1e-30f);
    float rcp = __frcp_rn(alpha), unit = alpha * p.a.softmaxScale * (kLog2e / 254.f);          // of the joined integers, as logits to base 2
    const bool finite = bits < 0x7f800000u && fabsf(unit) < INFINITY;
    if (fabsf(unit) > kWideUnit) {
        // logits may pass 2^20: a power of two as unit, up to twice as coarse, makes them exact
        const float wide = __uint_as_float(min((__float_as_uint(fabsf(unit)) + 0x7fffffu) & 0x7f800000u, 0x7f000000u));
        rcp *= fabsf(unit) / wide;
        unit = copysignf(wide, unit);
    }
    // adding 1.5 * 2^23 leaves the nearest integer in the low bits of the sum
    const uint64_t rcp2 = pack2(rcp, rcp), magic = pack2(12582912.f, 12582912.f), minus = pack2(-1.f, -1.f), low = pack2(254.f, 254.f);
    uint32_t hi[4], lo[4];
#pragma unroll
    for (int w = 0; w < 4; ++w) {
        uint32_t ch[4], cl[4];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            const uint64_t v = f[2 * w + e], h = fma2(v, rcp2, magic), l = fma2(fma2(v, rcp2, fma2(h, minus, magic)), low, magic);
            ch[2 * e] = (uint32_t)h; ch[2 * e + 1] = (uint32_t)(h >> 32);
            cl[2 * e] = (uint32_t)l; cl[2 * e + 1] = (uint32_t)(l >> 32);
        }
        hi[w] = __byte_perm(__byte_perm(ch[0], ch[1], 0x0040), __byte_perm(ch[2], ch[3], 0x0040), 0x5410);
        lo[w] = __byte_perm(__byte_perm(cl[0], cl[1], 0x0040), __byte_perm(cl[2], cl[3], 0x0040), 0x5410);
    }
    const uint64_t plane = 1024ull * p.s.octets, segment = kind * 4u + (lane >> 3);
    char *dst = p.at(p.s.codes) + segment * 2ull * plane + 1024ull * octet + row * 128u + (((lane & 7u) ^ row) << 4);
    *reinterpret_cast<uint4 *>(dst) = make_uint4(hi[0], hi[1], hi[2], hi[3]);
    *reinterpret_cast<uint4 *>(dst + plane) = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    if (lane == 0)
        reinterpret_cast<float *>(p.at(p.s.alphas))[(uint64_t)(kind * p.s.octets + octet) * kOctet + row] =
            finite ? unit : __uint_as_float(0x7fc00000u);
}

// Group descriptors of all slots, by one block; the head gets the number of live tokens, and no arrivals yet.
__device__ void describe_groups(const Tree &p)
{
    __shared__ uint32_t shared_live;
    const uint32_t per_token = p.a.heads / kOctet;
    const int32_t *cu = p.cu();
    const uint32_t live = live_requests(p, &shared_live);
    const uint32_t live_tokens = split::live_token_count(live ? cu[live] : 0, p.a.tokens);
    if (threadIdx.x == 0) { p.head()[1] = 0; p.head()[2] = live_tokens; p.head()[3] = live ? min((uint32_t)max(cu[0], 0), live_tokens) : 0u; }
    for (uint32_t i = threadIdx.x; i < p.s.slots; i += blockDim.x) {
        uint32_t lo = 0, hi = live ? live - 1u : 0u;
        while (lo < hi) {
            const uint32_t mid = (lo + hi + 1u) >> 1;
            if (slot_of((uint32_t)max(cu[mid], 0) * per_token, mid, 0) <= i) lo = mid; else hi = mid - 1u;
        }
        Group g = {};
        if (live) {
            const int32_t first = max(cu[lo], 0), n = min(cu[lo + 1], (int32_t)live_tokens) - first;
            const uint32_t base = slot_of((uint32_t)first * per_token, lo, 0), octets = n > 0 ? (uint32_t)n * per_token : 0u;
            if (i >= base && (i - base) * kGroupOctets < octets) {
                const uint32_t j = i - base;
                g.request = (int32_t)lo;
                g.first_octet = (int32_t)((uint32_t)first * per_token + j * kGroupOctets);
                g.octets = (int32_t)min(kGroupOctets, octets - j * kGroupOctets);
                g.prefix = p.seq()[lo] - (cu[lo + 1] - cu[lo]);
                g.drafted = min(n, (int32_t)kTreeDraft);
                const int64_t last = (int64_t)g.prefix + g.drafted, start = (int64_t)window_page(g.prefix, p.a.window) * kTreePage;
                // one tile at least, so that the rows of a group without a key are written
                g.ori_tiles = last > start ? (int32_t)((last - start + kTile - 1) / kTile) : 1;
                const int64_t table_rows = (int64_t)p.a.cmpTableWidth * kTreePage;
                int64_t rows = 0;
                if (p.a.ratio == 128u) rows = (int64_t)(max(g.prefix, 0) / 128) + (p.a.cmpPaths ? (int32_t)kTreeDraft : 0);
                g.cmp_rows = (int32_t)(rows < table_rows ? rows : table_rows);
                g.tiles = g.ori_tiles + (g.cmp_rows + (int32_t)kTile - 1) / (int32_t)kTile;
            }
        }
        p.groups()[i] = g;
    }
    __syncthreads();
}

// Block 0 plans the walk, the others encode: what is live matters to the plan alone, so the codes of
// padding rows are computed too (and never read).
__global__ void __launch_bounds__(kEncodeThreads) tree_encode_kernel(const __grid_constant__ Tree p)
{
    __shared__ __align__(16) float sm_scale[2 * kDim];        // channel 16 l + 4 i + e of a kind at 128 i + 4 l + e
    grid_dependency_launch_dependents();
    grid_dependency_wait();
    if (blockIdx.x == 0) {
        describe_groups(p);
        if (p.a.ratio != 4u) cut_tiles(p);                    // on ratio-4 layers the tiles are known once the lists are joined
        return;
    }
    const uint32_t lane = threadIdx.x & 31u, row = threadIdx.x >> 5, blocks = gridDim.x - 1u;
    auto fetch = [&](uint32_t octet, uint4 (&raw)[2]) {
        const uint4 *src = reinterpret_cast<const uint4 *>(p.a.q + ((uint64_t)octet * kOctet + row) * (kDim * 2u)) + lane * 2u;
        raw[0] = src[0];
        raw[1] = src[1];
    };
    uint32_t octet = blockIdx.x - 1u;
    uint4 raw[2];
    fetch(octet, raw);
    for (uint32_t i = threadIdx.x; i < p.s.kinds * kDim; i += kEncodeThreads) {
        const uint32_t c = i % kDim;
        sm_scale[i / kDim * kDim + (c >> 2 & 3u) * 128u + (c >> 4) * 4u + (c & 3u)] = __ldg(reinterpret_cast<const float *>(i < kDim ? p.a.oriScale : p.a.cmpScale) + c);
    }
    __syncthreads();
    for (; octet < p.s.octets; octet += blocks) {
        uint64_t q[8];
        const uint32_t *words = reinterpret_cast<const uint32_t *>(raw);
#pragma unroll
        for (int i = 0; i < 8; ++i) q[i] = pack2(__uint_as_float(words[i] << 16), __uint_as_float(words[i] & 0xffff0000u));
        if (octet + blocks < p.s.octets) fetch(octet + blocks, raw);       // the next octet's rows are on their way
#pragma unroll 1
        for (uint32_t kind = 0; kind < p.s.kinds; ++kind) encode_row(p, kind, octet, row, q, sm_scale);
    }
}

// ------------------------------------------------------------------ union of top-k lists
// One block per group.  Rows are ranked by the bits before theirs in a bitmap, so the list ascends whatever
// order the atomics ran in.  An entry carries its location (page * 32 + row in page, -1 when the page
// is missing) and, per octet, how often the octet's token names it.  A chain of some twelve dependent steps between
// barriers, so bound by latency: 64 groups of eight lists of 1024 take 13 us behind the encode kernel, 16 alone.
__global__ void __launch_bounds__(kUnionThreads, 1) tree_union_kernel(const __grid_constant__ Tree p)
{
    extern __shared__ uint32_t smem[];
    uint32_t *bitmap = smem, *base = bitmap + kUnionRows / 32u, *counts = base + kUnionRows / 32u;      // counts: UINT16 [entries][8]
    __shared__ uint32_t sums[33];
    grid_dependency_launch_dependents();
    grid_dependency_wait();
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, per_token = p.a.heads / kOctet;
    const Group g = p.groups()[blockIdx.x];
    if (g.octets) {
        const uint32_t first_token = (uint32_t)g.first_octet / per_token;
        const uint32_t tokens = ((uint32_t)(g.first_octet + g.octets) - 1u) / per_token - first_token + 1u;
        const uint32_t total = tokens * p.a.topk;             // at most 8 x 1024: eight entries a thread
        const int64_t table_rows = (int64_t)p.a.cmpTableWidth * kTreePage, named = (int64_t)(max(g.prefix, 0) / 4) + kTreeDraft;
        const uint32_t limit = (uint32_t)(named < table_rows ? named : table_rows);
        const int32_t *picks = reinterpret_cast<const int32_t *>(p.a.indices) + (uint64_t)first_token * p.a.topk;
        const int32_t *table = reinterpret_cast<const int32_t *>(p.a.cmpTable) + (uint64_t)g.request * p.a.cmpTableWidth;
        const uint64_t at = (uint64_t)g.first_octet * p.s.listed;
        int32_t *rows_out = reinterpret_cast<int32_t *>(p.at(p.s.rows)) + at;
        uint4 *counts_out = reinterpret_cast<uint4 *>(p.at(p.s.counts)) + at;
        uint32_t pick[8];
#pragma unroll
        for (uint32_t k = 0; k < 8; ++k) {
            const uint32_t i = threadIdx.x + k * kUnionThreads;
            const uint32_t v = i < total ? (uint32_t)picks[i] : 0xffffffffu;
            pick[k] = v < limit ? v : 0xffffffffu;
        }
        uint32_t listed = 0;
        for (uint32_t low = 0; low < limit; low += kUnionRows) {
            const uint32_t words = (min(limit - low, kUnionRows) + 31u) / 32u;
            for (uint32_t i = threadIdx.x; i < words; i += kUnionThreads) bitmap[i] = 0;
            __syncthreads();
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                const uint32_t r = pick[k] - low;
                if (pick[k] != 0xffffffffu && pick[k] >= low && r < kUnionRows) atomicOr(bitmap + r / 32u, 1u << (r & 31u));
            }
            __syncthreads();
            const uint32_t per = (words + kUnionThreads - 1u) / kUnionThreads;
            const uint32_t begin = min(threadIdx.x * per, words), end = min(begin + per, words);
            uint32_t sum = 0;
            for (uint32_t i = begin; i < end; ++i) sum += __popc(bitmap[i]);
            uint32_t incl = sum;
#pragma unroll
            for (int d = 1; d < 32; d <<= 1) {
                const uint32_t n = __shfl_up_sync(0xffffffffu, incl, d);
                if (lane >= (uint32_t)d) incl += n;
            }
            if (lane == 31) sums[warp] = incl;
            __syncthreads();
            if (warp == 0) {
                const uint32_t s = sums[lane];
                uint32_t si = s;
#pragma unroll
                for (int d = 1; d < 32; d <<= 1) {
                    const uint32_t n = __shfl_up_sync(0xffffffffu, si, d);
                    if (lane >= (uint32_t)d) si += n;
                }
                sums[lane] = si - s;
                if (lane == 31) sums[32] = si;
            }
            __syncthreads();
            uint32_t before = sums[warp] + incl - sum;
            const uint32_t found = sums[32];
            for (uint32_t i = begin; i < end; ++i) { base[i] = before; before += __popc(bitmap[i]); }
            for (uint32_t i = threadIdx.x; i < found * 4u; i += kUnionThreads) counts[i] = 0;
            __syncthreads();
#pragma unroll
            for (uint32_t k = 0; k < 8; ++k) {
                const uint32_t r = pick[k] - low;
                if (pick[k] == 0xffffffffu || pick[k] < low || r >= kUnionRows) continue;
                const uint32_t rank = base[r / 32u] + __popc(bitmap[r / 32u] & ((1u << (r & 31u)) - 1u));
                // every thread that names the row writes the same location
                const int32_t page = table[pick[k] / kTreePage];
                const bool there = (uint32_t)page < p.a.cmpPages;
                rows_out[listed + rank] = there ? (int32_t)((uint32_t)page * kTreePage + (pick[k] % kTreePage)) : -1;
                if (!there) continue;                         // a missing row counts for nobody
                const uint32_t token = first_token + (threadIdx.x + k * kUnionThreads) / p.a.topk;
                const int32_t o0 = max((int32_t)(token * per_token) - g.first_octet, 0);
                const int32_t o1 = min((int32_t)((token + 1u) * per_token) - g.first_octet, g.octets);
                for (int32_t o = o0; o < o1; ++o) atomicAdd(counts + rank * 4u + (uint32_t)o / 2u, (o & 1) ? 0x10000u : 1u);
            }
            __syncthreads();
            for (uint32_t i = threadIdx.x; i < found; i += kUnionThreads) counts_out[listed + i] = reinterpret_cast<const uint4 *>(counts)[i];
            listed += found;
            __syncthreads();
        }
        if (threadIdx.x == 0) {
            p.groups()[blockIdx.x].cmp_rows = (int32_t)listed;
            p.groups()[blockIdx.x].tiles = g.ori_tiles + (int32_t)((listed + kTile - 1u) / kTile);
        }
    }
    if (last_block(p, gridDim.x)) cut_tiles(p);
}

// ------------------------------------------------------------------ walk: common to the roles
struct WalkShared {
    uint32_t base;
    char *ptr;
    __device__ __forceinline__ uint32_t bar(uint32_t i) const { return base + kSmBars + 8u * i; }
    __device__ __forceinline__ volatile uint32_t *flags() const { return reinterpret_cast<volatile uint32_t *>(ptr + kSmFlags); }
    __device__ __forceinline__ float *floats(uint32_t offset) const { return reinterpret_cast<float *>(ptr + offset); }
};

// A bounded wait: false once a wait of the block has run out.  One copy of the polling loop per ROLE, because
// warps with different register allocations cannot share a function.
template <int ROLE>
__device__ __noinline__ bool walk_wait_slow(uint32_t bar, uint32_t parity, volatile uint32_t *flags)
{
    const long long start = clock64();
#pragma unroll 1
    for (uint32_t spin = 1;; ++spin) {
        if (mbar_try_wait(bar, parity)) return true;
        if ((spin & 63u) == 0) {
            if (flags[kFlagAbort]) return false;
            if (clock64() - start > (long long)kTreeWaitMillions * 1000000ll) { flags[kFlagAbort] = 1; return false; }
        }
    }
}
template <int ROLE>
__device__ __forceinline__ bool walk_wait(const WalkShared &sm, uint32_t bar_index, uint32_t parity)
{
    const uint32_t bar = sm.bar(bar_index);
    if (mbar_try_wait(bar, parity)) return true;
    return walk_wait_slow<ROLE>(bar, parity, sm.flags());
}

// The block's items in order: groups, the first and last possibly in part.  AHEAD: the next descriptor is read
// while the current item is worked on (eight registers that not every role has).
template <bool AHEAD>
struct Items {
    uint32_t slot, last_slot, last_tile, begin, end;
    Group g, next;
    __device__ __forceinline__ void step(const Tree &p)
    {
        ++slot;
        if (AHEAD) {
            g = next;
            next = load(p, slot + 1u);
        } else {
            g = load(p, slot);
        }
    }
    __device__ __forceinline__ Group load(const Tree &p, uint32_t at) const
    {
        Group v = {};
        if (at < p.s.slots) {
            const int4 *src = reinterpret_cast<const int4 *>(p.groups() + at);
            const int4 a = __ldcg(src), b = __ldcg(src + 1);
            v.request = a.x; v.first_octet = a.y; v.octets = a.z; v.prefix = a.w;
            v.drafted = b.x; v.ori_tiles = b.y; v.cmp_rows = b.z; v.tiles = b.w;
        }
        return v;
    }
    __device__ __forceinline__ bool open(const Tree &p, uint32_t from)
    {
        for (;; from = 0) {
            end = slot == last_slot ? last_tile : (uint32_t)g.tiles;
            begin = from;
            if (slot >= p.s.slots || slot > last_slot) return false;
            if (begin < end) return true;
            step(p);
        }
    }
    __device__ __forceinline__ bool first(const Tree &p)
    {
        const uint2 *cuts = reinterpret_cast<const uint2 *>(p.at(p.s.cuts)) + blockIdx.x;
        const uint2 a = __ldcg(cuts), b = __ldcg(cuts + 1);
        slot = a.x; last_slot = b.x; last_tile = b.y;
        g = load(p, slot);
        if (AHEAD) next = load(p, slot + 1u);
        return open(p, a.y);
    }
    __device__ __forceinline__ bool advance(const Tree &p)
    {
        step(p);
        return open(p, 0u);
    }
    __device__ __forceinline__ bool whole() const { return begin == 0 && end == (uint32_t)g.tiles; }
    // Partial results: a block has at most one piece that another block continues and one that continues
    // another's, hence two places per block.
    __device__ __forceinline__ uint32_t partial() const { return 2u * blockIdx.x + (begin == 0 ? 1u : 0u); }
};

// ------------------------------------------------------------------ walk: producers
// Two warps take the segments of the tiles in turn: 128 channels of 128 keys, 16 KB.  Pages come as
// whole boxes of 32 rows x 128 bytes; the listed rows of a ratio-4 layer by gathers of four rows, or
// row by row when the page stride is no multiple of a row.  Lanes look up pages and rows; boxes and gathers go
// out from one elected lane with operands that are the same in the whole warp (with two warps 51 cycles a box
// and 22 a gather, 78 and 33 when lanes issue their own).
template <bool LISTED>
__device__ void produce(const Tree &p, const WalkShared &sm, uint32_t mine, const CUtensorMap *ori_map, const CUtensorMap *cmp_map,
                        const CUtensorMap *row_map, bool gather)
{
    const uint32_t lane = threadIdx.x & 31u;
    const bool leader = elect_one();
    Items<true> it = {};
    uint32_t tile = 0;                                        // tiles of the block so far: this warp takes segments mine and mine + 2
    // Looks up tile j: lane l four rows of the list, or for l < 4 the tile's l-th page.
    int4 raw;
    auto look = [&](uint32_t j) {
        raw = make_int4(-1, -1, -1, -1);
        if (LISTED && j >= (uint32_t)it.g.ori_tiles) {
            const uint32_t row = (j - (uint32_t)it.g.ori_tiles) * kTile + 4u * lane;
            if (row < (uint32_t)it.g.cmp_rows)
                raw = __ldcg(reinterpret_cast<const int4 *>(p.at(p.s.rows) + 4ull * ((uint64_t)it.g.first_octet * p.s.listed + row)));
        } else {
            const bool ori = j < (uint32_t)it.g.ori_tiles;
            const int32_t *table = reinterpret_cast<const int32_t *>(ori ? p.a.oriTable : p.a.cmpTable);
            const uint32_t width = ori ? p.a.oriTableWidth : p.a.cmpTableWidth;
            const uint32_t index = (ori ? (uint32_t)window_page(it.g.prefix, p.a.window) + j * 4u : (j - (uint32_t)it.g.ori_tiles) * 4u) + lane;
            if (lane < 4 && index < width) raw.x = table[(uint64_t)it.g.request * width + index];
        }
    };
    for (bool more = it.first(p); more; more = it.advance(p)) {
        look(it.begin);
        for (uint32_t j = it.begin; j < it.end; ++j, ++tile) {
            const bool ori = j < (uint32_t)it.g.ori_tiles;
            // what the tile before has looked up for this one
            int32_t at[4] = {raw.x, raw.y, raw.z, raw.w};
            if (j + 1u < it.end) look(j + 1u);
            uint32_t there = 0, bytes;
            if (LISTED && !ori) {
                const uint32_t row = (j - (uint32_t)it.g.ori_tiles) * kTile + 4u * lane;
                uint32_t found = 0;
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (row + i >= (uint32_t)it.g.cmp_rows) at[i] = -1;
                    found += at[i] >= 0;
                }
                bytes = gather ? kSeg : 128u * __reduce_add_sync(0xffffffffu, found);
                if (gather) {
                    const uint32_t per_page = (uint32_t)(p.a.cmpStride / kDim);
#pragma unroll
                    for (int i = 0; i < 4; ++i)               // a missing row reads as zeros from beyond the map
                        at[i] = at[i] < 0 ? 0x7ffffff0 : (int32_t)((uint32_t)at[i] / kTreePage * per_page + (uint32_t)at[i] % kTreePage);
                }
            } else {
                there = __ballot_sync(0xffffffffu, (uint32_t)at[0] < (ori ? p.a.oriPages : p.a.cmpPages)) & 15u;
                bytes = 4096u * __popc(there);
            }
#pragma unroll 1
            for (uint32_t seg = mine; seg < 4u; seg += kProducers) {
                const uint32_t slot = (4u * tile + seg) % kRing;
                if (!walk_wait<2>(sm, kBarKeyEmpty + slot / 2u, ((tile >> 1) & 1u) ^ 1u)) return;
                __syncwarp();
                const uint32_t full = sm.bar(kBarKeyFull + slot), dst = sm.base + kSmKey + slot * kSeg;
                if (leader) {
                    if (seg == 0) sm.flags()[kFlagPages + (tile & 3u)] = there;
                    mbar_arrive_expect_tx(full, bytes);
                }
                if (LISTED && !ori) {
                    if (gather) {
#pragma unroll 8
                        for (uint32_t g = 0; g < 32u; ++g) {
                            const int32_t r0 = __shfl_sync(0xffffffffu, at[0], g), r1 = __shfl_sync(0xffffffffu, at[1], g);
                            const int32_t r2 = __shfl_sync(0xffffffffu, at[2], g), r3 = __shfl_sync(0xffffffffu, at[3], g);
                            if (leader) tma_gather4(dst + g * 512u, row_map, (int32_t)(seg * 128u), r0, r1, r2, r3, full);
                        }
                    } else {
                        __syncwarp();                         // the bytes are announced before any lane asks for some
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (at[i] >= 0)
                                tma_page_rows(dst + lane * 512u + i * 128u, row_map, (int32_t)(seg * 128u), at[i] % (int32_t)kTreePage,
                                              at[i] / (int32_t)kTreePage, full);
                    }
                } else {
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i) {
                        const int32_t page = __shfl_sync(0xffffffffu, at[0], i);
                        if (leader && ((there >> i) & 1u)) tma_page_rows(dst + i * 4096u, ori ? ori_map : cmp_map, (int32_t)(seg * 128u), 0, page, full);
                    }
                }
                __syncwarp();
            }
        }
    }
}

// ------------------------------------------------------------------ walk: issue
// Two warps issue one product each (an elected lane; the warp stays converged): a warp's serial work
// between two products, waits and commits, takes as long as the products, and would hold up the other kind.  What
// loops and addresses depend on is broadcast, so that the compiler sees one value for the warp and keeps
// the operand descriptors in uniform registers.
__device__ __forceinline__ uint32_t same(uint32_t v) { return __shfl_sync(0xffffffffu, v, 0); }

// S[128 keys, 128 code rows] = K . Q^T.  The query codes of an item's kind are one resident set of 64 KB; they
// are replaced once the last product that reads them has completed.
__device__ void issue_scores(const Tree &p, const WalkShared &sm, uint32_t tmem)
{
    constexpr uint32_t kScore = idesc_i8(128, kCodeRows, 0, 0);
    const bool leader = elect_one();
    const uint64_t keys = smem_desc(sm.base + kSmKey, 16u, 1024u, kSwizzle128), query = smem_desc(sm.base + kSmQuery, 16u, 1024u, kSwizzle128);
    Items<false> it;
    uint32_t t = 0, sets = 0;
    for (bool more = same(it.first(p)); more; more = same(it.advance(p))) {
        const uint32_t begin = same(it.begin), end = same(it.end), ori_tiles = same((uint32_t)it.g.ori_tiles);
        const uint32_t bytes = 1024u * same((uint32_t)it.g.octets), first_octet = same((uint32_t)it.g.first_octet);
        for (uint32_t j = begin; j < end; ++j, ++t) {
            if (j == begin || j == ori_tiles) {
                if (sets && !walk_wait<3>(sm, kBarQueryEmpty, (sets - 1u) & 1u)) return;
                if (leader) {
                    mbar_arrive_expect_tx(sm.bar(kBarQueryFull), 8u * bytes);
                    const uint64_t plane = 1024ull * p.s.octets;
                    const char *src = p.at(p.s.codes) + (j < ori_tiles ? 0ull : 8ull * plane) + 1024ull * first_octet;
#pragma unroll 1
                    for (uint32_t i = 0; i < 8; ++i)
                        bulk_load(sm.base + kSmQuery + (i >> 1) * kSeg + (i & 1u) * (kSeg / 2u), src + i * plane, bytes, sm.bar(kBarQueryFull));
                }
                __syncwarp();
                if (!walk_wait<3>(sm, kBarQueryFull, sets & 1u)) return;
                ++sets;
            }
            const uint32_t buf = t & 1u, ph = (t >> 1) & 1u;
            if (!walk_wait<3>(sm, kBarScoreFree + buf, ph ^ 1u)) return;
            tc_fence_after();
            const uint64_t a0 = keys + buf * ((4u * kSeg) >> 4);
            const uint32_t d = tmem + kColScore + buf * kCodeRows;
#pragma unroll
            for (uint32_t seg = 0; seg < 4; ++seg) {
                if (!walk_wait<3>(sm, kBarKeyFull + buf * 4u + seg, ph)) return;
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k)
                    if (leader) mma_i8(d, a0 + ((seg * kSeg + k * 32u) >> 4), query + ((seg * kSeg + k * 32u) >> 4), kScore, seg | k);
            }
            if (leader) {
                mma_commit(sm.bar(kBarScoreFull + buf));
                if (j + 1u == end || j + 1u == ori_tiles) mma_commit(sm.bar(kBarQueryEmpty));
            }
        }
    }
}

// O[128 channels, 128 code rows] = K^T . P for each of the four channel blocks, two blocks in tensor memory.
__device__ void issue_outputs(const Tree &p, const WalkShared &sm, uint32_t tmem)
{
    constexpr uint32_t kOut = idesc_i8(128, kCodeRows, 1, 1);
    const bool leader = elect_one();
    const uint64_t keys = smem_desc(sm.base + kSmKey, kSeg, 1024u, kSwizzle128), weights = smem_desc(sm.base + kSmWeight, kSeg, 1024u, kSwizzle128);
    Items<true> it;
    uint32_t tiles = 0;                                       // only their number matters here
    for (bool more = it.first(p); more; more = it.advance(p)) tiles += it.end - it.begin;
    tiles = same(tiles);
    for (uint32_t t = 0; t < tiles; ++t) {
        const uint32_t buf = t & 1u, ph = (t >> 1) & 1u;
        if (!walk_wait<3>(sm, kBarWeightReady + buf, ph)) return;
        const uint64_t a0 = keys + buf * ((4u * kSeg) >> 4), b0 = weights + buf * (kSeg >> 4);
#pragma unroll
        for (uint32_t block = 0; block < 4; ++block) {
            // use 2 t + (block >> 1) of this half of the output columns
            if (!walk_wait<3>(sm, kBarOutFree + (block & 1u), ((block >> 1) & 1u) ^ 1u)) return;
            tc_fence_after();
#pragma unroll
            for (uint32_t k = 0; k < 4; ++k)
                if (leader) mma_i8(tmem + kColOut + (block & 1u) * kCodeRows, a0 + ((block * kSeg + k * 4096u) >> 4), b0 + ((k * 4096u) >> 4), kOut, k);
            if (leader) {
                mma_commit(sm.bar(kBarOutFull + (block & 1u)));
                // the last reader of two segments, and with the second two of the weights
                if (block & 1u) mma_commit(sm.bar(kBarKeyEmpty + 2u * buf + (block >> 1)));
            }
        }
    }
}

// ------------------------------------------------------------------ walk: softmax (warps 0-7)
// Two halves of four warps; thread (half, key) has the key's logits of rows 32 half .. 32 half + 31, four
// octets, which it takes one after the other straight from tensor memory into weight codes.  That some
// logit lies above its reference shows in passing; then the octets concerned get new references (exact
// maxima) and are done again.  Maxima and sums over keys are warp reductions of integers, whose result
// does not depend on their order.
__device__ __forceinline__ bool softmax_sync(const WalkShared &sm, uint32_t half, uint32_t &phase)
{
    mbar_arrive(sm.bar(kBarSync + half));
    const bool ok = walk_wait<0>(sm, kBarSync + half, phase);
    phase ^= 1u;
    return ok;
}
__device__ __forceinline__ float exp2_approx(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Integers in the order of the floats they come from (and back).
__device__ __forceinline__ int32_t ordered(int32_t bits) { return bits ^ ((bits >> 31) & 0x7fffffff); }

template <bool LISTED>
__device__ void softmax(const Tree &p, const WalkShared &sm, uint32_t tmem)
{
    constexpr uint32_t kOctets = kGroupOctets / 2, kRows = kGroupRows / 2;         // of a half
    const uint32_t half = threadIdx.x >> 7, key = threadIdx.x & 127u, lane = key & 31u, warp = key >> 5;
    const uint32_t score = tmem + ((warp * 32u) << 16) + kColScore + half * kRows;
    volatile uint32_t *flags = sm.flags();
    float *ref = sm.floats(kSmRef) + half * kRows, *sums = sm.floats(kSmSum) + half * kRows;
    int32_t *top = reinterpret_cast<int32_t *>(sm.ptr + kSmTop) + half * kRows;
    const uint32_t per_token = p.a.heads / kOctet;
    uint32_t phase = 0, t = 0, vote = kFlagVote + half * 3u;
    Items<false> it;
    uint32_t items = 0;
    for (bool more = it.first(p); more; more = it.advance(p), ++items) {
        const uint32_t row0 = half * kRows;                   // first row of the half in the group
        const bool mine = key < kRows && row0 + key < (uint32_t)it.g.octets * kOctet;          // this thread looks after row `key` of the half
        float row_sum = 0.f;                                  // this warp's share of the denominator of row `lane`
        {
            uint64_t *path = reinterpret_cast<uint64_t *>(sm.ptr + kSmPath);
            float *alpha = sm.floats(kSmAlpha) + row0;
            if (key < kRows) {
                const uint64_t row = (uint64_t)it.g.first_octet * kOctet + row0 + key;
                const float *alphas = reinterpret_cast<const float *>(p.at(p.s.alphas));
                const float a = mine ? __ldcg(alphas + row) : 0.f;
                const float b = mine && p.s.kinds == 2u ? __ldcg(alphas + (uint64_t)p.s.octets * kOctet + row) : 0.f;
                // A query row that is not finite walks as zeros, so as not to make its octet's rows seek new
                // references at every tile; the NaN is in its denominator.
                const bool finite = a == a && b == b;
                alpha[key] = finite ? a : 0.f;
                alpha[kGroupRows + key] = finite ? b : 0.f;
                if (!finite) row_sum = __uint_as_float(0x7fc00000u);
                ref[key] = -kNoKey;
                top[key] = top[kGroupRows + key] = INT32_MIN;
            } else if (key < kRows + kOctets) {
                const uint32_t o = half * kOctets + key - kRows;
                uint64_t m = 0, c = 0;
                if (o < (uint32_t)it.g.octets) {
                    const uint32_t token = ((uint32_t)it.g.first_octet + o) / per_token;
                    m = reinterpret_cast<const uint64_t *>(p.a.paths)[token];
                    if (it.g.drafted < (int32_t)kTreeDraft) m &= (1ull << it.g.drafted) - 1ull;
                    if (p.a.cmpPaths) c = reinterpret_cast<const uint64_t *>(p.a.cmpPaths)[token];
                }
                path[o] = m;
                path[kGroupOctets + o] = c;
                reinterpret_cast<int32_t *>(path + 2 * kGroupOctets)[o] = __popcll(m);
            }
        }
        if (!softmax_sync(sm, half, phase)) return;
        float row_ref = kNoKey;                               // reference of row `lane`, the same in every warp of the half
        float later = 1.f;                                    // what the row's sums are multiplied by at the next tile
        const uint32_t present = (1u << max(min(it.g.octets - (int32_t)(half * kOctets), (int32_t)kOctets), 0)) - 1u;
        const int32_t whole_rows = max(it.g.prefix, 0) / 128;
        // how often the half's octets name this thread's row of listed tile j
        auto counts_of = [&](uint32_t j) {
            const uint32_t entry = (j - (uint32_t)it.g.ori_tiles) * kTile + key;
            if (entry >= (uint32_t)it.g.cmp_rows) return make_uint2(0, 0);
            return __ldcg(reinterpret_cast<const uint2 *>(p.at(p.s.counts)) + 2u * ((uint64_t)it.g.first_octet * p.s.listed + entry) + half);
        };
        uint2 ahead = make_uint2(0, 0);

        for (uint32_t j = it.begin; j < it.end; ++j, ++t) {
            const bool ori = j < (uint32_t)it.g.ori_tiles;
            const uint32_t buf = t & 1u, ph = (t >> 1) & 1u;
            // ---- which octets see this key, and on ratio-4 layers how often
            uint32_t sees = 0;
            uint2 count = make_uint2(0x00010001u, 0x00010001u);
            if (LISTED && !ori) {
                count = j == max(it.begin, (uint32_t)it.g.ori_tiles) ? counts_of(j) : ahead;
                if (j + 1u < it.end) ahead = counts_of(j + 1u);
                sees = (count.x & 0xffffu ? 1u : 0u) | (count.x >> 16 ? 2u : 0u) | (count.y & 0xffffu ? 4u : 0u) | (count.y >> 16 ? 8u : 0u);
            } else {
                // the page mask came with segment 0, which the scores have needed
                if (!walk_wait<0>(sm, kBarScoreFull + buf, ph)) return;
                const bool page = (flags[kFlagPages + (t & 3u)] >> warp) & 1u;
                const int32_t row = (int32_t)((ori ? j : j - (uint32_t)it.g.ori_tiles) * kTile + key);
                const uint64_t *path = reinterpret_cast<const uint64_t *>(sm.ptr + kSmPath) + half * kOctets;
                if (ori) {
                    const int32_t *length = reinterpret_cast<const int32_t *>(sm.ptr + kSmPath + 16u * kGroupOctets) + half * kOctets;
                    const int32_t drafted = window_page(it.g.prefix, p.a.window) * (int32_t)kTreePage + row - it.g.prefix;
#pragma unroll
                    for (uint32_t o = 0; o < kOctets; ++o) {
                        const bool seen = drafted < 0 ? drafted + (int32_t)p.a.window >= length[o]
                                                      : drafted < (int32_t)kTreeDraft && ((path[o] >> drafted) & 1ull);
                        sees |= seen ? 1u << o : 0u;
                    }
                } else if (row < whole_rows) {
                    sees = 0xfu;
                } else if (row - whole_rows < (int32_t)kTreeDraft) {
#pragma unroll
                    for (uint32_t o = 0; o < kOctets; ++o) sees |= (uint32_t)((path[kGroupOctets + o] >> (row - whole_rows)) & 1ull) << o;
                }
                sees = page ? sees & present : 0u;
            }

            if (LISTED && !walk_wait<0>(sm, kBarScoreFull + buf, ph)) return;
            // the weights of tile t - 2 have been read when its last two key segments have
            if (t >= 2u && !walk_wait<0>(sm, kBarKeyEmpty + 2u * buf + 1u, ph ^ 1u)) return;
            tc_fence_after();
            const float *alpha = sm.floats(kSmAlpha) + row0 + (ori ? 0u : kGroupRows);
            char *weights = sm.ptr + kSmWeight + buf * kSeg + key * 128u;
            const uint32_t columns = score + buf * kCodeRows;
            // What is added to the fine steps of this key's weights before they are cut off: over a warp's keys 32 values 8 apart,
            // in another order and with another offset in the next warp and tile.  `dithers` is their sum and the codes' bias.
            const uint32_t dither = (__brev(lane ^ j) >> 24) ^ (2u * warp + (j & 1u));
            const uint32_t dithers = 32u * (kCodeBias + (dither & 7u)) + 8u * 496u;
            // log2 of how often octet o counts this key: minus infinity where it does not see it
            auto bias_of = [&](uint32_t o) {
                float bias = (sees >> o) & 1u ? 0.f : -INFINITY;
                if (LISTED) {
                    const uint32_t n = ((o & 2u ? count.y : count.x) >> ((o & 1u) * 16u)) & 0xffffu;
                    if (n > 1u && bias == 0.f) bias = log2f((float)n);
                }
                return bias;
            };
            // One octet: integers joined exactly and converted once, log2 weights by packed FMAs, codes, their sums over
            // the warp, and the codes' bytes to shared memory.  True when some weight is above 1.
            uint32_t total = 0;
            auto codes = [&](uint32_t o, const uint32_t *hi, const uint32_t *lo) {
                const float bias = bias_of(o);
                const uint64_t bias2 = pack2(bias, bias), steps = pack2(kWeightSteps * kFine, kWeightSteps * kFine);
                const uint64_t magic = pack2(__uint_as_float(kCodeBias | dither), __uint_as_float(kCodeBias | dither));
                uint32_t pair[4], sum[8], seen_bits = 0;
#pragma unroll
                for (uint32_t q = 0; q < 4; q += 2) {
                    const ulonglong2 a = reinterpret_cast<const ulonglong2 *>(alpha)[o * 2u + q / 2u], m = reinterpret_cast<const ulonglong2 *>(ref)[o * 2u + q / 2u];
#pragma unroll
                    for (uint32_t e = 0; e < 2; ++e) {
                        const uint32_t r = 2u * (q + e);
                        const uint64_t x = fma2(pack2((float)((int32_t)hi[r] * 254 + (int32_t)lo[r]), (float)((int32_t)hi[r + 1] * 254 + (int32_t)lo[r + 1])),
                                                e ? a.y : a.x, add2(e ? m.y : m.x, bias2));
                        const uint64_t c = fma2(pack2(exp2_approx(low2(x)), exp2_approx(high2(x))), steps, magic);      // 2^23 + 256 (128 + code) + fraction + dither
                        const uint32_t d0 = (uint32_t)c, d1 = (uint32_t)(c >> 32);
                        seen_bits |= d0 | d1;
                        sum[r] = __reduce_add_sync(0xffffffffu, d0);
                        sum[r + 1] = __reduce_add_sync(0xffffffffu, d1);
                        pair[q + e] = __byte_perm(d0, d1, 0x6521);
                    }
                }
                const uint32_t chunk = half * 2u + (o >> 1), place = (o & 1u) * 8u;
                *reinterpret_cast<uint2 *>(weights + ((chunk ^ (key & 7u)) << 4) + place) =
                    make_uint2(__byte_perm(pair[0], pair[1], 0x7531), __byte_perm(pair[2], pair[3], 0x7531));
                *reinterpret_cast<uint2 *>(weights + (((4u + chunk) ^ (key & 7u)) << 4) + place) =
                    make_uint2(__byte_perm(pair[0], pair[1], 0x6420) ^ 0x80808080u, __byte_perm(pair[2], pair[3], 0x6420) ^ 0x80808080u);
                // lane 8 o + i keeps the sum of row i
                const uint32_t s01 = lane & 1u ? sum[1] : sum[0], s23 = lane & 1u ? sum[3] : sum[2], s45 = lane & 1u ? sum[5] : sum[4], s67 = lane & 1u ? sum[7] : sum[6];
                const uint32_t s03 = lane & 2u ? s23 : s01, s47 = lane & 2u ? s67 : s45, s = lane & 4u ? s47 : s03;
                if ((lane >> 3) == o) total = s;
                // a weight above 1 leaves the 15 bits of a code
                return (seen_bits & ~(0x4b000000u | 0x7fffffu)) != 0;
            };
            // Row maxima of octet pair o over this warp's keys, as integers in float order, into `top` (a buffer for even
            // and one for odd tiles, since a fast warp meets the next tile's maxima while a slow one reads).
            auto maxima = [&](uint32_t o, uint32_t above) {
                uint32_t hi[16], lo[16];
                tmem_ld16(columns + o * 8u, hi);
                tmem_ld16(columns + kGroupRows + o * 8u, lo);
                const float bias[2] = {bias_of(o), bias_of(o + 1u)};
                tmem_wait_ld();
                int32_t high = INT32_MIN;
#pragma unroll
                for (uint32_t i = 0; i < 16; ++i) {
                    const float x = fmaf((float)((int32_t)hi[i] * 254 + (int32_t)lo[i]), alpha[o * 8u + i], bias[i >> 3]);
                    const int32_t v = __reduce_max_sync(0xffffffffu, ordered(__float_as_int(x)));
                    if (lane == o * 8u + i) high = v;
                }
                // rows of an octet that no warp has flagged keep their reference: nothing else of theirs is redone
                if (lane >> 4 == o >> 1 && ((above >> (lane >> 3)) & 1u)) atomicMax(top + buf * kGroupRows + lane, high);
            };
            // Round 0 takes the references as they are (an item's first tile has none and skips it), round 1 redoes the
            // octets that got new ones.  The code exists once: the warps of this kernel share an instruction cache
            // that does not hold two copies.
            uint32_t todo = j == it.begin ? 0u : 0xfu, above = ~todo & 0xfu;
            bool moved = false;
#pragma unroll 1
            for (uint32_t round = 0;; ++round) {
#pragma unroll 1
                for (uint32_t o = 0; o < kOctets; o += 2) {   // two octets at a time, for loads and arithmetic to overlap
                    if (!((todo >> o) & 3u)) continue;        // a neighbour that did not move comes out as it was
                    uint32_t hi[16], lo[16];
                    tmem_ld16(columns + o * 8u, hi);
                    tmem_ld16(columns + kGroupRows + o * 8u, lo);
                    tmem_wait_ld();
                    const bool first = codes(o, hi, lo), second = codes(o + 1u, hi + 8, lo + 8);
                    above |= (first ? 1u << o : 0u) | (second ? 2u << o : 0u);
                }
                if (round) break;
                above = __reduce_or_sync(0xffffffffu, above);
                if (above) {                                  // only a warp that has such a weight can hold a new maximum
                    if (lane == 0) atomicOr(const_cast<uint32_t *>(flags) + vote, above);
#pragma unroll 1
                    for (uint32_t o = 0; o < kOctets; o += 2) if ((above >> o) & 3u) maxima(o, above);
                }
                if (!softmax_sync(sm, half, phase)) return;
                todo = flags[vote];
                const uint32_t zero = kFlagVote + half * 3u, low = __ballot_sync(0xffffffffu, later != 1.f);
                vote = vote == zero + 2u ? zero : vote + 1u;
                // the word after next was last read before the barrier just passed, and is set behind the next one
                if (key == 0) {
                    flags[vote == zero + 2u ? zero : vote + 1u] = 0;
                    flags[kFlagRescale + buf * 2u + half] = todo | (low & 0xffu ? 1u : 0u) | (low & 0xff00u ? 2u : 0u) | (low & 0xff0000u ? 4u : 0u) | (low >> 24 ? 8u : 0u);
                }
                if (!(todo | low)) break;
                float factor = later;
                later = 1.f;
                if (!todo) {
                    if (warp == 0) sm.floats(kSmFactor)[buf * kGroupRows + row0 + lane] = factor;
                    break;
                }
                // Every warp works out the new references by itself, from the maxima and the old ones in its
                // registers, and writes the same values; of the octets that are done again only.  Maxima left from
                // earlier tiles do not lie above the reference they have led to and move nothing; nor does a NaN.
                const float highest = __int_as_float(ordered(top[buf * kGroupRows + lane]));
                // the margin covers the rounding of the maximum, and no more: a row does not move because another one does
                if (((todo >> (lane >> 3)) & 1u) && highest > row_ref - fabsf(highest) * 0x1p-23f) {
                    const float next = highest + (j + 1u < it.end ? kHeadroom : 1.f), down = exp2_approx(row_ref - next);
                    row_ref = next;
                    ref[lane] = -next;
                    factor *= down;
                    row_sum *= down;
                    moved = true;
                }
                if (warp == 0) sm.floats(kSmFactor)[buf * kGroupRows + row0 + lane] = factor;
                __syncwarp();
            }
            tc_fence_before();
            mbar_arrive(sm.bar(kBarScoreFree + buf));
            fence_proxy_async_smem();
            mbar_arrive(sm.bar(kBarWeightReady + buf));
            row_sum = fmaf((float)(total - dithers), 1.f / kFine, row_sum);
            // Where a new maximum leaves little weight for others, the reference may be close to it from the next tile on:
            // where the second heaviest of the tile's four runs of 32 keys weighs less than the maximum.  (With twice and half the
            // maximum the C4 batch takes 79 and 78 us against 77.5, and errors are the same to 1e-4 up to half.)  Not for the sake
            // of one last tile (44.3 against 44.8 us on the window batch).
            if (todo && j + 2u < it.end) {
                uint8_t *spread = reinterpret_cast<uint8_t *>(sm.ptr + kSmSpread) + (row0 + lane) * 4u;
                spread[warp] = (uint8_t)(32 - __clz((int32_t)(total - dithers)));
                if (!softmax_sync(sm, half, phase)) return;
                const uint32_t bits = *reinterpret_cast<const uint32_t *>(spread);
                const uint32_t b0 = bits & 255u, b1 = (bits >> 8) & 255u, b2 = (bits >> 16) & 255u, b3 = bits >> 24;
                const uint32_t second = max(max(min(b0, b1), min(b2, b3)), min(max(b0, b1), max(b2, b3)));
                if (moved && second < kSpread) {
                    const float next = row_ref - (float)min(kSpread - second, 2u);
                    later = exp2_approx(row_ref - next);
                    row_ref = next;
                    row_sum *= later;
                    ref[lane] = -next;
                }
                __syncwarp();
            }
        }

        // ---- denominators: warp 0 looks after the rows and adds the other warps' shares in warp order
        if (!walk_wait<0>(sm, kBarDoneFree, (items & 1u) ^ 1u)) return;       // the last item's inverses have been read
        if (warp) sums[(warp - 1u) * kGroupRows + lane] = row_sum;
        if (!softmax_sync(sm, half, phase)) return;
        if (mine) {
            const uint64_t row = (uint64_t)it.g.first_octet * kOctet + row0 + key;
            const float m = row_ref;
            // logits beyond FP32 give NaN
            const float l = m == INFINITY ? __uint_as_float(0x7fc00000u) : ((row_sum + sums[key]) + sums[kGroupRows + key]) + sums[2u * kGroupRows + key];
            if (it.whole()) {
                const float sink = __ldg(reinterpret_cast<const float *>(p.a.sinks) + row % p.a.heads);
                const float sink2 = sink * kLog2e, at = fmaxf(m, sink2), own = exp2_approx(m - at);
                const float all_sum = l * own + (sink == -INFINITY ? 0.f : kWeightSteps * exp2_approx(sink2 - at));
                sm.floats(kSmSum)[row0 + key] = all_sum == 0.f ? 0.f : own / all_sum;
                if (p.a.lse)
                    reinterpret_cast<float *>(p.a.lse)[row] = all_sum == 0.f ? -INFINITY : (at + log2f(all_sum * (1.f / kWeightSteps))) * kLn2;
            } else {
                float *partial = reinterpret_cast<float *>(p.at(p.s.partials)) + (uint64_t)it.partial() * kPartial + kGroupRows * kDim + row0;
                partial[key] = l;
                partial[kGroupRows + key] = m;
            }
        }
        mbar_arrive(sm.bar(kBarDone));
    }
}

// ------------------------------------------------------------------ walk: accumulate (warps 8-15)
// Thread = channel of each 128-channel block, rows 32 h .. 32 h + 31: 128 running sums in registers.  The
// integers of a block are read, joined, scaled and added while the tensor core fills the other block.
__device__ void accumulate(const Tree &p, const WalkShared &sm, uint32_t tmem)
{
    const uint32_t index = threadIdx.x - kWarpAccumulate * 32u, h = index >> 7, channel = index & 127u, warp = channel >> 5;
    const uint32_t tmem_lane = tmem + ((warp * 32u) << 16) + kColOut + h * 32u;
    {
        // rows of no live token are cleared
        const uint32_t live = __ldcg(p.head() + 2) * p.a.heads, skipped = __ldcg(p.head() + 3) * p.a.heads, rows = p.a.tokens * p.a.heads;
        for (uint32_t i = blockIdx.x; i < skipped + rows - live; i += gridDim.x) {
            const uint32_t row = i < skipped ? i : live + i - skipped;
            if (index < 64u) reinterpret_cast<uint4 *>(p.a.out)[(uint64_t)row * 64u + index] = make_uint4(0, 0, 0, 0);
            if (p.a.lse && index == 64u) reinterpret_cast<float *>(p.a.lse)[row] = 0.f;
        }
    }
    Items<false> it;
    uint32_t t = 0, items = 0;
    for (bool more = it.first(p); more; more = it.advance(p), ++items) {
        uint64_t acc[4][16];                                  // pairs of rows
#pragma unroll
        for (int block = 0; block < 4; ++block)
#pragma unroll
            for (int r = 0; r < 16; ++r) acc[block][r] = 0;
        for (uint32_t j = it.begin; j < it.end; ++j, ++t) {
            const uint32_t buf = t & 1u, ph = (t >> 1) & 1u;
            if (!walk_wait<1>(sm, kBarWeightReady + buf, ph)) return;
            const float *scale = reinterpret_cast<const float *>(j < (uint32_t)it.g.ori_tiles ? p.a.oriScale : p.a.cmpScale) + channel;
            const uint32_t moved = sm.flags()[kFlagRescale + buf * 2u + h];
            if (moved) {
                const ulonglong2 *factor = reinterpret_cast<const ulonglong2 *>(sm.ptr + kSmFactor) + buf * 16u + h * 8u;
#pragma unroll
                for (int o = 0; o < 4; ++o) {
                    if (!((moved >> o) & 1u)) continue;
#pragma unroll
                    for (int q = 2 * o; q < 2 * o + 2; ++q) {
                        const ulonglong2 f = factor[q];
#pragma unroll
                        for (int block = 0; block < 4; ++block) {
                            acc[block][2 * q] = mul2(acc[block][2 * q], f.x);
                            acc[block][2 * q + 1] = mul2(acc[block][2 * q + 1], f.y);
                        }
                    }
                }
            }
#pragma unroll
            for (uint32_t block = 0; block < 4; ++block) {
                const uint32_t half = block & 1u;
                if (!walk_wait<1>(sm, kBarOutFull + half, (block >> 1) & 1u)) return;
                const float f = __ldg(scale + block * 128u);
                const uint64_t f2 = pack2(f, f);
                tc_fence_after();
#pragma unroll
                for (uint32_t c = 0; c < 4; ++c) {
                    uint32_t hi[8], lo[8];
                    tmem_ld8(tmem_lane + half * kCodeRows + c * 8u, hi);
                    tmem_ld8(tmem_lane + half * kCodeRows + kGroupRows + c * 8u, lo);
                    tmem_wait_ld();
                    if (c == 3) {
                        tc_fence_before();
                        mbar_arrive(sm.bar(kBarOutFree + half));
                    }
#pragma unroll
                    for (uint32_t i = 0; i < 4; ++i)
                        acc[block][c * 4u + i] = fma2(pack2((float)((int32_t)hi[2 * i] * 256 + (int32_t)lo[2 * i]),
                                                            (float)((int32_t)hi[2 * i + 1] * 256 + (int32_t)lo[2 * i + 1])), f2, acc[block][c * 4u + i]);
                }
            }
        }
        if (!walk_wait<1>(sm, kBarDone, items & 1u)) return;
        const uint32_t rows = (uint32_t)it.g.octets * kOctet;
        auto value = [&](uint32_t block, uint32_t r) { return r & 1u ? high2(acc[block][r / 2u]) : low2(acc[block][r / 2u]); };
        if (it.whole()) {
            const float *inverse = sm.floats(kSmSum) + h * 32u;
            __nv_bfloat16 *out = reinterpret_cast<__nv_bfloat16 *>(p.a.out) + ((uint64_t)it.g.first_octet * kOctet + h * 32u) * kDim + channel;
#pragma unroll
            for (uint32_t r = 0; r < 32; ++r) {
                if (h * 32u + r < rows) {
                    const float f = inverse[r];
#pragma unroll
                    for (uint32_t block = 0; block < 4; ++block) out[r * kDim + block * 128u] = __float2bfloat16_rn(value(block, r) * f);
                }
            }
        } else {
            float *partial = reinterpret_cast<float *>(p.at(p.s.partials)) + (uint64_t)it.partial() * kPartial + h * 32u * kDim + channel;
#pragma unroll
            for (uint32_t r = 0; r < 32; ++r)
                if (h * 32u + r < rows)
#pragma unroll
                    for (uint32_t block = 0; block < 4; ++block) partial[r * kDim + block * 128u] = value(block, r);
        }
        mbar_arrive(sm.bar(kBarDoneFree));
    }
}

// 7528 tiles of a C128 batch (101 GFLOP) take 164 us on 148 SMs, 51 tiles a block: the tensor pipe is active for 41 % of
// it.  A tile without a new reference takes the softmax warps 4100 cycles (over half of them for the weights), which is what
// bounds the walk; the life of a tile, from its fetch into one of two places to its last product, takes
// nearly twice that.  Tiles are 128 keys because the INT8 MMA is full at M = 128, and groups 64 rows because N = 128
// balances its operand reads with its arithmetic (64 cycles; N = 64 takes 48) and 64 KB of codes are what fits beside two tiles.
template <bool LISTED>
__global__ void __launch_bounds__(kWalkThreads, 1) tree_walk_kernel(const __grid_constant__ Tree p, const __grid_constant__ CUtensorMap ori_map,
                                                                     const __grid_constant__ CUtensorMap cmp_map,
                                                                     const __grid_constant__ CUtensorMap row_map, const uint32_t gather)
{
    extern __shared__ __align__(1024) char smem_walk[];
    WalkShared sm;
    sm.base = smem_addr(smem_walk);
    sm.ptr = smem_walk;
    const uint32_t warp = threadIdx.x >> 5;
    volatile uint32_t *flags = sm.flags();
    if (threadIdx.x == 0) {
        for (uint32_t i = 0; i < kRing; ++i) mbar_init(sm.bar(kBarKeyFull + i), 1);
        for (uint32_t i = 0; i < kRing / 2u; ++i) mbar_init(sm.bar(kBarKeyEmpty + i), 1);
        mbar_init(sm.bar(kBarQueryFull), 1);
        mbar_init(sm.bar(kBarQueryEmpty), 1);
        for (uint32_t i = 0; i < 2; ++i) {
            mbar_init(sm.bar(kBarScoreFull + i), 1); mbar_init(sm.bar(kBarScoreFree + i), 256);
            mbar_init(sm.bar(kBarWeightReady + i), 256);
            mbar_init(sm.bar(kBarOutFull + i), 1); mbar_init(sm.bar(kBarOutFree + i), 256);
        }
        mbar_init(sm.bar(kBarSync), 128);
        mbar_init(sm.bar(kBarSync + 1), 128);
        mbar_init(sm.bar(kBarDone), 256);
        mbar_init(sm.bar(kBarDoneFree), 256);
        for (uint32_t i = 0; i < 16; ++i) if (i != kFlagTmem) flags[i] = 0;
        fence_mbar_init();
    }
    if (warp == kWarpIssue) {
        tmem_alloc(sm.base + kSmFlags + 4u * kFlagTmem, kTmemAll);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = flags[kFlagTmem];
    grid_dependency_launch_dependents();
    grid_dependency_wait();

    if (warp < kWarpAccumulate) {
        registers_release<kRegsSoftmax>();
        softmax<LISTED>(p, sm, tmem);
    } else if (warp < kWarpIssue) {
        registers_acquire<kRegsAccumulate>();
        accumulate(p, sm, tmem);
    } else {
        registers_release<kRegsIssue>();
        if (warp == kWarpIssue) issue_scores(p, sm, tmem);
        else if (warp == kWarpIssue + 1u) issue_outputs(p, sm, tmem);
        else produce<LISTED>(p, sm, warp - kWarpProduce, &ori_map, &cmp_map, &row_map, gather != 0);
        __syncwarp();
    }
    tc_fence_before();
    __syncthreads();
    if (flags[kFlagAbort]) {
        // A wait ran out: copies and products already issued may still land in this block's memory, so it
        // stays for far longer than they can take before it gives that memory up.
        if (threadIdx.x == 0) p.head()[0] = kTreeTimedOut;
        for (uint32_t i = 0; i < 200u; ++i) __nanosleep(1000u);
        __syncthreads();
    }
    if (warp == kWarpIssue) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemAll);
    }
}

// ------------------------------------------------------------------ merge
// 147 cuts on 148 SMs leave up to 147 groups of two pieces or more, 128 KB each: 9 to 10 us, the chain cut -> data ->
// output and two waves of blocks.  Block (i, o): octet o of the group that cut i is the first to fall into.  Pieces are joined in piece
// order: M = max of the references and the sink, out = sum O 2^(ref - M) / (sum l 2^(ref - M) + sink).
__global__ void __launch_bounds__(kMergeThreads) tree_merge_kernel(const __grid_constant__ Tree p)
{
    grid_dependency_launch_dependents();
    grid_dependency_wait();
    const uint2 *cuts = reinterpret_cast<const uint2 *>(p.at(p.s.cuts));
    const uint32_t i = blockIdx.x + 1u, octet = blockIdx.y;
    const uint2 before = __ldcg(cuts + i - 1u), cut = __ldcg(cuts + i), after = __ldcg(cuts + i + 1u);
    // nothing to join, or an earlier cut has the group
    if (cut.y == 0 || cut.x >= p.s.slots || (before.x == cut.x && before.y != 0)) return;
    const float *partials = reinterpret_cast<const float *>(p.at(p.s.partials));
    const uint32_t row = octet * kOctet + (threadIdx.x >> 5), lane = threadIdx.x & 31u;
    auto piece = [&](uint32_t q) { return partials + (uint64_t)(q == 0 ? 2u * (i - 1u) + 1u : 2u * (i - 1u + q)) * kPartial; };
    // The first two pieces, which most groups have no more of, are requested before the group is known: where
    // they lie depends on the cut alone (rows the group does not have are read in vain).
    constexpr uint32_t kSums = kGroupRows * kDim, kRefs = kSums + kGroupRows;
    float4 v[2][4];
    float refs[2], sums[2];
#pragma unroll
    for (uint32_t q = 0; q < 2; ++q) {
        refs[q] = __ldcg(piece(q) + kRefs + row);
        sums[q] = __ldcg(piece(q) + kSums + row);
#pragma unroll
        for (int k = 0; k < 4; ++k) v[q][k] = __ldcg(reinterpret_cast<const float4 *>(piece(q) + row * kDim) + k * 32 + lane);
    }
    const Group g = p.groups()[cut.x];
    if (octet >= (uint32_t)g.octets) return;
    uint32_t pieces = 2;
    for (uint2 next = after; i + pieces - 1u < p.grid && next.x == cut.x && next.y != 0; next = __ldcg(cuts + i + pieces - 1u)) ++pieces;
    const uint64_t global_row = (uint64_t)g.first_octet * kOctet + row;
    const float sink = __ldg(reinterpret_cast<const float *>(p.a.sinks) + global_row % p.a.heads), sink2 = sink * kLog2e;
    float at = fmaxf(sink2, fmaxf(refs[0], refs[1]));
#pragma unroll 4
    for (uint32_t q = 2; q < pieces; ++q) at = fmaxf(at, __ldcg(piece(q) + kRefs + row));
    float total = sink == -INFINITY ? 0.f : kWeightSteps * exp2_approx(sink2 - at);
    float acc[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) acc[k] = 0.f;
    auto join = [&](float ref, float sum, const float4 (&o)[4]) {
        const float f = exp2_approx(ref - at);
        total = fmaf(sum, f, total);
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            acc[4 * k] = fmaf(o[k].x, f, acc[4 * k]); acc[4 * k + 1] = fmaf(o[k].y, f, acc[4 * k + 1]);
            acc[4 * k + 2] = fmaf(o[k].z, f, acc[4 * k + 2]); acc[4 * k + 3] = fmaf(o[k].w, f, acc[4 * k + 3]);
        }
    };
    join(refs[0], sums[0], v[0]);
    join(refs[1], sums[1], v[1]);
#pragma unroll 2
    for (uint32_t q = 2; q < pieces; ++q) {
        const float *src = piece(q);
        float4 o[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) o[k] = __ldcg(reinterpret_cast<const float4 *>(src + row * kDim) + k * 32 + lane);
        join(__ldcg(src + kRefs + row), __ldcg(src + kSums + row), o);
    }
    const float inverse = total == 0.f ? 0.f : 1.f / total;
    __nv_bfloat162 *out = reinterpret_cast<__nv_bfloat162 *>(reinterpret_cast<__nv_bfloat16 *>(p.a.out) + global_row * kDim);
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        out[(k * 32 + lane) * 2] = __floats2bfloat162_rn(acc[4 * k] * inverse, acc[4 * k + 1] * inverse);
        out[(k * 32 + lane) * 2 + 1] = __floats2bfloat162_rn(acc[4 * k + 2] * inverse, acc[4 * k + 3] * inverse);
    }
    if (p.a.lse && lane == 0)
        reinterpret_cast<float *>(p.a.lse)[global_row] = total == 0.f ? -INFINITY : (at + log2f(total * (1.f / kWeightSteps))) * kLn2;
}

// ------------------------------------------------------------------ host
using TreeEncodeTiled = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *, const cuuint64_t *,
                                     const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave, CUtensorMapSwizzle,
                                     CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
TreeEncodeTiled tree_encode_tiled()
{
    static std::atomic<void *> cached{nullptr};
    void *fn = cached.load(std::memory_order_acquire);
    if (fn == nullptr) {
        cudaDriverEntryPointQueryResult status;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &status) != cudaSuccess ||
            status != cudaDriverEntryPointSuccess)
            return nullptr;
        cached.store(fn, std::memory_order_release);
    }
    return reinterpret_cast<TreeEncodeTiled>(fn);
}

// Pages as [pages, 32 rows, 512 bytes], boxes of `rows` rows x 128 bytes; or, with rows = 0, the whole pool as rows of
// 512 bytes for gathers (ids beyond it read as zeros).
bool tree_map(CUtensorMap *map, uint64_t base, uint64_t stride, uint32_t pages, uint32_t rows)
{
    const TreeEncodeTiled encode = tree_encode_tiled();
    if (encode == nullptr) return false;
    const cuuint32_t ones[3] = {1, 1, 1};
    if (rows == 0) {
        const cuuint64_t dims[2] = {kDim, 0x7ffffff0ull}, strides[1] = {kDim};
        const cuuint32_t box[2] = {128, 1};
        return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, reinterpret_cast<void *>(base), dims, strides, box, ones,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
    const cuuint64_t dims[3] = {kDim, kTreePage, pages}, strides[2] = {kDim, stride};
    const cuuint32_t box[3] = {128, rows, 1};
    return encode(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 3, reinterpret_cast<void *>(base), dims, strides, box, ones,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

template <class... Params, class... Args>
cudaError_t tree_launch(void (*kernel)(Params...), dim3 grid, uint32_t threads, uint32_t smem, cudaStream_t stream, const Args &...args)
{
    cudaLaunchConfig_t config = {};
    config.gridDim = grid;
    config.blockDim = dim3(threads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attribute[1];
    attribute[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attribute[0].val.programmaticStreamSerializationAllowed = 1;
    config.attrs = attribute;
    config.numAttrs = programmatic_launch_enabled() ? 1u : 0u;
    return cudaLaunchKernelEx(&config, kernel, args...);
}

// The opt-in to large dynamic shared memory, once per device and kernel.
template <class Kernel>
cudaError_t tree_opt_in(Kernel kernel, uint32_t smem, std::atomic<uint64_t> &configured)
{
    int device = 0;
    cudaError_t e = cudaGetDevice(&device);
    if (e != cudaSuccess) return e;
    const uint64_t bit = device >= 0 && device < kMaxDevices ? 1ull << device : 0ull;
    if (bit && (configured.load(std::memory_order_relaxed) & bit)) return cudaSuccess;
    e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)smem);
    if (e == cudaSuccess) configured.fetch_or(bit, std::memory_order_relaxed);
    return e;
}

constexpr uint32_t kUnionSmem = 2u * (kUnionRows / 32u) * 4u + 8192u * 16u;      // bitmap, ranks, counts of 8 x 1024 entries

int tree_launch_all(const TreeAttentionArgs &a, cudaStream_t stream, int sms)
{
    Tree p;
    p.a = a;
    p.s = tree_space(a.tokens, a.heads, a.batch, a.ratio, a.topk);
    p.grid = (uint32_t)sms < split::kMaxCtas ? (uint32_t)sms : split::kMaxCtas;
    // A window layer's groups of two or three tiles stay whole and need no merge kernel: 16.9 against 17.8 us for one
    // request of 8 tokens (whose two tiles could run side by side), 44.2 against 46.0 us for 48 of 1 to 63 with 16 heads,
    // 16.9 against 17.9 us for four requests and a window of 200 rows.
    const uint32_t window_tiles = (a.window + kTreeDraft + kTreePage - 2u) / kTile + 1u;
    p.splits = a.ratio != 1u || window_tiles > kWholeTiles;
    const bool listed = a.ratio == 4u;
    const bool gather = a.cmpStride % kDim == 0 && (uint64_t)a.cmpPages * (a.cmpStride / kDim) < 0x7ffffff0ull;
    CUtensorMap ori_map, cmp_map, row_map;
    if (!tree_map(&ori_map, a.ori, a.oriStride, a.oriPages, kTreePage) || !tree_map(&cmp_map, a.cmp, a.cmpStride, a.cmpPages, kTreePage) ||
        !tree_map(&row_map, a.cmp, a.cmpStride, a.cmpPages, listed && gather ? 0u : 1u))
        return SHAREDKV_EINVAL;
    static std::atomic<uint64_t> walk_pages{0}, walk_rows{0}, unions{0};
    const uint32_t encode_blocks = p.s.octets < 4u * (uint32_t)sms ? p.s.octets : 4u * (uint32_t)sms;      // four fill an SM
    cudaError_t e = tree_launch(tree_encode_kernel, dim3(encode_blocks + 1u), kEncodeThreads, 0u, stream, p);
    if (e == cudaSuccess && listed) {
        e = tree_opt_in(tree_union_kernel, kUnionSmem, unions);
        if (e == cudaSuccess) e = tree_launch(tree_union_kernel, dim3(p.s.slots), kUnionThreads, kUnionSmem, stream, p);
        if (e == cudaSuccess) e = tree_opt_in(tree_walk_kernel<true>, kWalkSmem, walk_rows);
        if (e == cudaSuccess) e = tree_launch(tree_walk_kernel<true>, dim3(p.grid), kWalkThreads, kWalkSmem, stream, p, ori_map, cmp_map, row_map, (uint32_t)gather);
    } else if (e == cudaSuccess) {
        e = tree_opt_in(tree_walk_kernel<false>, kWalkSmem, walk_pages);
        if (e == cudaSuccess) e = tree_launch(tree_walk_kernel<false>, dim3(p.grid), kWalkThreads, kWalkSmem, stream, p, ori_map, cmp_map, row_map, 0u);
    }
    if (e == cudaSuccess && p.splits && p.grid > 1u) e = tree_launch(tree_merge_kernel, dim3(p.grid - 1u, kGroupOctets), kMergeThreads, 0u, stream, p);
    return (int)e;
}

}  // namespace

uint64_t tree_workspace_bytes(uint32_t tokens, uint32_t heads, uint32_t batch, uint32_t ratio, uint32_t topk)
{
    return tree_space(tokens, heads, batch, ratio, topk).bytes;
}

int tree_status(const void *workspace, cudaStream_t stream)
{
    if (workspace == nullptr) return SHAREDKV_EINVAL;
    uint32_t status = 0;
    cudaError_t e = cudaMemcpyAsync(&status, workspace, sizeof(status), cudaMemcpyDeviceToHost, stream);
    if (e == cudaSuccess) e = cudaStreamSynchronize(stream);
    if (e != cudaSuccess) return (int)e;
    return status == kTreeTimedOut ? SHAREDKV_ETIMEDOUT : SHAREDKV_OK;
}

int tree_attention(const TreeAttentionArgs *args, cudaStream_t stream)
{
    if (args == nullptr) return SHAREDKV_EINVAL;
    TreeAttentionArgs a = *args;
    if (a.tokens == 0) return SHAREDKV_OK;
    if (a.ratio != 1u && a.ratio != 4u && a.ratio != 128u) return SHAREDKV_EINVAL;
    if (a.heads == 0 || a.heads % kOctet || a.heads > 128u || a.window == 0 || a.window > 65536u) return SHAREDKV_EINVAL;
    if (a.batch == 0) {                                       // every row is padding
        if (!a.out || a.out % 16u || a.lse % 4u) return SHAREDKV_EINVAL;
        const uint64_t rows = (uint64_t)a.tokens * a.heads;
        cudaError_t e = cudaMemsetAsync(reinterpret_cast<void *>(a.out), 0, rows * kDim * 2u, stream);
        if (e == cudaSuccess && a.lse) e = cudaMemsetAsync(reinterpret_cast<void *>(a.lse), 0, rows * 4u, stream);
        return (int)e;
    }
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
    const int sms = device_sm_count();
    if (sms <= 0) return (int)cudaErrorInvalidDevice;
    return tree_launch_all(a, stream, sms);
}

}  // namespace sharedkv
