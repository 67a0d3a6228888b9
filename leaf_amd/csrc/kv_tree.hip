// The plan of a step of drafted trees, and the end of one (include/leafhip.h:
// lh_kv_tree, lh_kv_keep).
//
// What bounds both is a launch: the plan of 24 trees of 8 rows takes 4.0 us and of
// 250 of 64 rows 4.1, the lengths and blocks of 16 or 64 requests 3.9 (6.3 where a wave
// copied one request's blocks after the other's).
#include <algorithm>

#include "kv8.h"

namespace leafhip {
namespace {

// Ancestors by doubling: a row's mask takes its parent's, then its parent's
// parent's parent's.. until no row has one left; a row's depth is the number of
// its ancestors.  A thread has a row, its masks stand in LDS.
constexpr int kMostWords = kTreeRows / 64;
__global__ __launch_bounds__(kTreeRows) void kv_tree_kernel(KvTreeCall p) {
    extern __shared__ uint64_t masks[];             // [rows][words]
    __shared__ int above[kTreeRows];
    const Kv8Request q = kv8_request(p.batch, blockIdx.x);
    const int i = threadIdx.x, words = p.words;
    int up = -1;
    uint64_t own[kMostWords];
    if (i < q.rows) {
        up = p.parents[q.start + i];
        if (up < 0 || up >= i) up = -1;
        above[i] = up;
#pragma unroll
        for (int w = 0; w < kMostWords; ++w) {
            own[w] = i >> 6 == w ? 1ull << (i & 63) : 0;
            if (w < words) masks[i * words + w] = own[w];
        }
    }
    while (__syncthreads_or(up >= 0)) {
        if (up >= 0) {
#pragma unroll
            for (int w = 0; w < kMostWords; ++w)
                if (w < words) own[w] |= masks[up * words + w];
            up = above[up];
        }
        __syncthreads();
        if (i < q.rows) {
            above[i] = up;
#pragma unroll
            for (int w = 0; w < kMostWords; ++w)
                if (w < words) masks[i * words + w] = own[w];
        }
    }
    if (i >= q.rows) return;
    int depth = -1;
#pragma unroll
    for (int w = 0; w < kMostWords; ++w) {
        if (w >= words) continue;
        depth += __popcll(own[w]);
        p.masks[(size_t)(q.start + i) * words + w] = own[w];
    }
    p.batch.positions[q.start + i] = q.length - q.rows + depth;
}

// lh_kv_keep: one workgroup sums the blocks that the requests give back.
constexpr int kKeepThreads = 1024;
constexpr int kPerThread = 4;                       // LH_KV_MAX_REQUESTS <= 4 * 1024
constexpr int kFewBlocks = 4;
__global__ __launch_bounds__(kKeepThreads) void kv_keep_kernel(KvKeepCall p) {
    const KvBatchView& b = p.batch;
    __shared__ int given[kKeepThreads * kPerThread], first[kKeepThreads * kPerThread];   // before each request; its first table entry
    __shared__ int waves[kKeepThreads / 64];
    const int n = b.requests, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int count = min(max(*b.free_count, 0), b.blocks);
    const long long room = (long long)b.width << b.block_shift;
    int gives[kPerThread], mine = 0;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int r = threadIdx.x * kPerThread + j;
        gives[j] = 0;
        if (r >= n) continue;
        const int length = b.lengths[r], rows = b.rows[r], kept = p.kept[r];
        const bool fits = rows > 0 && rows <= length && length <= room && kept >= 0 && kept <= rows;
        const int after = fits ? length - rows + kept : length;
        if (fits) {
            first[r] = (after + b.block - 1) >> b.block_shift;
            gives[j] = ((length + b.block - 1) >> b.block_shift) - first[r];
        }
        p.lengths[r] = after;
        mine += gives[j];
    }
    int s = mine;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int below = __shfl_up(s, o, 64);
        if (lane >= o) s += below;
    }
    if (lane == 63) waves[wave] = s;
    __syncthreads();
    int at = s - mine, all = 0;
    for (int w = 0; w < kKeepThreads / 64; ++w) {
        if (w < wave) at += waves[w];
        all += waves[w];
    }
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        given[threadIdx.x * kPerThread + j] = at;
        at += gives[j];
    }
    const int returned = min(all, b.blocks - count);
    if (threadIdx.x == 0) *b.free_left = count + returned;
    __syncthreads();
    // a wave looks at 64 requests: a lane copies its own's table entries where they are few, the wave those of the others
    for (int base = wave * 64; base < n; base += kKeepThreads) {
        const int r = base + lane, blocks = r >= n ? 0 : (r + 1 < kKeepThreads * kPerThread ? given[r + 1] : all) - given[r];
        const bool few = blocks <= kFewBlocks;
        if (few && blocks > 0) {
            const int* row = b.table + (size_t)r * b.width + first[r];
            int ids[kFewBlocks];
#pragma unroll
            for (int j = 0; j < kFewBlocks; ++j) ids[j] = row[min(j, blocks - 1)];
#pragma unroll
            for (int j = 0; j < kFewBlocks; ++j)
                if (j < blocks && given[r] + j < returned) b.free_blocks[count + given[r] + j] = ids[j];
        }
        for (uint64_t some = __ballot(!few); some; some &= some - 1) {
            const int from = __builtin_ctzll(some), to = given[base + from];
            const int here = min(__shfl(blocks, from, 64), returned - to);
            const int* row = b.table + (size_t)(base + from) * b.width + first[base + from];
            for (int j = lane; j < here; j += 64) b.free_blocks[count + to + j] = row[j];
        }
    }
}

}  // namespace

void launch_kv_tree(const KvTreeCall& call, hipStream_t stream) {
    const int threads = (call.batch.max_rows + 63) / 64 * 64;
    kv_tree_kernel<<<call.batch.requests, threads, (size_t)8 * call.words * threads, stream>>>(call);
}

void launch_kv_keep(const KvKeepCall& call, hipStream_t stream) { kv_keep_kernel<<<1, kKeepThreads, 0, stream>>>(call); }

}  // namespace leafhip
