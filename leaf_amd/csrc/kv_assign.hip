// Block tables and slot maps of a step, from the requests' lengths
// (include/leafhip.h: lh_kv_assign).
//
// With held = ceil(cached / B) and, for the requests that fit, need =
// ceil((cached + fresh) / B) - held, everything follows from three prefix sums
// over the requests: rows (starts), blocks given back by ended requests, and
// blocks needed.  A request is taken in when its inclusive sum of needs is at
// most the free blocks; the u-th needed block is entry free - 1 - u of the
// stack with the returned blocks behind it.
//
// Every workgroup forms the sums for all requests (they fit its LDS) and
// writes a share of what they say, each output by the thread that finds its
// request by bisection: tokens, table entries and returned blocks are spread
// evenly however ragged the requests are.  A returned block is read from its
// owner's table row, not from the stack, so that no workgroup reads what
// another writes; what the caller may update in place (lengths, free_left) is
// written by the only workgroup, or by a second launch.
//
// What bounds it: the latency of a launch (5 us) and of some dependent loads and
// sums: 24 requests of one token take 6.5 us, 2000 9, 1000 of which 50 return some 6,250 blocks
// 13, 40 prompts of 15,600 tokens together 7.7 and 5 for the second launch.
#include <algorithm>

#include "kv8.h"

namespace leafhip {
namespace {

constexpr int kThreads = 1024;
constexpr int kPerThread = 4;                       // requests a thread sums: LH_KV_MAX_REQUESTS <= 4 * 1024
constexpr int kGroupTokens = 2048;                  // tokens that one workgroup writes; 15,600 take it 16.8 us, eight and the second launch 13.0
constexpr int kSmallRows = 4;

// Exclusive prefix sums over the workgroup of each thread's value, and their total.
template <typename T>
__device__ __forceinline__ T scan_block(T v, long long* scratch, T& total) {
    T* waves = (T*)scratch;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T below = __shfl_up(s, o, 64);
        if (lane >= o) s += below;
    }
    __syncthreads();
    if (lane == 63) waves[wave] = s;
    __syncthreads();
    T before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < kThreads / 64; ++w) {
        const T one = waves[w];
        if (w < wave) before += one;
        total += one;
    }
    return before + s - v;
}

// The last index in [0, n) whose value is at most `what` (values ascend, the first is 0).
__device__ __forceinline__ int find_last(const int* values, int n, int what) {
    int low = 0, high = n;
    while (high - low > 1) {
        const int mid = (low + high) / 2;
        if (values[mid] <= what) low = mid;
        else high = mid;
    }
    return low;
}

// DIRECT: the only workgroup, which writes the lengths and the free count too.
// FINAL: the second launch of several, which writes only those.
// SMALL: no request has more than kSmallRows new tokens, so it needs one block at most, and the thread that sums a
// request writes its tokens and its block too: no bisection, which is a dozen dependent reads (24 requests 6.5 us for 7.4).
template <bool DIRECT, bool FINAL, bool SMALL>
__global__ __launch_bounds__(kThreads) void kv_assign_kernel(KvBatchView b) {
    extern __shared__ int lds[];
    __shared__ long long waves[kThreads / 64];
    const int n = b.requests;
    int* starts = lds;                              // exclusive sums: rows,
    int* needed = lds + n;                          // blocks needed by requests that fit,
    int* given = lds + 2 * n;                       // blocks given back;
    int* cached = lds + 3 * n;                      // -1: not taken in
    const int count = min(max(*b.free_count, 0), b.blocks);
    const long long room = (long long)b.width << b.block_shift;

    int c[kPerThread], f[kPerThread], held[kPerThread];
    long long mine_rows = 0;
    int mine_given = 0;                             // (blocks: at most the table's entries, which an int counts)
    const int first = threadIdx.x * kPerThread;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int r = first + j;
        c[j] = r < n ? b.cached[r] : 0;
        f[j] = r < n ? b.fresh[r] : 0;
        held[j] = (int)((min(max((long long)c[j], 0LL), room) + b.block - 1) >> b.block_shift);
        mine_rows += max(f[j], 0);
        mine_given += f[j] < 0 ? held[j] : 0;
    }
    long long all_rows;
    int all_given, all_needed;
    long long at_row = scan_block(mine_rows, waves, all_rows);
    int at_given = scan_block(mine_given, waves, all_given);
    const int returned = min(all_given, b.blocks - count);
    const int free_blocks = count + returned;
    int need[kPerThread];
    int mine_needed = 0;
    long long row = at_row;
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const long long after = (long long)c[j] + max(f[j], 0);
        row += max(f[j], 0);
        const bool fits = f[j] >= 0 && c[j] >= 0 && after <= room && f[j] <= b.max_rows && row <= b.tokens;
        need[j] = fits ? (int)((after + b.block - 1) >> b.block_shift) - held[j] : -1;
        mine_needed += max(need[j], 0);
    }
    int at_needed = scan_block(mine_needed, waves, all_needed);
    const int first_row = (int)min(at_row, (long long)b.tokens), first_needed = at_needed;
    int takes_of = 0;                               // a bit for each of the thread's requests
    int used = 0;                                   // inclusive sum of the last request taken in
#pragma unroll
    for (int j = 0; j < kPerThread; ++j) {
        const int r = first + j;
        const int upto = at_needed + max(need[j], 0);
        const bool takes = need[j] >= 0 && (need[j] == 0 || upto <= free_blocks);
        if (takes && need[j] > 0) used = upto;
        takes_of |= takes << j;
        if (r < n) {
            const int start = (int)min(at_row, (long long)b.tokens);
            starts[r] = start;
            needed[r] = at_needed;
            given[r] = at_given;
            cached[r] = takes ? c[j] : -1;
            if (DIRECT || FINAL) {
                b.starts[r] = start;
                b.rows[r] = takes ? f[j] : 0;
                b.lengths[r] = f[j] < 0 ? 0 : c[j] + (takes ? f[j] : 0);
                if (r == n - 1) b.starts[n] = (int)min(at_row + max(f[j], 0), (long long)b.tokens);
            }
        }
        at_row += max(f[j], 0);
        at_needed = upto;
        at_given += f[j] < 0 ? held[j] : 0;
    }
    // the blocks that are used, over all threads
    {
        int m = used;
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) m = max(m, __shfl_xor(m, o, 64));
        __syncthreads();
        if ((threadIdx.x & 63) == 0) waves[threadIdx.x >> 6] = m;
        __syncthreads();
        for (int w = 0; w < kThreads / 64; ++w) m = max(m, (int)waves[w]);
        used = m;
    }
    if ((DIRECT || FINAL) && threadIdx.x == 0) *b.free_left = free_blocks - used;
    if (FINAL) return;

    // block g of those given back: its owner's table row, from the first
    auto returned_block = [&](int g) {
        const int r = find_last(given, n, g);
        return b.table[(size_t)r * b.width + (g - given[r])];
    };
    auto taken_block = [&](int u) {                 // the u-th block that the requests need
        const int entry = free_blocks - 1 - u;
        return entry < count ? b.free_blocks[entry] : returned_block(entry - count);
    };
    auto held_of = [&](int r) { return (cached[r] + b.block - 1) >> b.block_shift; };

    const long long thread = blockIdx.x * kThreads + threadIdx.x, threads = gridDim.x * kThreads;
    const int rows = (int)min(all_rows, (long long)b.tokens);
    if (SMALL) {
        int t = first_row, u = first_needed;
        // (the blocks of all four requests first, then what depends on them)
        int held_id[kPerThread], new_id[kPerThread];
#pragma unroll
        for (int j = 0; j < kPerThread; ++j) {
            const bool takes = takes_of >> j & 1;
            const int before = (c[j] - 1) >> b.block_shift;        // the block of its last token
            held_id[j] = takes && c[j] > 0 && f[j] > 0 ? b.table[(size_t)(first + j) * b.width + before] : -1;
            new_id[j] = takes && need[j] > 0 ? taken_block(u) : -1;
            u += max(need[j], 0);
        }
#pragma unroll
        for (int j = 0; j < kPerThread; ++j) {
            const bool takes = takes_of >> j & 1;
            if (takes && need[j] > 0) b.table[(size_t)(first + j) * b.width + held[j]] = new_id[j];
            for (int i = 0; i < f[j]; ++i, ++t) {
                if (t >= b.tokens) break;
                const int position = c[j] + i, id = position >> b.block_shift < held[j] ? held_id[j] : new_id[j];
                const bool known = takes && (unsigned)id < (unsigned)b.blocks;
                b.positions[t] = takes ? position : -1;
                b.slots[t] = known ? (id << b.block_shift) + (position & (b.block - 1)) : -1;
            }
        }
        for (int t = rows + threadIdx.x; t < b.tokens; t += kThreads) b.positions[t] = b.slots[t] = -1;
    } else {
        for (long long at = thread; at < b.tokens; at += threads) {
            const int t = (int)at;
            int position = -1, slot = -1;
            if (t < rows) {
                const int r = find_last(starts, n, t);
                if (cached[r] >= 0) {
                    position = cached[r] + (t - starts[r]);
                    const int entry = position >> b.block_shift, held = held_of(r);
                    const int id = entry < held ? b.table[(size_t)r * b.width + entry] : taken_block(needed[r] + entry - held);
                    if ((unsigned)id < (unsigned)b.blocks) slot = (id << b.block_shift) + (position & (b.block - 1));
                }
            }
            b.positions[t] = position;
            b.slots[t] = slot;
        }
        for (long long at = thread; at < used; at += threads) {
            const int u = (int)at;
            const int r = find_last(needed, n, u);
            b.table[(size_t)r * b.width + held_of(r) + (u - needed[r])] = taken_block(u);
        }
    }
    // returned blocks: a wave looks at 64 requests and copies the rows of those that have ended
    const int lane = threadIdx.x & 63;
    for (int base = (int)(thread >> 6) * 64; base < n; base += (int)threads) {
        const int r = base + lane, end = r + 1 < n ? given[r + 1] : all_given, blocks = r < n ? end - given[r] : 0;
        for (uint64_t ended = __ballot(blocks > 0); ended; ended &= ended - 1) {
            const int from = __builtin_ctzll(ended), first_block = given[base + from];
            const int here = min(__shfl(blocks, from, 64), returned - first_block);
            const int* row = b.table + (size_t)(base + from) * b.width;
#pragma unroll 4
            for (int j = lane; j < here; j += 64) b.free_blocks[count + first_block + j] = row[j];
        }
    }
}

}  // namespace

void launch_kv_assign(const KvBatchView& b, hipStream_t stream) {
    const size_t lds = (size_t)4 * b.requests * sizeof(int);
    if (b.tokens <= kGroupTokens) {
        if (b.max_rows <= kSmallRows) kv_assign_kernel<true, false, true><<<1, kThreads, lds, stream>>>(b);
        else kv_assign_kernel<true, false, false><<<1, kThreads, lds, stream>>>(b);
        return;
    }
    const int groups = std::min((b.tokens + kGroupTokens - 1) / kGroupTokens, 256);
    kv_assign_kernel<false, false, false><<<groups, kThreads, lds, stream>>>(b);
    kv_assign_kernel<false, true, false><<<1, kThreads, lds, stream>>>(b);
}

}  // namespace leafhip
