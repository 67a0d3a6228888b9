// The kept rows of drafted trees moved together in the caches of a model's
// layers (include/leafhip.h: lh_kv8_compact).
//
// Kept row k of a request moves from place path[k] >= k of its new rows to
// place k.  A workgroup takes a request's KV head of one layer, and the blocks
// that receive rows one after the other: it gathers a block's rows in LDS, then
// writes them.  What a block gives to a later one does not exist (rows only move
// forward), so a block can be written before the next is read.
#include "kv8.h"

namespace leafhip {
namespace {

constexpr int kThreads = 256;

// A code under the scale `old`, under `scale`, both powers of two for E4M3.
template <bool E4M3>
__device__ __forceinline__ uint8_t moved_code(uint8_t code, float old, float scale) {
    if (old == scale || !finite_f32(scale)) return code;
    if (E4M3) return (uint8_t)e4m3_pair(__builtin_amdgcn_cvt_f32_fp8(code, 0) * (old / scale), 0.0f);
    return (uint8_t)(int)__builtin_rint((double)(int8_t)code * (double)old / (double)scale);
}

template <bool E4M3>
__global__ __launch_bounds__(kThreads) void kv8_compact_kernel(Kv8CompactCall p) {
    extern __shared__ __align__(16) uint8_t codes[];   // [tokens of a block][dim]
    __shared__ int source[128];                        // of each token: where it comes from, in tokens of the pool; -1: nowhere
    __shared__ float scale_of[128];                    // and its block's scale there
    __shared__ float largest;
    const KvBatchView& b = p.batch;
    const int request = blockIdx.y, kvh = blockIdx.x, kv_heads = p.kv_heads, dim = p.dim, block = b.block, shift = b.block_shift;
    const Kv8Request q = kv8_request(b, request);
    const int kept = p.kept[request];
    if (q.rows <= 0 || kept <= 0 || kept > q.rows) return;
    const int* path = p.path + q.start;
    const int* table = b.table + (size_t)request * b.width;
    const Kv8Layer& layer = p.layers[blockIdx.z];
    // the path ascends within the rows; the first row that moves
    int first = kept;
    bool wrong = false;
    for (int k = threadIdx.x; k < kept; k += kThreads) {
        const int at = path[k];
        wrong = wrong || at < 0 || at >= q.rows || (k && at <= path[k - 1]);
        if (at != k) first = min(first, k);
    }
    if (__syncthreads_or(wrong)) return;
    __shared__ int firsts[kThreads / 64];
    for (int o = 32; o > 0; o >>= 1) first = min(first, __shfl_xor(first, o, 64));
    if ((threadIdx.x & 63) == 0) firsts[threadIdx.x >> 6] = first;
    __syncthreads();
    for (int w = 0; w < kThreads / 64; ++w) first = min(first, firsts[w]);
    if (first == kept) return;
    const int before = q.length - q.rows;
    for (int entry = (before + first) >> shift; entry <= (before + kept - 1) >> shift; ++entry) {
        const int id = table[entry];
        if ((unsigned)id >= (unsigned)b.blocks) continue;
        const int start = entry << shift, from = max(before - start, 0), to = min(before + kept - start, block);
        for (int which = 0; which < 2; ++which) {
            float* const scales = which ? layer.value_scales : layer.key_scales;
            uint8_t* const all = which ? layer.values : layer.keys;
            float* const scale_at = scales + (size_t)id * kv_heads + kvh;
            uint8_t* const mine = all + ((size_t)id * kv_heads + kvh) * block * dim;
            const int token_stride = which ? 1 : dim, dim_stride = which ? block : 1;
            const float old = *scale_at;
            if (threadIdx.x < 128) {
                const int slot = threadIdx.x;
                int comes = -1;
                float scale = 0.0f;
                if (slot >= from && slot < to) {
                    const int position = before + path[start + slot - before], page = table[position >> shift];
                    if ((unsigned)page < (unsigned)b.blocks) {
                        comes = (page << shift) + (position & (block - 1));
                        scale = scales[(size_t)page * kv_heads + kvh];
                    }
                }
                source[slot] = comes;
                scale_of[slot] = scale;
            }
            __syncthreads();
            if (threadIdx.x < 64) {
                float most = from > 0 ? old : 0.0f;
                bool spoilt = !(most >= 0.0f && most < INFINITY);
                for (int slot = threadIdx.x; slot < block; slot += 64) {
                    const float scale = source[slot] >= 0 ? scale_of[slot] : 0.0f;
                    spoilt = spoilt || !(scale >= 0.0f && scale < INFINITY);
                    most = fmaxf(most, scale);
                }
                most = wave_max_f32(most);
                spoilt = __any(spoilt);
                if (threadIdx.x == 0) largest = spoilt ? NAN : most;
            }
            __syncthreads();
            const float scale = largest;
            // gather
            const int tokens = to - from;
            for (int i = threadIdx.x; i < tokens * dim; i += kThreads) {
                const int slot = from + (which ? i % tokens : i / dim), d = which ? i / tokens : i % dim;
                const int comes = source[slot];
                if (comes < 0) continue;
                const uint8_t* of = all + ((size_t)(comes >> shift) * kv_heads + kvh) * block * dim;
                const uint8_t code = of[(size_t)(comes & (block - 1)) * token_stride + d * dim_stride];
                codes[slot * dim + d] = moved_code<E4M3>(code, scale_of[slot], scale);
            }
            // the block's earlier tokens follow its scale
            if (from > 0 && scale > old)
                for (int i = threadIdx.x; i < from * dim; i += kThreads) {
                    const int slot = which ? i % from : i / dim, d = which ? i / from : i % dim;
                    uint8_t* at = mine + slot * token_stride + d * dim_stride;
                    *at = moved_code<E4M3>(*at, old, scale);
                }
            __syncthreads();
            for (int i = threadIdx.x; i < tokens * dim; i += kThreads) {
                const int slot = from + (which ? i % tokens : i / dim), d = which ? i / tokens : i % dim;
                if (source[slot] >= 0) mine[slot * token_stride + d * dim_stride] = codes[slot * dim + d];
            }
            if (threadIdx.x == 0) *scale_at = scale;
            __syncthreads();
        }
    }
}

}  // namespace

void launch_kv8_compact(const Kv8CompactCall& call, int layers, hipStream_t stream) {
    const dim3 grid(call.kv_heads, call.batch.requests, layers);
    const size_t lds = (size_t)call.batch.block * call.dim;
    if (call.e4m3) kv8_compact_kernel<true><<<grid, kThreads, lds, stream>>>(call);
    else kv8_compact_kernel<false><<<grid, kThreads, lds, stream>>>(call);
}

}  // namespace leafhip
