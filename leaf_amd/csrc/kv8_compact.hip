// The kept rows of drafted trees moved together in the caches of a model's
// layers (include/leafhip.h: lh_kv8_compact).
//
// Kept row k of a request moves from place path[k] >= k of its new rows to
// place k.  A wave takes the keys or the values of a request's KV head in one
// layer, and in them the blocks that receive rows, one after the other.  Rows only
// move forward: what row k overwrites, no later row comes from.  So a wave can
// move rows in their order, some at a time, each loaded before any of them
// is stored, and needs neither a copy nor a barrier.
//
// What bounds it: six dependent loads (the request, its path, its table, scales,
// codes) behind the launch.  64 requests of 8 rows, 4 KV heads of 64 in 22 layers (INT8,
// 11,264 waves, of which the GPU holds some 7,200) take 13.7 us, 16 of 64 rows, 2 heads in 24
// layers (E4M3) 7.1.  With a workgroup for a request's KV head, its rows through LDS and barriers:
// 21 and 10.4; with a wave for keys and values together 13.0 and 8.4.
#include "kv8.h"

namespace leafhip {
namespace {

constexpr int kWaves = 4;
constexpr int kTogether = 16;                       // values of a dim that a lane moves at a time

// Codes under the scale `old`, under `scale`, both powers of two for E4M3; `inverse` is about 1 / scale.
template <bool E4M3>
__device__ __forceinline__ uint32_t moved_code(uint32_t code, float old, float scale, double inverse) {
    if (E4M3) return e4m3_pair(__builtin_amdgcn_cvt_f32_fp8(code & 0xFFu, 0) * (old / scale), 0.0f) & 0xFFu;
    // the nearest whole number, ties to even, as in nearest_i8: x and the rest are exact
    const double x = (double)(int8_t)code * (double)old;
    double q = __builtin_rint(x * inverse);
    const double rest = fma(-q, (double)scale, x), twice = 2.0 * __builtin_fabs(rest);
    if (twice > (double)scale || (twice == (double)scale && ((int)q & 1))) q += __builtin_copysign(1.0, rest);
    return (uint32_t)(int)q & 0xFFu;
}
template <bool E4M3>
__device__ __forceinline__ uint32_t moved_word(uint32_t word, float old, float scale, double inverse) {
    uint32_t out = 0;
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
        out = out >> 8 | moved_code<E4M3>(word, old, scale, inverse) << 24;
        word >>= 8;
    }
    return out;
}

template <bool E4M3>
__global__ __launch_bounds__(64 * kWaves) void kv8_compact_kernel(Kv8CompactCall p) {
    const KvBatchView& b = p.batch;
    const int lane = threadIdx.x & 63, kv_heads = p.kv_heads, dim = p.dim, block = b.block, shift = b.block_shift;
    const int unit = __builtin_amdgcn_readfirstlane(blockIdx.x * kWaves + (threadIdx.x >> 6));
    const bool which = unit & 1;                    // values
    const int kvh = unit / 2 % kv_heads, request = unit / 2 / kv_heads;
    if (request >= b.requests) return;
    const Kv8Request q = kv8_request(b, request);
    const int kept = p.kept[request];
    if (q.rows <= 0 || kept <= 0 || kept > q.rows) return;
    const int* path = p.path + q.start;
    const int* table = b.table + (size_t)request * b.width;
    const Kv8Layer& layer = p.layers[blockIdx.y];
    float* const scales = which ? layer.value_scales : layer.key_scales;
    uint8_t* const all = which ? layer.values : layer.keys;
    // the path ascends within the rows; from the first row that moves on all do
    int first = kept;
    bool wrong = false;
    for (int base = 0; base < kept; base += 64) {
        const int k = base + lane, at = k < kept ? path[k] : 0, previous = k < kept && k ? path[k - 1] : -1;
        wrong = wrong || (k < kept && (at <= previous || at >= q.rows));
        const uint64_t moves = __ballot(k < kept && at != k);
        if (moves && first == kept) first = base + __builtin_ctzll(moves);
    }
    if (__any(wrong) || first == kept) return;
    const int before = q.length - q.rows, mask = block - 1;
    const size_t head_bytes = (size_t)block * dim;
    for (int entry = (before + first) >> shift; entry <= (before + kept - 1) >> shift; ++entry) {
        const int id = table[entry];
        if ((unsigned)id >= (unsigned)b.blocks) continue;
        const int start = entry << shift, from = max(before - start, 0), to = min(before + kept - start, block), tokens = to - from;
        const size_t own = (size_t)id * kv_heads + kvh;
        // where the block's kept rows come from: rows `lane` and 64 + lane of them, in tokens of the pool, and these blocks' scales
        int comes[2];
        float given[2], most = 0.0f;
        bool spoilt = false;
        const float old = scales[own];
        if (from > 0) {
            most = old;
            spoilt = !(old >= 0.0f && old < INFINITY);
        }
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int i = lane + 64 * j;
            comes[j] = -1;
            given[j] = 0.0f;
            if (i >= tokens) continue;
            const int position = before + path[start + from + i - before], page = table[position >> shift];
            if ((unsigned)page >= (unsigned)b.blocks) continue;
            comes[j] = (page << shift) + (position & mask);
            given[j] = scales[(size_t)page * kv_heads + kvh];
            spoilt = spoilt || !(given[j] >= 0.0f && given[j] < INFINITY);
            most = fmaxf(most, given[j]);
        }
        spoilt = __any(spoilt);
        const float scale = spoilt ? NAN : wave_max_f32(most);
        const double inverse = 1.0 / (double)scale;
        // (a spoilt block's codes stay as they come)
        auto differs = [&](float other) { return !spoilt && other != scale; };
        uint8_t* const mine = all + own * head_bytes;
        if (!which) {
            // 16 codes of a row to a lane
            const int pieces = dim / 16;
            for (int base = 0; base < tokens * pieces; base += 64) {
                const int u = base + lane, i = u / pieces, d = 16 * (u - i * pieces);
                const int low = __shfl(comes[0], i & 63, 64), high = __shfl(comes[1], i & 63, 64), at = i < 64 ? low : high;
                const float low_scale = __shfl(given[0], i & 63, 64), high_scale = __shfl(given[1], i & 63, 64);
                const float other = i < 64 ? low_scale : high_scale;
                const bool moves = u < tokens * pieces && at >= 0;
                v4u codes{};
                if (moves) codes = *(const v4u*)(all + ((size_t)(at >> shift) * kv_heads + kvh) * head_bytes + (size_t)(at & mask) * dim + d);
                if (moves && differs(other))
#pragma unroll
                    for (int w = 0; w < 4; ++w) codes[w] = moved_word<E4M3>(codes[w], other, scale, inverse);
                if (moves) *(v4u*)(mine + (size_t)(from + i) * dim + d) = codes;
            }
            if (from > 0 && differs(old))           // the block's earlier tokens follow its scale
                for (int u = lane; u < from * (dim / 4); u += 64) {
                    uint32_t* at = (uint32_t*)mine + u;
                    *at = moved_word<E4M3>(*at, old, scale, inverse);
                }
        } else {
            // a dim's tokens to a lane
            for (int d0 = 0; d0 < dim; d0 += 64) {  // (all lanes come round together: they read each other's registers)
                const int d = d0 + lane;
                const bool has = d < dim;
                uint8_t* const line = mine + (size_t)d * block;
                for (int base = 0; base < tokens; base += kTogether) {
                    uint32_t codes[kTogether];
#pragma unroll
                    for (int i = 0; i < kTogether; ++i) {
                        const int at = base + i < tokens ? __builtin_amdgcn_readlane(base + i < 64 ? comes[0] : comes[1], (base + i) & 63) : -1;
                        codes[i] = has && at >= 0 ? all[((size_t)(at >> shift) * kv_heads + kvh) * head_bytes + (size_t)d * block + (at & mask)] : 0;
                    }
#pragma unroll
                    for (int i = 0; i < kTogether; ++i) {
                        if (base + i >= tokens) continue;
                        const int n = (base + i) & 63;
                        if (__builtin_amdgcn_readlane(base + i < 64 ? comes[0] : comes[1], n) < 0) continue;
                        const float other = __int_as_float(__builtin_amdgcn_readlane(__float_as_int(base + i < 64 ? given[0] : given[1]), n));
                        if (has) line[from + base + i] = (uint8_t)(differs(other) ? moved_code<E4M3>(codes[i], other, scale, inverse) : codes[i]);
                    }
                }
                if (has && from > 0 && differs(old))
                    for (int base = 0; base < from; base += 16) {
                        v4u codes = *(const v4u*)(line + base);
#pragma unroll
                        for (int w = 0; w < 4; ++w) {
                            const int n = min(from - base - 4 * w, 4);   // of the word's tokens, earlier ones
                            if (n <= 0) continue;
                            const uint32_t moved = moved_word<E4M3>(codes[w], old, scale, inverse), later = n < 4 ? ~0u << 8 * n : 0;
                            codes[w] = (moved & ~later) | (codes[w] & later);
                        }
                        *(v4u*)(line + base) = codes;
                    }
            }
        }
        if (lane == 0) scales[own] = scale;
    }
}

}  // namespace

void launch_kv8_compact(const Kv8CompactCall& call, int layers, hipStream_t stream) {
    const int64_t units = (int64_t)call.batch.requests * call.kv_heads * 2;
    const dim3 grid((uint32_t)((units + kWaves - 1) / kWaves), layers);
    if (call.e4m3) kv8_compact_kernel<true><<<grid, 64 * kWaves, 0, stream>>>(call);
    else kv8_compact_kernel<false><<<grid, 64 * kWaves, 0, stream>>>(call);
}

}  // namespace leafhip
