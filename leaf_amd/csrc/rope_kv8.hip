// RoPE and the append of a step's keys and values to an 8-bit cache in blocks
// (include/leafhip.h: lh_rope_kv8).
//
// A block's scale covers all of its tokens, so the unit of work is a run: the
// step's tokens that fall into one block, of one KV head.  A run is found from
// the slots alone, and worked on by its first token's workgroup.  The run's largest
// magnitude gives the scale; a scale that grows moves the codes of the block's
// earlier tokens.  Where a skipped token parts a block's tokens, they are
// several runs, one after the other.
#include <algorithm>

#include "kv8.h"

namespace leafhip {
namespace {

struct Token {
    int slot, position;                             // slot -1: skipped
};
__device__ __forceinline__ Token token_of(const RopeKv8Call& p, int t) {
    Token k{-1, 0};
    if (t < 0 || t >= p.batch.tokens) return k;
    const int slot = p.batch.slots[t], position = p.batch.positions[t];
    if (slot >= 0 && slot < p.batch.blocks << p.batch.block_shift && position >= 0 && position < p.positions)
        k = Token{slot, position};
    return k;
}

// Value d of a head's row, rotated (the products and their sum each rounded).
__device__ __forceinline__ float rotated(const float* row, int d, const float* c, const float* s, int half) {
    if (d < half) return row[d] * c[d] - row[d + half] * s[d];
    if (d < 2 * half) return row[d] * c[d - half] + row[d - half] * s[d - half];
    return row[d];
}

// A bit for each slot of a block.
struct BlockBits {
    uint64_t low, high;
    __device__ __forceinline__ uint64_t from(int i) const {    // 64 of them
        return i >= 64 ? high >> (i - 64) : i ? low >> i | high << (64 - i) : low;
    }
    __device__ __forceinline__ int first() const { return low ? __builtin_ctzll(low) : 64 + __builtin_ctzll(high); }
    // Set bits in a row from i.
    __device__ __forceinline__ int run(int i) const {
        const uint64_t gaps = ~from(i);
        if (gaps) return __builtin_ctzll(gaps);
        const uint64_t later = i ? 0 : high;             // (64 from i > 0 on are the last)
        return 64 + (~later ? __builtin_ctzll(~later) : 64);
    }
    // The first set bit from i on; 128 where there is none.
    __device__ __forceinline__ int next(int i) const {
        for (; i < 128; i += 64) {
            const uint64_t b = from(i);
            if (b) return i + __builtin_ctzll(b);
        }
        return 128;
    }
};

__global__ __launch_bounds__(64) void rope_kv8_kernel(RopeKv8Call p) {
    const int t = blockIdx.x, lane = threadIdx.x, half = p.rotary / 2, dim = p.cache.dim, block = p.batch.block;
    const int kv_heads = p.cache.kv_heads, group = p.heads / kv_heads, h = blockIdx.y;
    const size_t width = (size_t)(p.heads + 2 * kv_heads) * dim;
    const Token own = token_of(p, t);
    if (own.slot < 0) return;
    {
        const float* c = p.cosines + (size_t)own.position * half;
        const float* s = p.sines + (size_t)own.position * half;
        for (int i = lane; i < group * dim; i += 64) {
            const int q = h * group + i / dim, d = i % dim;
            p.q_heads[((size_t)q * p.batch.tokens + t) * dim + d] = rotated(p.qkv + t * width + (size_t)q * dim, d, c, s, half);
        }
    }
    // which of the block's slots have a token in this step: the rows beside this one
    const int place = own.slot & (block - 1);
    auto taken = [&](int i) { return i < block && token_of(p, t - place + i).slot == own.slot - place + i; };
    const BlockBits bits{__ballot(taken(lane)), block > 64 ? __ballot(taken(64 + lane)) : 0};
    if (bits.first() < place) return;                    // the first of them works on the block
    const size_t at = (size_t)(own.slot >> p.batch.block_shift) * kv_heads + h;
    for (int offset = place; offset < block; ) {
        const int run = bits.run(offset), row = t - place + offset;
        for (int which = 0; which < 2; ++which) {        // keys, values
            uint8_t* codes = (which ? p.cache.values : p.cache.keys) + at * block * dim;
            float* scales = which ? p.cache.value_scales : p.cache.key_scales;
            const float* rows = p.qkv + (size_t)(p.heads + which * kv_heads + h) * dim;
            auto value = [&](int i, int d) {
                const float* x = rows + (size_t)(row + i) * width;
                if (which) return x[d];
                const size_t pos = p.batch.positions[row + i];
                return rotated(x, d, p.cosines + pos * half, p.sines + pos * half, half);
            };
            auto code = [&](int i, int d) -> uint8_t& { return codes[which ? (size_t)d * block + i : (size_t)i * dim + d]; };
            uint32_t most = 0;                           // magnitudes as bits: their order, NaN above all
            for (int i = lane; i < run * dim; i += 64) most = max(most, __float_as_uint(value(i / dim, i % dim)) & 0x7fffffffu);
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) most = max(most, (uint32_t)__shfl_xor((int)most, o, 64));
            const float top = __uint_as_float(most), old = offset ? scales[at] : 0.0f;
            const bool whole = finite_f32(top) && finite_f32(old);
            const float need = p.cache.e4m3 ? e4m3_scale(top) : fmaxf(top / 127.0f, 1e-12f);
            const float scale = fmaxf(need, old), inverse = p.cache.e4m3 ? inverse_of_power(scale) : 1.0f / scale;
            if (whole && offset && scale > old)
                for (int i = lane; i < offset * dim; i += 64) {
                    uint8_t& c = code(i / dim, i % dim);
                    if (p.cache.e4m3) c = (uint8_t)e4m3_pair(__builtin_amdgcn_cvt_f32_fp8(c, 0) * (old * inverse), 0.0f);
                    else c = (uint8_t)(int)__builtin_rint((double)(int8_t)c * (double)old / (double)scale);
                }
            for (int i = lane; i < run * dim; i += 64) {
                const float x = value(i / dim, i % dim);
                uint8_t c = 0;
                if (whole) c = p.cache.e4m3 ? (uint8_t)e4m3_pair(x * inverse, 0.0f) : (uint8_t)nearest_i8(x, scale, inverse);
                code(offset + i / dim, i % dim) = c;
            }
            __syncthreads();                             // the next run reads these
            if (lane == 0) scales[at] = whole ? scale : NAN;
        }
        __syncthreads();
        offset = bits.next(offset + run);
    }
}

}  // namespace

void launch_rope_kv8(const RopeKv8Call& call, hipStream_t stream) {
    rope_kv8_kernel<<<dim3(call.batch.tokens, call.cache.kv_heads), 64, 0, stream>>>(call);
}

}  // namespace leafhip
