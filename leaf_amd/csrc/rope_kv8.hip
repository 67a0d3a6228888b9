// RoPE and the append of a step's keys and values to an 8-bit cache in blocks
// (include/leafhip.h: lh_rope_kv8).
//
// A block's scale covers all of its tokens, so the unit of work is a run: the
// step's tokens that fall into one block, of one KV head.  A run is found from
// the slots alone, and worked on by its first token's workgroup.  The run's largest
// magnitude gives the scale; a scale that grows moves the codes of the block's
// earlier tokens.  Where a skipped token parts a block's tokens, they are
// several runs, one after the other.
//
// Keys are stored row by row, values with a dim's tokens together, as attention
// reads them.  A thread takes four dims of four slots: a word of four codes for
// each, stored along the dims for keys and along the slots for values.
//
// What bounds it: the latency of dependent loads (slots and positions, the rows
// beside them, the values, their scale, and, past one group of slots a thread,
// the values again) and cold code: with loops unrolled
// over 16 slots, 100 KB of it, the same calls took two to three times as long.  64 single tokens of
// 32 heads of 64 over 4 take 7.7 us, 2048 tokens of 14 heads over 2 15.6 (18 MB, of which
// the queries 14.7), a chunk of 500 beside 47 single tokens, 32 heads of 128 over 8, 22;
// 4096 tokens of those 73 (235 MB at 3.2 TB/s, 46 of them the queries').
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
        const uint64_t later = i < 64 ? high >> i : 0;   // those from i + 64 on
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

// Four values of a head's row from d on, rotated; QUADS: half is a multiple of four.
template <bool QUADS>
__device__ __forceinline__ v4f rotated4(const float* row, int d, const float* c, const float* s, int half) {
    const v4f x = *(const v4f*)(row + d);
    if (!half) return x;
    v4f out = x;
    if (QUADS) {
        // (a quad that is not turned takes what it loads from the first ones, for nothing: no branch parts the loads)
        const bool turned = d < 2 * half, low = d < half;
        const int i = !turned ? 0 : low ? d : d - half, partner = !turned ? 0 : low ? d + half : d - half;
        const v4f co = *(const v4f*)(c + i), si = *(const v4f*)(s + i), y = *(const v4f*)(row + partner);
        const v4f a = x * co, b = y * si;
#pragma unroll
        for (int e = 0; e < 4; ++e) out[e] = !turned ? x[e] : low ? a[e] - b[e] : a[e] + b[e];
    } else {
        for (int e = 0; e < 4; ++e) out[e] = rotated(row, d + e, c, s, half);
    }
    return out;
}

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kGroup = 4;                           // slots of a unit, by four dims: what a thread takes at a time
// Groups of slots by quads of dims of a block that one wave takes; more are the workgroup's.  With 32 / 128 / 512: 64 tokens
// in a block of 64 (heads of 64) 8.9 / 11.5 / 15.2 us, 4096 tokens in blocks of 16 (heads of 128) 67 / 56 / 42, of 64 39 / 39 / 123.
constexpr int kWaveUnits = 128;

// A token that is the first of its block in this step.
struct Leader {
    int row, slot;                                  // row -1: none
    BlockBits bits;                                 // the slots of the block that have a token
};

// Four codes of an earlier token, moved from scale `old` to `scale`.  One code after the other: the loop's code
// is fetched cold by nearly every call, and runs only where a scale has grown.
template <bool E4M3>
__device__ __forceinline__ uint32_t moved(uint32_t word, float old, float scale, float inverse) {
    uint32_t out = 0;
#pragma unroll 1
    for (int i = 0; i < 4; ++i) {
        uint32_t c;
        if (E4M3) c = e4m3_pair(__builtin_amdgcn_cvt_f32_fp8(word & 0xFFu, 0) * (old * inverse), 0.0f);
        else c = (uint32_t)(int)__builtin_rint((double)(int8_t)(word & 0xFFu) * (double)old / (double)scale);
        out = out >> 8 | c << 24;
        word >>= 8;
    }
    return out;
}

// One run of a block's keys or values by a team of threads (a wave, or the workgroup): slots [offset, offset + run),
// whose rows are those from `base` on, at `positions` [slot].  Two passes over its values, which stay in registers
// where no thread has two groups.
template <bool QUADS, bool E4M3>
__device__ __forceinline__ void append_run(const RopeKv8Call& p, int kvh, bool which, int base, const int* positions, size_t at,
                                           int offset, int run, bool team, uint32_t* most) {
    const int thread = team ? threadIdx.x : threadIdx.x & 63, threads = team ? kThreads : 64;
    const int half = p.rotary / 2, dim = p.cache.dim, block = p.batch.block, kv_heads = p.cache.kv_heads, quads = dim / 4;
    const size_t width = (size_t)(p.heads + 2 * kv_heads) * dim;
    float* const scale_at = (which ? p.cache.value_scales : p.cache.key_scales) + at;
    uint8_t* const codes = (which ? p.cache.values : p.cache.keys) + at * block * dim;
    const float old = offset ? *scale_at : 0.0f;
    // a thread: always the same quad of dims, of every abreast-th group of slots
    const int own = thread / quads, d = (thread - own * quads) * 4, abreast = threads / quads;
    const int end = (offset + run + kGroup - 1) / kGroup, begin = own < abreast ? offset / kGroup + own : end;
    const float* rows = p.qkv + (size_t)(p.heads + which * kv_heads + kvh) * dim + (long long)base * width;
    v4f x[kGroup];
    auto load = [&](int g) {
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
            // (slots outside the run: its nearest one)
            const int slot = min(max(g * kGroup + i, offset), offset + run - 1);
            const float* row = rows + slot * width;
            if (which) {
                x[i] = *(const v4f*)(row + d);
            } else {
                const size_t turn = (size_t)positions[slot] * half;
                x[i] = rotated4<QUADS>(row, d, p.cosines + turn, p.sines + turn, half);
            }
        }
    };
    uint32_t top = 0;                               // magnitudes as bits: their order, NaN above all
#pragma unroll 1
    for (int g = begin; g < end; g += abreast) {
        load(g);
#pragma unroll
        for (int i = 0; i < kGroup; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) top = max(top, __float_as_uint(x[i][e]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if (team) {
        __syncthreads();                            // the last run's are read
        if ((threadIdx.x & 63) == 0) most[threadIdx.x >> 6] = top;
        __syncthreads();
        for (int w = 0; w < kWaves; ++w) top = max(top, most[w]);
    }
    const float largest = __uint_as_float(top);
    float scale = fmaxf(E4M3 ? e4m3_scale(largest) : fmaxf(largest / 127.0f, 1e-12f), old);
    const bool fine = finite_f32(largest) && finite_f32(old);
    const float inverse = E4M3 ? inverse_of_power(scale) : 1.0f / scale;
    if (thread == 0) *scale_at = fine ? scale : NAN;
    if (offset && fine && scale > old) {
        // the earlier tokens' words, those of keys [slot][dim / 4], of values [dim][slot / 4]
        const int words = which ? (offset + 3) / 4 : quads, lines = which ? dim : offset, pitch = which ? block : dim;
#pragma unroll 1
        for (int i = thread; i < words * lines; i += threads) {
            const int w = i % words;
            uint8_t* to = codes + (size_t)(i / words) * pitch + 4 * w;
            const uint32_t word = moved<E4M3>(*(const uint32_t*)to, old, scale, inverse);
            const int n = which ? offset - 4 * w : 4;
            if (n >= 4) *(uint32_t*)to = word;
            else                                    // the others are the run's
                for (int e = 0; e < n; ++e) to[e] = (uint8_t)(word >> 8 * e);
        }
    }
#pragma unroll 1
    for (int g = begin; g < end; g += abreast) {
        if (end - offset / kGroup > abreast) load(g);
        uint32_t word[kGroup];                      // of each slot, its four dims
#pragma unroll
        for (int i = 0; i < kGroup; ++i) {
            if (E4M3) {
                word[i] = e4m3_pair(x[i][0] * inverse, x[i][1] * inverse) | e4m3_pair(x[i][2] * inverse, x[i][3] * inverse) << 16;
            } else {
                word[i] = 0;
#pragma unroll
                for (int e = 0; e < 4; ++e) word[i] |= ((uint32_t)nearest_i8(x[i][e], scale, inverse) & 0xFFu) << 8 * e;
            }
            if (!fine) word[i] = 0;
        }
        const int from = max(offset - g * kGroup, 0), to = min(offset + run - g * kGroup, kGroup);
        if (!which) {
#pragma unroll
            for (int i = 0; i < kGroup; ++i)
                if (i >= from && i < to) *(uint32_t*)(codes + (size_t)(g * kGroup + i) * dim + d) = word[i];
            continue;
        }
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            uint8_t* at_dim = codes + (size_t)(d + e) * block + g * kGroup;
            const uint32_t line = (word[0] >> 8 * e & 0xFFu) | (word[1] >> 8 * e & 0xFFu) << 8 | (word[2] >> 8 * e & 0xFFu) << 16 |
                                  word[3] >> 8 * e << 24;
            if (to - from == kGroup) *(uint32_t*)at_dim = line;
            else
#pragma unroll
                for (int i = 0; i < kGroup; ++i)
                    if (i >= from && i < to) at_dim[i] = (uint8_t)(line >> 8 * i);
        }
    }
}

// A thread's share of a token's queries: the same rotated quad with its partner, or copied quad, of four heads, whose
// loads are in flight together; without QUADS single values.
constexpr int kHeads = 4;
template <bool QUADS>
__host__ __device__ inline int query_items(const RopeKv8Call& p) {
    return (p.heads + kHeads - 1) / kHeads * (p.rotary / 2 + p.cache.dim - p.rotary) / (QUADS ? 4 : 1);
}
// Workgroup `group` of `groups`: some tokens whole, or a part of one.
template <bool QUADS>
__device__ __forceinline__ void rotate_queries(const RopeKv8Call& p, int group, int groups) {
    constexpr int step = QUADS ? 4 : 1;
    const int half = p.rotary / 2, dim = p.cache.dim, turned = half / step, per_head = turned + (dim - p.rotary) / step;
    const int items = query_items<QUADS>(p), abreast = max(1, kThreads / items), parts = (items + kThreads - 1) / kThreads;
    const size_t width = (size_t)(p.heads + 2 * p.cache.kv_heads) * dim;
    for (long long g = group; ; g += groups) {
        const long long t0 = g / parts * abreast;
        if (t0 >= p.batch.tokens) return;
        const int own = parts > 1 ? 0 : threadIdx.x / items, item = (int)(g % parts) * kThreads + threadIdx.x - own * items;
        const Token token = token_of(p, (int)min(t0 + own, (long long)p.batch.tokens));
        if (own >= abreast || item >= items || token.slot < 0) continue;
        const int t = (int)t0 + own, h = item / per_head * kHeads, i = item % per_head, heads = min(kHeads, p.heads - h);
        const size_t pitch = (size_t)p.batch.tokens * dim;
        const float* row = p.qkv + t * width + (size_t)h * dim;
        float* to = p.q_heads + (size_t)h * pitch + (size_t)t * dim;
        const int d = i < turned ? step * i : p.rotary + step * (i - turned);
        const float* c = p.cosines + (size_t)token.position * half;
        const float* s = p.sines + (size_t)token.position * half;
        if (QUADS) {
            const int partner = i < turned ? d + half : d;
            v4f a[kHeads], b[kHeads], co{}, si{};
            if (i < turned) {
                co = *(const v4f*)(c + d);
                si = *(const v4f*)(s + d);
            }
#pragma unroll
            for (int k = 0; k < kHeads; ++k) {
                const float* from = row + min(k, heads - 1) * dim;
                a[k] = *(const v4f*)(from + d);
                b[k] = *(const v4f*)(from + partner);
            }
#pragma unroll
            for (int k = 0; k < kHeads; ++k) {
                if (k >= heads) continue;
                if (i < turned) {
                    *(v4f*)(to + k * pitch + d) = a[k] * co - b[k] * si;
                    *(v4f*)(to + k * pitch + partner) = b[k] * co + a[k] * si;
                } else {
                    *(v4f*)(to + k * pitch + d) = a[k];
                }
            }
        } else {
            for (int k = 0; k < heads; ++k) {
                const float* from = row + k * dim;
                to[k * pitch + d] = rotated(from, d, c, s, half);
                if (i < turned) to[k * pitch + d + half] = rotated(from, d + half, c, s, half);
            }
        }
    }
}

struct Launch {
    int cache_groups;                               // the first workgroups, of the cache's keys and values
    int each;                                       // tokens that a wave of these looks at
    int teams;                                      // whether a block's tokens of a step may be more than one wave should take
};

// The first workgroups take some tokens of a KV head's keys or values each, `each` for a wave: a block's tokens by the
// wave of the first of them, or by the workgroup where they are many.  The others rotate the queries.
template <bool QUADS, bool E4M3>
__global__ __launch_bounds__(kThreads, 4) void rope_kv8_kernel(RopeKv8Call p, Launch how) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, kv_heads = p.cache.kv_heads, block = p.batch.block;
    const int group = blockIdx.x;
    if (group >= how.cache_groups) {
        rotate_queries<QUADS>(p, group - how.cache_groups, gridDim.x - how.cache_groups);
        return;
    }
    __shared__ Leader leaders[kWaves];
    __shared__ int positions[kWaves][128];
    __shared__ uint32_t most[kWaves];
    const bool which = group & 1;
    const int kvh = group / 2 % kv_heads, t0 = (group / 2 / kv_heads * kWaves + wave) * how.each;
    uint64_t candidates = 1;
    if (how.each > 1) {
        // a token that follows the one before it in a block is not the block's first: one look at both settles most
        bool first = false;
        if (lane < how.each) {
            const Token token = token_of(p, t0 + lane), before = token_of(p, t0 + lane - 1);
            first = token.slot >= 0 && !(before.slot == token.slot - 1 && before.slot >= 0 && token.slot & (block - 1));
        }
        candidates = __ballot(first);
        if (!__syncthreads_or(candidates != 0)) return;
    }
#pragma unroll 1
    for (int turn = 0; turn < how.each; ++turn) {
        Leader own{-1, 0, {0, 0}};
        bool many = false;
        if (candidates >> turn & 1) {
            // which of the block's slots have a token in this step: of the rows beside this one
            const int t = t0 + turn;
            const Token low = token_of(p, t - 63 + lane), high = token_of(p, t + 1 + lane);
            const int slot = __shfl(low.slot, 63, 64), place = slot & (block - 1);
            auto taken = [&](int i) {
                const int row = 63 - place + i, from = row & 63;   // of the rows in `low` and `high`
                const int ls = __shfl(low.slot, from, 64), hs = __shfl(high.slot, from, 64);
                const int lp = __shfl(low.position, from, 64), hp = __shfl(high.position, from, 64);
                Token k{row < 64 ? ls : hs, row < 64 ? lp : hp};
                if (block > 64 && (row < 0 || row >= 128)) k = token_of(p, t - place + i);
                positions[wave][i] = k.position;
                return i < block && k.slot == slot - place + i;
            };
            const BlockBits bits{__ballot(taken(lane)), block > 64 ? __ballot(taken(64 + lane)) : 0};
            if (slot >= 0 && bits.first() == place) {
                own = Leader{t, slot, bits};
                const int last = bits.high ? 127 - __builtin_clzll(bits.high) : 63 - __builtin_clzll(bits.low);
                many = how.teams && (last / kGroup - place / kGroup + 1) * (p.cache.dim / 4) > kWaveUnits;
            }
        }
        bool any_many = false;
        if (how.teams) {
            if (lane == 0) leaders[wave] = many ? own : Leader{-1, 0, {0, 0}};
            any_many = __syncthreads_or(many);
        }
        // a wave its own block, then all of them together the large ones
#pragma unroll 1
        for (int w = -1; w < (any_many ? kWaves : 0); ++w) {
            const bool team = w >= 0;
            const Leader l = team ? leaders[w] : many ? Leader{-1, 0, {0, 0}} : own;
            if (l.row < 0) continue;
            const int place = l.slot & (block - 1);
            const size_t at = (size_t)(l.slot >> p.batch.block_shift) * kv_heads + kvh;
            for (int offset = place; offset < block; ) {
                const int run = l.bits.run(offset);
                append_run<QUADS, E4M3>(p, kvh, which, l.row - place, positions[team ? w : wave], at, offset, run, team, most);
                offset = l.bits.next(offset + run);
                if (offset >= block) break;
                __threadfence_block();              // the next run reads what this one wrote
                if (team) __syncthreads();
            }
        }
        if (how.teams && how.each > 1) __syncthreads();   // leaders and positions are read
    }
}

// Workgroups for the cache's part before a wave looks at several tokens (up to eight), about those that the GPU holds at once.
// With 256 / 512 / 1024: 2048 tokens of 2 heads of 64 22 / 13 / 18 us, a chunk of 500 beside 47 single tokens 35 / 21 / 21.
constexpr int kMostGroups = 512;

}  // namespace

void launch_rope_kv8(const RopeKv8Call& call, hipStream_t stream) {
    const bool quads = call.rotary % 8 == 0;
    const int items = quads ? query_items<true>(call) : query_items<false>(call);
    const int kv = 2 * call.cache.kv_heads, tokens = call.batch.tokens;
    Launch how;
    how.each = (int)std::min<int64_t>(std::max<int64_t>(((int64_t)tokens * kv / kWaves + kMostGroups - 1) / kMostGroups, 1), 8);
    how.cache_groups = (tokens + kWaves * how.each - 1) / (kWaves * how.each) * kv;
    const int slots = std::min(call.batch.block, call.batch.max_rows);
    how.teams = (slots + 2 * kGroup - 2) / kGroup * (call.cache.dim / 4) > kWaveUnits;
    const size_t abreast = std::max(1, kThreads / items), parts = (items + kThreads - 1) / kThreads;
    const size_t query_groups = std::min<size_t>((tokens + abreast - 1) / abreast * parts, 1 << 20);
    const dim3 grid((uint32_t)(how.cache_groups + query_groups));
    if (quads && call.cache.e4m3) rope_kv8_kernel<true, true><<<grid, kThreads, 0, stream>>>(call, how);
    else if (quads) rope_kv8_kernel<true, false><<<grid, kThreads, 0, stream>>>(call, how);
    else if (call.cache.e4m3) rope_kv8_kernel<false, true><<<grid, kThreads, 0, stream>>>(call, how);
    else rope_kv8_kernel<false, false><<<grid, kThreads, 0, stream>>>(call, how);
}

}  // namespace leafhip
