// Causal grouped-query attention of a ragged batch over an 8-bit cache in
// blocks (include/leafhip.h: lh_attention_kv8), on the f16 matrix cores with
// f32 accuracy.
//
// Operands.  A code is an f16 value exactly (8 bits fit 11).  A query row is
// scaled by a power of two so that its largest value is below 2^15 and taken as
// hi + lo, two f16 values of together 22 bits, and a weight likewise: two
// products each for Q K^T and P V, summed in f32 (an f32 operand as bf16 values
// would need three).
//
// Scales.  The score of a key is (q . code) c with c = query scale * key scale *
// log2(e) / sqrt(dim).  A value's scale is 2^e f with 1 <= f < 2: weights are
// formed as t = 2^(score + e - b + 8), relative to the largest weight times value
// scale rather than the largest weight, so that w = t f, which is what meets the
// value codes, keeps its 22 bits wherever it counts however far the scales of
// blocks are apart, and the sum of weights adds t 2^-e.  b is a whole number per
// row, at most 6 below the largest score + e so far (w < 2^15), so most steps
// rescale nothing and a rescale is exact.
//
// Layout.  A step is 64 keys.  S^T = K Q^T by v_mfma_f32_16x16x32_f16 with lane
// l = 16 lq + li: row li of its tile j of keys is key 16 (li / 4) + 4 j + li % 4
// of the step, so that lane l then holds the scores of query row li for the 16
// keys 16 lq + 4 j + r in a row: P is the other operand of O^T = V^T P^T without
// leaving its registers, V's lanes read 16 codes of one dim (the cache keeps a
// dim's tokens together), and a lane's 16 keys lie in one block, with one scale.
// Both K and V come as 16-byte loads; a key's dims are permuted alike in Q.
#include <algorithm>

#include "kv8.h"

namespace leafhip {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

constexpr int kStep = 64;                           // keys
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kFewRows = 16;                        // rows of a KV head in one tile
constexpr float kNoBase = -1e30f;
constexpr float kSlack = 6.0f, kLift = 8.0f;

// 16 codes as two operands.
template <bool E4M3>
__device__ __forceinline__ void widen(v4u codes, v8h& a, v8h& b) {
    v2h h[8];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if (E4M3) {
            h[2 * i] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[i], 1.0f, false);
            h[2 * i + 1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8(codes[i], 1.0f, true);
        } else {
            // 0x6400 + (code + 128) is 1024 + code + 128
            const uint32_t u = codes[i] ^ 0x80808080u;
            const v2h offset = v2h{(_Float16)-1152.0f, (_Float16)-1152.0f};
            h[2 * i] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) + offset;
            h[2 * i + 1] = __builtin_bit_cast(v2h, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) + offset;
        }
    }
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        a[2 * i] = h[i].x; a[2 * i + 1] = h[i].y;
        b[2 * i] = h[4 + i].x; b[2 * i + 1] = h[4 + i].y;
    }
}

// x = hi + lo to 22 bits, toward zero.
__device__ __forceinline__ void split2(float x, float y, v2h& hi, v2h& lo) {
    hi = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_pkrtz(x, y));
    lo = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_pkrtz(x - (float)hi.x, y - (float)hi.y));
}

// A query row's operands for its lanes (one of four), and what its products are to be multiplied by.
template <int CC, bool FULL>
__device__ __forceinline__ void load_query(const float* q, int dim, int lq, float scale, v8h (&hi)[CC][2], v8h (&lo)[CC][2], float& c) {
    v4f f[CC][4];
    float most = 0.0f;
    bool spoilt = false;
#pragma unroll
    for (int cc = 0; cc < CC; ++cc)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int d = 64 * cc + 16 * lq;
            f[cc][e] = FULL || d < dim ? *(const v4f*)(q + d + 4 * e) : v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                most = fmaxf(most, __builtin_fabsf(f[cc][e][i]));
                spoilt = spoilt || !finite_f32(f[cc][e][i]);
            }
        }
    if (spoilt) most = INFINITY;
    most = max_xor32(max_xor16(most));
    // 2^k with the largest value in [2^14, 2^15) (from 2^-100 up; zeros and smaller values need none)
    const int exponent = max((int)(__float_as_uint(most) >> 23), 127 - 100);
    const float up = __uint_as_float((uint32_t)min(127 + 14 + 127 - exponent, 254) << 23);
    const float down = __uint_as_float((uint32_t)max(exponent - 14, 1) << 23);
#pragma unroll
    for (int cc = 0; cc < CC; ++cc)
#pragma unroll
        for (int e = 0; e < 4; ++e)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                v2h h, l;
                split2(f[cc][e][2 * i] * up, f[cc][e][2 * i + 1] * up, h, l);
                const int at = 4 * (e & 1) + 2 * i;
                hi[cc][e >> 1][at] = h.x; hi[cc][e >> 1][at + 1] = h.y;
                lo[cc][e >> 1][at] = l.x; lo[cc][e >> 1][at + 1] = l.y;
            }
    c = finite_f32(most) ? down * scale * 1.4426950408889634f : NAN;
}

// What a lane's 16 keys of a step need of their block.
struct KeyScales {
    float key, value;                               // NaN where the block spoils the rows that see it
};

// The keys of one request and KV head.
struct Keys {
    const int* table;
    const uint8_t *keys, *values;
    const float *key_scales, *value_scales;
    int shift, blocks, kv_heads, kvh, dim, end;     // end: keys of the request

    __device__ __forceinline__ int block_of(int key) const { return table[min(key, end - 1) >> shift]; }
    __device__ __forceinline__ bool known(int id) const { return (unsigned)id < (unsigned)blocks; }
    __device__ __forceinline__ size_t at(int id) const { return (size_t)(known(id) ? id : 0) * kv_heads + kvh; }
    __device__ __forceinline__ KeyScales scales(int id) const {
        const size_t i = at(id);
        KeyScales s{key_scales[i], value_scales[i]};
        const bool fine = known(id);
        if (!fine || !(s.key >= 0.0f && s.key < INFINITY)) s.key = NAN;
        if (!fine || !(s.value >= 0.0f && s.value < INFINITY)) s.value = NAN;
        return s;
    }
    // Tile j of 16 keys: 16 codes of key 16 (li / 4) + 4 j + li % 4 from dim d on; id: the block of key 16 (li / 4).
    template <bool FULL>
    __device__ __forceinline__ v4u load_key(int id, int step, int j, int li, int d) const {
        const int place = (step * kStep + 16 * (li >> 2) + 4 * j + (li & 3)) & ((1 << shift) - 1);
        if (!FULL && d >= dim) return v4u{0, 0, 0, 0};
        return *(const v4u*)(keys + ((at(id) << shift) + place) * dim + d);
    }
    // 16 keys from 16 lq of dim d; id: the block of key 16 lq.
    __device__ __forceinline__ v4u load_value(int id, int step, int lq, int d) const {
        const int place = (step * kStep + 16 * lq) & ((1 << shift) - 1);
        return *(const v4u*)(values + ((at(id) * dim + d) << shift) + place);
    }
};

// Codes of `keys` tokens, the others zero.
__device__ __forceinline__ v4u first_codes(v4u codes, int keys) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int n = keys - 4 * i;
        codes[i] = n >= 4 ? codes[i] : n <= 0 ? 0u : codes[i] & ((1u << 8 * n) - 1);
    }
    return codes;
}

// A row's online softmax: its base and its sum (this lane's keys).
struct Softmax {
    float base = kNoBase, sum = 0.0f;
};

// A step's scores to weights: acc [tile][r] are the products of key 4 tile + r of the lane's 16.
// MASKED: of these only keys [from, to) are visible.  Rescales o where the base moves.
template <bool MASKED, int TILES>
__device__ __forceinline__ void weigh(v4f (&acc)[4], float c, KeyScales s, Softmax& m, v4f (&o)[TILES], int tiles, int from, int to,
                                      v8h (&hi)[2], v8h (&lo)[2]) {
    const int exponent = min(max((int)(__float_as_uint(s.value) >> 23) - 127, -64), 64);
    const float e = (float)exponent, down = __uint_as_float((uint32_t)(127 - exponent) << 23), f = s.value * down;
    c *= s.key;
    c = c < 1e-37f ? 1e-37f : c;                    // (a masked key is minus infinity times it)
    if (MASKED) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r)
                if (4 * j + r < from || 4 * j + r >= to) acc[j][r] = -INFINITY;
    }
    float top = acc[0][0];
#pragma unroll
    for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int r = 0; r < 4; ++r) top = fmaxf(top, acc[j][r]);
    top = fmaf(top, c, e);
    top = max_xor32(max_xor16(top));
    if (__any(top > m.base + kSlack)) {
        const float base = top > m.base + kSlack ? __builtin_ceilf(top) : m.base;
        const float alpha = __builtin_amdgcn_exp2f(m.base - base);
        m.base = base;
        m.sum *= alpha;
#pragma unroll
        for (int t = 0; t < TILES; ++t)
            if (t < tiles) o[t] = o[t] * alpha;
    }
    const float shift = e + (kLift - m.base);
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float t = __builtin_amdgcn_exp2f(fmaf(acc[j][r], c, shift));
            w[r] = t * f;
            if (MASKED && (4 * j + r < from || 4 * j + r >= to)) t = w[r] = 0.0f;
            sum += t;
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            v2h h, l;
            split2(w[2 * i], w[2 * i + 1], h, l);
            const int at = 4 * (j & 1) + 2 * i;
            hi[j >> 1][at] = h.x; hi[j >> 1][at + 1] = h.y;
            lo[j >> 1][at] = l.x; lo[j >> 1][at + 1] = l.y;
        }
    }
    m.sum = fmaf(sum, down, m.sum);
}

// How a batch's work is shared out.  A request's rows of a KV head make tiles of
// `tile_rows`; a tile's keys are cut into equal parts of at most `per` steps,
// per chosen so that all parts of the batch are about `target` workgroups.
struct Share {
    int tile_rows, target, least;                   // least: steps a part has at least
    int few;                                        // requests of at most kFewRows rows (1) or of more (0)
};
__device__ __forceinline__ int tiles_of(const Kv8Request& q, int group, const Share& share) {
    const int rows = q.rows * group;
    if (rows == 0 || (rows <= kFewRows) != (share.few != 0)) return 0;
    return (rows + share.tile_rows - 1) / share.tile_rows;
}
// Steps of the longest tile of a request.
__device__ __forceinline__ int steps_of(const Kv8Request& q, int window) {
    const int first = window ? max(0, q.length - q.rows + 1 - window) : 0;
    return (q.length + kStep - 1) / kStep - first / kStep;
}

struct Item {
    int request, tile, part, parts, first;          // first: number of the request's first item of its KV head
    Kv8Request q;
};

// Which part of which tile of which request is item `index` (of one KV head);
// request -1: none.  Every workgroup sums the whole batch, 256 requests at a time.
__device__ __forceinline__ Item find_item(const KvBatchView& b, int kv_heads, int group, int window, const Share& share, int index,
                                          int& per) {
    __shared__ int sums[kWaves];
    __shared__ Item found;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    auto steps = [&](const Kv8Request& q) { return tiles_of(q, group, share) * steps_of(q, window); };
    Kv8Request mine{0, 0, 0};
    long long total = 0;
    for (int r = threadIdx.x; r < b.requests; r += kThreads) {
        mine = kv8_request(b, r);
        total += steps(mine);
    }
    // (in f32: a share of work, not a sum that anything else depends on)
    float all = wave_sum_f32((float)total);
    __shared__ float totals[kWaves];
    if (lane == 0) totals[wave] = all;
    if (threadIdx.x == 0) found.request = -1;
    __syncthreads();
    all = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all += totals[w];
    per = max(share.least, (int)fminf(all * (float)kv_heads / (float)share.target + 1.0f, 1e9f));
    int before = 0;
    for (int base = 0; base < b.requests; base += kThreads) {
        const int r = base + threadIdx.x;
        if (b.requests > kThreads) mine = r < b.requests ? kv8_request(b, r) : Kv8Request{0, 0, 0};
        const int tiles = tiles_of(mine, group, share), parts = (steps_of(mine, window) + per - 1) / per;
        const int items = tiles ? tiles * parts : 0;
        int s = items;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int below = __shfl_up(s, o, 64);
            if (lane >= o) s += below;
        }
        if (lane == 63) sums[wave] = s;
        __syncthreads();
        int start = before + s - items, all_items = 0;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) start += sums[w];
            all_items += sums[w];
        }
        if (index >= start && index < start + items) {
            const int i = index - start;
            // the longest tiles (the last) first
            found = Item{r, tiles - 1 - i / parts, i % parts, parts, start, mine};
        }
        before += all_items;
        __syncthreads();
        if (index < before) break;
    }
    return found;
}

__device__ __forceinline__ Keys keys_of(const AttentionKv8Call& p, int request, int kvh, int end) {
    const KvBatchView& b = p.batch;
    return Keys{b.table + (size_t)request * b.width, p.cache.keys, p.cache.values, p.cache.key_scales, p.cache.value_scales,
                b.block_shift, b.blocks, p.cache.kv_heads, kvh, p.cache.dim, end};
}

// Partial results: a tile of rows by dim floats and each row's (base, sum), one after the other by item.
__device__ __forceinline__ float* partial_rows(const AttentionKv8Call& p, size_t item, int tile_rows) {
    return p.partial + 64 + p.batch.requests + item * tile_rows * (p.cache.dim + 2);
}

// ---- at most 16 rows of a KV head (single tokens): each wave takes every fourth step, straight from memory
template <int CC, bool FULL, bool E4M3>
__global__ __launch_bounds__(kThreads) void attention_kv8_few_kernel(AttentionKv8Call p, Share share) {
    constexpr int TILES = 4 * CC;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, li = lane & 15, lq = lane >> 4;
    const int kv_heads = p.cache.kv_heads, group = p.heads / kv_heads, dim = FULL ? 64 * CC : p.cache.dim;
    const int kvh = blockIdx.x % kv_heads, tiles = FULL ? TILES : dim / 16;
    int per;
    const Item item = find_item(p.batch, kv_heads, group, p.window, share, blockIdx.x / kv_heads, per);
    if (item.request < 0) return;
    const Kv8Request& q = item.q;
    const int rows = q.rows * group, row = min(li, rows - 1);
    const int token = q.start + row / group, head = kvh * group + row % group;
    const int position = q.length - q.rows + row / group;
    const int low = q.length - q.rows;                             // of the first row
    const int first = p.window ? max(0, low + 1 - p.window) / kStep : 0;
    const int steps = (q.length + kStep - 1) / kStep - first;
    const int begin = first + (int)((long long)item.part * steps / item.parts);
    const int end = first + (int)((long long)(item.part + 1) * steps / item.parts);
    const Keys keys = keys_of(p, item.request, kvh, q.length);

    v4u kr[4][CC], vr[TILES];
    KeyScales scales;
    auto load_keys = [&](int id, int step) {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int cc = 0; cc < CC; ++cc) kr[j][cc] = keys.load_key<FULL>(id, step, j, li, 64 * cc + 16 * lq);
    };
    auto load_values = [&](int id, int step) {
#pragma unroll
        for (int t = 0; t < TILES; ++t)
            if (FULL || t < tiles) vr[t] = keys.load_value(id, step, lq, 16 * t + li);
        scales = keys.scales(id);
    };
    auto block_k = [&](int step) { return keys.block_of(step * kStep + 16 * (li >> 2)); };
    auto block_v = [&](int step) { return keys.block_of(step * kStep + 16 * lq); };

    v8h qh[CC][2], ql[CC][2];
    float c;
    int step = begin + wave, ik = block_k(step), iv = block_v(step);
    load_query<CC, FULL>(p.q_heads + ((size_t)head * p.batch.tokens + token) * dim, dim, lq, p.scale, qh, ql, c);
    if (step < end) {
        load_keys(ik, step);
        load_values(iv, step);
        ik = block_k(step + kWaves);
        iv = block_v(step + kWaves);
    }
    v4f o[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) o[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    Softmax m;
    for (; step < end; step += kWaves) {
        v4f acc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            acc[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int cc = 0; cc < CC; ++cc) {
                v8h k[2];
                widen<E4M3>(kr[j][cc], k[0], k[1]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[h], ql[cc][h], acc[j], 0, 0, 0);
                    acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[h], qh[cc][h], acc[j], 0, 0, 0);
                }
            }
        }
        const bool more = step + kWaves < end;
        if (more) load_keys(ik, step + kWaves);
        v8h hi[2], lo[2];
        const int at = step * kStep + 16 * lq;                     // the lane's first key
        if (step * kStep + kStep > low + 1 || p.window) {          // the wave's rows see different keys
            const int from = p.window ? position + 1 - p.window - at : 0;
            weigh<true>(acc, c, scales, m, o, tiles, from, position + 1 - at, hi, lo);
            // (codes that no token wrote, or of no block, may be NaN, which no weight of zero stops)
            const int written = scales.value == scales.value ? q.length - at : 0;
#pragma unroll
            for (int t = 0; t < TILES; ++t)
                if (FULL || t < tiles) vr[t] = first_codes(vr[t], written);
        } else {
            weigh<false>(acc, c, scales, m, o, tiles, 0, 16, hi, lo);
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t)
            if (FULL || t < tiles) {
                v8h v[2];
                widen<E4M3>(vr[t], v[0], v[1]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[h], lo[h], o[t], 0, 0, 0);
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[h], hi[h], o[t], 0, 0, 0);
                }
            }
        if (more) {
            load_values(iv, step + kWaves);
            ik = block_k(step + 2 * kWaves);
            iv = block_v(step + 2 * kWaves);
        }
    }

    // ---- the four waves' states together; wave w then has the tiles t % 4 = w
    __shared__ v4f values[kWaves][TILES][64];
    __shared__ float bases[kWaves][16], sums[kWaves][16];
    m.sum = add_xor32(add_xor16(m.sum));
    if (lq == 0) {
        bases[wave][li] = m.base;
        sums[wave][li] = m.sum;
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t)
        if (FULL || t < tiles) values[wave][t][lane] = o[t];
    __syncthreads();
    float base = kNoBase, sum = 0.0f, alpha[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) base = fmaxf(base, bases[w][li]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        alpha[w] = __builtin_amdgcn_exp2f(bases[w][li] - base);
        sum = fmaf(sums[w][li], alpha[w], sum);
    }
    if (p.partial && threadIdx.x == 0) {
        // for the merge: parts' steps, and the first item of the request
        if (blockIdx.x == 0) *(int*)p.partial = per;
        if (item.parts > 1 && item.part == 0 && kvh == 0) ((int*)p.partial)[64 + item.request] = item.first;
    }
    if (li >= rows) return;
    const bool whole = item.parts == 1;
    float* part = whole ? nullptr : partial_rows(p, (size_t)(item.first + item.part) * kv_heads + kvh, share.tile_rows) + (size_t)li * (dim + 2);
    if (part && wave == 0 && lq == 0) {
        part[dim] = base;
        part[dim + 1] = sum;
    }
    for (int t = wave; t < tiles; t += kWaves) {
        v4f x = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const v4f v = values[w][t][lane];
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = fmaf(v[r], alpha[w], x[r]);
        }
        const int d = 16 * t + 4 * lq;
        if (whole) {
            *(v4f*)(p.out + ((size_t)token * p.heads + head) * dim + d) = v4f{x[0] / sum, x[1] / sum, x[2] / sum, x[3] / sum};
        } else {
#pragma unroll
            for (int r = 0; r < 4; ++r) part[d + r] = x[r];
        }
    }
}

// ---- rows whose keys were parted: one wave a row
__global__ __launch_bounds__(kThreads) void attention_kv8_merge_kernel(AttentionKv8Call p, Share share) {
    const int group = p.heads / p.cache.kv_heads, dim = p.cache.dim, lane = threadIdx.x & 63;
    const int request = blockIdx.x, kvh = blockIdx.y;
    const Kv8Request q = kv8_request(p.batch, request);
    const int tiles = tiles_of(q, group, share);
    if (!tiles) return;
    const int per = *(const int*)p.partial, steps = steps_of(q, p.window), parts = (steps + per - 1) / per;
    if (parts == 1) return;
    const int first = ((const int*)p.partial)[64 + request];
    for (int row = threadIdx.x >> 6; row < q.rows * group; row += kWaves) {
        const int tile = row / share.tile_rows;
        const float* part = partial_rows(p, (size_t)(first + (tiles - 1 - tile) * parts) * p.cache.kv_heads + kvh, share.tile_rows) +
                            (size_t)(row % share.tile_rows) * (dim + 2);
        const size_t stride = (size_t)p.cache.kv_heads * share.tile_rows * (dim + 2);
        float base = kNoBase, sum = 0.0f, x[4] = {0.0f, 0.0f, 0.0f, 0.0f};
        for (int i = 0; i < parts; ++i) base = fmaxf(base, part[i * stride + dim]);
        for (int i = 0; i < parts; ++i) {
            const float alpha = __builtin_amdgcn_exp2f(part[i * stride + dim] - base);
            sum = fmaf(part[i * stride + dim + 1], alpha, sum);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (lane + 64 * k < dim) x[k] = fmaf(part[i * stride + lane + 64 * k], alpha, x[k]);
        }
        float* out = p.out + ((size_t)(q.start + row / group) * p.heads + kvh * group + row % group) * dim;
#pragma unroll
        for (int k = 0; k < 4; ++k)
            if (lane + 64 * k < dim) out[lane + 64 * k] = x[k] / sum;
    }
}

// One wave a row (token, head), a key at a time.
__global__ __launch_bounds__(64) void attention_kv8_row_kernel(AttentionKv8Call p) {
    const KvBatchView& b = p.batch;
    const int t = blockIdx.x, h = blockIdx.y, lane = threadIdx.x, dim = p.cache.dim;
    const int kv_heads = p.cache.kv_heads, kvh = h / (p.heads / kv_heads);
    Kv8Request q{0, 0, 0};
    int r = 0;
    for (int base = 0; base < b.requests; base += 64) {
        Kv8Request mine{0, 0, 0};
        if (base + lane < b.requests) mine = kv8_request(b, base + lane);
        const uint64_t found = __ballot(t >= mine.start && t < mine.start + mine.rows);
        if (!found) continue;
        const int from = __builtin_ctzll(found);
        r = base + from;
        q = Kv8Request{__shfl(mine.start, from, 64), __shfl(mine.rows, from, 64), __shfl(mine.length, from, 64)};
        break;
    }
    if (q.rows * (p.heads / kv_heads) <= kFewRows) return;
    const int last = q.length - q.rows + (t - q.start), first = p.window ? max(0, last + 1 - p.window) : 0;
    float x[4], o[4] = {0.0f, 0.0f, 0.0f, 0.0f}, m = -INFINITY, l = 0.0f;
    bool spoilt = false;
#pragma unroll
    for (int c = 0; c < 4; ++c) {
        x[c] = lane + 64 * c < dim ? p.q_heads[((size_t)h * b.tokens + t) * dim + lane + 64 * c] : 0.0f;
        spoilt = spoilt || !finite_f32(x[c]);
    }
    spoilt = __any(spoilt);
    auto decode = [&](uint8_t c) { return p.cache.e4m3 ? __builtin_amdgcn_cvt_f32_fp8(c, 0) : (float)(int8_t)c; };
    for (int k = first; k <= last; ++k) {
        int id = b.table[(size_t)r * b.width + (k >> b.block_shift)];
        const bool known = (unsigned)id < (unsigned)b.blocks;
        if (!known) id = 0;
        const size_t at = (size_t)id * kv_heads + kvh;
        const int place = k & (b.block - 1);
        float s = 0.0f;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (lane + 64 * c < dim)
                s = fmaf(x[c], decode(p.cache.keys[(at * b.block + place) * dim + lane + 64 * c]), s);
        s = wave_sum_f32(s) * (p.cache.key_scales[at] * p.scale);
        const float sv = p.cache.value_scales[at];
        spoilt = spoilt || !known || !finite_f32(s) || !finite_f32(sv);
        const float top = fmaxf(m, s), a = expf(m - top), e = expf(s - top);
        m = top;
        l = l * a + e;
#pragma unroll
        for (int c = 0; c < 4; ++c)
            if (lane + 64 * c < dim)
                o[c] = o[c] * a + e * sv * decode(p.cache.values[(at * dim + lane + 64 * c) * b.block + place]);
    }
#pragma unroll
    for (int c = 0; c < 4; ++c)
        if (lane + 64 * c < dim)
            p.out[((size_t)t * p.heads + h) * dim + lane + 64 * c] = spoilt ? NAN : o[c] / l;
}

constexpr int kTarget = 768;                        // workgroups that the parts of a batch are cut for

Share few_share(const AttentionKv8Call&) { return Share{kFewRows, kTarget, kWaves, 1}; }

// At most this many items: a request's parts are fewer than its steps / per + 1.
size_t most_items(const AttentionKv8Call& call, const Share& share) {
    const size_t kv = call.cache.kv_heads;
    const size_t longest = ((size_t)call.batch.width * call.batch.block + kStep - 1) / kStep + 1;
    const size_t parts = std::min<size_t>((share.target + kv - 1) / kv + call.batch.requests,
                                          call.batch.requests * ((longest + share.least - 1) / share.least));
    return parts * kv;
}

template <int CC, bool FULL>
void launch_few(const AttentionKv8Call& call, const Share& share, hipStream_t stream) {
    const int grid = (int)most_items(call, share);
    if (call.cache.e4m3) attention_kv8_few_kernel<CC, FULL, true><<<grid, kThreads, 0, stream>>>(call, share);
    else attention_kv8_few_kernel<CC, FULL, false><<<grid, kThreads, 0, stream>>>(call, share);
}

}  // namespace

size_t attention_kv8_workspace_bytes(const AttentionKv8Call& call) {
    const Share share = few_share(call);
    return 4 * (64 + call.batch.requests + most_items(call, share) * share.tile_rows * (call.cache.dim + 2));
}

void launch_attention_kv8(const AttentionKv8Call& call, hipStream_t stream) {
    const int group = call.heads / call.cache.kv_heads, dim = call.cache.dim;
    if (group <= kFewRows) {
        const Share share = few_share(call);
        switch ((dim + 63) / 64 * 2 + (dim % 64 == 0)) {
        case 2: launch_few<1, false>(call, share, stream); break;
        case 3: launch_few<1, true>(call, share, stream); break;
        case 4: launch_few<2, false>(call, share, stream); break;
        case 5: launch_few<2, true>(call, share, stream); break;
        case 6: launch_few<3, false>(call, share, stream); break;
        case 7: launch_few<3, true>(call, share, stream); break;
        case 8: launch_few<4, false>(call, share, stream); break;
        default: launch_few<4, true>(call, share, stream); break;
        }
        attention_kv8_merge_kernel<<<dim3(call.batch.requests, call.cache.kv_heads), kThreads, 0, stream>>>(call, share);
    }
    if (call.batch.max_rows * group > kFewRows)
        attention_kv8_row_kernel<<<dim3(call.batch.tokens, call.heads), 64, 0, stream>>>(call);
}

}  // namespace leafhip
