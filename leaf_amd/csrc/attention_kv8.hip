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
// log2(e) / sqrt(dim); its weight is u = 2^(score - a + 8).  What meets the value
// codes is w = u v 2^-d of a value scale v = 2^e f, 1 <= f < 2: relative to the
// largest weight times value scale, so that it keeps its 22 bits wherever it counts
// however far the scales of blocks are apart, while the sum is of u, in which a key
// counts whatever its value's scale is.  a and d are whole numbers per row, a at most 6
// below the largest score and d at most 6 below the largest score - a + e so far
// (u < 2^14, w < 2^15), so most steps rescale nothing and a rescale is exact.  A row's
// output is its sum of w times codes, times 2^d, over its sum of u.  score - a + 8 is one
// fused operation where what the rounding of a's own score left out is little; past
// 2^22, where it grows to more than w has room for, scores are rounded before a is taken.
//
// Layout.  A step is 64 keys.  S^T = K Q^T by v_mfma_f32_16x16x32_f16 with lane
// l = 16 lq + li: row li of its tile j of keys is key 16 (li / 4) + 4 j + li % 4
// of the step, so that lane l then holds the scores of query row li for the 16
// keys 16 lq + 4 j + r in a row: P is the other operand of O^T = V^T P^T without
// leaving its registers, V's lanes read 16 codes of one dim (the cache keeps a
// dim's tokens together), and a lane's 16 keys lie in one block, with one scale.
// Both K and V come as 16-byte loads; a key's dims are permuted alike in Q.
//
// Two kernels: attention_kv8_few_kernel takes requests of at most 16 rows of a KV
// head and reads the cache straight into registers; attention_kv8_rows_kernel takes
// the others, or every request (see kManyTokens), and shares what it widens through
// LDS.  The keys of a tile of rows are cut into
// parts where a batch has too few tiles for the GPU, and a second launch joins
// the parts.  Lengths are known on the device only: every workgroup sums the
// batch and finds its own part (dependent loads, part of the 7 us that the smallest call takes).
#include <algorithm>
#include <atomic>
#include <climits>

#include "kv8.h"

namespace leafhip {
namespace {

typedef _Float16 v8h __attribute__((ext_vector_type(8)));
typedef _Float16 v2h __attribute__((ext_vector_type(2)));

constexpr int kStep = 64;                           // keys
constexpr int kWaves = 4;
constexpr int kThreads = 64 * kWaves;
constexpr int kFewRows = 16;                        // rows of a KV head in one tile
constexpr int kHeader = 4;                          // integers before a plan's requests
constexpr float kNoBase = -3e38f;
constexpr float kSlack = 6.0f, kLift = 8.0f;
constexpr float kFar = 4194304.0f;                  // 2^22: a score's rounding is an eighth below it (w has room for one)

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

// x = hi + lo to 22 bits, toward zero; x - hi in one instruction with hi as it is, an f16 half of a register.
__device__ __forceinline__ void split2(float x, float y, v2h& hi, v2h& lo) {
    hi = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_pkrtz(x, y));
    float dx, dy;
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel_hi:[1,0,0]" : "=v"(dx) : "v"(hi), "v"(x));
    asm("v_fma_mix_f32 %0, %1, -1.0, %2 op_sel:[1,0,0] op_sel_hi:[1,0,0]" : "=v"(dy) : "v"(hi), "v"(y));
    lo = __builtin_bit_cast(v2h, __builtin_amdgcn_cvt_pkrtz(dx, dy));
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
    float key, value;
    bool known;                                     // a block of the pool
    // NaN where the block spoils the rows that see it.  (Apart from the loads: what looks at a value waits for it, and
    // a step's are loaded a step ahead.)
    __device__ __forceinline__ KeyScales checked() const {
        return KeyScales{known && key >= 0.0f && key < INFINITY ? key : NAN,
                         known && value >= 0.0f && value < INFINITY ? value : NAN, known};
    }
};

// The keys of one request and KV head, for one lane.  A block's codes of a KV head are block * dim consecutive bytes,
// those of all heads `stride`; a step begins at the start of a block or 64 tokens into one of 128.
struct Keys {
    const int* table;
    const uint8_t *keys, *values;                   // of the KV head, in block 0
    const float *key_scales, *value_scales;
    uint32_t stride, kv_heads;
    int shift, blocks, dim, end;                    // end: keys of the request
    uint32_t key_lane, value_lane;                  // offset of the lane's first code in a block
    int key_group, value_group;                     // the lane's first key of a step, of its row of keys and its column of values

    __device__ __forceinline__ Keys(const AttentionKv8Call& p, int request, int kvh, int end_, int dim_, int li, int lq) {
        const KvBatchView& b = p.batch;
        table = b.table + (size_t)request * b.width;
        shift = b.block_shift;
        blocks = b.blocks;
        kv_heads = p.cache.kv_heads;
        dim = dim_;
        end = end_;
        const int mask = (1 << shift) - 1;
        stride = kv_heads * (uint32_t)dim << shift;
        keys = p.cache.keys + (size_t)kvh * (dim << shift);
        values = p.cache.values + (size_t)kvh * (dim << shift);
        key_scales = p.cache.key_scales + kvh;
        value_scales = p.cache.value_scales + kvh;
        key_group = 16 * (li >> 2);
        value_group = 16 * lq;
        key_lane = ((key_group & mask) + (li & 3)) * dim + 16 * lq;
        value_lane = (li << shift) + (value_group & mask);
    }
    __device__ __forceinline__ int block_of(int key) const { return table[(uint32_t)min(key, end - 1) >> shift]; }
    // The blocks of the lane's keys in a step: where its row of keys and its column of values are.
    __device__ __forceinline__ int key_block(int step) const { return block_of(step * kStep + key_group); }
    __device__ __forceinline__ int value_block(int step) const { return block_of(step * kStep + value_group); }
    __device__ __forceinline__ bool known(int id) const { return (unsigned)id < (unsigned)blocks; }
    __device__ __forceinline__ uint32_t in_block(int step) const { return step * kStep & ((1 << shift) - 1); }
    __device__ __forceinline__ KeyScales scales(int id) const {
        const uint64_t i = (uint64_t)(known(id) ? (uint32_t)id : 0u) * kv_heads;
        return KeyScales{key_scales[i], value_scales[i], known(id)};
    }
    // Where the lane's codes of a step begin.
    __device__ __forceinline__ const uint8_t* key_codes(int id, int step) const {
        return keys + (uint64_t)(known(id) ? (uint32_t)id : 0u) * stride + (key_lane + in_block(step) * dim);
    }
    __device__ __forceinline__ const uint8_t* value_codes(int id, int step) const {
        return values + (uint64_t)(known(id) ? (uint32_t)id : 0u) * stride + (value_lane + in_block(step));
    }
    // 16 codes from dim 64 cc + 16 lq on of key 16 (li / 4) + 4 j + li % 4 (FULL: dim is a multiple of 64).
    template <bool FULL>
    __device__ __forceinline__ v4u load_key(const uint8_t* codes, int j, int cc, int lq) const {
        if (!FULL && 64 * cc + 16 * lq >= dim) return v4u{0, 0, 0, 0};
        return *(const v4u*)(codes + 4 * j * dim + 64 * cc);
    }
    // 16 keys from 16 lq on of dim 16 t + li.
    __device__ __forceinline__ v4u load_value(const uint8_t* codes, int t) const { return *(const v4u*)(codes + (16 * t << shift)); }
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

// A row's online softmax: the bases of its weights and of its outputs (a and d above), and its sum (this lane's keys).
struct Softmax {
    float base = kNoBase, lift = 0.0f, sum = 0.0f;
    bool far = false;                               // of the wave: whether a base is past kFar
};

// What a row's outputs are multiplied by.
__device__ __forceinline__ float output_scale(float lift, float sum) { return __builtin_amdgcn_ldexpf(1.0f / sum, (int)lift); }
// The same of a part, of which a row may see no key.
__device__ __forceinline__ float part_scale(float lift, float sum) { return sum == 0.0f ? 0.0f : output_scale(lift, sum); }

// A step's scores to weights: acc [tile][r] are the products of key 4 tile + r of the lane's 16.
// MASKED: of these only keys [from, to) are visible.  Rescales sum and o where their bases move.
template <bool MASKED, int TILES>
__device__ __forceinline__ void weigh(v4f (&acc)[4], float c, KeyScales s, Softmax& m, v4f (&o)[TILES], int from, int to,
                                      v8h (&hi)[2], v8h (&lo)[2]) {
    const float e = (float)((int)(__float_as_uint(s.value) >> 23) - 127);
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
    top *= c;
    if (__any(top - m.base > kSlack || (top - m.base) + e > m.lift + kSlack)) {   // (a row's four lanes have the same bases)
        const float row_top = max_xor32(max_xor16(top));
        const float base = row_top - m.base > kSlack ? __builtin_ceilf(row_top) : m.base, moved = m.base - base;
        const float most = max_xor32(max_xor16((top - base) + e));
        // (the outputs' own base, base + lift, moves only where it has to)
        const float kept = m.lift + moved, lift = most > kept + kSlack ? __builtin_ceilf(most) : kept;
        const float alpha = __builtin_amdgcn_exp2f(kept - lift);
        m.sum *= __builtin_amdgcn_exp2f(moved);
        m.base = base;
        m.lift = lift;
        m.far = __any(__builtin_fabsf(base) > kFar && base != kNoBase);
#pragma unroll
        for (int t = 0; t < TILES; ++t) o[t] = o[t] * alpha;
    }
    float f = __builtin_amdgcn_ldexpf(s.value, -(int)m.lift);
    f = f > 0x1p127f ? 0x1p127f : f;                // (only where every u is below 2^-112; zero times infinity it may not be)
    const float shift = kLift - m.base;
    if (m.far) {
        const bool far = __builtin_fabsf(m.base) > kFar;           // a row's own: all of its waves weigh a score alike
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[j][r] = far ? (acc[j][r] * c - m.base) + kLift : fmaf(acc[j][r], c, shift);
    } else {
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) acc[j][r] = fmaf(acc[j][r], c, shift);
    }
    float sum = 0.0f;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        float w[4];
#pragma unroll
        for (int r = 0; r < 4; ++r) {
            float u = __builtin_amdgcn_exp2f(acc[j][r]);
            w[r] = u * f;
            if (MASKED && (4 * j + r < from || 4 * j + r >= to)) u = w[r] = 0.0f;
            sum += u;
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
    m.sum += sum;
}

// How a batch's work is shared out.  A request's rows of a KV head make tiles of
// `tile_rows`; a tile's steps are cut into equal parts of at most `per`, per
// chosen so that all parts of the batch are about `target` workgroups.  A request
// has workgroups for as many parts of each tile as its longest tile has.
struct Share {
    int tile_rows, target, least;                   // least: steps a part has at least
    int from, to;                                   // takes the requests of from..to rows of a KV head
    int items, slots;                               // of a KV head, that there are workgroups, and partial results, for
    size_t at;                                      // where its partial results begin: in floats
};
__device__ __forceinline__ int tiles_of(const Kv8Request& q, int group, const Share& share) {
    const int rows = q.rows * group;
    if (rows < share.from || rows > share.to) return 0;
    return (rows + share.tile_rows - 1) / share.tile_rows;
}
// The steps that a tile's rows see.
struct Steps {
    int begin, end;
};
__device__ __forceinline__ Steps steps_of(const Kv8Request& q, int group, int window, int tile_rows, int tile) {
    const int r0 = tile * tile_rows, last = min(r0 + tile_rows, q.rows * group) - 1, before = q.length - q.rows;
    return Steps{window ? max(0, before + r0 / group + 1 - window) / kStep : 0, (before + last / group) / kStep + 1};
}
// No tile of a request has more.
__device__ __forceinline__ int most_steps(const Kv8Request& q, int group, int window, int tile_rows) {
    const int all = (q.length - 1) / kStep + 1;
    return window ? (int)min((long long)all, ((long long)window + tile_rows / group) / kStep + 3) : all;
}
__device__ __forceinline__ int parts_of(int steps, int per) { return (steps + per - 1) / per; }

struct Item {
    int request, tile, part, slot;                  // slot: of the tile's first part among the KV head's partial results
    Kv8Request q;
};

// Which part of which tile of which request is item `index` (of one KV head);
// request -1: none.  Every workgroup sums the whole batch, a request a thread.
// The plan of a batch, for the merge, stands before the partial results: `per`, then each request's first slot.
__device__ __forceinline__ Item find_item(const AttentionKv8Call& p, int group, const Share& share, int index, int& per) {
    const KvBatchView& b = p.batch;
    const int window = p.window;
    __shared__ uint64_t sums[kWaves];
    __shared__ Item found;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    auto steps = [&](const Kv8Request& q) {
        return (float)tiles_of(q, group, share) * (float)most_steps(q, group, window, share.tile_rows);
    };
    Kv8Request mine{0, 0, 0};
    float all = 0.0f;
    for (int r = threadIdx.x; r < b.requests; r += kThreads) {
        mine = kv8_request(b, r);
        all += steps(mine);
    }
    all = wave_sum_f32(all);
    __shared__ float totals[kWaves];
    if (lane == 0) totals[wave] = all;
    if (threadIdx.x == 0) found.request = -1;
    __syncthreads();
    all = 0.0f;
#pragma unroll
    for (int w = 0; w < kWaves; ++w) all += totals[w];
    per = max(share.least, (int)fminf(all * (float)p.cache.kv_heads / (float)share.target * 1.0001f + 1.0f, 1e9f));
    // items, and of these the partial results (kept for tiles of several parts), before each request: two sums in one
    uint64_t before = 0;
    for (int base = 0; base < b.requests; base += kThreads) {
        const int r = base + threadIdx.x;
        if (b.requests > kThreads) mine = r < b.requests ? kv8_request(b, r) : Kv8Request{0, 0, 0};
        const int tiles = tiles_of(mine, group, share), parts = parts_of(most_steps(mine, group, window, share.tile_rows), per);
        // (what a batch's rows allow is far below the limits; requests that claim the same rows may not reach into the other sum)
        const uint64_t items = tiles ? min((long long)tiles * parts, 1LL << 27) : 0;
        const uint64_t own = items << 24 | (parts > 1 ? min((uint32_t)items, 4095u) : 0);
        uint64_t s = own;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const uint64_t below = __shfl_up((unsigned long long)s, o, 64);
            if (lane >= o) s += below;
        }
        if (lane == 63) sums[wave] = s;
        __syncthreads();
        uint64_t start = before + s - own;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) start += sums[w];
            before += sums[w];
        }
        const long long i = (long long)index - (long long)(start >> 24);
        const int slot = (int)(start & 0xFFFFFF);
        if (i >= 0 && i < (long long)items) {
            // the longest tiles (the last) first
            found = Item{r, tiles - 1 - (int)i / parts, (int)i % parts, slot + (int)i / parts * parts, mine};
        }
        // the first workgroup leaves the plan for the merge
        if (blockIdx.x == 0 && r < b.requests) ((int*)p.partial)[share.at + kHeader + r] = slot;
        if (blockIdx.x == 0 && r == 0) ((int*)p.partial)[share.at] = per;
        __syncthreads();
        if ((long long)index < (long long)(before >> 24) && blockIdx.x) break;
    }
    return found;
}

// Partial results: of each item its rows' outputs, rows by dim floats; behind all of them each row's base and sum.
__device__ __forceinline__ float* partial_values(const AttentionKv8Call& p, const Share& share, size_t item) {
    return p.partial + share.at + (kHeader + p.batch.requests + 3) / 4 * 4 + item * share.tile_rows * p.cache.dim;
}
__device__ __forceinline__ v2f* partial_sums(const AttentionKv8Call& p, const Share& share, size_t item) {
    return (v2f*)partial_values(p, share, (size_t)share.slots * p.cache.kv_heads) + item * share.tile_rows;
}

// ---- at most 16 rows of a KV head (single tokens): each wave takes every fourth step, straight from memory
// 64 requests of 200 to 4096 tokens, 32 heads of 128 over 8: 69 us and 5 for the
// join, 281 MB at 4.1 TB/s.  What bounds it is latency: without its arithmetic an
// earlier state took 65 of 77 us in all.  A CU has waves for 66% of the kernel's cycles,
// and issues vector instructions for 41% of those, 320 of some 680 a step of 64 keys
// widening codes (INT8, heads of 128).  A part is some eight steps a wave behind four
// dependent loads (its place, the query, the first table entries, the first codes); how
// much of the rest is these starts and how much parts that end unevenly is not shown.
// 8 requests of 16000 tokens take 57 us, 4.6 TB/s.
template <int CC, bool FULL, bool E4M3>
__global__ __launch_bounds__(kThreads, CC == 1 ? 3 : CC == 2 ? 2 : 1) void attention_kv8_few_kernel(AttentionKv8Call p, Share share) {
    constexpr int TILES = 4 * CC;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, lq = lane >> 4;
    const int kv_heads = p.cache.kv_heads, group = p.heads / kv_heads, dim = FULL ? 64 * CC : p.cache.dim;
    const int kvh = blockIdx.x % kv_heads, tiles = FULL ? TILES : dim / 16;
    int per;
    const Item item = find_item(p, group, share, blockIdx.x / kv_heads, per);
    if (item.request < 0) return;
    const Kv8Request& q = item.q;
    const int rows = q.rows * group, row = min(li, rows - 1);
    const int token = q.start + row / group, head = kvh * group + row % group;
    const int position = q.length - q.rows + row / group;
    const int low = q.length - q.rows;                             // of the first row
    const Steps seen = steps_of(q, group, p.window, share.tile_rows, 0);
    const int steps = seen.end - seen.begin, parts = parts_of(steps, per);
    if (item.part >= parts || (parts > 1 && item.slot > share.slots - parts)) return;
    const int begin = seen.begin + (int)((long long)item.part * steps / parts);
    const int end = seen.begin + (int)((long long)(item.part + 1) * steps / parts);
    const Keys keys(p, item.request, kvh, q.length, dim, li, lq);

    // Every load is issued a step ahead, as soon as its registers are free, and none under a condition, after which a
    // wait for an older one would be for all: past its end a wave loads its last step again.
    v4u kr[4][CC], vr[TILES];
    KeyScales scales;
    auto load_keys = [&](int id, int step) {
        const uint8_t* codes = keys.key_codes(id, step);
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int cc = 0; cc < CC; ++cc) kr[j][cc] = keys.load_key<FULL>(codes, j, cc, lq);
    };
    auto load_values = [&](int id, int step) {
        const uint8_t* codes = keys.value_codes(id, step);
#pragma unroll
        for (int t = 0; t < TILES; ++t) vr[t] = keys.load_value(codes, FULL ? t : min(t, tiles - 1));
        scales = keys.scales(id);
    };

    v8h qh[CC][2], ql[CC][2];
    float c;
    int step = begin + wave;
    const int last = step < end ? step + (end - 1 - step) / kWaves * kWaves : begin;
    auto after = [&](int s) { return min(s, last); };
    int ik = keys.key_block(after(step)), iv = keys.value_block(after(step));
    load_query<CC, FULL>(p.q_heads + ((size_t)head * p.batch.tokens + token) * dim, dim, lq, p.scale, qh, ql, c);
    load_keys(ik, after(step));
    load_values(iv, after(step));
    ik = keys.key_block(after(step + kWaves));
    iv = keys.value_block(after(step + kWaves));
    v4f o[TILES];
#pragma unroll
    for (int t = 0; t < TILES; ++t) o[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    Softmax m;
    for (; step < end; step += kWaves) {
        v4f acc[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int cc = 0; cc < CC; ++cc) {
            v8h k[4][2];
#pragma unroll
            for (int j = 0; j < 4; ++j) widen<E4M3>(kr[j][cc], k[j][0], k[j][1]);
            // (no product waits for the one before it)
#pragma unroll
            for (int h = 0; h < 2; ++h) {
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[j][h], ql[cc][h], acc[j], 0, 0, 0);
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[j][h], qh[cc][h], acc[j], 0, 0, 0);
            }
        }
        load_keys(ik, after(step + kWaves));
        ik = keys.key_block(after(step + 2 * kWaves));
        v8h hi[2], lo[2];
        const KeyScales now = scales.checked();
        const int at = step * kStep + 16 * lq;                     // the lane's first key
        if (step * kStep + kStep > low + 1 || p.window) {          // the wave's rows see different keys
            const int from = p.window ? position + 1 - p.window - at : 0;
            weigh<true>(acc, c, now, m, o, from, position + 1 - at, hi, lo);
            // (codes that no token wrote, or of no block, may be NaN, which no weight of zero stops)
            const int written = now.known ? q.length - at : 0;
#pragma unroll
            for (int t = 0; t < TILES; ++t) vr[t] = first_codes(vr[t], written);
        } else {
            weigh<false>(acc, c, now, m, o, 0, 16, hi, lo);
        }
#pragma unroll
        for (int t = 0; t < TILES; ++t)
            if (FULL || t <= 4 * CC - 4 || t < tiles) {            // (a head has more than 64 (CC - 1) dims)
                v8h v[2];
                widen<E4M3>(vr[t], v[0], v[1]);
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[h], lo[h], o[t], 0, 0, 0);
                    o[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[h], hi[h], o[t], 0, 0, 0);
                }
            }
        load_values(iv, after(step + kWaves));
        iv = keys.value_block(after(step + 2 * kWaves));
    }

    // ---- the four waves' states together; wave w then has the tiles t % 4 = w
    __shared__ v4f values[kWaves][TILES][64];
    __shared__ float bases[kWaves][16], lifts[kWaves][16], sums[kWaves][16];
    m.sum = add_xor32(add_xor16(m.sum));
    if (lq == 0) {
        bases[wave][li] = m.base;
        lifts[wave][li] = m.lift;
        sums[wave][li] = m.sum;
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t)
        if (FULL || t < tiles) values[wave][t][lane] = o[t];
    __syncthreads();
    float base = kNoBase, lift = -INFINITY, sum = 0.0f, alpha[kWaves];
#pragma unroll
    for (int w = 0; w < kWaves; ++w) base = fmaxf(base, bases[w][li]);
#pragma unroll
    for (int w = 0; w < kWaves; ++w) {
        const float below = bases[w][li] - base;
        sum = fmaf(sums[w][li], __builtin_amdgcn_exp2f(below), sum);
        alpha[w] = below + lifts[w][li];
        lift = fmaxf(lift, alpha[w]);
    }
#pragma unroll
    for (int w = 0; w < kWaves; ++w) alpha[w] = __builtin_amdgcn_exp2f(alpha[w] - lift);
    if (li >= rows) return;
    const size_t slot = (size_t)(item.slot + item.part) * kv_heads + kvh;
    float* to = p.out + ((size_t)token * p.heads + head) * dim;
    float scale = output_scale(lift, sum);
    if (parts > 1) {
        to = partial_values(p, share, slot) + (size_t)li * dim;
        scale = part_scale(lift, sum);
        if (wave == 0 && lq == 0) partial_sums(p, share, slot)[li] = v2f{base, sum};
    }
    for (int t = wave; t < tiles; t += kWaves) {
        v4f x = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const v4f v = values[w][t][lane];
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = fmaf(v[r], alpha[w], x[r]);
        }
        *(v4f*)(to + 16 * t + 4 * lq) = x * scale;
    }
}

// ---- more rows of a KV head: tiles of 64, 16 for a wave, K and V widened once for all of them through LDS
// 512 tokens behind 7001 keys, 32 heads of 128 over 8 (E4M3): 137 to 147 us, about
// 10 of them the join's; 2048 tokens of 14 heads of 64 over 2 (INT8): 44 to 46, 7 the join's.
// What bounds the chunk is issue: a CU has waves for 87% of the kernel's cycles, and of those
// other vector instructions (252 a step of 16 scores a lane, some 80 of them widening codes)
// take 41% and MFMAs 42%.  The prompt leaves CUs idle first: they have waves for 59% of the
// cycles, of which vector instructions take 57% and MFMAs 22%.  Its tiles see from one step
// to all, while parts are cut, and workgroups launched, for tiles as long as the last.  Two row tiles
// a wave (54 us for the prompt, 138 for the chunk, with spills), three or four waves a
// SIMD in fewer registers (47 and 169), and eight waves in two groups half a step apart, one
// in its products while the other is in its softmax (62 and 143), gave nothing.
constexpr int kTileRows = 16 * kWaves;

template <int CC, bool FULL, bool E4M3>
__global__ __launch_bounds__(kThreads, CC <= 2 ? 2 : 1) void attention_kv8_rows_kernel(AttentionKv8Call p, Share share) {
    constexpr int TILES = 4 * CC;
    constexpr int kOperand = 64 * 16;                              // bytes of one operand of a wave
    constexpr int kKeyBytes = 4 * CC * 2 * kOperand, kBuffer = 2 * kKeyBytes;
    extern __shared__ __align__(16) uint8_t lds[];                 // two of [tile of keys][cc][half][lane], [tile of dims][half][lane]
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), li = lane & 15, lq = lane >> 4;
    const int kv_heads = p.cache.kv_heads, group = p.heads / kv_heads, dim = FULL ? 64 * CC : p.cache.dim;
    const int kvh = blockIdx.x % kv_heads, tiles = FULL ? TILES : dim / 16;
    int per;
    const Item item = find_item(p, group, share, blockIdx.x / kv_heads, per);
    if (item.request < 0) return;
    const Kv8Request& q = item.q;
    const int rows = q.rows * group, w0 = item.tile * kTileRows + 16 * wave;   // the wave's first row
    const int before = q.length - q.rows;                          // position of the first row
    const Steps seen = steps_of(q, group, p.window, kTileRows, item.tile);
    const int steps = seen.end - seen.begin, parts = parts_of(steps, per);
    if (item.part >= parts || (parts > 1 && item.slot > share.slots - parts)) return;
    const int begin = seen.begin + (int)((long long)item.part * steps / parts);
    const int end = seen.begin + (int)((long long)(item.part + 1) * steps / parts);
    const Keys keys(p, item.request, kvh, q.length, dim, li, lq);
    const int row = min(w0 + li, rows - 1), token = q.start + row / group, head = kvh * group + row % group;
    const int position = before + row / group;
    v8h qh[CC][2], ql[CC][2];
    float c;
    load_query<CC, FULL>(p.q_heads + ((size_t)head * p.batch.tokens + token) * dim, dim, lq, p.scale, qh, ql, c);
    // of the wave's rows: the first sees every key up to `low`, the last none after `high`
    const int low = before + min(w0, rows - 1) / group;
    const int high = w0 < rows ? before + min(w0 + 15, rows - 1) / group : -1;

    // staging: wave w widens tile w of the keys and the tiles w, w + 4.. of the dims
    v4u kr[CC], vr[CC];
    bool known = true;
    auto load = [&](int step, int ik, int iv) {
        const uint8_t *kc = keys.key_codes(ik, step), *vc = keys.value_codes(iv, step);
        known = keys.known(iv);
#pragma unroll
        for (int cc = 0; cc < CC; ++cc) {
            kr[cc] = keys.load_key<FULL>(kc, wave, cc, lq);
            vr[cc] = keys.load_value(vc, FULL ? wave + 4 * cc : min(wave + 4 * cc, tiles - 1));
        }
    };
    auto store = [&](int step) {
        uint8_t* buffer = lds + (step & 1) * kBuffer;
        // (codes that no token wrote, or of no block, may be NaN, which no weight of zero stops)
        const bool clear = E4M3 && (step * kStep + kStep > q.length || !__all(known));
#pragma unroll
        for (int cc = 0; cc < CC; ++cc) {
            v8h a, b;
            widen<E4M3>(kr[cc], a, b);
            v8h* to = (v8h*)(buffer + ((wave * CC + cc) * 2) * kOperand) + lane;
            to[0] = a;
            to[64] = b;
            if (clear) vr[cc] = first_codes(vr[cc], known ? q.length - (step * kStep + 16 * lq) : 0);
            widen<E4M3>(vr[cc], a, b);
            to = (v8h*)(buffer + kKeyBytes + ((wave + 4 * cc) * 2) * kOperand) + lane;
            to[0] = a;
            to[64] = b;
        }
    };

    v4f o[TILES];
    Softmax m;
#pragma unroll
    for (int t = 0; t < TILES; ++t) o[t] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
    // Every load is used a step later and none issued under a condition, after which a wait for an older one would be
    // for all; past the end they are the last block's and not used.
    load(begin, keys.key_block(begin), keys.value_block(begin));
    store(begin);
    load(begin + 1, keys.key_block(begin + 1), keys.value_block(begin + 1));
    KeyScales scales = keys.scales(keys.value_block(begin));
    int ik = keys.key_block(begin + 2), iv = keys.value_block(begin + 2), is = keys.value_block(begin + 1);
    lds_barrier();
    for (int step = begin; step < end; ++step) {
        const uint8_t* buffer = lds + (step & 1) * kBuffer;
        store(step + 1);
        load(step + 2, ik, iv);
        ik = keys.key_block(step + 3);
        iv = keys.value_block(step + 3);
        const KeyScales now = scales.checked();
        const bool idle = step * kStep > high || (p.window && step * kStep + kStep <= low + 1 - p.window);
        if (!idle) {
            v4f acc[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[j] = v4f{0.0f, 0.0f, 0.0f, 0.0f};
            // (no product waits for the one before it)
#pragma unroll
            for (int cc = 0; cc < CC; ++cc)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    v8h k[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) k[j] = *((const v8h*)(buffer + ((j * CC + cc) * 2 + h) * kOperand) + lane);
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[j], ql[cc][h], acc[j], 0, 0, 0);
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k[j], qh[cc][h], acc[j], 0, 0, 0);
                }
            v8h hi[2], lo[2];
            const int at = step * kStep + 16 * lq;
            if (step * kStep + kStep > low + 1 || (p.window && step * kStep <= high - p.window)) {
                const int from = p.window ? position + 1 - p.window - at : 0;
                weigh<true>(acc, c, now, m, o, from, position + 1 - at, hi, lo);
            } else {
                weigh<false>(acc, c, now, m, o, 0, 16, hi, lo);
            }
#pragma unroll
            for (int t0 = 0; t0 < TILES; t0 += 4) {
                if (!FULL && t0 >= tiles) continue;                // (tiles past the last: copies of it, not kept)
#pragma unroll
                for (int h = 0; h < 2; ++h) {
                    v8h v[4];
#pragma unroll
                    for (int t = 0; t < 4; ++t) v[t] = *((const v8h*)(buffer + kKeyBytes + ((t0 + t) * 2 + h) * kOperand) + lane);
#pragma unroll
                    for (int t = 0; t < 4; ++t) o[t0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[t], lo[h], o[t0 + t], 0, 0, 0);
#pragma unroll
                    for (int t = 0; t < 4; ++t) o[t0 + t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v[t], hi[h], o[t0 + t], 0, 0, 0);
                }
            }
        }
        scales = keys.scales(is);
        is = keys.value_block(step + 2);
        lds_barrier();                                             // (the next loads stay in flight)
    }

    const float sum = add_xor32(add_xor16(m.sum));
    if (w0 + li >= rows) return;
    float* to = p.out + ((size_t)token * p.heads + head) * dim;
    float scale = output_scale(m.lift, sum);
    if (parts > 1) {
        const size_t slot = (size_t)(item.slot + item.part) * kv_heads + kvh;
        to = partial_values(p, share, slot) + (size_t)(16 * wave + li) * dim;
        scale = part_scale(m.lift, sum);
        if (lq == 0) partial_sums(p, share, slot)[16 * wave + li] = v2f{m.base, sum};
    }
#pragma unroll
    for (int t = 0; t < TILES; ++t)
        if (FULL || t < tiles) *(v4f*)(to + 16 * t + 4 * lq) = o[t] * scale;
}

// A row's parts together: its base, and its sum relative to that.
__device__ __forceinline__ void add_part(v2f part, float& base, float& total) {
    const float most = fmaxf(base, part.x);
    total = fmaf(total, __builtin_amdgcn_exp2f(base - most), part.y * __builtin_amdgcn_exp2f(part.x - most));
    base = most;
}
// What a part's outputs count for: at most one, so that no output is too large or too small for the sum.
__device__ __forceinline__ float part_share(v2f part, float base, float inverse) {
    return part.y * __builtin_amdgcn_exp2f(part.x - base) * inverse;
}

// ---- rows whose keys were parted, of at most 16 rows of a KV head: a wave for each token and head, every lane four
// values of one part at a time
__global__ __launch_bounds__(1024) void attention_kv8_few_merge_kernel(AttentionKv8Call p, Share share) {
    const int group = p.heads / p.cache.kv_heads, dim = p.cache.dim, lane = threadIdx.x & 63;
    const int request = blockIdx.x, kvh = blockIdx.y;
    const Kv8Request q = kv8_request(p.batch, request);
    if (!tiles_of(q, group, share)) return;
    const int* plan = (const int*)p.partial + share.at;
    const Steps seen = steps_of(q, group, p.window, share.tile_rows, 0);
    const int parts = parts_of(seen.end - seen.begin, plan[0]), item = plan[kHeader + request];
    // (requests that claim the same rows can have more parts than there is room for: such rows stay undefined)
    if (parts == 1 || item < 0 || item > share.slots - parts) return;
    const size_t kv_heads = p.cache.kv_heads, slot = (size_t)item * kv_heads + kvh;
    const size_t sum_stride = kv_heads * share.tile_rows, stride = sum_stride * dim;
    // lanes: (part i0 + lane / quads, quad lane % quads) of rows of up to 64 quads
    const int quads = dim / 4, abreast = 64 / quads, quad = lane % quads, own = lane / quads;
    for (int row = threadIdx.x >> 6; row < q.rows * group; row += blockDim.x >> 6) {
        const v2f* sums = partial_sums(p, share, slot) + row;
        const float* values = partial_values(p, share, slot) + (size_t)row * dim;
        float base = kNoBase, total = 0.0f;
        for (int i = lane; i < parts; i += 64) add_part(sums[i * sum_stride], base, total);
        const float own_base = base;
        base = wave_max_f32(base);
        const float inverse = 1.0f / wave_sum_f32(total * __builtin_amdgcn_exp2f(own_base - base));
        v4f x = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        if (own < abreast) {
#pragma unroll 4
            for (int i = own; i < parts; i += abreast) {
                const float share_of = part_share(sums[i * sum_stride], base, inverse);
                const v4f v = *(const v4f*)(values + i * stride + 4 * quad);
#pragma unroll
                for (int r = 0; r < 4; ++r) x[r] = fmaf(v[r], share_of, x[r]);
            }
        }
        // the parts abreast together, in their order
        v4f all = v4f{0.0f, 0.0f, 0.0f, 0.0f};
        for (int k = 0; k < abreast; ++k)
#pragma unroll
            for (int r = 0; r < 4; ++r) all[r] += __shfl(x[r], k * quads + quad, 64);
        if (own == 0) *(v4f*)(p.out + ((size_t)(q.start + row / group) * p.heads + kvh * group + row % group) * dim + 4 * quad) = all;
    }
}

// ---- the same of more rows: some workgroups a tile, a thread for four values of a row
constexpr int kMergeSplit = 4;                      // workgroups of a tile (2 / 4 / 8: a chunk beside decoding requests 45 / 44 / 48 us)
__global__ __launch_bounds__(kThreads) void attention_kv8_rows_merge_kernel(AttentionKv8Call p, Share share) {
    __shared__ int sums_of[kWaves], found[5];
    const int group = p.heads / p.cache.kv_heads, dim = p.cache.dim, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int kvh = blockIdx.x / kMergeSplit % p.cache.kv_heads, index = blockIdx.x / kMergeSplit / p.cache.kv_heads;
    // tile `index` of the batch
    if (threadIdx.x == 0) found[0] = -1;
    __syncthreads();
    int before = 0;
    for (int base = 0; base < p.batch.requests; base += kThreads) {
        const int r = base + threadIdx.x;
        const Kv8Request mine = r < p.batch.requests ? kv8_request(p.batch, r) : Kv8Request{0, 0, 0};
        const int tiles = tiles_of(mine, group, share);
        int s = tiles;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const int below = __shfl_up(s, o, 64);
            if (lane >= o) s += below;
        }
        if (lane == 63) sums_of[wave] = s;
        __syncthreads();
        int start = before + s - tiles;
        for (int w = 0; w < kWaves; ++w) {
            if (w < wave) start += sums_of[w];
            before += sums_of[w];
        }
        if (index >= start && index < start + tiles) {
            found[0] = r;
            found[1] = tiles - 1 - (index - start);
            found[2] = mine.start;
            found[3] = mine.rows;
            found[4] = mine.length;
        }
        __syncthreads();
        if (index < before) break;
    }
    if (found[0] < 0) return;
    const int request = found[0], tile = found[1];
    const Kv8Request q{found[2], found[3], found[4]};
    const int* plan = (const int*)p.partial + share.at;
    const int per = plan[0], first = plan[kHeader + request];
    const Steps seen = steps_of(q, group, p.window, share.tile_rows, tile);
    const int parts = parts_of(seen.end - seen.begin, per);
    const int item = first + (tiles_of(q, group, share) - 1 - tile) * parts_of(most_steps(q, group, p.window, share.tile_rows), per);
    if (parts == 1 || item < 0 || item > share.slots - parts) return;
    const size_t kv_heads = p.cache.kv_heads, slot = (size_t)item * kv_heads + kvh;
    const size_t sum_stride = kv_heads * share.tile_rows, stride = sum_stride * dim;
    const int r0 = tile * share.tile_rows, rows = min(share.tile_rows, q.rows * group - r0), quads = dim / 4;
    for (int u = blockIdx.x % kMergeSplit * kThreads + threadIdx.x; u < rows * quads; u += kMergeSplit * kThreads) {
        const int row = u / quads, quad = u % quads;
        const v2f* sums = partial_sums(p, share, slot) + row;
        const float* values = partial_values(p, share, slot) + (size_t)row * dim + 4 * quad;
        float base = kNoBase, total = 0.0f;
        v4f x = v4f{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int i = 0; i < parts; ++i) add_part(sums[i * sum_stride], base, total);
        const float inverse = 1.0f / total;
#pragma unroll 4
        for (int i = 0; i < parts; ++i) {
            const float share_of = part_share(sums[i * sum_stride], base, inverse);
            const v4f v = *(const v4f*)(values + i * stride);
#pragma unroll
            for (int r = 0; r < 4; ++r) x[r] = fmaf(v[r], share_of, x[r]);
        }
        *(v4f*)(p.out + ((size_t)(q.start + (r0 + row) / group) * p.heads + kvh * group + (r0 + row) % group) * dim + 4 * quad) = x;
    }
}

// Workgroups that a batch's keys are cut for, about those that the GPU holds at once: more are more partial results and
// more starts, fewer leave CUs idle.  Of few rows, with 512 / 768 / 1024: heads of 64, 100 requests 23 / 26 / 27 us, heads
// of 128, 64 ragged requests 73 / 68 / 74 and 8 long ones 57 / 67 / 62; of many rows, heads of 64, a prompt of 2048
// tokens 54 / 46 / 47, heads of 128, a chunk of 512 138 / 152 / 150.
constexpr int few_target(int cc) { return cc <= 2 ? 512 : 256; }
constexpr int rows_target(int cc) { return cc == 1 ? 768 : cc == 2 ? 512 : 256; }
// Steps of a part at least, with 4 / 8: one request of 4095 tokens 10.9 / 12.5 us (a part's wave has one or two steps);
// eight prompts of 300 tokens 37 / 27 (none is parted with 8; 16 costs a chunk beside decoding requests 47 for 44).
constexpr int kFewLeast = 4, kRowsLeast = 8;
// Rows of the step for each request from which the kernel of many rows takes every request: one launch in place of
// two, one after the other, although it has a request of one token in a tile of 64.  At 13 a request it takes 75 us for 73
// (heads of 128) and at 8 30 for 40 (heads of 64), at 3.5 203 for 151 and 39 for 45; between 3.5 and 8 nothing was
// measured.  The host knows the batch's sizes alone, so padding rows count: 64 single tokens in 512 rows take 110 us for
// 74 (heads of 128) and 43 for 24 (heads of 64) where max_rows lets the rows be one request's.
constexpr int kManyTokens = 6;

// At most this many tiles, and items, of a KV head: a tile's parts are at most its steps / per + 1.
int most_tiles(const AttentionKv8Call& call, const Share& share) {
    const size_t group = call.heads / call.cache.kv_heads;
    size_t tiles = std::min(call.batch.requests, call.batch.tokens);
    if (share.tile_rows > kFewRows) tiles += (size_t)call.batch.tokens * group / share.tile_rows;
    return (int)tiles;
}
int most_items(const AttentionKv8Call& call, const Share& share) {
    const size_t kv = call.cache.kv_heads, tiles = most_tiles(call, share);
    const size_t longest = ((size_t)call.batch.width * call.batch.block + kStep - 1) / kStep + 1;
    return (int)std::min<size_t>((share.target + kv - 1) / kv + tiles, tiles * ((longest + share.least - 1) / share.least));
}

// Partial results: a tile of several parts has more steps than `per`, so at most twice its steps / per.
int most_slots(const AttentionKv8Call& call, const Share& share) {
    return std::min(share.items, 2 * ((share.target + call.cache.kv_heads - 1) / call.cache.kv_heads) + 1);
}

size_t partial_floats(const AttentionKv8Call& call, const Share& share) {
    return (kHeader + call.batch.requests + 3) / 4 * 4 + (size_t)share.slots * call.cache.kv_heads * share.tile_rows * (call.cache.dim + 2);
}

// Which kernel takes which requests, and where in the workspace.
struct Shares {
    Share few, many;
    size_t floats;
};
Shares shares_of(const AttentionKv8Call& call) {
    const int group = call.heads / call.cache.kv_heads;
    const bool only_many = group > kFewRows || call.batch.tokens / kManyTokens >= call.batch.requests;
    const bool only_few = (size_t)call.batch.max_rows * group <= kFewRows;
    const int cc = (call.cache.dim + 63) / 64;
    Shares s{{kFewRows, few_target(cc), kFewLeast, 1, kFewRows, 0, 0, 0},
             {kTileRows, rows_target(cc), kRowsLeast, only_many ? 1 : kFewRows + 1, INT_MAX, 0, 0, 0}, 0};
    if (only_few || !only_many) {
        s.few.items = most_items(call, s.few);
        s.few.slots = most_slots(call, s.few);
        s.many.at = (partial_floats(call, s.few) + 3) / 4 * 4;
        s.floats = s.many.at;
    }
    if (!only_few) {
        s.many.items = most_items(call, s.many);
        s.many.slots = most_slots(call, s.many);
        s.floats = s.many.at + partial_floats(call, s.many);
    }
    return s;
}

template <int CC, bool FULL, bool E4M3>
void launch(const AttentionKv8Call& call, const Share& share, hipStream_t stream) {
    const int grid = share.items * call.cache.kv_heads;
    if (share.tile_rows == kFewRows) {
        attention_kv8_few_kernel<CC, FULL, E4M3><<<grid, kThreads, 0, stream>>>(call, share);
        return;
    }
    constexpr int kLds = 2 * 16 * CC * 1024;
    constexpr auto kernel = attention_kv8_rows_kernel<CC, FULL, E4M3>;
    if (kLds >= 65536) {                            // more than the default, with the static arrays: allowed once a device
        static std::atomic<uint64_t> allowed{0};
        int device = 0;
        (void)hipGetDevice(&device);
        if (!(allowed >> (device & 63) & 1) &&
            hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, kLds) == hipSuccess)
            allowed |= 1ull << (device & 63);
    }
    kernel<<<grid, kThreads, kLds, stream>>>(call, share);
}

template <int CC, bool FULL>
void launch(const AttentionKv8Call& call, const Share& share, hipStream_t stream) {
    if (call.cache.e4m3) launch<CC, FULL, true>(call, share, stream);
    else launch<CC, FULL, false>(call, share, stream);
}

}  // namespace

size_t attention_kv8_workspace_bytes(const AttentionKv8Call& call) { return 4 * shares_of(call).floats; }

void launch_attention_kv8(const AttentionKv8Call& call, hipStream_t stream) {
    const int dim = call.cache.dim, group = call.heads / call.cache.kv_heads;
    const Shares shares = shares_of(call);
    for (const Share& share : {shares.few, shares.many}) {
        if (!share.items) continue;
        switch ((dim + 63) / 64 * 2 + (dim % 64 == 0)) {
        case 2: launch<1, false>(call, share, stream); break;
        case 3: launch<1, true>(call, share, stream); break;
        case 4: launch<2, false>(call, share, stream); break;
        case 5: launch<2, true>(call, share, stream); break;
        case 6: launch<3, false>(call, share, stream); break;
        case 7: launch<3, true>(call, share, stream); break;
        case 8: launch<4, false>(call, share, stream); break;
        default: launch<4, true>(call, share, stream); break;
        }
    }
    // (no tile is parted that has no more steps than a part at least)
    const size_t steps = ((size_t)call.batch.width << call.batch.block_shift) / kStep + 1;
    if (shares.few.items && steps > (size_t)kFewLeast)
        attention_kv8_few_merge_kernel<<<dim3(call.batch.requests, call.cache.kv_heads),
                                         64 * (int)std::min<int64_t>(kFewRows, (int64_t)group * call.batch.max_rows), 0, stream>>>(call, shares.few);
    if (shares.many.items && steps > (size_t)kRowsLeast)
        attention_kv8_rows_merge_kernel<<<most_tiles(call, shares.many) * call.cache.kv_heads * kMergeSplit, kThreads, 0, stream>>>(
            call, shares.many);
}

}  // namespace leafhip
