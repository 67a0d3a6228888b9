// Causal grouped-query attention of a ragged batch over an 8-bit cache in
// blocks (include/leafhip.h: lh_attention_kv8).
#include <algorithm>

#include "kv8.h"

namespace leafhip {
namespace {

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
    if (!q.rows) return;
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

}  // namespace

size_t attention_kv8_workspace_bytes(const AttentionKv8Call&) { return 0; }

void launch_attention_kv8(const AttentionKv8Call& call, hipStream_t stream) {
    attention_kv8_row_kernel<<<dim3(call.batch.tokens, call.heads), 64, 0, stream>>>(call);
}

}  // namespace leafhip
