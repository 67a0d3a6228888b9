// Which drafted tokens of a step stand, and the token behind them
// (include/leafhip.h: lh_verify_drafts).
//
// With w(x) = 2^((l(x) - m) c) of a row's logits l, m their largest and c =
// log2(e) / T, the target's probabilities are w / Z, the draft's v / Y.  A row's
// first k children refused leave the target's weights r = max(w - K v, 0), K = C Z /
// Y with C = 0 at first and C + (sum of r) / Z after each (a maximum of
// differences with zero, one in the other, is one with their sum); of drafts
// without probabilities, w without the refused tokens.  A child with token x is
// taken if u (sum of r) v(x) / Y < r(x), or u (sum of r) < r(x).
//
// All sums and weights are 64-bit: the last token is the one at whose weight the
// sums in order pass u times all, and among 10^5 tokens an f32 sum would often be
// on the other side of it.
//
// A workgroup walks a request's tree and reads only the rows on its way.  Each
// wave has a contiguous share of the vocabulary: the shares' sums say where the
// last token is, and its share alone is read again.
#include "kv8.h"

namespace leafhip {
namespace {

constexpr int kThreads = 1024;
constexpr int kWaves = kThreads / 64;
constexpr int kBatch = 16;                          // values that a thread has in flight
constexpr int kTable = 64;                          // powers of two of a step

// 2^y for y <= 0 (0 below 2^-1000), to 1e-15: table[j] = 2^(j / 64), 2^f by its series for |f| <= 1/128.
__device__ __forceinline__ double power(double y, const double* table) {
    const double shift = 6755399441055744.0 / kTable;              // 1.5 * 2^52 / 64: the sum's last bit is 1/64
    const double t = fmax(y, -1000.0) + shift, f = fmax(y, -1000.0) - (t - shift);
    const int n = __double2loint(t);                               // 64 y to the nearest
    double s = 1.3333558146428443e-3;                              // ln2^k / k!
    s = fma(s, f, 9.618129107628477e-3);
    s = fma(s, f, 5.550410866482158e-2);
    s = fma(s, f, 2.402265069591007e-1);
    s = fma(s, f, 6.931471805599453e-1);
    s = fma(s, f, 1.0);
    s *= table[n & (kTable - 1)];
    const double p = __hiloint2double(__double2hiint(s) + ((n >> 6) << 20), __double2loint(s));
    return y < -1000.0 ? 0.0 : p;
}

// A row of logits in weights.
struct Row {
    const float* logits;
    float most;
    double total;                                   // the sum of its weights
};

struct Shared {
    double table[kTable];
    double sums[kWaves];                            // of each share: of what is left,
    double whole[kWaves];                           // of the target's weights
    double scan[kWaves];
    float tops[kWaves];
    int where[kWaves];
    int parents[kTreeRows], ids[kTreeRows], refused[kTreeRows];
    float accept[kTreeRows];
    int found;
};

// What the walk is at: the target's row, the draft's, and what refusals have left.
struct State {
    Row target, draft;
    bool bad;                                       // no distribution
    int best;                                       // greedy: the first largest
    double scale;                                   // K; 0: nothing refused
    double used;                                    // C
    double left;                                    // the sum of r
    int refusals;                                   // tokens in `refused`
};

__device__ __forceinline__ double weight(const Row& row, int x, double c, const double* table) {
    return power(((double)row.logits[x] - (double)row.most) * c, table);
}

// The sum of v over the workgroup's waves, each wave's in `sums` too.
__device__ __forceinline__ double sum_shares(double v, double* sums) {
    v = wave_sum_f64(v);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sums[threadIdx.x >> 6] = v;
    __syncthreads();
    double all = 0.0;
    for (int w = 0; w < kWaves; ++w) all += sums[w];
    return all;
}

struct Walk {
    const VerifyCall& p;
    Shared& s;
    double c;                                       // log2(e) / T
    int share;                                      // values of a wave's share

    __device__ __forceinline__ int begin(int wave) const { return min(wave * share, p.vocab); }

    // A row's largest value, its first place, and the sum of its weights (each share's in `sums`); false: no distribution.
    __device__ bool measure(Row& row, int& best, bool greedy, double* sums) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, end = begin(wave + 1);
        float most = -INFINITY;
        int at = p.vocab;
        double sum = 0.0;
        bool wrong = false;
        for (int base = begin(wave) + lane; base < end; base += 64 * kBatch) {
            float l[kBatch], top = -INFINITY;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) l[i] = base + 64 * i < end ? row.logits[base + 64 * i] : -INFINITY;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) {
                wrong = wrong || !(l[i] < INFINITY);
                top = fmaxf(top, l[i]);
            }
            if (greedy) {
                if (top > most) {
#pragma unroll
                    for (int i = kBatch - 1; i >= 0; --i)
                        if (l[i] == top) at = base + 64 * i;
                    most = top;
                }
                continue;
            }
            if (top > most) {
                if (most > -INFINITY) sum *= power(((double)most - (double)top) * c, s.table);
                most = top;
            }
            if (most == -INFINITY) continue;
#pragma unroll
            for (int i = 0; i < kBatch; ++i) sum += l[i] > -INFINITY ? power(((double)l[i] - (double)most) * c, s.table) : 0.0;
        }
        float top = wave_max_f32(most);
        int place = most == top ? at : p.vocab;
        for (int o = 32; o > 0; o >>= 1) place = min(place, __shfl_xor(place, o, 64));
        if (lane == 0) {
            s.tops[wave] = top;
            s.where[wave] = place;
        }
        wrong = __syncthreads_or(wrong);
        top = s.tops[0];
        for (int w = 1; w < kWaves; ++w) top = fmaxf(top, s.tops[w]);
        best = p.vocab;
        for (int w = kWaves - 1; w >= 0; --w)
            if (s.tops[w] == top) best = s.where[w];
        row.most = top;
        if (wrong || top == -INFINITY) return false;
        if (greedy) {
            __syncthreads();
            return true;
        }
        if (most > -INFINITY) sum *= power(((double)most - (double)top) * c, s.table);
        row.total = sum_shares(sum, sums);
        return true;
    }

    // What is left of value x.
    __device__ __forceinline__ double left_of(const State& z, int x) const {
        double r = weight(z.target, x, c, s.table);
        if (z.scale > 0.0) r = fmax(r - z.scale * weight(z.draft, x, c, s.table), 0.0);
        for (int i = 0; i < z.refusals; ++i)
            if (s.refused[i] == x) r = 0.0;
        return r;
    }

    // The sum of what is left, of every share.
    __device__ double measure_left(const State& z) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, end = begin(wave + 1);
        double sum = 0.0;
        for (int base = begin(wave) + lane; base < end; base += 64 * kBatch / 2) {
            float l[kBatch / 2], d[kBatch / 2];
#pragma unroll
            for (int i = 0; i < kBatch / 2; ++i) {
                l[i] = base + 64 * i < end ? z.target.logits[base + 64 * i] : -INFINITY;
                d[i] = base + 64 * i < end ? z.draft.logits[base + 64 * i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < kBatch / 2; ++i)
                sum += fmax(power(((double)l[i] - (double)z.target.most) * c, s.table) -
                            z.scale * power(((double)d[i] - (double)z.draft.most) * c, s.table), 0.0);
        }
        return sum_shares(sum, s.sums);
    }

    // The share of a refused token anew.
    __device__ double measure_share(const State& z, int x) const {
        const int wave = x / share, end = begin(wave + 1);
        double sum = 0.0;
        for (int i = begin(wave) + threadIdx.x; i < end; i += kThreads) sum += left_of(z, i);
        sum = sum_shares(sum, s.scan);
        if (threadIdx.x == 0) s.sums[wave] = sum;
        __syncthreads();
        double all = 0.0;
        for (int w = 0; w < kWaves; ++w) all += s.sums[w];
        return all;
    }

    // The first token at which the sums in order pass u times all.
    __device__ int choose(const State& z, float u, const double* sums) const {
        double all = 0.0;
        for (int w = 0; w < kWaves; ++w) all += sums[w];
        const double goal = (double)fminf(fmaxf(u, 0.0f), 1.0f) * all;
        double before = 0.0;
        int wave = -1, last = 0;
        double last_before = 0.0;
        for (int w = 0; w < kWaves && wave < 0; ++w) {
            if (sums[w] > 0.0) {
                last = w;
                last_before = before;
            }
            if (before + sums[w] > goal) wave = w;
            else before += sums[w];
        }
        if (wave < 0) {                             // (u is 1)
            wave = last;
            before = last_before;
        }
        // the share's values, some in order to a thread
        const int from = begin(wave), end = begin(wave + 1), each = (end - from + kThreads - 1) / kThreads;
        const int own = min(from + (int)threadIdx.x * each, end), own_end = min(own + each, end);
        double sum = 0.0;
        for (int i = own; i < own_end; ++i) sum += left_of(z, i);
        double upto = sum;
        for (int o = 1; o < 64; o <<= 1) {
            const double below = __shfl_up(upto, o, 64);
            if ((int)(threadIdx.x & 63) >= o) upto += below;
        }
        __syncthreads();
        if ((threadIdx.x & 63) == 63) s.scan[threadIdx.x >> 6] = upto;
        if (threadIdx.x == 0) s.found = p.vocab;
        __syncthreads();
        double start = before + upto - sum;
        for (int w = 0; w < (int)(threadIdx.x >> 6); ++w) start += s.scan[w];
        // a token of the thread that passes it; and the share's last one that is left, where rounding lets none
        int passes = p.vocab, last_left = -1;
        for (int i = own; i < own_end; ++i) {
            const double r = left_of(z, i);
            start += r;
            if (r > 0.0) {
                last_left = i;
                if (start > goal && passes == p.vocab) passes = i;
            }
        }
        atomicMin(&s.found, passes);
        __syncthreads();
        const int found = s.found;
        __syncthreads();
        if (found < p.vocab) return found;
        if (threadIdx.x == 0) s.found = -1;
        __syncthreads();
        atomicMax(&s.found, last_left);
        __syncthreads();
        return s.found;
    }
};

__global__ __launch_bounds__(kThreads) void verify_kernel(VerifyCall p) {
    __shared__ Shared s;
    const int request = blockIdx.x, lane = threadIdx.x & 63;
    const int start = p.batch.starts[request];
    int rows = p.batch.rows[request];
    if (rows < 0 || rows > p.batch.max_rows || start < 0 || start > p.batch.tokens - rows) rows = 0;
    if (rows == 0) {
        if (threadIdx.x == 0) {
            p.kept[request] = 0;
            p.next[request] = -1;
        }
        return;
    }
    for (int i = threadIdx.x; i < rows; i += kThreads) {
        s.parents[i] = p.parents[start + i];
        s.ids[i] = p.ids[start + i];
        s.accept[i] = p.accept[start + i];
        p.path[start + i] = i ? -1 : 0;
    }
    if (threadIdx.x < kTable) s.table[threadIdx.x] = exp2((double)threadIdx.x / kTable);
    __syncthreads();
    const float temperature = p.temperatures[request];
    const bool greedy = temperature == 0.0f;
    const Walk walk{p, s, 1.4426950408889634 / (double)temperature, (p.vocab + kWaves - 1) / kWaves};
    State z{};
    bool known = false;                             // the row's distributions are measured
    int row = 0, kept = 1;
    auto look = [&]() {
        const size_t at = (size_t)(start + row) * p.vocab;
        z.target.logits = p.logits + at;
        z.draft.logits = p.draft ? p.draft + at : nullptr;
        z.scale = z.used = 0.0;
        z.refusals = 0;
        z.bad = !(temperature >= 0.0f && temperature < INFINITY) || !walk.measure(z.target, z.best, greedy, s.sums);
        if (!z.bad && !greedy) {
            z.left = z.target.total;
            if (threadIdx.x < kWaves) s.whole[threadIdx.x] = s.sums[threadIdx.x];
            __syncthreads();
        }
        known = true;
    };
    bool draft_known = false;
    for (int i = 1; ; ++i) {
        // the next child
        int child = rows;
        for (int base = i; base < rows && child == rows; base += 64) {
            const uint64_t some = __ballot(base + lane < rows && s.parents[min(base + lane, rows - 1)] == row);
            if (some) child = base + __builtin_ctzll(some);
        }
        if (child == rows) break;
        i = child;
        const int x = s.ids[i];
        const float u = s.accept[i];
        bool taken = u < 0.0f;
        if (!taken) {
            if (!known) look();
            if (z.bad) break;
            if ((unsigned)x >= (unsigned)p.vocab) continue;
            if (greedy) {
                taken = x == z.best;
            } else {
                double of_draft = 1.0;
                if (z.draft.logits) {
                    if (!draft_known) {
                        int unused;
                        z.bad = !walk.measure(z.draft, unused, false, s.scan);
                        if (z.bad) break;
                        draft_known = true;
                    }
                    of_draft = weight(z.draft, x, walk.c, s.table) / z.draft.total;
                }
                taken = (double)u * z.left * of_draft < walk.left_of(z, x);
                if (!taken && z.draft.logits) {
                    z.used += z.left / z.target.total;
                    z.scale = z.used * z.target.total / z.draft.total;
                    z.left = walk.measure_left(z);
                } else if (!taken) {
                    __syncthreads();
                    if (threadIdx.x == 0) s.refused[z.refusals] = x;
                    ++z.refusals;
                    __syncthreads();
                    z.left = walk.measure_share(z, x);
                }
            }
        }
        if (taken) {
            if (threadIdx.x == 0) p.path[start + kept] = i;
            ++kept;
            row = i;
            known = draft_known = false;
            z.bad = false;
        }
    }
    if (!known) look();
    int next = -1;
    if (!z.bad && greedy) {
        next = z.best;
    } else if (!z.bad) {
        const bool some = z.left > 0.0;
        if (!some) {
            z.scale = 0.0;
            z.refusals = 0;
        }
        next = walk.choose(z, p.sample[request], some ? s.sums : s.whole);
    }
    if (threadIdx.x == 0) {
        p.kept[request] = kept;
        p.next[request] = next;
    }
}

}  // namespace

size_t verify_workspace_bytes(const VerifyCall&) { return 0; }

void launch_verify(const VerifyCall& call, hipStream_t stream) {
    verify_kernel<<<call.batch.requests, kThreads, 0, stream>>>(call);
}

}  // namespace leafhip
