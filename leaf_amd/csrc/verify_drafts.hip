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
// on the other side of it.  p and q are good to some 1.5e-13 of themselves (`power`), so
// what is left of a token after n refusals is good to some (n + 1) 1e-12 of the whole,
// not of what is left.
//
// A walk's rows come one after the other, and only those on its way are read
// (unless all are few: then a launch measures them beforehand, see kAhead).
// Several workgroups share a request: each has a segment of the vocabulary, and
// all of them walk.  What a walk needs of the whole vocabulary (a row's largest
// value and sums, the sum of what a refusal has left) they exchange through slots
// in memory, one for each segment and exchange of the walk, each word of which
// tells by itself whether it has been written.  A workgroup that does not find
// another's words in time (it may not have started) computes them itself: the
// same operations on the same values give the same words, and no workgroup
// depends on another's progress.
//
// What bounds it: the latency of an exchange, some 6 us of loads, reductions, a
// store and the others' loads that see it, for each row and refusal of the longest
// walk; with 64 requests, 32000 tokens and both models' logits 9 us a row, of which 3 to 4 are 16
// MB of logits and, by count, 2 are 64-bit arithmetic.  64 trees of 8 rows take 41 us, 16 of 26 over 151936
// tokens 38 to 40, 100 greedy chains of 4 over 49152 28.5, a chain of 5 by itself 18 to 21.  Loading
// the row that a walk may come to next while it waits made all of them slower (48 us for the 41 with a quarter of it,
// 67 with all): the words that it waits for come behind those loads.
#include <algorithm>
#include <atomic>
#include <cfloat>
#include <cstdlib>

#include "kv8.h"

namespace leafhip {
namespace {

constexpr int kThreads = 512;
constexpr int kWaves = kThreads / 64;
constexpr int kMostSegments = 128;
constexpr int kWords = 3;                           // of a slot
constexpr int kBatch = 4;                           // values of a row that a thread has in flight
constexpr int kTable = 256;                         // powers of two of a step
constexpr int kHeld = 16;                           // values of a row that a thread keeps the weights of, in LDS
constexpr uint64_t kEmpty = ~0ull;                  // a word that is not written: no value's bits (NaN is stored as kNaN)
constexpr uint32_t kNaN = 0x7fc00000u;

// 2^y for y <= 0 (0 below 2^-1000), to 1.5e-13: table[j] = 2^(j / 256), 2^f by its series for |f| <= 1/512.
__device__ __forceinline__ double power(double y, const double* table) {
    const double shift = 6755399441055744.0 / kTable;              // 1.5 * 2^52 / 256: the sum's last bit is 1/256
    const double t = y + shift, f = y - (t - shift);
    const int n = __double2loint(t);                               // 256 y to the nearest
    double s = 5.550410866482158e-2;                               // ln2^k / k!
    s = fma(s, f, 2.402265069591007e-1);
    s = fma(s, f, 6.931471805599453e-1);
    s = fma(s, f, 1.0);
    s *= table[n & (kTable - 1)];
    const double p = __hiloint2double(__double2hiint(s) + ((n >> 8) << 20), __double2loint(s));
    return y < -1000.0 ? 0.0 : p;
}

// Reductions over a wave without the LDS: rotations in rows of 16 lanes, then swaps of rows.  Every lane gets the result.
template <int N>
__device__ __forceinline__ uint32_t rotated16(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_update_dpp(0, (int)x, 0x120 + N, 0xf, 0xf, true);
}
__device__ __forceinline__ float all_max(float x) {
    x = fmaxf(x, __uint_as_float(rotated16<8>(__float_as_uint(x))));
    x = fmaxf(x, __uint_as_float(rotated16<4>(__float_as_uint(x))));
    x = fmaxf(x, __uint_as_float(rotated16<2>(__float_as_uint(x))));
    x = fmaxf(x, __uint_as_float(rotated16<1>(__float_as_uint(x))));
    return max_xor32(max_xor16(x));
}
__device__ __forceinline__ int all_min(int x) {
    x = min(x, (int)rotated16<8>((uint32_t)x));
    x = min(x, (int)rotated16<4>((uint32_t)x));
    x = min(x, (int)rotated16<2>((uint32_t)x));
    x = min(x, (int)rotated16<1>((uint32_t)x));
    auto p = __builtin_amdgcn_permlane16_swap((uint32_t)x, (uint32_t)x, false, false);
    x = min((int)p[0], (int)p[1]);
    p = __builtin_amdgcn_permlane32_swap((uint32_t)x, (uint32_t)x, false, false);
    return min((int)p[0], (int)p[1]);
}
template <int N>
__device__ __forceinline__ double add_rotated16(double x) {
    return x + __hiloint2double((int)rotated16<N>((uint32_t)__double2hiint(x)), (int)rotated16<N>((uint32_t)__double2loint(x)));
}
__device__ __forceinline__ double all_sum(double x) {
    x = add_rotated16<1>(add_rotated16<2>(add_rotated16<4>(add_rotated16<8>(x))));
    auto h = __builtin_amdgcn_permlane16_swap((uint32_t)__double2hiint(x), (uint32_t)__double2hiint(x), false, false);
    auto l = __builtin_amdgcn_permlane16_swap((uint32_t)__double2loint(x), (uint32_t)__double2loint(x), false, false);
    x = __hiloint2double((int)h[0], (int)l[0]) + __hiloint2double((int)h[1], (int)l[1]);
    h = __builtin_amdgcn_permlane32_swap((uint32_t)__double2hiint(x), (uint32_t)__double2hiint(x), false, false);
    l = __builtin_amdgcn_permlane32_swap((uint32_t)__double2loint(x), (uint32_t)__double2loint(x), false, false);
    return __hiloint2double((int)h[0], (int)l[0]) + __hiloint2double((int)h[1], (int)l[1]);
}

struct Shared {
    double table[kTable];
    uint64_t words[kWords][kMostSegments];          // of an exchange
    double whole[kMostSegments], left[kMostSegments];   // of each segment: the sum of the target's weights, and of what is left
    double sums[2][kWaves];                         // of each wave's share of the segment in hand
    float tops[2][kWaves];
    int where[kWaves];
    int parents[kTreeRows], ids[kTreeRows], refused[kTreeRows];
    float accept[kTreeRows];
    int found;
};

struct How {
    int segments, size;                             // of the vocabulary, and values of one: a multiple of kWaves
    bool ahead;                                     // a launch before the walk measures every row
    long long wait;                                 // cycles until a workgroup computes what others owe
};
// The workspace: slots [2 tokens exchanges][segment][kWords], a request's from 2 starts on (a walk looks at each row once
// at most, and refuses each once at most); behind them, where rows are measured ahead, their words [tokens][segment][kWords].
__device__ __forceinline__ uint64_t* slots_of(const VerifyCall& p, const How& how, int start) {
    return (uint64_t*)p.workspace + (size_t)2 * start * how.segments * kWords;
}
__device__ __forceinline__ uint64_t* words_of(const VerifyCall& p, const How& how, int token) {
    return slots_of(p, how, p.batch.tokens) + (size_t)token * how.segments * kWords;
}

// One walk, by one of its workgroups.  Every workgroup of a request holds the same values here.
// HELD: a segment has at most kHeld values for a thread, whose weights stay in LDS while the walk is at their row.
template <bool HELD>
struct Walk {
    const VerifyCall& p;
    Shared& s;
    const How& how;
    uint64_t* slots;                                // the walk's: [exchange][segment][kWords]
    int own, start;
    double c;                                       // log2(e) / T
    bool greedy;

    int exchange = 0;                               // the next one
    // of the row that the walk is at
    const float *target = nullptr, *drafted = nullptr;   // drafted: null where no child is tried against it
    float most_w = 0.0f, most_v = 0.0f;             // m
    double total_w = 0.0, total_v = 0.0;            // Z, Y
    int best = 0;                                   // greedy: the first largest
    double scale = 0.0, used = 0.0, left = 0.0;     // K, C and the sum of r
    int refusals = 0;
    // HELD: the segment whose weights are kept, relative to the wave's largest values
    int held = -1;
    float held_w = 0.0f, held_v = 0.0f;
    double* weights = nullptr;                      // [2][kHeld][kThreads]

    __device__ __forceinline__ Walk(const VerifyCall& p_, Shared& s_, const How& how_, uint64_t* slots_, int own_, int start_, float temperature)
        : p(p_), s(s_), how(how_), slots(slots_), own(own_), start(start_), c(1.4426950408889634 / (double)temperature),
          greedy(temperature == 0.0f) {}

    __device__ __forceinline__ double weight(float l, float most) const { return power(((double)l - (double)most) * c, s.table); }

    // A wave's share of a segment.
    __device__ __forceinline__ int share_begin(int segment, int wave) const { return min(segment * how.size + how.size / kWaves * wave, p.vocab); }

    // A wave's share of a segment, some values at a time, the next ones under way meanwhile: use(values of the row, of
    // the draft's, the first one's place and the share's end, behind which values are minus infinity).
    template <bool BOTH, int BATCH, typename Use>
    __device__ __forceinline__ void stream(int segment, Use use) const {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, end = share_begin(segment, wave + 1);
        int base = share_begin(segment, wave) + lane;
        float l[BATCH], d[BATCH], nl[BATCH], nd[BATCH];
        auto load = [&](int from, float (&a)[BATCH], float (&b)[BATCH]) {
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                const int x = min(from + 64 * i, p.vocab - 1);
                a[i] = target[x];
                if (BOTH) b[i] = drafted[x];
            }
        };
        load(base, l, d);
        for (; base - lane < end; base += 64 * BATCH) {
            load(base + 64 * BATCH, nl, nd);
#pragma unroll
            for (int i = 0; i < BATCH; ++i)
                if (base + 64 * i >= end) l[i] = d[i] = -INFINITY;
            use(l, d, base);
#pragma unroll
            for (int i = 0; i < BATCH; ++i) {
                l[i] = nl[i];
                d[i] = nd[i];
            }
        }
    }

    // A lane's largest value so far, and the sum of its weights relative to that.
    struct Part {
        float most = -FLT_MAX;
        double sum = 0.0;
        bool wrong = false;
    };
    __device__ __forceinline__ void add(const float (&l)[kBatch], Part& part) const {
        float top = l[0];
#pragma unroll
        for (int i = 0; i < kBatch; ++i) {
            part.wrong = part.wrong || !(l[i] < INFINITY);
            top = fmaxf(top, l[i]);
        }
        if (__any(top > part.most)) {
            const float higher = fmaxf(top, part.most);
            part.sum *= weight(part.most, higher);
            part.most = higher;
        }
#pragma unroll
        for (int i = 0; i < kBatch; ++i) part.sum += weight(l[i], part.most);
    }

    // The words of a segment's slot: largest values (at least -FLT_MAX), and sums of the weights relative to them (in
    // `sums` those of each wave's share).
    __device__ __forceinline__ void measure(int segment, uint64_t (&out)[kWords]) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const bool draft = drafted != nullptr;
        Part a_w, a_v;
        int at = p.vocab;
        float top_w, top_v = -FLT_MAX;
        double sum_w = 0.0, sum_v = 0.0;
        if (greedy) {
            a_w.most = -INFINITY;
            stream<false, 2 * kBatch>(segment, [&](const float (&l)[2 * kBatch], const float (&)[2 * kBatch], int base) {
#pragma unroll
                for (int i = 0; i < 2 * kBatch; ++i) {
                    a_w.wrong = a_w.wrong || !(l[i] < INFINITY);
                    if (l[i] > a_w.most) {
                        a_w.most = l[i];
                        at = base + 64 * i;
                    }
                }
            });
            top_w = all_max(a_w.wrong ? INFINITY : a_w.most);      // (plus infinity: no distribution)
            at = all_min(a_w.most == top_w ? at : p.vocab);
        } else if (HELD && draft) {
            const int begin = share_begin(segment, wave), end = share_begin(segment, wave + 1);
            float l[kHeld], d[kHeld];
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                const int x = min(begin + lane + 64 * i, p.vocab - 1);
                l[i] = target[x];
                d[i] = drafted[x];
            }
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                if (begin + lane + 64 * i >= end) l[i] = d[i] = -INFINITY;
                a_w.wrong = a_w.wrong || !(l[i] < INFINITY);
                a_v.wrong = a_v.wrong || !(d[i] < INFINITY);
                a_w.most = fmaxf(a_w.most, l[i]);
                a_v.most = fmaxf(a_v.most, d[i]);
            }
            held = segment;
            held_w = top_w = all_max(a_w.wrong ? INFINITY : a_w.most);
            held_v = top_v = all_max(a_v.wrong ? INFINITY : a_v.most);
#pragma unroll
            for (int i = 0; i < kHeld; ++i) {
                if (begin + 64 * i >= end) continue;
                const double w = weight(l[i], top_w), v = weight(d[i], top_v);
                weights[i * kThreads + threadIdx.x] = w;
                weights[(kHeld + i) * kThreads + threadIdx.x] = v;
                sum_w += w;
                sum_v += v;
                if (i % 4 == 3) __builtin_amdgcn_sched_barrier(0);   // (more at a time need more registers than there are)
            }
            sum_w = all_sum(sum_w);
            sum_v = all_sum(sum_v);
        } else {
            if (draft)
                stream<true, kBatch>(segment, [&](const float (&l)[kBatch], const float (&d)[kBatch], int) {
                    add(l, a_w);
                    add(d, a_v);
                });
            else
                stream<false, kBatch>(segment, [&](const float (&l)[kBatch], const float (&)[kBatch], int) { add(l, a_w); });
            top_w = all_max(a_w.wrong ? INFINITY : a_w.most);
            sum_w = all_sum(a_w.sum * weight(a_w.most, top_w));
            if (draft) {
                top_v = all_max(a_v.wrong ? INFINITY : a_v.most);
                sum_v = all_sum(a_v.sum * weight(a_v.most, top_v));
            }
        }
        __syncthreads();                            // the last exchange is read
        if (lane == 0) {
            s.tops[0][wave] = top_w;
            s.tops[1][wave] = top_v;
            s.sums[0][wave] = sum_w;
            s.sums[1][wave] = sum_v;
            s.where[wave] = at;
        }
        __syncthreads();
        // the waves' together: a lane a wave
        const int i = lane & (kWaves - 1);
        const float a = s.tops[0][i], b = s.tops[1][i];
        top_w = all_max(a);
        top_v = all_max(b);
        out[0] = (uint64_t)(top_v == INFINITY ? kNaN : __float_as_uint(top_v)) << 32 | (top_w == INFINITY ? kNaN : __float_as_uint(top_w));
        out[2] = 0;
        if (greedy) {
            out[1] = (uint64_t)all_min(a == top_w ? s.where[i] : p.vocab);
            return;
        }
        out[1] = __double_as_longlong(all_sum(lane < kWaves ? s.sums[0][i] * weight(a, top_w) : 0.0));
        if (draft) out[2] = __double_as_longlong(all_sum(lane < kWaves ? s.sums[1][i] * weight(b, top_v) : 0.0));
    }

    // What is left of value x, of logits l and d.
    __device__ __forceinline__ double left_of(int x, float l, float d) const {
        double r = weight(l, most_w);
        if (scale > 0.0) r = fmax(r - scale * weight(d, most_v), 0.0);
        for (int i = 0; i < refusals; ++i)
            if (s.refused[i] == x) r = 0.0;
        return r;
    }
    __device__ __forceinline__ double left_of(int x) const { return left_of(x, target[x], scale > 0.0 ? drafted[x] : 0.0f); }

    // The sum of what is left of a segment (in `sums` of each wave's share).
    __device__ __forceinline__ void measure_left(int segment, uint64_t (&out)[kWords]) {
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        double sum = 0.0;
        if (HELD && scale > 0.0) {
            if (held != segment) measure(segment, out);            // (so that whoever computes a word gets its bits)
            const int begin = share_begin(segment, wave), end = share_begin(segment, wave + 1);
            const double fw = weight(held_w, most_w), fv = scale * weight(held_v, most_v);
#pragma unroll
            for (int i = 0; i < kHeld; ++i)         // (a value behind the end weighs nothing)
                if (begin + 64 * i < end)
                    sum += fmax(weights[i * kThreads + threadIdx.x] * fw - weights[(kHeld + i) * kThreads + threadIdx.x] * fv, 0.0);
        } else if (scale > 0.0)
            stream<true, kBatch>(segment, [&](const float (&l)[kBatch], const float (&d)[kBatch], int) {
#pragma unroll
                for (int i = 0; i < kBatch; ++i) sum += fmax(weight(l[i], most_w) - scale * weight(d[i], most_v), 0.0);
            });
        else
            stream<false, kBatch>(segment, [&](const float (&l)[kBatch], const float (&)[kBatch], int base) {
#pragma unroll
                for (int i = 0; i < kBatch; ++i) sum += left_of(base + 64 * i, l[i], 0.0f);
            });
        sum = all_sum(sum);
        __syncthreads();                            // the last exchange is read
        if (lane == 0) s.sums[0][wave] = sum;
        __syncthreads();
        out[0] = __double_as_longlong(all_sum(lane < kWaves ? s.sums[0][lane & (kWaves - 1)] : 0.0));
        out[1] = out[2] = 0;
    }

    // An exchange: of a row's largest values and sums, or (LEFT) of what is left, of every segment or of `only` one.
    template <bool LEFT>
    __device__ __forceinline__ void trade(int only) {
        constexpr int words = LEFT ? 1 : kWords;
        const int segments = how.segments;
        uint64_t* const slot = slots + (size_t)exchange * segments * kWords;
        ++exchange;
        bool waited = segments == 1;
        int segment = only < 0 ? own : only;
        bool computes = segment == own;             // (another's word is waited for first)
        for (;;) {
            if (computes) {
                uint64_t out[kWords];
                if (LEFT) measure_left(segment, out);
                else measure(segment, out);
                if (threadIdx.x < words) {
                    uint64_t word = out[0];
                    if (threadIdx.x == 1) word = out[1];
                    if (threadIdx.x == 2) word = out[2];
                    if (word == kEmpty) word = kNaN;    // (some NaN's bits: no distribution)
                    s.words[threadIdx.x][segment] = word;
                    if (segments > 1 && segment == own)
                        __hip_atomic_store(slot + segment * kWords + threadIdx.x, word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                }
            } else {
                __syncthreads();                    // the last exchange is read
            }
            if (!waited) {
                for (int i = threadIdx.x; i < segments * words; i += kThreads) {
                    const int of = i / words, word = i - of * words;
                    if (of == own || (only >= 0 && of != only)) continue;
                    const long long begin = clock64();
                    uint64_t got;
                    do {
                        got = __hip_atomic_load(slot + of * kWords + word, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    } while (got == kEmpty && clock64() - begin < how.wait);
                    s.words[word][of] = got;
                }
                waited = true;
            }
            __syncthreads();
            // a segment whose words have not come
            int missing = segments;
            for (int i = threadIdx.x & 63; i < segments; i += 64)
                for (int j = 0; j < words; ++j)
                    if ((only < 0 || i == only) && s.words[j][i] == kEmpty) missing = min(missing, i);
            missing = all_min(missing);
            if (missing == segments) return;
            segment = missing;
            computes = true;
        }
    }

    // The distributions at a row; false: there is none.
    template <bool AHEAD>
    __device__ __forceinline__ bool look(int row, bool draft) {
        target = p.logits + (size_t)(start + row) * p.vocab;
        drafted = draft ? p.draft + (size_t)(start + row) * p.vocab : nullptr;
        scale = used = 0.0;
        refusals = 0;
        held = -1;
        if (AHEAD) {
            __syncthreads();                        // the last exchange is read
            const uint64_t* words = words_of(p, how, start + row);
            for (int i = threadIdx.x; i < how.segments * kWords; i += kThreads) s.words[i % kWords][i / kWords] = words[i];
            __syncthreads();
        } else {
            trade<false>(-1);
        }
        const int lane = threadIdx.x & 63, segments = how.segments;
        float a[kMostSegments / 64], b[kMostSegments / 64];
        most_w = greedy ? -INFINITY : -FLT_MAX;
        most_v = -FLT_MAX;
        bool wrong = false;
#pragma unroll
        for (int k = 0; k < kMostSegments / 64; ++k) {
            const bool some = lane + 64 * k < segments;
            const uint64_t tops = some ? s.words[0][lane + 64 * k] : 0xff800000ff800000ull;
            a[k] = __uint_as_float((uint32_t)tops);
            b[k] = __uint_as_float((uint32_t)(tops >> 32));
            wrong = wrong || a[k] != a[k] || (draft && b[k] != b[k]);
            most_w = fmaxf(most_w, a[k]);
            most_v = fmaxf(most_v, b[k]);
        }
        most_w = all_max(most_w);
        most_v = all_max(most_v);
        if (__any(wrong)) return false;
        if (greedy) {
            best = p.vocab;
#pragma unroll
            for (int k = 0; k < kMostSegments / 64; ++k)
                if (lane + 64 * k < segments && a[k] == most_w) best = min(best, (int)s.words[1][lane + 64 * k]);
            best = all_min(best);
            return most_w > -INFINITY;
        }
        total_w = total_v = 0.0;
#pragma unroll
        for (int k = 0; k < kMostSegments / 64; ++k) {
            const int i = lane + 64 * k;
            if (i >= segments) continue;
            const double sum = __longlong_as_double(s.words[1][i]) * weight(a[k], most_w);
            if (threadIdx.x < 64) s.whole[i] = s.left[i] = sum;
            total_w += sum;
            if (draft) total_v += __longlong_as_double(s.words[2][i]) * weight(b[k], most_v);
        }
        total_w = all_sum(total_w);
        if (draft) total_v = all_sum(total_v);
        left = total_w;
        return total_w > 0.0 && (!draft || total_v > 0.0);   // (minus infinity everywhere)
    }

    // A refused child of the row, whose token has r left: what is left then.
    __device__ __forceinline__ void refuse(int x, double r) {
        const bool draft = drafted != nullptr;
        const int of = x / how.size;
        bool asks = true;
        __syncthreads();                            // `left` is written
        if (draft) {
            used += left / total_w;
            scale = used * total_w / total_v;
        } else {
            // One segment has less.  A difference that is not small beside the sum is as good as a new sum, and needs no exchange.
            const double after = s.left[of] - r;
            asks = !(after >= s.whole[of] * 0x1p-10);
            __syncthreads();                        // `left` is read
            if (threadIdx.x == 0) {
                s.refused[refusals] = x;
                s.left[of] = after;
            }
            ++refusals;
            __syncthreads();
        }
        const int only = draft ? -1 : of;
        if (asks) trade<true>(only);
        left = 0.0;
        for (int i = threadIdx.x & 63; i < how.segments; i += 64) {
            const double sum = asks && (draft || i == of) ? __longlong_as_double(s.words[0][i]) : s.left[i];
            if (asks && threadIdx.x < 64) s.left[i] = sum;
            left += sum;
        }
        left = all_sum(left);
    }

    // What a child's token, of logits l and d, has left, and whether it is taken.
    __device__ __forceinline__ bool takes(int x, float u, float l, float d, double& r) const {
        r = weight(l, most_w);
        double of_draft = 1.0;
        if (drafted) {
            const double y = weight(d, most_v);
            of_draft = y / total_v;
            if (scale > 0.0) r = fmax(r - scale * y, 0.0);
        }
        for (int i = 0; i < refusals; ++i)
            if (s.refused[i] == x) r = 0.0;
        return (double)u * left * of_draft < r;
    }

    // Of n sums in order, the one at which they pass a goal, and what is before it; past all, the last that is not zero.
    __device__ static __forceinline__ int passed(const double* sums, int n, double goal, double& before) {
        double upto = before, last_before = before;
        int last = 0;
        for (int i = 0; i < n; ++i) {
            const double sum = sums[i];
            if (sum > 0.0) {
                last = i;
                last_before = upto;
            }
            if (upto + sum > goal) break;           // (then it is not zero)
            upto += sum;
        }
        before = last_before;
        return last;
    }

    // The first token at which the sums in order pass u times all, in the workgroup that has its segment; -1 in others.
    __device__ __forceinline__ int choose(float u) {
        __syncthreads();                            // `left` is written
        const bool none = !(left > 0.0);
        if (none) {
            scale = 0.0;
            refusals = 0;
        }
        const double* sums = none ? s.whole : s.left;
        double all = 0.0;
        for (int i = 0; i < how.segments; ++i) all += sums[i];
        const double goal = (double)fminf(fmaxf(u, 0.0f), 1.0f) * all;
        double before = 0.0;
        const int segment = passed(sums, how.segments, goal, before);
        if (segment != own) return -1;
        uint64_t unused[kWords];
        measure_left(own, unused);                  // the waves' shares
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        const int share = passed(s.sums[0], kWaves, goal, before);
        // of the wave's share some values in order to a thread
        const int from = share_begin(own, share), end = share_begin(own, share + 1), each = (end - from + kThreads - 1) / kThreads;
        const int mine = min(from + (int)threadIdx.x * each, end), mine_end = min(mine + each, end);
        // What is left of a value has to be what measure_left has summed, bit for bit: after many refusals all that is left may
        // be of the size of a weight's rounding, and a share whose sum is not zero must have a value that is not.
        const bool kept = HELD && scale > 0.0;
        const double fw = kept ? weight(s.tops[0][share], most_w) : 0.0, fv = kept ? scale * weight(s.tops[1][share], most_v) : 0.0;
        auto rest_of = [&](int x) {
            if (!kept) return left_of(x);
            const int at = ((x - from) >> 6) * kThreads + 64 * share + ((x - from) & 63);   // of the share's wave: as it was stored
            return fmax(weights[at] * fw - weights[kHeld * kThreads + at] * fv, 0.0);
        };
        double sum = 0.0;
        for (int x = mine; x < mine_end; ++x) sum += rest_of(x);
        double upto = sum;
#pragma unroll
        for (int o = 1; o < 64; o <<= 1) {
            const double below = __shfl_up(upto, o, 64);
            if (lane >= o) upto += below;
        }
        if (lane == 63) s.sums[1][wave] = upto;
        if (threadIdx.x == 0) s.found = p.vocab;
        __syncthreads();
        double at = before + upto - sum;
        for (int i = 0; i < wave; ++i) at += s.sums[1][i];
        int passes = p.vocab, last_left = -1;
        for (int x = mine; x < mine_end; ++x) {
            const double r = rest_of(x);
            at += r;
            if (!(r > 0.0)) continue;
            last_left = x;
            if (at > goal && passes == p.vocab) passes = x;
        }
        passes = all_min(passes);
        if (lane == 0) atomicMin(&s.found, passes);
        __syncthreads();
        passes = s.found;
        if (passes < p.vocab) return passes;
        // rounding lets none pass: the share's last token that is left
        __syncthreads();
        if (threadIdx.x == 0) s.found = -1;
        __syncthreads();
        atomicMax(&s.found, last_left);
        __syncthreads();
        return s.found;
    }
};

// A request's rows, [start, start + rows); rows is 0 where the arrays name rows that the batch has no room for.
struct Rows {
    int start, rows;
};
__device__ __forceinline__ Rows rows_of(const KvBatchView& b, int request) {
    Rows r{b.starts[request], b.rows[request]};
    if (r.rows < 0 || r.rows > b.max_rows || r.start < 0 || r.start > b.tokens - r.rows) r.rows = 0;
    return r;
}

// Every row's words, each segment by a workgroup; and the slots that the walk needs, empty.
__global__ __launch_bounds__(kThreads, 2) void verify_rows_kernel(VerifyCall p, How how) {
    __shared__ Shared s;
    const int segment = blockIdx.x % how.segments, row = blockIdx.x / how.segments % p.batch.max_rows;
    const int request = blockIdx.x / how.segments / p.batch.max_rows;
    const Rows own = rows_of(p.batch, request);
    if (row >= own.rows) return;
    const float temperature = p.temperatures[request];
    uint64_t* const slots = slots_of(p, how, own.start) + (size_t)2 * row * how.segments * kWords;
    if (threadIdx.x < 2 * kWords) slots[(threadIdx.x / kWords * how.segments + segment) * kWords + threadIdx.x % kWords] = kEmpty;
    if (threadIdx.x < kTable) s.table[threadIdx.x] = exp2((double)threadIdx.x / kTable);
    Walk<false> walk(p, s, how, nullptr, segment, own.start, temperature);
    bool parent = false;                            // of a row behind
    for (int i = row + 1 + threadIdx.x; i < own.rows; i += kThreads) parent = parent || p.parents[own.start + i] == row;
    parent = __syncthreads_or(parent);
    walk.target = p.logits + (size_t)(own.start + row) * p.vocab;
    walk.drafted = p.draft && parent && !walk.greedy ? p.draft + (size_t)(own.start + row) * p.vocab : nullptr;
    uint64_t out[kWords];
    walk.measure(segment, out);
    if (threadIdx.x == 0)
#pragma unroll
        for (int i = 0; i < kWords; ++i) words_of(p, how, own.start + row)[(size_t)segment * kWords + i] = out[i];
}

template <bool AHEAD, bool HELD>
__global__ __launch_bounds__(kThreads, 2) void verify_kernel(VerifyCall p, How how) {
    __shared__ Shared s;
    extern __shared__ double weights[];
    const int request = blockIdx.x / how.segments, own = blockIdx.x % how.segments, lane = threadIdx.x & 63;
    const Rows mine = rows_of(p.batch, request);
    const int start = mine.start, rows = mine.rows;
    if (rows == 0) {
        if (own == 0 && threadIdx.x == 0) {
            p.kept[request] = 0;
            p.next[request] = -1;
        }
        return;
    }
    const float temperature = p.temperatures[request];
    Walk<HELD> walk(p, s, how, slots_of(p, how, start), own, start, temperature);
    walk.weights = weights;
    for (int i = threadIdx.x; i < rows; i += kThreads) {
        s.parents[i] = p.parents[start + i];
        s.ids[i] = p.ids[start + i];
        s.accept[i] = p.accept[start + i];
        if (own == 0) p.path[start + i] = i ? -1 : 0;
    }
    if (threadIdx.x < kTable) s.table[threadIdx.x] = exp2((double)threadIdx.x / kTable);
    __syncthreads();
    const bool with_draft = p.draft && !walk.greedy;
    // The next child of a row, from row i on, that a walk tries or takes without a test; rows: none.
    auto child_of = [&](int row, int i) {
        for (int base = i; base < rows; base += 64) {
            const int at = min(base + lane, rows - 1);
            const bool fits = base + lane < rows && s.parents[at] == row && (s.accept[at] < 0.0f || (unsigned)s.ids[at] < (unsigned)p.vocab);
            const uint64_t some = __ballot(fits);
            if (some) return base + __builtin_ctzll(some);
        }
        return rows;
    };
    int row = 0, kept = 1;
    bool known = false, wrong = !(temperature >= 0.0f && temperature < INFINITY);
    for (int child = child_of(0, 1); ; child = child_of(row, child + 1)) {
        bool taken = child < rows && s.accept[child] < 0.0f;
        if (!taken) {
            const int x = child < rows ? s.ids[child] : 0;
            float l = 0.0f, d = 0.0f;
            if (child < rows && !walk.greedy) {
                const size_t at = (size_t)(start + row) * p.vocab + x;
                l = p.logits[at];
                if (with_draft) d = p.draft[at];
            }
            if (!known && !wrong) wrong = !walk.template look<AHEAD>(row, with_draft && child < rows);
            known = true;
            if (wrong || child == rows) break;
            double r;
            taken = walk.greedy ? x == walk.best : walk.takes(x, s.accept[child], l, d, r);
            if (!taken && !walk.greedy) walk.refuse(x, r);
        }
        if (taken) {
            if (own == 0 && threadIdx.x == 0) p.path[start + kept] = child;
            ++kept;
            row = child;
            known = false;
        }
    }
    int next = -1;
    if (!wrong) next = walk.greedy ? (own == 0 ? walk.best : -1) : walk.choose(p.sample[request]);
    if (threadIdx.x != 0) return;
    if (own == 0) p.kept[request] = kept;
    if (next >= 0 || (wrong && own == 0)) p.next[request] = next;
}

__global__ void empty_slots_kernel(uint64_t* slots, size_t count) {
    for (size_t i = (size_t)blockIdx.x * blockDim.x + threadIdx.x; i < count; i += (size_t)gridDim.x * blockDim.x) slots[i] = kEmpty;
}

// Workgroups that the requests' vocabularies are cut for: as many as the GPU has CUs, of at least 2048 values each; twice as
// many where each had more than 32768.  With 256 / 512: 64 trees of 8 rows over 32000 tokens, both models' logits, 41 / 62
// us, 100 chains of 4 over 49152 greedy 28.5 / 28.8, 100 chains of 4 over 151936 136 / 104.
constexpr int kTarget = 256, kLeast = 2048, kLong = 32768;
// Bytes of logits up to which every row is measured ahead of the walk, side by side, although it may not come to all
// of them.  Ahead / as the walk comes, us.  Both models' logits, 32000 tokens: a chain of 8 rows that all stand (2 MB) 28 / 59,
// 16 (33 MB) 43 / 61 and 43 / 60 where half stand, 64 (131 MB, which stay in the last-level cache) 66 / 75, 71 / 74; but 64 trees of 8 rows in
// three states in turn (3 times 113 MB) 75 / 41.  One model's: 40 chains of 4 over 49152 (31 MB) sampled 30 / 34, greedy
// 17.5 / 21.6; 100 (79 MB) 49 / 58 and 26 / 29; 100 greedy over 151936 (243 MB) 53 / 50, 52.5 / 46 where they end early; 16 trees of 26 rows over
// 151936 sampled (214 MB) 107 / 41.  So wide trees decide: ahead reads rows that no walk comes to.  Between 33 and 113 MB trees were not
// measured, and chains, above all greedy ones, would gain some us up to about 100.
constexpr double kAhead = 32 << 20;

// How.wait: LEAF_VERIFY_WAIT as it is when the library is loaded (later launches of any thread do not look at the
// environment).  Never longer than the default: whoever is waited for may not be able to start before the waiting ones end.
constexpr long long kLongestWait = 200000;
const long long kWait = [] {
    const char* given = std::getenv("LEAF_VERIFY_WAIT");
    char* end = nullptr;
    const long long cycles = given ? std::strtoll(given, &end, 10) : kLongestWait;
    return given && end == given ? kLongestWait : std::clamp(cycles, 0LL, kLongestWait);
}();
How how_of(const VerifyCall& call) {
    const int each = std::max(1, kTarget / call.batch.requests), target = call.vocab / each > kLong ? 2 * kTarget : kTarget;
    const int most = std::min({(call.vocab + kLeast - 1) / kLeast, kMostSegments, std::max(1, target / call.batch.requests)});
    How how{most, 0, false, kWait};
    how.size = ((call.vocab + most - 1) / most + kWaves - 1) / kWaves * kWaves;
    how.segments = (call.vocab + how.size - 1) / how.size;
    // (not where its workgroups, for max_rows of every request, are mostly for rows that no request has)
    how.ahead = call.batch.max_rows > 1 && (double)call.batch.tokens * call.vocab * (call.draft ? 8 : 4) <= kAhead &&
                (int64_t)call.batch.requests * call.batch.max_rows <= 4LL * call.batch.tokens;
    return how;
}
size_t workspace_words(const VerifyCall& call, const How& how) {
    if (how.segments == 1 && !how.ahead) return 0;
    return (size_t)(how.ahead ? 3 : 2) * call.batch.tokens * how.segments * kWords;
}

}  // namespace

size_t verify_workspace_bytes(const VerifyCall& call) { return 8 * workspace_words(call, how_of(call)); }

void launch_verify(const VerifyCall& call, hipStream_t stream) {
    const How how = how_of(call);
    const int grid = call.batch.requests * how.segments;
    if (how.ahead) {
        verify_rows_kernel<<<grid * call.batch.max_rows, kThreads, 0, stream>>>(call, how);
        verify_kernel<true, false><<<grid, kThreads, 0, stream>>>(call, how);
        return;
    }
    if (const size_t words = workspace_words(call, how))
        empty_slots_kernel<<<(int)std::min<size_t>((words + 1023) / 1024, 1024), 256, 0, stream>>>((uint64_t*)call.workspace, words);
    if (!call.draft || how.size > kThreads * kHeld) {
        verify_kernel<false, false><<<grid, kThreads, 0, stream>>>(call, how);
        return;
    }
    constexpr int kLds = 2 * kHeld * kThreads * (int)sizeof(double);
    static std::atomic<uint64_t> allowed{0};        // more than the default: allowed once a device
    int device = 0;
    (void)hipGetDevice(&device);
    if (!(allowed >> (device & 63) & 1) &&
        hipFuncSetAttribute(reinterpret_cast<const void*>(verify_kernel<false, true>), hipFuncAttributeMaxDynamicSharedMemorySize, kLds) == hipSuccess)
        allowed |= 1ull << (device & 63);
    verify_kernel<false, true><<<grid, kThreads, kLds, stream>>>(call, how);
}

}  // namespace leafhip
