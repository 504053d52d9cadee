// The best continuations of a request's beams.  Beam b with score s_b continues with token t at
//     s_b + x_bt - lse_b,   lse_b = log sum_t exp x_bt,
// and the `wanted` largest over all beams and tokens of a request are chosen, equal ones by the lowest b * vocabulary + t.
//
// The logits are read once and stay in registers: a CTA takes one slice of a row after the other, and leaves their maximum, the sum of their
// exponentials and their `wanted` largest logits (within a beam the order of logits is the order of scores); a second kernel, a CTA a
// request, joins the CTAs' sums and ranks what they left.  Candidates of different beams are compared in 64 bits (an fp32 score of -20 has steps of 2e-6): a
// score is its beam's, and its logit's distance from the row's largest, exactly, less the logarithm of the row's sum.  That sum is of fp32 exponentials of
// base 2, fp32 within a thread and 64-bit from there on, and its logarithm is right to 1e-7 (32 rows of 9,000 to 50,000 logits of
// standard deviations of 0.1 to 6: off by 5.9e-8 at most): beams that lie nearer to one another than that are ordered by rounding.
//
// The `wanted` largest of a set, without sorting it: every warp gives the four largest of its lanes' own maxima, and the wanted-th largest of these 32 elements (all of
// them different ones) bounds what is chosen: no chosen element lies below it, and the few at or above it are ranked by counting.  (Above 32 wanted: the least of the warps'
// eighth largest.)  So many equal elements that they do not fit the list are chosen one after the other (8 rows of 152,064 logits, all but 100 masked by a finite value: 64 us
// instead of 13; by -inf, which is never chosen: 13).
#include <cfloat>

#include "common.cuh"
#include "packed.cuh"

using namespace mlb;

MLB_DEFINE_LAST_ERROR()

namespace {

constexpr int THREADS = 256;
constexpr int PER = 32;                          // logits a thread holds
constexpr int SLICE = THREADS * PER;
constexpr int MAX_WANTED = 64;
constexpr int MAX_BEAMS = 32;
constexpr int LIST = 1024;
constexpr int WARPS = THREADS / 32;
constexpr float LOG2E = 1.4426950408889634f;

struct SelectParams {
    const void* logits;      // [requests * beams, ld]
    long long ld;
    const float* scores;     // [requests, beams]
    const int* ended;        // [requests, beams] or null
    int end_token, vocab, beams, wanted, parts, group;      // a part: `group` slices of a row
    // what the parts leave
    double* part_ref;        // [rows, parts]         the largest logit
    double* part_sum;        // [rows, parts]         of e^(x - ref)
    int* part_bad;           // [rows, parts]
    float* part_value;       // [rows, parts, wanted], falling; -inf: none
    int* part_token;         // [rows, parts, wanted]
    float* out_scores;       // [requests, wanted]
    int* out_parents;
    int* out_tokens;
};

// a before b in the order of choice
template <typename V>
__device__ __forceinline__ bool before(V va, long long ia, V vb, long long ib) { return va > vb || (va == vb && ia < ib); }

template <typename V>
struct Ranking {
    V value[LIST];
    int index[LIST];
    int count;
    V best[WARPS];
    int best_index[WARPS];
    V last;
    int last_index;
};

__device__ __forceinline__ unsigned sortable(float v) {
    const unsigned b = __float_as_uint(v);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);       // larger float <-> larger key (-0 below 0: a bound between them would part equals)
}
__device__ __forceinline__ float unsorted(unsigned k) { return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k); }

// A bound that the `wanted` largest elements of the CTA do not lie below, from the threads' largest ones (none is NaN).  Two steps with a
// barrier between them.
struct Bounds {
    unsigned top[WARPS][8];
};
__device__ __forceinline__ void give_tops(Bounds& s, float mine, int wanted) {
    const unsigned lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    unsigned key = sortable(mine + 0.0f);                      // (-0 + 0 is 0)
    const int rounds = wanted > 32 ? 8 : 4;
    for (int i = 0; i < rounds; ++i) {
        const unsigned found = __reduce_max_sync(0xffffffffu, key);
        if (lane == 0) s.top[warp][i] = found;
        if (lane == __ffs(__ballot_sync(0xffffffffu, key == found)) - 1) key = 0u;
    }
}
__device__ __forceinline__ float take_bound(const Bounds& s, int wanted) {
    const unsigned lane = threadIdx.x & 31;
    if (wanted > 32) {
        unsigned least = 0xffffffffu;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) least = min(least, s.top[w][7]);
        return unsorted(least);
    }
    const unsigned key = s.top[lane >> 2][lane & 3];
    int larger = 0;
#pragma unroll
    for (int o = 1; o < 32; ++o) {
        const unsigned other = __shfl_sync(0xffffffffu, key, (lane + o) & 31);
        larger += other > key || (other == key && ((lane + o) & 31) < lane) ? 1 : 0;
    }
    return unsorted(__shfl_sync(0xffffffffu, key, __ffs(__ballot_sync(0xffffffffu, larger == wanted - 1)) - 1));
}

// How many places of the list a thread's `hits` elements get, and the first of them: one atomic a warp.
template <typename V>
__device__ __forceinline__ int take_places(Ranking<V>& s, int hits) {
    const int lane = threadIdx.x & 31;
    int sum = hits;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int other = __shfl_up_sync(0xffffffffu, sum, o);
        if (lane >= o) sum += other;
    }
    int first = 0;
    if (lane == 31 && sum) first = atomicAdd(&s.count, sum);
    return __shfl_sync(0xffffffffu, first, 31) + sum - hits;
}

// Ranks the s.count elements of the list, or, if they were too many for it, chooses from all of the threads' elements one after the other; emit(rank, value, index) is called
// once for each of the `wanted` first.  `each(visit)` calls visit(value, index) for the thread's own elements.  Returns how many there were.
template <typename V, typename Each, typename Emit>
__device__ __forceinline__ int rank_list(Ranking<V>& s, int wanted, Each each, Emit emit) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int count = s.count;
    if (count <= LIST) {
        // eight lanes an element, each against every eighth other one
        for (int i0 = 0; i0 < count; i0 += THREADS / 8) {
            const int i = i0 + tid / 8;
            const V v = s.value[min(i, count - 1)];
            const int index = s.index[min(i, count - 1)];
            int rank = 0;
#pragma unroll 4
            for (int j = tid % 8; j < count; j += 8) rank += before(s.value[j], s.index[j], v, index) ? 1 : 0;
#pragma unroll
            for (int o = 1; o < 8; o <<= 1) rank += __shfl_xor_sync(0xffffffffu, rank, o);
            if (tid % 8 == 0 && i < count && rank < wanted) emit(rank, v, index);
        }
        return min(count, wanted);
    }
    const V none = (V)-INFINITY;
    V last = (V)INFINITY;
    int last_index = -1, rank = 0;
    for (; rank < wanted; ++rank) {
        V v = none;
        int index = 0x7fffffff;
        each([&](V x, int i) {
            if (x > none && before(last, last_index, x, i) && before(x, i, v, index)) { v = x; index = i; }
        });
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) {
            const V ov = __shfl_xor_sync(0xffffffffu, v, o);
            const int oi = __shfl_xor_sync(0xffffffffu, index, o);
            if (before(ov, oi, v, index)) { v = ov; index = oi; }
        }
        if (lane == 0) { s.best[warp] = v; s.best_index[warp] = index; }
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < WARPS; ++w)
                if (before(s.best[w], s.best_index[w], v, index)) { v = s.best[w]; index = s.best_index[w]; }
            s.last = v;
            s.last_index = index;
        }
        __syncthreads();
        last = s.last;
        last_index = s.last_index;
        if (last == none) break;
        if (tid == 0) emit(rank, last, last_index);
    }
    return rank;
}

// pieces of 16 bytes
template <typename T> struct Row;
template <> struct Row<float> {
    static constexpr int W = 4;
    static __device__ __forceinline__ void unpack(const uint4& x, float* v) {
        v[0] = __uint_as_float(x.x); v[1] = __uint_as_float(x.y); v[2] = __uint_as_float(x.z); v[3] = __uint_as_float(x.w);
    }
};
template <> struct Row<__nv_bfloat16> {
    static constexpr int W = 8;
    static __device__ __forceinline__ void unpack(const uint4& x, float* v) {
        const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
};

__device__ __forceinline__ float max_nan(float a, float b, float c) {       // NaN where one of them is
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
__device__ __forceinline__ float exp2_approx(float x) {
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));      // (what is below 2^-126 adds nothing to a sum that is at least 1)
    return r;
}

typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float lo, float hi) { return ((f32x2)__float_as_uint(hi) << 32) | __float_as_uint(lo); }
__device__ __forceinline__ float low(f32x2 v) { return __uint_as_float((unsigned)v); }
__device__ __forceinline__ float high(f32x2 v) { return __uint_as_float((unsigned)(v >> 32)); }

// WIDE: rows begin at multiples of 16 bytes and are read in pieces of 16.
//
// The first slice gives the bound, and from there on a slice costs its reading, a maximum and an exponential an element: what is above the bound goes on
// the list as it comes, and the list is ranked once, at the end.  Threads sum relative to their own maximum, which is subtracted first: the largest term is 1
// exactly, so a row with one continuation has the logarithm 0, and rows of the type's lowest values keep their distances.  A thread's pieces of the next slice come into its own places in shared memory while this one is worked on; nobody
// else reads them, so nobody waits for anybody.
//
// What bounds it: with few rows a slice a CTA, and the way from the launch to the ranked list (8 rows of 151,936: 13 us with the join).  With many rows no one thing: 160
// rows of 152,064 fp32 logits, a fifth of them not read (78 MB), take 30 us with the join, of which reading alone is 15, the join 6, the bound 2.6, the list 2.6, its
// ranking 2.3 and the exponentials 1.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(THREADS, 4) select_slices_kernel(SelectParams p) {
    pdl_prologue();
    __shared__ Ranking<float> s;
    __shared__ Bounds bounds;
    __shared__ double s_sum[WARPS];
    __shared__ float s_ref[WARPS];
    constexpr int W = WIDE ? Row<T>::W : 1, PIECES = PER / W;
    const int part = blockIdx.x, row = blockIdx.y, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    // a beam that has ended or is dead is not read
    if ((p.ended && p.ended[row]) || p.scores[row] == -INFINITY) return;
    const size_t at = (size_t)row * p.parts + part;
    const T* const x = (const T*)p.logits + (size_t)row * p.ld;
    const int begin = part * p.group * SLICE, end = (int)min((long long)p.vocab, (long long)begin + (long long)p.group * SLICE);
    if (tid == 0) s.count = 0;
    // the warps' tops want elements in every warp: pieces that do not go round the CTA once are dealt out to the warps in turn
    auto place_of = [&](int count) { return count > THREADS * W ? tid : lane * WARPS + warp; };
    extern __shared__ __align__(16) unsigned char next_s[];
    uint4* const next = reinterpret_cast<uint4*>(next_s) + tid;       // piece k: next[k * THREADS]
    const unsigned next_at = (unsigned)__cvta_generic_to_shared(next);
    auto ask = [&](int from) {
        const int count = min(SLICE, end - from), place = place_of(count);
        if (count == SLICE) {
            const T* const at = x + from + tid * W;
#pragma unroll
            for (int k = 0; k < PIECES; ++k)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(next_at + k * THREADS * 16), "l"(at + k * THREADS * W) : "memory");
            return;
        }
#pragma unroll 1
        for (int k = 0; k < PIECES; ++k) {
            const int i = (k * THREADS + place) * W, there = min(W, count - i);
            if (there > 0)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(next_at + k * THREADS * 16), "l"(x + from + i),
                             "r"(there * (int)sizeof(T)) : "memory");
        }
    };
    if (WIDE) ask(begin);
    float bound = -FLT_MAX;                       // (-inf is never chosen)
    bool bad = false;
    float top = -INFINITY;                        // the thread's largest so far
    double sum = 0.0;                             // of e^(x - top)
    for (int from = begin; from < end; from += SLICE) {
        const int count = min(SLICE, end - from), place = place_of(count);
        float v[PER];
        if (WIDE) {
            asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
            for (int k = 0; k < PIECES; ++k) Row<T>::unpack(next[k * THREADS], v + k * W);
            if (count < SLICE) {
#pragma unroll
                for (int k = 0; k < PIECES; ++k)
#pragma unroll
                    for (int c = 0; c < W; ++c)
                        if ((k * THREADS + place) * W + c >= count) v[k * W + c] = -INFINITY;
            }
            if (from + SLICE < end) ask(from + SLICE);
        } else {
#pragma unroll
            for (int k = 0; k < PER; ++k) v[k] = k * THREADS + place < count ? to_f32(x[from + k * THREADS + place]) : -INFINITY;
        }
        // groups of eight neighbours, and their largest
        float most[4];
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            const float* const u = v + g * 8;
            most[g] = max_nan(max_nan(u[0], u[1], u[2]), max_nan(u[3], u[4], u[5]), max_nan(u[6], u[7], u[7]));
        }
        const float mine = max_nan(max_nan(most[0], most[1], most[2]), most[3], most[3]);
        bad |= !(mine < INFINITY);
        if (mine > top) {
            sum = top == -INFINITY ? 0.0 : sum * (double)exp2_approx((top - mine) * LOG2E);
            top = mine;
        }
        if (top > -INFINITY) {
            // two to an instruction, each rounded as always
            const f32x2 scale = pair(LOG2E, LOG2E), shift = pair(-top, -top);
            f32x2 sums = 0ull;
#pragma unroll
            for (int k = 0; k < PER; k += 2) {
                f32x2 e;
                asm("{\n\t.reg .b64 d;\n\tadd.rn.f32x2 d, %1, %3;\n\tmul.rn.f32x2 %0, d, %2;\n\t}" : "=l"(e) : "l"(pair(v[k], v[k + 1])), "l"(scale), "l"(shift));
                e = pair(exp2_approx(low(e)), exp2_approx(high(e)));
                asm("add.rn.f32x2 %0, %0, %1;" : "+l"(sums) : "l"(e));
            }
            sum += (double)(low(sums) + high(sums));
        }
        float least = bound;
        if (bound == -FLT_MAX) {                  // (the same in all threads) no slice so far had `wanted` elements
            give_tops(bounds, bad ? -INFINITY : mine, p.wanted);
            __syncthreads();
            bound = fmaxf(take_bound(bounds, p.wanted), -FLT_MAX);
            // this slice's equals count, later ones come behind them
            least = bound;
            if (bound > -FLT_MAX) bound = unsorted(sortable(bound) + 1u);
            __syncthreads();                      // (the tops may be given again)
        }
        // (few warps have any, and those have them in one of the four groups whose maxima are there)
#pragma unroll
        for (int g = 0; g < 4; ++g) {
            if (!__any_sync(0xffffffffu, most[g] >= least)) continue;
#pragma unroll
            for (int k = g * 8; k < g * 8 + 8; ++k)
                if (v[k] >= least) {
                    const int to = atomicAdd(&s.count, 1);
                    if (to < LIST) { s.value[to] = v[k]; s.index[to] = from + (k / W * THREADS + place) * W + k % W; }
                }
        }
    }
    float warp_ref = top;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) warp_ref = fmaxf(warp_ref, __shfl_xor_sync(0xffffffffu, warp_ref, o));
    if (lane == 0) s_ref[warp] = warp_ref;
    if (__syncthreads_or(bad)) {
        if (tid == 0) p.part_bad[at] = 1;
        return;
    }
    float all_ref = -INFINITY;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) all_ref = fmaxf(all_ref, s_ref[w]);
    sum = top == -INFINITY ? 0.0 : sum * (double)exp2_approx((top - all_ref) * LOG2E);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) s_sum[warp] = sum;
    float* const values = p.part_value + at * p.wanted;
    int* const tokens = p.part_token + at * p.wanted;
    const int found = rank_list<float>(s, p.wanted,
        [&](auto visit) {
            for (int i = begin + tid; i < end; i += THREADS) visit(to_f32(x[i]), i);
        },
        [&](int rank, float value, int index) { values[rank] = value; tokens[rank] = index; });
    for (int i = found + tid; i < p.wanted; i += THREADS) values[i] = -INFINITY;
    __syncthreads();
    if (tid == 0) {
        sum = 0.0;
#pragma unroll
        for (int w = 0; w < WARPS; ++w) sum += s_sum[w];
        p.part_bad[at] = 0;
        p.part_ref[at] = all_ref;
        p.part_sum[at] = sum;
    }
}

// What the parts left: up to AHEAD elements a thread are asked for at once, before the sums are joined (a call of few beams has that many; of more, the
// rest is read when it is looked at).  A chain of round trips to memory and shared memory and no bandwidth: 6 us for 32 requests of 5 beams.
constexpr int AHEAD = 12;
__global__ void __launch_bounds__(THREADS) select_join_kernel(SelectParams p) {
    pdl_prologue();
    __shared__ Ranking<double> s;
    __shared__ Bounds bounds;
    __shared__ double s_ref[MAX_BEAMS], s_shift[MAX_BEAMS];       // a candidate's score: shift + (x - ref); of an ended beam shift
    __shared__ int s_kind[MAX_BEAMS];            // 0: dead, 1: live, 2: ended
    __shared__ int s_bad;
    const int request = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int B = p.beams, parts = p.parts, wanted = p.wanted, each_beam = parts * wanted, total = B * each_beam;
    const float* const values = p.part_value + (size_t)request * total;
    const int* const tokens = p.part_token + (size_t)request * total;
    // A thread's k-th element.  Lists fall, so every warp gets other places of the lists in every round.
    auto element = [&](int k) { return k * THREADS + ((tid + 32 * k) & (THREADS - 1)); };
    float ahead[AHEAD];
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
        if (k * THREADS < total) ahead[k] = element(k) < total ? values[element(k)] : -INFINITY;
    if (tid == 0) { s_bad = 0; s.count = 0; }
    __syncthreads();
    for (int b = warp; b < B; b += WARPS) {
        const size_t row = (size_t)request * B + b;
        const float score = p.scores[row];
        const int ended = p.ended ? p.ended[row] : 0;
        // the first 32 parts' words are asked for together; those of a beam that has none are not looked at
        const size_t at = row * parts + min(lane, parts - 1);
        const int bad0 = p.part_bad[at];
        const double ref0 = p.part_ref[at];
        const double sum0 = p.part_sum[at];
        int kind = score == -INFINITY ? 0 : ended ? 2 : 1;
        double shift = (double)score, ref = -INFINITY;
        bool bad = !(score < INFINITY);
        if (kind == 1) {
            for (int i = lane; i < parts; i += 32) {
                const int part_bad = i < 32 ? bad0 : p.part_bad[row * parts + i];
                bad |= part_bad != 0;
                if (!part_bad) ref = fmax(ref, i < 32 ? ref0 : p.part_ref[row * parts + i]);
            }
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) ref = fmax(ref, __shfl_xor_sync(0xffffffffu, ref, o));
            if (!__any_sync(0xffffffffu, bad)) {
                double sum = 0.0;
                for (int i = lane; i < parts; i += 32) {
                    const double r = i < 32 ? ref0 : p.part_ref[row * parts + i];
                    if (r > -INFINITY) sum += (i < 32 ? sum0 : p.part_sum[row * parts + i]) * exp(r - ref);
                }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (ref == -INFINITY) kind = 0;
                else shift -= log(sum);
            }
        }
        if (__any_sync(0xffffffffu, bad) && lane == 0) s_bad = 1;
        if (lane == 0) { s_kind[b] = kind; s_ref[b] = ref; s_shift[b] = shift; }
    }
    __syncthreads();
    float* const out_scores = p.out_scores + (size_t)request * wanted;
    int* const out_parents = p.out_parents + (size_t)request * wanted;
    int* const out_tokens = p.out_tokens + (size_t)request * wanted;
    if (s_bad) {                                  // a logit or a score that is no number, or +inf: nothing of the request can be ranked
        for (int i = tid; i < wanted; i += THREADS) { out_scores[i] = NAN; out_parents[i] = out_tokens[i] = -1; }
        return;
    }
    // the score of element i, whose value is v; an ended beam has one, in its first place
    const float beams_per_element = 1.0f / (float)each_beam;
    auto beam_of = [&](int i) {                   // i / each_beam: the estimate is at most one off
        const int b = (int)((float)i * beams_per_element);
        return b + ((b + 1) * each_beam <= i ? 1 : 0) - (b * each_beam > i ? 1 : 0);
    };
    auto score_of = [&](int i, float v) -> double {
        const int b = beam_of(i);
        const int kind = s_kind[b];
        if (kind == 1) return v > -INFINITY ? s_shift[b] + ((double)v - s_ref[b]) : -INFINITY;
        return kind == 2 && i == b * each_beam ? s_shift[b] : -INFINITY;
    };
    auto index_of = [&](int i) {
        const int b = beam_of(i);
        return b * p.vocab + (s_kind[b] == 1 ? tokens[i] : p.end_token);
    };
    // visit(score, element) for the thread's own elements, `all` of them or those that were asked for ahead
    double score[AHEAD];
    double mine = -INFINITY;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) {
        score[k] = -INFINITY;
        if (k * THREADS < total) {
            if (element(k) < total) score[k] = score_of(element(k), ahead[k]);
            mine = fmax(mine, score[k]);
        }
    }
    for (int k = AHEAD; k * THREADS < total; ++k)
        if (element(k) < total) mine = fmax(mine, score_of(element(k), values[element(k)]));
    // (the bound goes by the scores rounded down to fp32: what is at or above it so is at or above it)
    give_tops(bounds, __double2float_rd(mine), wanted);
    __syncthreads();
    const double bound = (double)fmaxf(take_bound(bounds, wanted), -FLT_MAX);
    int hits = 0;
#pragma unroll
    for (int k = 0; k < AHEAD; ++k) hits += score[k] >= bound ? 1 : 0;
    int to = take_places(s, hits);
#pragma unroll
    for (int k = 0; k < AHEAD; ++k)
        if (score[k] >= bound) {
            if (to < LIST) { s.value[to] = score[k]; s.index[to] = element(k); }
            ++to;
        }
    for (int i = AHEAD * THREADS + tid; i < total; i += THREADS) {
        const double v = score_of(i, values[i]);
        if (v >= bound) {
            const int at = atomicAdd(&s.count, 1);
            if (at < LIST) { s.value[at] = v; s.index[at] = i; }
        }
    }
    __syncthreads();
    // elements to tokens, where they are on the list
    for (int i = tid; i < min(s.count, LIST); i += THREADS) s.index[i] = index_of(s.index[i]);
    __syncthreads();
    const int found = rank_list<double>(s, wanted,
        [&](auto visit) {
            for (int i = tid; i < total; i += THREADS) {
                const double v = score_of(i, values[i]);
                if (v > -INFINITY) visit(v, index_of(i));
            }
        },
        [&](int rank, double value, int index) {
            out_scores[rank] = (float)value;
            out_parents[rank] = index / p.vocab;
            out_tokens[rank] = index % p.vocab;
        });
    for (int i = found + tid; i < wanted; i += THREADS) { out_scores[i] = -INFINITY; out_parents[i] = out_tokens[i] = -1; }
}

// Slices of a row that a CTA takes: with many rows two waves of CTAs, four a multiprocessor at a time, which is what fits it (a CTA's first slice costs more than the
// others, and ended beams leave gaps: 32 requests of 5 beams over 152,064, a fifth ended, one wave 33.7 us, two 31.0, four 32.1).
int group_of(int rows, int vocab) {
    const int slices = (vocab + SLICE - 1) / SLICE, parts = sm_count() * 8 / rows;
    return parts >= slices ? 1 : parts <= 1 ? slices : (slices + parts - 1) / parts;
}
int parts_of(int vocab, int group) { return (int)((vocab + (long long)SLICE * group - 1) / ((long long)SLICE * group)); }

long long aligned(long long bytes) { return (bytes + 15) / 16 * 16; }

template <typename T>
void launch_slices(const SelectParams& p, int rows, cudaStream_t stream) {
    // (160 rows of 50,256 fp32, bf16 logits in pieces 19.1, 18.0 us; of 50,257 element by element 17.8, 19.1; 8 rows 10.7, 10.4 and 10.5, 11.3)
    const bool wide = ((uintptr_t)p.logits & 15) == 0 && p.ld * sizeof(T) % 16 == 0;
    if (wide) launch_kernel(select_slices_kernel<T, true>, dim3(p.parts, rows), THREADS, SLICE * sizeof(T), stream, p);
    else launch_kernel(select_slices_kernel<T, false>, dim3(p.parts, rows), THREADS, 0, stream, p);
}

// bytes of scratch that a call of these sizes needs
long long scratch_of(int requests, int beams, int vocab, int wanted) {
    const long long slots = (long long)requests * beams * parts_of(vocab, 1);
    return 2 * aligned(slots * 8) + aligned(slots * 4) + 2 * aligned(slots * wanted * 4);
}

}  // namespace

MLB_EXPORT int mlb_beam_select(const void* logits, int dtype, long long ld, const float* scores, const int* ended, int end_token, int requests, int beams,
                               int vocab, int wanted, float* out_scores, int* out_parents, int* out_tokens, void* scratch, long long scratch_bytes,
                               cudaStream_t stream) {
    if (requests < 0 || beams <= 0 || beams > MAX_BEAMS || vocab <= 0 || vocab > (1 << 30) || ld < vocab || wanted <= 0 || wanted > MAX_WANTED)
        return fail(MLB_UNSUPPORTED_SIZE, "beam_select: %d requests of %d beams, vocabulary %d, %d wanted (at most %d beams, %d wanted)", requests, beams,
                    vocab, wanted, MAX_BEAMS, MAX_WANTED);
    if ((long long)beams * vocab >= (1ll << 31) || (long long)requests * beams > 65535)
        return fail(MLB_UNSUPPORTED_SIZE, "beam_select: %d requests of %d beams over %d tokens are too many", requests, beams, vocab);
    if (ended && (end_token < 0 || end_token >= vocab)) return fail(MLB_INVALID_ARGUMENT, "beam_select: end token %d outside the vocabulary", end_token);
    if (requests == 0) return MLB_OK;
    if (scratch_bytes < scratch_of(requests, beams, vocab, wanted) || ((uintptr_t)scratch & 15))
        return fail(MLB_INVALID_ARGUMENT, "beam_select: the scratch is too small or not aligned");
    SelectParams p{};
    p.logits = logits; p.ld = ld; p.scores = scores; p.ended = ended; p.end_token = end_token; p.vocab = vocab; p.beams = beams; p.wanted = wanted;
    p.group = group_of(requests * beams, vocab);
    p.parts = parts_of(vocab, p.group);
    p.out_scores = out_scores; p.out_parents = out_parents; p.out_tokens = out_tokens;
    const int rows = requests * beams;
    const long long slots = (long long)rows * p.parts;
    char* at = (char*)scratch;
    p.part_sum = (double*)at; at += aligned(slots * 8);
    p.part_ref = (double*)at; at += aligned(slots * 8);
    p.part_bad = (int*)at; at += aligned(slots * 4);
    p.part_value = (float*)at; at += aligned(slots * wanted * 4);
    p.part_token = (int*)at;
    if (dtype == MLB_BF16) launch_slices<__nv_bfloat16>(p, rows, stream);
    else if (dtype == MLB_F32) launch_slices<float>(p, rows, stream);
    else return fail(MLB_INVALID_ARGUMENT, "beam_select: logits are fp32 or bf16");
    int status = check_launch("beam_select slices");
    if (status != MLB_OK) return status;
    launch_kernel(select_join_kernel, requests, THREADS, 0, stream, p);
    return check_launch("beam_select join");
}

MLB_PACKED(mlb_beam_select)
