// The best continuations of a request's beams.  Beam b with score s_b continues with token t at
//     s_b + x_bt - lse_b,   lse_b = log sum_t exp x_bt,
// and the `wanted` largest over all beams and tokens of a request are chosen, equal ones by the lowest b * vocabulary + t.
//
// The logits are read once and stay in registers: a CTA takes a slice of a row, leaves the slice's maximum, the sum of its
// exponentials and its `wanted` largest logits (within a beam the order of logits is the order of scores); a second kernel, a CTA a
// request, joins the slices' sums and ranks what the slices left.  Sums are fp32 within a thread and 64-bit from there on, and
// candidates of different beams are compared in 64 bits: an fp32 score of -20 has steps of 2e-6, and beams that lie
// nearer than that would be ordered by rounding.
//
// The `wanted` largest of a set, without sorting it: of the threads' own maxima the wanted-th largest is a bound that no chosen
// element lies below; the few elements at or above it are ranked by counting.  (So many equal elements that they do not fit
// the list: chosen one after the other.)
#include "common.cuh"

using namespace mlb;

MLB_DEFINE_LAST_ERROR()

namespace {

constexpr int THREADS = 256;
constexpr int PER = 32;                          // logits a thread holds
constexpr int SLICE = THREADS * PER;
constexpr int MAX_WANTED = 64;
constexpr int MAX_BEAMS = 32;
constexpr int LIST = 2048;

struct SelectParams {
    const void* logits;      // [requests * beams, ld]
    long long ld;
    const float* scores;     // [requests, beams]
    const int* ended;        // [requests, beams] or null
    int end_token, vocab, beams, wanted, parts;
    // what the slices leave
    float* part_max;         // [rows, parts]
    double* part_sum;        // [rows, parts]
    int* part_bad;           // [rows, parts]
    float* part_value;       // [rows, parts, wanted], falling; -inf: none
    int* part_token;         // [rows, parts, wanted]
    float* out_scores;       // [requests, wanted]
    int* out_parents;
    int* out_tokens;
};

__device__ __forceinline__ double block_sum_f64(double v, double* scratch) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    if (lane == 0) scratch[warp] = v;
    __syncthreads();
    v = lane < THREADS / 32 ? scratch[lane] : 0.0;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// a before b in the order of choice
template <typename V>
__device__ __forceinline__ bool before(V va, long long ia, V vb, long long ib) { return va > vb || (va == vb && ia < ib); }

// The `wanted` first of the elements of all threads (value > -inf) in the order of choice; emit(rank, value, index) is called once for
// each.  `each(visit)` calls visit(value, index) for the thread's own elements, the same ones each time.  `mine` is the largest of the thread's
// own values (-inf: none).  Indices are distinct.
template <typename V>
struct Ranking {
    V top[THREADS];
    V value[LIST];
    int index[LIST];
    V bound;
    int count;
    V best[THREADS / 32];
    int best_index[THREADS / 32];
    V last;
    int last_index;
};

template <typename V, typename Each, typename Emit>
__device__ __forceinline__ void choose(Ranking<V>& s, int wanted, V mine, Each each, Emit emit) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const V none = (V)-INFINITY;
    s.top[tid] = mine;
    if (tid == 0) { s.count = 0; s.bound = none; }
    __syncthreads();
    int larger = 0;
#pragma unroll 8
    for (int j = 0; j < THREADS; ++j) larger += (s.top[j] > mine || (s.top[j] == mine && j < tid)) ? 1 : 0;
    if (larger == wanted - 1) s.bound = mine;
    __syncthreads();
    const V bound = s.bound;
    if (mine >= bound && mine > none) {
        each([&](V v, int i) {
            if (v >= bound && v > none) {
                const int at = atomicAdd(&s.count, 1);
                if (at < LIST) { s.value[at] = v; s.index[at] = i; }
            }
        });
    }
    __syncthreads();
    const int count = s.count;
    if (count <= LIST) {
        for (int i = tid; i < count; i += THREADS) {
            const V v = s.value[i];
            const int index = s.index[i];
            int rank = 0;
            for (int j = 0; j < count && rank < wanted; ++j) rank += before(s.value[j], s.index[j], v, index) ? 1 : 0;
            if (rank < wanted) emit(rank, v, index);
        }
        __syncthreads();
        return;
    }
    // more equal elements than the list holds: one after the other
    V last = (V)INFINITY;
    int last_index = -1;
    for (int rank = 0; rank < wanted; ++rank) {
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
            for (int w = 1; w < THREADS / 32; ++w)
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
    __syncthreads();
}

template <typename T> struct Row;
template <> struct Row<float> {
    static constexpr int W = 4;
    static __device__ __forceinline__ void load(const float* p, float* v) {
        const float4 x = *reinterpret_cast<const float4*>(p);
        v[0] = x.x; v[1] = x.y; v[2] = x.z; v[3] = x.w;
    }
};
template <> struct Row<__nv_bfloat16> {
    static constexpr int W = 8;
    static __device__ __forceinline__ void load(const __nv_bfloat16* p, float* v) {
        const uint4 x = *reinterpret_cast<const uint4*>(p);
        const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
};

// WIDE: rows begin at multiples of 16 bytes and are read in pieces of 16.
template <typename T, bool WIDE>
__global__ void __launch_bounds__(THREADS) select_slices_kernel(SelectParams p) {
    pdl_prologue();
    __shared__ Ranking<float> s;
    __shared__ double s_sum[32];
    __shared__ float s_max[32];
    constexpr int W = WIDE ? Row<T>::W : 1;
    const int part = blockIdx.x, row = blockIdx.y, tid = threadIdx.x;
    // a beam that has ended or is dead is not read
    if ((p.ended && p.ended[row]) || p.scores[row] == -INFINITY) return;
    const int from = part * SLICE, count = min(SLICE, p.vocab - from);
    const T* const x = (const T*)p.logits + (size_t)row * p.ld + from;
    float v[PER];
#pragma unroll
    for (int k = 0; k < PER / W; ++k) {
        const int i = (k * THREADS + tid) * W;
        if (WIDE && i + W <= count) {
            Row<T>::load(x + i, v + k * W);
        } else {
#pragma unroll
            for (int c = 0; c < W; ++c) v[k * W + c] = i + c < count ? to_f32(x[i + c]) : -INFINITY;
        }
    }
    float mine = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int k = 0; k < PER; ++k) {
        mine = fmaxf(mine, v[k]);
        bad |= !(v[k] < INFINITY);
    }
    const int any_bad = __syncthreads_or(bad);
    const size_t at = (size_t)row * p.parts + part;
    if (any_bad) {
        if (tid == 0) p.part_bad[at] = 1;
        return;
    }
    const int lane = tid & 31, warp = tid >> 5;
    float top = warp_max(mine);
    if (lane == 0) s_max[warp] = top;
    __syncthreads();
    top = warp_max(lane < THREADS / 32 ? s_max[lane] : -INFINITY);
    float sum = 0.0f;
    if (mine > -INFINITY) {
#pragma unroll
        for (int k = 0; k < PER; ++k) sum += expf(v[k] - top);
    }
    const double total = block_sum_f64((double)sum, s_sum);
    if (tid == 0) { p.part_bad[at] = 0; p.part_max[at] = top; p.part_sum[at] = total; }
    float* const values = p.part_value + at * p.wanted;
    int* const tokens = p.part_token + at * p.wanted;
    for (int i = tid; i < p.wanted; i += THREADS) values[i] = -INFINITY;
    __syncthreads();
    choose<float>(s, p.wanted, mine,
                  [&](auto visit) {
#pragma unroll
                      for (int k = 0; k < PER / W; ++k)
#pragma unroll
                          for (int c = 0; c < W; ++c) visit(v[k * W + c], (k * THREADS + tid) * W + c);
                  },
                  [&](int rank, float value, int index) { values[rank] = value; tokens[rank] = from + index; });
}

__global__ void __launch_bounds__(THREADS) select_join_kernel(SelectParams p) {
    pdl_prologue();
    extern __shared__ unsigned char dyn[];
    Ranking<double>& s = *reinterpret_cast<Ranking<double>*>(dyn);
    __shared__ double s_shift[MAX_BEAMS];        // score - lse; of an ended beam its score
    __shared__ int s_kind[MAX_BEAMS];            // 0: dead, 1: live, 2: ended
    __shared__ int s_bad;
    const int request = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int B = p.beams, parts = p.parts, wanted = p.wanted;
    if (tid == 0) s_bad = 0;
    for (int i = tid; i < wanted; i += THREADS) {
        p.out_scores[(size_t)request * wanted + i] = -INFINITY;
        p.out_parents[(size_t)request * wanted + i] = -1;
        p.out_tokens[(size_t)request * wanted + i] = -1;
    }
    __syncthreads();
    for (int b = warp; b < B; b += THREADS / 32) {
        const size_t row = (size_t)request * B + b;
        const float score = p.scores[row];
        int kind = score == -INFINITY ? 0 : (p.ended && p.ended[row]) ? 2 : 1;
        double shift = (double)score;
        bool bad = !(score < INFINITY);
        if (kind == 1) {
            float top = -INFINITY;
            for (int i = lane; i < parts; i += 32) {
                bad |= p.part_bad[row * parts + i] != 0;
                if (!p.part_bad[row * parts + i]) top = fmaxf(top, p.part_max[row * parts + i]);
            }
            top = warp_max(top);
            if (!__any_sync(0xffffffffu, bad)) {
                double sum = 0.0;
                if (top > -INFINITY)
                    for (int i = lane; i < parts; i += 32) {
                        const float m = p.part_max[row * parts + i];
                        if (m > -INFINITY) sum += p.part_sum[row * parts + i] * exp((double)m - (double)top);
                    }
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
                if (top == -INFINITY) kind = 0;
                shift -= (double)top + log(sum);
            }
        }
        if (__any_sync(0xffffffffu, bad) && lane == 0) s_bad = 1;
        if (lane == 0) { s_kind[b] = kind; s_shift[b] = shift; }
    }
    __syncthreads();
    if (s_bad) {                                  // a logit or a score that is no number, or +inf: nothing of the request can be ranked
        for (int i = tid; i < wanted; i += THREADS) p.out_scores[(size_t)request * wanted + i] = NAN;
        return;
    }
    // a thread's own candidates: every THREADS-th of [beam][part][wanted] (an ended beam: its first place only)
    const int each_beam = parts * wanted, total = B * each_beam;
    const float* const values = p.part_value + (size_t)request * total;
    const int* const tokens = p.part_token + (size_t)request * total;
    auto each = [&](auto visit) {
        for (int i = tid; i < total; i += THREADS) {
            const int b = i / each_beam;
            if (s_kind[b] == 1) {
                const float v = values[i];
                if (v > -INFINITY) visit(s_shift[b] + (double)v, b * p.vocab + tokens[i]);
            } else if (s_kind[b] == 2 && i == b * each_beam) {
                visit(s_shift[b], b * p.vocab + p.end_token);
            }
        }
    };
    double mine = -INFINITY;
    each([&](double v, int) { mine = fmax(mine, v); });
    choose<double>(s, wanted, mine, each, [&](int rank, double value, int index) {
        const size_t at = (size_t)request * wanted + rank;
        p.out_scores[at] = (float)value;
        p.out_parents[at] = index / p.vocab;
        p.out_tokens[at] = index % p.vocab;
    });
}

int parts_of(int vocab) { return (vocab + SLICE - 1) / SLICE; }

long long aligned(long long bytes) { return (bytes + 15) / 16 * 16; }

template <typename T>
void launch_slices(const SelectParams& p, int rows, cudaStream_t stream) {
    const bool wide = ((uintptr_t)p.logits & 15) == 0 && p.ld * sizeof(T) % 16 == 0;
    if (wide) launch_kernel(select_slices_kernel<T, true>, dim3(p.parts, rows), THREADS, 0, stream, p);
    else launch_kernel(select_slices_kernel<T, false>, dim3(p.parts, rows), THREADS, 0, stream, p);
}

// bytes of scratch that a call of these sizes needs
long long scratch_of(int requests, int beams, int vocab, int wanted) {
    const long long slots = (long long)requests * beams * parts_of(vocab);
    return aligned(slots * 8) + 2 * aligned(slots * 4) + 2 * aligned(slots * wanted * 4);
}

}  // namespace

MLB_EXPORT int mlb_beam_select(const void* logits, int dtype, long long ld, const float* scores, const int* ended, int end_token, int requests, int beams,
                               int vocab, int wanted, float* out_scores, int* out_parents, int* out_tokens, void* scratch, long long scratch_bytes,
                               cudaStream_t stream) {
    if (requests < 0 || beams <= 0 || beams > MAX_BEAMS || vocab <= 0 || ld < vocab || wanted <= 0 || wanted > MAX_WANTED)
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
    p.parts = parts_of(vocab);
    p.out_scores = out_scores; p.out_parents = out_parents; p.out_tokens = out_tokens;
    const int rows = requests * beams;
    const long long slots = (long long)rows * p.parts;
    char* at = (char*)scratch;
    p.part_sum = (double*)at; at += aligned(slots * 8);
    p.part_max = (float*)at; at += aligned(slots * 4);
    p.part_bad = (int*)at; at += aligned(slots * 4);
    p.part_value = (float*)at; at += aligned(slots * wanted * 4);
    p.part_token = (int*)at;
    if (dtype == MLB_BF16) launch_slices<__nv_bfloat16>(p, rows, stream);
    else if (dtype == MLB_F32) launch_slices<float>(p, rows, stream);
    else return fail(MLB_INVALID_ARGUMENT, "beam_select: logits are fp32 or bf16");
    int status = check_launch("beam_select slices");
    if (status != MLB_OK) return status;
    static bool configured[MAX_DEVICES] = {};
    const int d = device_index();
    if (!configured[d]) {
        if (cudaFuncSetAttribute(select_join_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)sizeof(Ranking<double>)) != cudaSuccess)
            return check_launch("beam_select: shared memory");
        configured[d] = true;
    }
    launch_kernel(select_join_kernel, requests, THREADS, sizeof(Ranking<double>), stream, p);
    return check_launch("beam_select join");
}
