// Attention of trees of drafted tokens over the paged cache: each sequence brings n nodes (tokens proposed for the places behind
// its `length` cached ones), whose keys and values lie in its pages at places length .. length + n - 1.  A node sees the cached
// keys and the nodes above it (and itself), said by a row of bits:
//     key place j <  length:      seen when j > position - window            (position = length + depth in the tree)
//     key place length + j:       seen when bit j of the node's mask is set and position_j > position - window
//     o = sum softmax(scale q . k) v over the keys seen, fp32; no key seen: zeros.
//
//   draft_masks_kernel        the masks and positions from the nodes' parents, once a step
//   draft_attention_kernel    any type, head size and page size, fp32 FMAs
//   draft_join_kernel         joins the shares of the keys where they were split
//
// The tensor-core kernel for bf16 heads of 64 and 128 is csrc/drafts_tc.cu.
#include <algorithm>

#include "common.cuh"
#include "packed.cuh"

using namespace mlb;

MLB_DEFINE_LAST_ERROR()

namespace {

constexpr int MAX_NODES = 256;
constexpr int MAX_WORDS = MAX_NODES / 32;

// ------------------------------------------------------------------------------ masks
// A thread a node, walking up; a parent is an earlier node of the sequence or -1, so a walk ends.  A launch's time and little more (3.5 us alone for 16 trees of up to 64 nodes).
__global__ void __launch_bounds__(MAX_NODES) draft_masks_kernel(const int* __restrict__ parents, const int* __restrict__ starts, const int* __restrict__ lengths,
                                                                int tokens, int words, int* __restrict__ masks, int* __restrict__ positions, int* __restrict__ places,
                                                                int* error_flag) {
    pdl_prologue();
    __shared__ int s_parent[MAX_NODES];
    __shared__ unsigned s_bits[MAX_NODES * (MAX_WORDS + 1)];
    const int a = blockIdx.x, i = threadIdx.x;
    const int start = starts[a], length = lengths[a];
    int n = starts[a + 1] - start;
    if (n < 0 || n > words * 32 || start < 0 || start + n > tokens) {
        if (i == 0 && error_flag) atomicExch(error_flag, 3);
        n = 0;
    }
    if (i < n) {
        int parent = parents[start + i];
        if (parent < -1 || parent >= i) {
            if (error_flag) atomicExch(error_flag, 3);
            parent = -1;
        }
        s_parent[i] = parent;
    }
    __syncthreads();
    if (i >= n) return;
    unsigned* const bits = s_bits + i * (words | 1);           // an odd pitch: neighbouring threads in different banks
    for (int w = 0; w < words; ++w) bits[w] = 0u;
    int depth = -1;
    for (int node = i; node >= 0; node = s_parent[node]) {
        bits[node >> 5] |= 1u << (node & 31);
        ++depth;
    }
    for (int w = 0; w < words; ++w) masks[(size_t)(start + i) * words + w] = (int)bits[w];
    positions[start + i] = length + depth;
    if (places) places[start + i] = length + i;
}

// ------------------------------------------------------------------------------ attention
constexpr int THREADS = 128;                   // of a group: four warps that share a tile of keys
constexpr int ROWS = 16;                       // (node, head) rows of one kv head a CTA works on; a warp of a group has four
constexpr int KEYS = 32;                       // keys a tile: a lane each
// What bounds these sizes is the way of one warp through a tile, not the arithmetic or the memory, so a CTA has several groups, each with a tile of its own, and they
// join in shared memory.  (As many as fit it: two for fp32 heads beyond 128.)  Keys are split over CTAs as well while there are too few of them.  Three sequences of 100 to 700
// keys and trees of 3 to 13 nodes, 12 fp32 heads of 128: 20.1 us with masks and join, with two groups 22.7, with one 33.3; a launch, a chain of two tiles and the join.
template <typename T, int DMAX> constexpr int groups() { return DMAX * (int)sizeof(T) > 512 ? 2 : 4; }

struct DraftParams {
    const void* q;           // [T, ldq]
    const void* pages;       // [num_pages, 2, NKV, page_size, D]
    void* out;               // [T, NH * D]
    const int* starts;       // [A + 1]
    const int* lengths;      // [A]
    const int* positions;    // [T]
    const int* masks;        // [T, words]
    const int* table;        // [A, max_blocks]
    int words, max_blocks, num_pages, page_size;
    int heads, kv_heads, group, dim, window, row_tiles;
    int reach;               // keys that a row of the table has blocks for
    int share;               // keys of one share, a multiple of KEYS
    int shares;
    int tokens, max_nodes;
    float scale;
    float* part_out;         // [shares, T * NH, D]     unnormalised
    float2* part_norm;       // [shares, T * NH]        maximum, sum
    int* error_flag;
};

// the first key that any node of a sequence may see
__device__ __forceinline__ int first_key(int length, int window) { return window > 0 ? max(0, length - window + 1) : 0; }

// PIECES: the cache's rows are copied in pieces of 16 bytes, asynchronously, a tile ahead of the one that is worked on; else element by element.
// Keys and values lie in shared memory in the cache's type.  COLS columns and RPT rows a thread in the second product.
template <typename T> __device__ __forceinline__ void unpack(const uint4& x, float (&v)[16 / sizeof(T)]) {
    const unsigned w[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        if constexpr (sizeof(T) == 4) v[i] = __uint_as_float(w[i]);
        else { v[2 * i] = __uint_as_float(w[i] << 16); v[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
    }
}

template <typename T, int DMAX> constexpr int tile_bytes() { return KEYS * (2 * DMAX + 16 / (int)sizeof(T)) * (int)sizeof(T); }
template <typename T, int DMAX> constexpr int attention_smem() { return ROWS * DMAX * 4 + groups<T, DMAX>() * tile_bytes<T, DMAX>(); }

__device__ __forceinline__ void group_sync(int group) { asm volatile("bar.sync %0, %1;" ::"r"(group + 1), "n"(THREADS) : "memory"); }
__device__ __forceinline__ bool group_or(int group, bool mine) {
    int any;
    asm volatile("{\n\t.reg .pred p, q;\n\tsetp.ne.s32 p, %1, 0;\n\tbar.red.or.pred q, %2, %3, p;\n\tselp.s32 %0, 1, 0, q;\n\t}"
                 : "=r"(any) : "r"(mine ? 1 : 0), "r"(group + 1), "n"(THREADS) : "memory");
    return any != 0;
}

template <typename T, int DMAX, bool PIECES>
__global__ void __launch_bounds__(groups<T, DMAX>() * THREADS, 1) draft_attention_kernel(DraftParams p) {
    pdl_prologue();
    constexpr int GROUPS = groups<T, DMAX>();
    constexpr int COLS = DMAX > 128 ? 2 : 1;
    constexpr int RPT = DMAX >= 128 ? ROWS : DMAX / 8;         // 32: 4, 64: 8
    constexpr int EPP = 16 / sizeof(T);                        // elements a piece
    constexpr int PITCH = DMAX + EPP;                          // of a key row: neighbouring lanes' pieces in different banks
    constexpr int P = DMAX / EPP, MINE = KEYS * P / THREADS;   // pieces of a row, and a thread's of a tile
    static_assert(KEYS * P % THREADS == 0, "whole rounds of pieces");
    static_assert(ROWS * DMAX * 4 <= tile_bytes<T, DMAX>(), "a group's result fits where its tile was");
    extern __shared__ __align__(16) unsigned char smem[];
    float* const q_s = reinterpret_cast<float*>(smem);         // [ROWS][DMAX]
    __shared__ __align__(16) float p_s[GROUPS][ROWS][KEYS];
    __shared__ float alpha_s[GROUPS][ROWS], sum_s[GROUPS][ROWS], max_s[GROUPS][ROWS];
    __shared__ unsigned mask_s[ROWS][MAX_WORDS];
    __shared__ int pos_s[ROWS];
    const int lane = threadIdx.x & 31, group = threadIdx.x / THREADS, tid = threadIdx.x % THREADS, warp = tid >> 5;
    T* const k_s = reinterpret_cast<T*>(smem + ROWS * DMAX * 4 + group * tile_bytes<T, DMAX>());      // [KEYS][PITCH]
    T* const v_s = k_s + KEYS * PITCH;                         // [KEYS][DMAX]
    const int share = blockIdx.x, seq = blockIdx.z;
    const int kvh = blockIdx.y / p.row_tiles, row0 = (blockIdx.y % p.row_tiles) * ROWS;
    const int start = p.starts[seq], n = p.starts[seq + 1] - start, length = p.lengths[seq];
    const int G = p.group, D = p.dim;
    const int rows = min(ROWS, n * G - row0);
    if (rows <= 0) return;
    if (start < 0 || start + n > p.tokens) {                   // rows that are not there
        if (threadIdx.x == 0 && p.error_flag) atomicExch(p.error_flag, 3);
        return;
    }
    if (length < 0 || length > p.reach - n) {                  // keys that are not
        if (threadIdx.x == 0 && p.error_flag) atomicExch(p.error_flag, 2);
        return;
    }
    if (n > p.max_nodes && threadIdx.x == 0 && p.error_flag) atomicExch(p.error_flag, 3);      // the grid has no rows for the last of them
    // The shares begin at the first key that a row may see (positions are at least `length`); the last one takes what is left, so that a
    // sequence longer than the caller said costs time and nothing else.
    const int lo = first_key(length, p.window), total = length + n;
    const int key_begin = lo / KEYS * KEYS + share * p.share;
    const int key_end = share == p.shares - 1 ? total : min(total, key_begin + p.share);
    if (share > 0 && key_begin >= total) return;

    const size_t plane = (size_t)p.page_size * D, page_stride = 2 * plane * p.kv_heads, v_offset = plane * p.kv_heads;
    const int* const table = p.table + (size_t)seq * p.max_blocks;
    // where the row of the lane's key begins in the pool; -1: no row may see it, or it has no page
    auto place_of = [&](int key) -> long long {
        if (key < lo || key >= key_end) return -1;
        const int block = key / p.page_size;
        const int page = table[block];
        if (page < 0 || page >= p.num_pages) {
            if (p.error_flag) atomicExch(p.error_flag, 2);
            return -1;
        }
        return (long long)((size_t)page * page_stride + (size_t)kvh * plane + (size_t)(key % p.page_size) * D);
    };
    auto ask = [&](long long place) {                          // the pieces of a tile's keys and values
#pragma unroll
        for (int i = 0; i < MINE; ++i) {
            const int e = tid + i * THREADS, key = e / P, c = e % P * EPP;
            const long long at = __shfl_sync(0xffffffffu, place, key);
            const bool there = at >= 0 && c < D;
            const T* const from = (const T*)p.pages + (there ? at + c : 0);
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(k_s + key * PITCH + c)), "l"(from),
                         "r"(there ? 16 : 0) : "memory");
            asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"((unsigned)__cvta_generic_to_shared(v_s + key * DMAX + c)), "l"(from + (there ? v_offset : 0)),
                         "r"(there ? 16 : 0) : "memory");
        }
    };
    const int first = key_begin + group * KEYS;
    long long place = place_of(first + lane);
    if (PIECES && first < key_end) ask(place);
    for (int r = threadIdx.x >> 5; r < ROWS; r += GROUPS * THREADS / 32) {
        const int node = start + (row0 + min(r, rows - 1)) / G, head = kvh * G + (row0 + min(r, rows - 1)) % G;
        const T* const q = (const T*)p.q + ((size_t)node * p.heads + head) * D;
#pragma unroll
        for (int c = lane; c < DMAX; c += 32) q_s[r * DMAX + c] = r < rows && c < D ? to_f32(q[c]) : 0.0f;
        if (lane < p.words) mask_s[r][lane] = r < rows ? (unsigned)p.masks[(size_t)node * p.words + lane] : 0u;
        if (lane == 0) pos_s[r] = p.positions[node];
    }
    __syncthreads();

    float acc[RPT][COLS];
#pragma unroll
    for (int r = 0; r < RPT; ++r)
#pragma unroll
        for (int c = 0; c < COLS; ++c) acc[r][c] = 0.0f;
    // second product: this thread's first row and column
    const int my_row = DMAX >= 128 ? 0 : (tid / DMAX) * RPT, my_col = DMAX >= 128 ? tid : tid % DMAX;
    float m[4], l[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) { m[i] = -INFINITY; l[i] = 0.0f; }

    for (int base = first; base < key_end; base += GROUPS * KEYS) {
        const int key = base + lane;
        const int where = place < 0 ? -1 : key < length ? key : p.positions[start + key - length];      // the position of the lane's key; -1: not there
        bool odd = false;                                      // a value that is not finite: it may not meet the zero weight of a row that does not see it
        if (PIECES) {
            asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll
            for (int i = 0; i < MINE; ++i) {                   // (the pieces this thread brought)
                const int e = tid + i * THREADS;
                float v[EPP];
                unpack<T>(*reinterpret_cast<const uint4*>(v_s + e / P * DMAX + e % P * EPP), v);
#pragma unroll
                for (int c = 0; c < EPP; ++c) odd |= !(fabsf(v[c]) < INFINITY);
            }
        } else {
            for (int j = warp; j < KEYS; j += THREADS / 32) {
                const long long at = __shfl_sync(0xffffffffu, place, j);
                for (int c = lane; c < DMAX; c += 32) {
                    const bool there = at >= 0 && c < D;
                    const T k = there ? ((const T*)p.pages)[at + c] : from_f32<T>(0.0f), v = there ? ((const T*)p.pages)[at + v_offset + c] : from_f32<T>(0.0f);
                    k_s[j * PITCH + c] = k;
                    v_s[j * DMAX + c] = v;
                    odd |= !(fabsf(to_f32(v)) < INFINITY);
                }
            }
        }
        odd = group_or(group, odd);
        place = place_of(key + GROUPS * KEYS);                 // of the next tile, on its way
        // scores: a lane a key, the warp's four rows
        float s[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll 4
        for (int c = 0; c < DMAX; c += EPP) {
            float k[EPP];
            unpack<T>(*reinterpret_cast<const uint4*>(k_s + lane * PITCH + c), k);
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < EPP; j += 4) {
                    const float4 q4 = *reinterpret_cast<const float4*>(q_s + (warp * 4 + i) * DMAX + c + j);
                    s[i] = fmaf(q4.x, k[j], fmaf(q4.y, k[j + 1], fmaf(q4.z, k[j + 2], fmaf(q4.w, k[j + 3], s[i]))));
                }
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int r = warp * 4 + i;
            bool seen = where >= 0 && r < rows && (p.window <= 0 || where > pos_s[r] - p.window);
            if (key >= length) seen = seen && ((mask_s[r][min((key - length) >> 5, MAX_WORDS - 1)] >> ((key - length) & 31)) & 1u) && (key - length) < p.words * 32;
            const float x = seen ? s[i] * p.scale : -INFINITY;
            const float m_new = fmaxf(m[i], warp_max(x));
            const float e = x == -INFINITY ? 0.0f : expf(x - m_new);
            const float alpha = m[i] == -INFINITY ? 0.0f : expf(m[i] - m_new);
            l[i] = l[i] * alpha + warp_sum(e);
            m[i] = m_new;
            p_s[group][r][lane] = e;
            if (lane == 0) alpha_s[group][r] = alpha;
        }
        group_sync(group);
#pragma unroll
        for (int r = 0; r < RPT; ++r)
#pragma unroll
            for (int c = 0; c < COLS; ++c) acc[r][c] *= alpha_s[group][my_row + r];
        if (odd) {
            for (int j = 0; j < KEYS; ++j)
#pragma unroll
                for (int r = 0; r < RPT; ++r) {
                    const float e = p_s[group][my_row + r][j];
#pragma unroll
                    for (int c = 0; c < COLS; ++c)
                        if (e != 0.0f) acc[r][c] = fmaf(e, to_f32(v_s[j * DMAX + my_col + c * 128]), acc[r][c]);
                }
        } else {
#pragma unroll 2
            for (int j = 0; j < KEYS; j += 4) {
                float v[4][COLS];
#pragma unroll
                for (int i = 0; i < 4; ++i)
#pragma unroll
                    for (int c = 0; c < COLS; ++c) v[i][c] = to_f32(v_s[(j + i) * DMAX + my_col + c * 128]);
#pragma unroll
                for (int r = 0; r < RPT; ++r) {
                    const float4 e = *reinterpret_cast<const float4*>(&p_s[group][my_row + r][j]);
#pragma unroll
                    for (int c = 0; c < COLS; ++c) acc[r][c] = fmaf(e.w, v[3][c], fmaf(e.z, v[2][c], fmaf(e.y, v[1][c], fmaf(e.x, v[0][c], acc[r][c]))));
                }
            }
        }
        group_sync(group);                                     // this tile's rows and weights were read
        if (PIECES && base + GROUPS * KEYS < key_end) ask(place);
    }
    // the groups join
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < 4; ++i) { sum_s[group][warp * 4 + i] = l[i]; max_s[group][warp * 4 + i] = m[i]; }
    }
    float* const mine_s = reinterpret_cast<float*>(k_s);       // [ROWS][DMAX]
#pragma unroll
    for (int r = 0; r < RPT; ++r)
#pragma unroll
        for (int c = 0; c < COLS; ++c) mine_s[(my_row + r) * DMAX + my_col + c * 128] = acc[r][c];
    __syncthreads();
    const size_t all_rows = (size_t)p.tokens * p.heads;
    for (int e = threadIdx.x; e < rows * DMAX; e += GROUPS * THREADS) {
        const int r = e / DMAX, col = e % DMAX;
        if (col >= D) continue;
        float top = -INFINITY, sum = 0.0f, o = 0.0f;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) top = fmaxf(top, max_s[g][r]);
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            const float w = max_s[g][r] == -INFINITY ? 0.0f : expf(max_s[g][r] - top);
            sum += sum_s[g][r] == sum_s[g][r] ? sum_s[g][r] * w : NAN;
            if (w != 0.0f) o = fmaf(w, reinterpret_cast<const float*>(smem + ROWS * DMAX * 4 + g * tile_bytes<T, DMAX>())[e], o);
        }
        const size_t row = (size_t)(start + (row0 + r) / G) * p.heads + kvh * G + (row0 + r) % G;
        if (p.shares == 1) {
            const float inv = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : NAN;
            ((T*)p.out)[row * D + col] = from_f32<T>(o * inv);
        } else {
            p.part_out[((size_t)share * all_rows + row) * D + col] = o;
            if (col == 0) p.part_norm[(size_t)share * all_rows + row] = make_float2(top, sum);
        }
    }
}

// A warp a row: the shares in their order, their weights found by the lanes together.
template <typename T>
__global__ void __launch_bounds__(THREADS) draft_join_kernel(DraftParams p) {
    pdl_prologue();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, seq = blockIdx.y;
    const int start = p.starts[seq], n = p.starts[seq + 1] - start;
    const int at = blockIdx.x * (THREADS / 32) + warp;
    if (at >= n * p.heads || start < 0 || start + n > p.tokens) return;
    const size_t row = (size_t)start * p.heads + at, all_rows = (size_t)p.tokens * p.heads;
    const int length = p.lengths[seq], keys = length + n - first_key(length, p.window) / KEYS * KEYS;
    if (length < 0 || length > p.reach - n) return;
    const int shares = min(p.shares, (keys + p.share - 1) / p.share);
    const float2 mine = lane < shares ? p.part_norm[lane * all_rows + row] : make_float2(-INFINITY, 0.0f);       // of the first 32 shares
    float top = mine.x;
    for (int s = lane + 32; s < shares; s += 32) top = fmaxf(top, p.part_norm[s * all_rows + row].x);
    top = warp_max(top);
    float acc[8] = {0, 0, 0, 0, 0, 0, 0, 0}, sum = 0.0f;
    for (int s0 = 0; s0 < shares; s0 += 32) {
        const float2 norm = s0 == 0 ? mine : s0 + lane < shares ? p.part_norm[(s0 + lane) * all_rows + row] : make_float2(-INFINITY, 0.0f);
        const float weight = norm.x == -INFINITY ? 0.0f : expf(norm.x - top), part = norm.x == -INFINITY ? (norm.y == norm.y ? 0.0f : NAN) : norm.y * weight;
        const int here = min(32, shares - s0);
#pragma unroll 4
        for (int s = 0; s < here; ++s) {
            const float w = __shfl_sync(0xffffffffu, weight, s);
            sum += __shfl_sync(0xffffffffu, part, s);
            const float* const o = p.part_out + ((size_t)(s0 + s) * all_rows + row) * p.dim;
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (w != 0.0f && lane + 32 * i < p.dim) acc[i] = fmaf(w, o[lane + 32 * i], acc[i]);
        }
    }
    const float inv = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : NAN;
    T* const out = (T*)p.out + row * p.dim;
#pragma unroll
    for (int i = 0; i < 8; ++i)
        if (lane + 32 * i < p.dim) out[lane + 32 * i] = from_f32<T>(acc[i] * inv);
}

template <typename T, int DMAX, bool PIECES>
int launch_attention(const DraftParams& p, int sequences, cudaStream_t stream) {
    constexpr int bytes = attention_smem<T, DMAX>();
    static bool configured[MAX_DEVICES] = {};
    const int d = device_index();
    if (!configured[d]) {
        if (cudaFuncSetAttribute(draft_attention_kernel<T, DMAX, PIECES>, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes) != cudaSuccess)
            return check_launch("draft_attention: shared memory");
        configured[d] = true;
    }
    launch_kernel(draft_attention_kernel<T, DMAX, PIECES>, dim3(p.shares, p.row_tiles * p.kv_heads, sequences), groups<T, DMAX>() * THREADS, bytes, stream, p);
    return check_launch("draft_attention");
}
template <typename T, bool PIECES>
int launch_attention(const DraftParams& p, int sequences, cudaStream_t stream) {
    if (p.dim <= 32) return launch_attention<T, 32, PIECES>(p, sequences, stream);
    if (p.dim <= 64) return launch_attention<T, 64, PIECES>(p, sequences, stream);
    if (p.dim <= 128) return launch_attention<T, 128, PIECES>(p, sequences, stream);
    return launch_attention<T, 256, PIECES>(p, sequences, stream);
}

template <typename T>
int run_attention(const DraftParams& p, int sequences, int max_nodes, cudaStream_t stream) {
    const bool pieces = p.dim * sizeof(T) % 16 == 0 && ((uintptr_t)p.pages & 15) == 0;
    const int status = pieces ? launch_attention<T, true>(p, sequences, stream) : launch_attention<T, false>(p, sequences, stream);
    if (status != MLB_OK || p.shares == 1) return status;
    const int rows = THREADS / 32;
    launch_kernel(draft_join_kernel<T>, dim3((max_nodes * p.heads + rows - 1) / rows, sequences), THREADS, 0, stream, p);
    return check_launch("draft_join");
}

}  // namespace

MLB_EXPORT int mlb_draft_masks(const int* parents, const int* starts, const int* lengths, int tokens, int sequences, int words, int* masks, int* positions,
                               int* places, int* error_flag, cudaStream_t stream) {
    if (sequences < 0 || words <= 0 || words > MAX_WORDS) return fail(MLB_UNSUPPORTED_SIZE, "draft_masks: %d words a mask (at most %d)", words, MAX_WORDS);
    if (sequences == 0) return MLB_OK;
    launch_kernel(draft_masks_kernel, sequences, words * 32, 0, stream, parents, starts, lengths, tokens, words, masks, positions, places, error_flag);
    return check_launch("draft_masks");
}

// scratch: shares > 1: [shares, T * NH] float2, then [shares, T * NH, D] fp32
MLB_EXPORT int mlb_draft_attention(const void* q, const void* pages, void* out, int dtype, const int* starts, const int* lengths, const int* positions,
                                   const int* masks, int words, const int* table, int max_blocks, int num_pages, int page_size, int tokens, int sequences,
                                   int max_nodes, int heads, int kv_heads, int dim, float scale, int window, int share, int shares, void* scratch,
                                   int* error_flag, cudaStream_t stream) {
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || dim <= 0 || dim > 256)
        return fail(MLB_UNSUPPORTED_SIZE, "draft_attention: heads %d/%d of %d elements", heads, kv_heads, dim);
    if (words <= 0 || words > MAX_WORDS || max_nodes <= 0 || max_nodes > words * 32)
        return fail(MLB_UNSUPPORTED_SIZE, "draft_attention: %d nodes in masks of %d words (at most %d)", max_nodes, words, MAX_WORDS);
    if (num_pages <= 0 || page_size <= 0 || max_blocks <= 0 || tokens < 0 || sequences < 0 || window < 0) return fail(MLB_INVALID_ARGUMENT, "draft_attention: bad sizes");
    if (share <= 0 || share % KEYS != 0 || shares <= 0 || (shares > 1 && !scratch) || ((uintptr_t)scratch & 7)) return fail(MLB_INVALID_ARGUMENT, "draft_attention: bad shares");
    const int group = heads / kv_heads, row_tiles = (max_nodes * group + ROWS - 1) / ROWS;
    if (sequences > 65535 || row_tiles * kv_heads > 65535) return fail(MLB_UNSUPPORTED_SIZE, "draft_attention: too many sequences or rows");
    if (tokens == 0 || sequences == 0) return MLB_OK;
    DraftParams p{q, pages, out, starts, lengths, positions, masks, table, words, max_blocks, num_pages, page_size, heads, kv_heads, group, dim, window,
                  row_tiles, (int)std::min((long long)max_blocks * page_size, 1ll << 30), share, shares, tokens, max_nodes, scale, nullptr, nullptr, error_flag};
    p.part_norm = (float2*)scratch;
    p.part_out = (float*)scratch + (size_t)2 * shares * tokens * heads;
    if (dtype == MLB_F32) return run_attention<float>(p, sequences, max_nodes, stream);
    if (dtype == MLB_BF16) return run_attention<__nv_bfloat16>(p, sequences, max_nodes, stream);
    return fail(MLB_INVALID_ARGUMENT, "draft_attention: fp32 or bf16");
}

MLB_PACKED(mlb_draft_masks)
MLB_PACKED(mlb_draft_attention)
