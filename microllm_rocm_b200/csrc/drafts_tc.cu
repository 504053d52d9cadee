// Attention of drafted trees over the paged bf16 cache on the fifth-generation tensor cores, heads of 64 or 128 (-DHEAD_DIM).  What a
// row sees and how the shares of the keys are laid out is csrc/drafts.cu's; P is rounded to bf16 for the second product.
//
// A CTA takes one kv head of one sequence: the rows (node, head of the group) of up to 2 x floor(128 / group) nodes, and one share of
// the keys in tiles of 128.  It holds two streams of work, each with four softmax warps (a thread a row), its own scores and its own
// accumulator in tensor memory:
//     rows for one tile of 128 or fewer:  both streams have the same rows; one takes the even key tiles, the other the odd ones, and they meet at the end
//     more rows:                          a stream a row tile, both over every key tile, which is loaded once for the two
// so that one stream's softmax runs beside the other's products.  Warps:
//     warp 0      TMA: the queries (a box of heads x nodes, rows in the order node * group + head), then key and value tiles page by page
//                 into a ring, in the order in which the products need them
//     warp 1      one thread issues tcgen05.mma: S = Q K^T; O += P V with P in tensor memory.  P overwrites the scores it was made of; the next scores of a stream
//                 are issued behind the product that reads P, so "scores are there" also says that the accumulator is (the tensor pipe runs in order)
//     warps 2-9   softmax of stream (warp - 2) / 4: mask in the tiles that need one, running maximum and sum in fp32 with base-2
//                 exponentials, the accumulator rescaled only when a row's maximum has grown by 2^8
// In tiles that not every row sees alike the value rows are looked through: one that holds a number which is not finite is cleared for the product (0 * NaN
// would reach rows that do not see it) and the rows that do see it become NaN; value rows that nobody sees are cleared too.
//
// Every wait on an mbarrier is bounded; when a bound is hit the error flag is raised, the CTA waits (bounded) for the copies in flight, frees
// its tensor memory and returns.
#include "common.cuh"

#include <cuda.h>

#ifndef HEAD_DIM
#error "compile with -DHEAD_DIM=64 or 128"
#endif

using namespace mlb;

MLB_DEFINE_LAST_ERROR()

namespace {

constexpr int D = HEAD_DIM;
static_assert(D == 64 || D == 128, "HEAD_DIM must be 64 or 128");
constexpr int BM = 128;                      // rows of a stream (MMA M)
constexpr int BN = 128;                      // keys a tile
constexpr int SPANS = D / 64;                // 64-element (128-byte) column spans of a row
constexpr int ROW_BYTES = 128;               // one swizzle span
constexpr int Q_BYTES = SPANS * BM * ROW_BYTES;
constexpr int KV_BYTES = SPANS * BN * ROW_BYTES;
constexpr int SLOTS = D == 128 ? 5 : 8;
constexpr int SMEM_BYTES = 2 * Q_BYTES + SLOTS * KV_BYTES + 1024;
static_assert(SMEM_BYTES + 512 <= 227 * 1024, "a CTA's shared memory, its barriers among it");
constexpr int THREADS = 320;
constexpr int STREAM_COLS = 256;             // tensor memory of a stream: scores (then P as bf16 pairs) [0, 128), accumulator [128, 128 + D)
constexpr int TMEM_COLS = 2 * STREAM_COLS;
constexpr int O_COL = BN;
constexpr int SPIN_LIMIT = 1 << 21;          // polls of up to 2 us each
constexpr int MAX_PAGES_PER_TILE = 16;
constexpr int MAX_WORDS = 8;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_STEP = 8.0f;

struct TcParams {
    __nv_bfloat16* out;             // [T, NH * D]
    const int* starts;              // [A + 1]
    const int* lengths;             // [A]
    const int* positions;           // [T]
    const int* masks;               // [T, words]
    const int* table;               // [A, max_blocks]
    int words, max_blocks, num_pages, page_size, pages_per_tile;
    int heads, kv_heads, group, tile_nodes, pairs, window, max_nodes;
    int share;                      // keys of a share, a multiple of BN
    int shares, tokens;
    float scale_log2;
    float* part_out;                // [shares, T * NH, D]
    float2* part_norm;              // [shares, T * NH]
    int* error_flag;
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, int count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
    uint32_t ok;
    // the hint (ns) lets the hardware park the thread until the phase completes instead of spinning on shared memory
    asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\tselp.u32 %0, 1, 0, p;\n\t}"
                 : "=r"(ok) : "r"(bar), "r"(parity), "r"(2000u) : "memory");
    return ok != 0;
}
// false when the bound was hit (the caller gives up and the flag tells the host)
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, int* error_flag, int code) {
    for (int i = 0; i < SPIN_LIMIT; ++i)
        if (mbar_try_wait(bar, parity)) return true;
    if (error_flag) atomicCAS(error_flag, 0, code);          // the first failure is the one worth reporting
    return false;
}
// true in exactly one lane of the (converged) warp
__device__ __forceinline__ bool elect_one() {
    uint32_t pred;
    asm volatile("{\n\t.reg .pred P;\n\telect.sync _|P, 0xffffffff;\n\tselp.u32 %0, 1, 0, P;\n\t}" : "=r"(pred));
    return pred != 0;
}
__device__ __forceinline__ void tma_load_2d(uint32_t dst, const CUtensorMap* map, int c0, int c1, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(bar) : "memory");
}

// Shared-memory operand descriptors, 128-byte swizzle.  Rows are 128 bytes, groups of 8 rows
// 1024 bytes apart (the stride byte offset).  K-major: a row is an M/N index and holds 64
// contraction elements.  MN-major: a row is a contraction index and holds 64 M/N elements; the
// next 64 M/N elements are `lead_bytes` further on.
__device__ __forceinline__ uint64_t desc_k_major(uint32_t addr) {
    uint64_t d = 0;
    d |= (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)1 << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
__device__ __forceinline__ uint64_t desc_mn_major(uint32_t addr, uint32_t lead_bytes) {
    uint64_t d = 0;
    d |= (uint64_t)((addr & 0x3FFFFu) >> 4);
    d |= (uint64_t)((lead_bytes >> 4) & 0x3FFFu) << 16;
    d |= (uint64_t)(1024 >> 4) << 32;
    d |= (uint64_t)1 << 46;
    d |= (uint64_t)2 << 61;
    return d;
}
// kind::f16 instruction descriptor: fp32 accumulator, bf16 A (K-major) and B
__device__ __forceinline__ uint32_t idesc(int n, bool b_mn_major) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn_major ? (1u << 16) : 0u) | ((uint32_t)(n >> 3) << 17) |
           ((uint32_t)(BM >> 4) << 24);
}
__device__ __forceinline__ void umma(uint32_t tmem_d, uint64_t a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "l"(a), "l"(b), "r"(id), "r"(accumulate) : "memory");
}
// the same with the A operand in tensor memory (lane = row, a 32-bit column = two neighbouring bf16 of the contraction)
__device__ __forceinline__ void umma_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t b, uint32_t id, uint32_t accumulate) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
                 "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}"
                 ::"r"(tmem_d), "r"(tmem_a), "l"(b), "r"(id), "r"(accumulate) : "memory");
}
__device__ __forceinline__ void umma_commit(uint32_t bar) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
                 "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),
                   "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),
                   "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
                 "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
                   "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
                   "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
                 : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

__device__ __forceinline__ float fast_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
}

// The largest of a row's scores: eight chains of three operands a step.
template <int N>
__device__ __forceinline__ float row_max(const uint32_t (&s)[N]) {
    float m[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) m[k] = fmaxf(__uint_as_float(s[2 * k]), __uint_as_float(s[2 * k + 1]));
#pragma unroll
    for (int c = 16; c < N; c += 2) m[(c >> 1) & 7] = fmaxf(fmaxf(m[(c >> 1) & 7], __uint_as_float(s[c])), __uint_as_float(s[c + 1]));
    return fmaxf(fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3])), fmaxf(fmaxf(m[4], m[5]), fmaxf(m[6], m[7])));
}

// P = 2^(s * scale + shift) of N of a row's scores, as bf16 pairs in s[0 .. N / 2); returns the sum of the fp32 terms: neighbours first, then four
// chains of them.  Scaling and summing go two to an instruction, each rounded as always.
template <int N>
__device__ __forceinline__ float row_exp2(uint32_t (&s)[N], float scale, float shift) {
    typedef unsigned long long f32x2;
    auto pair = [](uint32_t lo, uint32_t hi) { return ((f32x2)hi << 32) | lo; };
    const f32x2 scale2 = pair(__float_as_uint(scale), __float_as_uint(scale)), shift2 = pair(__float_as_uint(shift), __float_as_uint(shift));
    f32x2 chains[2] = {0ull, 0ull};          // chains 0 and 1, 2 and 3
#pragma unroll
    for (int c = 0; c < N; c += 4) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            f32x2 x;
            asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(x) : "l"(pair(s[c + i], s[c + i + 1])), "l"(scale2), "l"(shift2));
            p[i] = fast_exp2(__uint_as_float((uint32_t)x));
            p[i + 1] = fast_exp2(__uint_as_float((uint32_t)(x >> 32)));
        }
        f32x2 neighbours;
        asm("add.rn.f32x2 %0, %1, %2;" : "=l"(neighbours) : "l"(pair(__float_as_uint(p[0]), __float_as_uint(p[2]))), "l"(pair(__float_as_uint(p[1]), __float_as_uint(p[3]))));
        asm("add.rn.f32x2 %0, %0, %1;" : "+l"(chains[(c >> 2) & 1]) : "l"(neighbours));
        s[c / 2] = pack_bf16(p[0], p[1]);
        s[c / 2 + 1] = pack_bf16(p[2], p[3]);
    }
    auto sum = [](f32x2 v) { return __uint_as_float((uint32_t)v) + __uint_as_float((uint32_t)(v >> 32)); };
    return sum(chains[0]) + sum(chains[1]);
}


__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
                 ::"r"(dst), "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(bar) : "memory");
}

// bits [from, to) of a 32-bit word, either end anywhere
__device__ __forceinline__ unsigned bit_range(int from, int to) {
    const unsigned upper = to <= 0 ? 0u : to >= 32 ? 0xffffffffu : (1u << to) - 1u;
    const unsigned lower = from <= 0 ? 0u : from >= 32 ? 0xffffffffu : (1u << from) - 1u;
    return upper & ~lower;
}

// the keys of a sequence that a CTA's share holds, in tiles
struct Span {
    int lo, total, first, count;    // the first key any node may see, all keys, the first tile and how many
};
__device__ __forceinline__ Span span_of(const TcParams& p, int length, int n, int share) {
    Span s;
    s.lo = p.window > 0 ? max(0, length - p.window + 1) : 0;
    s.total = length + n;
    const int per = p.share / BN;
    s.first = s.lo / BN + share * per;
    const int tiles = (s.total + BN - 1) / BN - s.first;
    s.count = max(0, share == p.shares - 1 ? tiles : min(tiles, per));
    return s;
}

__global__ void __launch_bounds__(THREADS, 1)
draft_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv, TcParams p) {
    pdl_launch_dependents();
    extern __shared__ unsigned char smem_dyn[];
    __shared__ __align__(8) unsigned long long q_full, slot_full[SLOTS], slot_empty[SLOTS], s_full[2], p_full[2], o_full[2], v_checked[2], norms_there;
    __shared__ uint32_t tmem_base_s;
    __shared__ int failed_s;
    __shared__ unsigned odd_s[2][2][4];           // [stream][turn & 1]: which of a tile's value rows are not finite

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = (smem_u32(smem_dyn) + 1023u) & ~1023u;     // the swizzle pattern wants 1024-byte alignment
    const uint32_t q_s = base;
    const uint32_t ring_s = q_s + 2 * Q_BYTES;
    // the rows' maxima and sums, for streams that share the rows: there the second query tile's place is free
    float2* const norm_s = reinterpret_cast<float2*>(smem_dyn + (base - smem_u32(smem_dyn)) + Q_BYTES);

    pdl_wait();                  // (the sequence's extents may be the kernel before's)
    // ---- what this CTA works on (uniform)
    const int share = blockIdx.x, seq = blockIdx.z;
    const int kvh = blockIdx.y / p.pairs, pair = blockIdx.y % p.pairs;
    const int token0 = p.starts[seq], n = p.starts[seq + 1] - token0, length = p.lengths[seq];
    const int node0 = pair * 2 * p.tile_nodes;                       // the first node of this CTA's rows
    if (n <= node0) return;
    if (n > p.max_nodes && threadIdx.x == 0 && p.error_flag) atomicExch(p.error_flag, 3);
    const Span span = span_of(p, length, n, share);
    if (span.count == 0) return;                                     // (never share 0; the join knows)
    const int n_tiles = span.count;
    const bool paired = n - node0 > p.tile_nodes;                    // a row tile a stream; else the streams share the key tiles
    // stream s: its tiles are t = t0, t0 + dt, ..
    const int dt = paired ? 1 : 2;

    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&q_full), 1);
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(smem_u32(&slot_full[s]), 1);
            mbar_init(smem_u32(&slot_empty[s]), 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(smem_u32(&s_full[s]), 1);
            mbar_init(smem_u32(&p_full[s]), 4);          // one arrival per softmax warp
            mbar_init(smem_u32(&o_full[s]), 1);
            mbar_init(smem_u32(&v_checked[s]), paired ? 8 : 4);
        }
        mbar_init(smem_u32(&norms_there), 8);
        failed_s = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&tmem_base_s)), "r"((uint32_t)TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = tmem_base_s;

    // Ring items in order of need.  Shared key tiles: K0 K1 V0 K2 V1 K3 ..; a row tile a stream: K0 V0 K1 V1 ..
    // The items walk like this for all who count them: prologue K(0 .. dt - 1), then for every t: V(t), K(t + dt).
    const int prologue = min(dt, n_tiles);
    int issued = 0;

    if (warp == 0) {
        // ------------------------------------------------------------------ producer (whole warp)
        if (lane == 0) {
            const int boxes = paired ? 2 : 1;
            mbar_expect_tx(smem_u32(&q_full), boxes * SPANS * p.tile_nodes * p.group * ROW_BYTES);
            for (int b = 0; b < boxes; ++b)
#pragma unroll
                for (int s = 0; s < SPANS; ++s)
                    tma_load_3d(q_s + b * Q_BYTES + s * BM * ROW_BYTES, &map_q, s * 64, kvh * p.group, token0 + node0 + b * p.tile_nodes, smem_u32(&q_full));
        }
        const int* table = p.table + (size_t)seq * p.max_blocks;
        auto lookup = [&](int tile) {                     // lane g: the page of block g of a tile
            const int block = (span.first + tile) * p.pages_per_tile + lane;
            return (lane < p.pages_per_tile && block < p.max_blocks) ? __ldg(table + block) : -1;
        };
        bool ok = true;
        int item = 0;                                     // = issued
        auto load = [&](int tile, int is_v) {
            lag_point();
            int page = lookup(tile);
            const int slot = item % SLOTS;
            if (item >= SLOTS) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&slot_empty[slot]), ((item / SLOTS) - 1) & 1, p.error_flag, 41)) != 0;
            if (!ok) return;
            const uint32_t bar = smem_u32(&slot_full[slot]);
            if (lane == 0) mbar_expect_tx(bar, KV_BYTES);
            __syncwarp();
            if (lane < p.pages_per_tile) {
                if (page < 0 || page >= p.num_pages) {
                    // a page that holds a key some row may see has to exist; the others are masked
                    const int first_key = ((span.first + tile) * p.pages_per_tile + lane) * p.page_size;
                    if (first_key < span.total && first_key + p.page_size > span.lo && p.error_flag) atomicExch(p.error_flag, 2);
                    page = 0;
                }
                const int row = ((page * 2 + is_v) * p.kv_heads + kvh) * p.page_size;
                const uint32_t dst = ring_s + slot * KV_BYTES + lane * p.page_size * ROW_BYTES;
#pragma unroll
                for (int s = 0; s < SPANS; ++s) tma_load_2d(dst + s * BN * ROW_BYTES, &map_kv, s * 64, row, bar);
            }
            ++item;
            issued = item;
        };
        for (int t = 0; t < prologue && ok; ++t) load(t, 0);
        for (int t = 0; t < n_tiles && ok; ++t) {
            load(t, 1);
            if (ok && t + dt < n_tiles) load(t + dt, 0);
        }
        if (!ok && lane == 0) failed_s = 1;
    } else if (warp == 1) {
        // ------------------------------------------------------------------ MMA issue: the warp walks converged, one lane issues
        const uint32_t idesc_qk = idesc(BN, false), idesc_pv = idesc(D, true);
        auto wait_warp = [&](unsigned long long* bar, uint32_t parity, int code) {
            return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, p.error_flag, code)) != 0;
        };
        bool ok = n_tiles == 0 || wait_warp(&q_full, 0, 42);
        int item = 0;                                      // ring items are consumed in the order they were loaded
        auto full = [&](int i, int code) { return wait_warp(&slot_full[i % SLOTS], (i / SLOTS) & 1, code); };
        auto issue_qk = [&](int s, int i, bool last_use) { // stream s's scores from ring item i
            const uint32_t kb = ring_s + (i % SLOTS) * KV_BYTES, qb = q_s + (paired ? s * Q_BYTES : 0);
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < D / 16; ++ks) {
                    const uint32_t off = (ks / 4) * (BM * ROW_BYTES) + (ks % 4) * 32;
                    umma(tmem_base + (uint32_t)(s * STREAM_COLS), desc_k_major(qb + off), desc_k_major(kb + off), idesc_qk, ks > 0);
                }
                if (last_use) umma_commit(smem_u32(&slot_empty[i % SLOTS]));
                umma_commit(smem_u32(&s_full[s]));
            }
            __syncwarp();
        };
        auto issue_pv = [&](int s, int i, bool first, bool last, bool last_use) {
            const uint32_t vb = ring_s + (i % SLOTS) * KV_BYTES;
            if (elect_one()) {
#pragma unroll
                for (int ks = 0; ks < BN / 16; ++ks)           // 16 keys = 8 columns of P
                    umma_ts(tmem_base + (uint32_t)(s * STREAM_COLS + O_COL), tmem_base + (uint32_t)(s * STREAM_COLS + ks * 8),
                            desc_mn_major(vb + ks * 16 * ROW_BYTES, BN * ROW_BYTES), idesc_pv, (!first || ks > 0) ? 1u : 0u);
                if (last_use) umma_commit(smem_u32(&slot_empty[i % SLOTS]));
                if (last) umma_commit(smem_u32(&o_full[s]));
            }
            __syncwarp();
        };
        if (paired) {
            if (ok && n_tiles > 0) {
                ok = full(item, 43);
                if (ok) {
                    issue_qk(0, item, false);
                    issue_qk(1, item, true);
                    ++item;
                }
            }
            for (int t = 0; t < n_tiles && ok; ++t) {
                lag_point();
                const bool last = t + 1 == n_tiles;
                ok = wait_warp(&p_full[0], t & 1, 44) && full(item, 45);
                if (!ok) break;
                tc_fence_after();
                issue_pv(0, item, t == 0, last, false);
                if (!last) {
                    ok = full(item + 1, 46);
                    if (!ok) break;
                    issue_qk(0, item + 1, false);
                }
                ok = wait_warp(&p_full[1], t & 1, 47);
                if (!ok) break;
                tc_fence_after();
                issue_pv(1, item, t == 0, last, true);
                if (!last) issue_qk(1, item + 1, true);
                item += 2;
            }
        } else {
            for (int t = 0; t < prologue && ok; ++t) {
                ok = full(item, 48);
                if (!ok) break;
                issue_qk(t, item, true);
                ++item;
            }
            for (int t = 0; t < n_tiles && ok; ++t) {
                lag_point();
                const int s = t & 1;
                ok = wait_warp(&p_full[s], (t >> 1) & 1, 49) && full(item, 50);
                if (!ok) break;
                tc_fence_after();
                issue_pv(s, item, t < 2, t + 2 >= n_tiles, true);
                ++item;
                if (t + 2 < n_tiles) {
                    ok = full(item, 51);
                    if (!ok) break;
                    issue_qk(s, item, true);
                    ++item;
                }
            }
        }
        if (!ok && lane == 0) failed_s = 1;
    } else {
        // ------------------------------------------------------------------ softmax, one thread per row
        const int stream = (warp - 2) >> 2;
        const int quarter = warp & 3;                     // the tensor-memory lanes this warp may touch
        const int r = quarter * 32 + lane;
        const int my_node0 = node0 + (paired ? stream * p.tile_nodes : 0);
        const int rows = min(p.tile_nodes, n - my_node0) * p.group;
        const bool active = quarter * 32 < rows;          // (the warp) else its rows are nobody's
        const bool mine = r < rows;
        const int node = my_node0 + (mine ? r / p.group : 0), head = kvh * p.group + (mine ? r % p.group : 0);
        const int pos = p.positions[token0 + node];
        const int lo_r = p.window > 0 ? max(0, pos - p.window + 1) : 0;
        const uint32_t tmem = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)(stream * STREAM_COLS);
        float m_used = -INFINITY, l = 0.0f;
        bool sees_odd = false, ok = true;
        auto wait_all = [&](unsigned long long* bar, uint32_t parity, int code) {
            return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, p.error_flag, code)) != 0;
        };
        // A tile that not every row sees alike holds a node, or a cached key in front of some node's window.  The latest position is at
        // most length + n - 1.
        const int window_end = p.window > 0 ? max(0, span.total - p.window) : 0;
        int turn = 0, looked = 0;                         // the stream's tiles, and those of them that were looked through
        for (int t = paired ? 0 : stream; t < n_tiles; t += dt, ++turn) {
            const int kbase = (span.first + t) * BN;
            const bool edge = kbase + BN > length || kbase < window_end;
            lag_point();
            ok = wait_all(&s_full[stream], turn & 1, 52);
            if (!ok) break;
            tc_fence_after();
            unsigned seen[4];
            if (edge) {
#pragma unroll
                for (int w = 0; w < 4; ++w) seen[w] = 0u;
                if (mine) {
                    const int j0 = kbase - length;        // the node at column 0, if any
                    const int* const row = p.masks + (size_t)(token0 + node) * p.words;
#pragma unroll
                    for (int w = 0; w < 4; ++w) {
                        const int first = kbase + w * 32, j = j0 + w * 32;
                        unsigned bits = bit_range(lo_r - first, length - first);             // cached keys
                        if (j + 31 >= 0 && j < n) {
                            // the 32 mask bits from bit j on (j may be negative)
                            const int at = j >> 5;        // rounds down
                            const unsigned low = at >= 0 && at < p.words ? (unsigned)row[at] : 0u, high = at + 1 >= 0 && at + 1 < p.words ? (unsigned)row[at + 1] : 0u;
                            unsigned nodes = __funnelshift_r(low, high, (unsigned)(j & 31)) & bit_range(-j, n - j);
                            if (p.window > 0 && lo_r > length) {
                                // a window shorter than the tree is deep
                                for (unsigned left = nodes; left; left &= left - 1) {
                                    const int b = __ffs(left) - 1;
                                    if (p.positions[token0 + j + b] < lo_r) nodes &= ~(1u << b);
                                }
                            }
                            bits |= nodes;
                        }
                        seen[w] = bits;
                    }
                }
            }
            if (active) {
                // Half a row at a time, read twice (for the maximum, for the exponentials): a whole one does not fit the registers that 10 warps leave a thread.
                constexpr int HALF = BN / 2;
                uint32_t sr[HALF];
                auto half_row = [&](int h) {
#pragma unroll
                    for (int c = 0; c < HALF / 32; ++c) tmem_ld32(tmem + (uint32_t)(h * HALF + c * 32), sr + c * 32);
                    tmem_wait_ld();
                    if (edge) {
#pragma unroll
                        for (int c = 0; c < HALF; ++c)
                            if (!((seen[h * 2 + (c >> 5)] >> (c & 31)) & 1u)) sr[c] = __float_as_uint(-INFINITY);
                    }
                };
                half_row(0);
                float top = row_max(sr);
                half_row(1);
                top = fmaxf(top, row_max(sr));
                const float m_new = fmaxf(m_used, top * p.scale_log2);
                const bool grow = m_new > m_used + RESCALE_STEP;      // also true for the first finite maximum
                const float alpha = grow ? (m_used == -INFINITY ? 0.0f : fast_exp2(m_used - m_new)) : 1.0f;
                if (turn > 0 && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
                    for (int c = 0; c < D / 32; ++c) {
                        uint32_t o[32];
                        tmem_ld32(tmem + (uint32_t)(O_COL + c * 32), o);
                        tmem_wait_ld();
#pragma unroll
                        for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                        tmem_st32(tmem + (uint32_t)(O_COL + c * 32), o);
                    }
                }
                if (grow) { l *= alpha; m_used = m_new; }
                const float shift = m_used == -INFINITY ? 0.0f : -m_used;
                // the second half is still in the registers; the first half's P goes where the first half was, so it is the first to go back
                uint32_t keep[HALF / 2];
                l += row_exp2(sr, p.scale_log2, shift);
#pragma unroll
                for (int i = 0; i < HALF / 2; ++i) keep[i] = sr[i];
                half_row(0);
                l += row_exp2(sr, p.scale_log2, shift);
                tmem_st32(tmem, sr);
                tmem_st32(tmem + (uint32_t)(HALF / 2), keep);
                tmem_wait_st();
            }
            if (edge) {
                // the tile's value rows: warp q of a stream looks through and clears keys 32 q .. 32 q + 31 (where both streams read the tile, stream 0's warps do)
                const int v_item = paired ? 1 + 2 * t : n_tiles == 1 ? 1 : 2 + t + min(t, n_tiles - 2);
                const int owner = paired ? 0 : stream, key = kbase + r;
                const bool nobodys = key >= span.total || key < span.lo;
                const uint32_t vrow = ring_s + (v_item % SLOTS) * KV_BYTES + r * ROW_BYTES;
                unsigned mark = 0u;
                if (stream == owner) {
                    ok = wait_all(&slot_full[v_item % SLOTS], (v_item / SLOTS) & 1, 53);
                    if (!ok) break;
                    bool odd = false;
                    if (!nobodys) {
                        uint32_t worst = 0u;              // an exponent of all ones is the largest there is
#pragma unroll
                        for (int i = 0; i < SPANS * 8; ++i) {
                            uint32_t v[4];
                            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                                         : "r"(vrow + (i / 8) * (BN * ROW_BYTES) + (i % 8) * 16));
#pragma unroll
                            for (int k = 0; k < 4; ++k) worst = __vmaxu2(worst, v[k] & 0x7f807f80u);
                        }
                        odd = (worst & 0x7f80u) == 0x7f80u || (worst >> 16) == 0x7f80u;
                    }
                    mark = __ballot_sync(0xffffffffu, odd);
                    if (lane == 0) odd_s[owner][looked & 1][quarter] = mark;
                    if (odd || nobodys) {
#pragma unroll 1
                        for (int i = 0; i < SPANS * 8; ++i)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vrow + (i / 8) * (BN * ROW_BYTES) + (i % 8) * 16), "r"(0u) : "memory");
                    }
                    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // for the tensor core
                }
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&v_checked[owner]));
                ok = wait_all(&v_checked[owner], looked & 1, 54);
                if (!ok) break;
#pragma unroll
                for (int w = 0; w < 4; ++w) sees_odd |= (seen[w] & *(volatile unsigned*)&odd_s[owner][looked & 1][w]) != 0u;
                ++looked;
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&p_full[stream]));
        }
        // ---- the rows' results.  Streams that share the rows meet: each takes half of the columns of both accumulators.
        float weight[2] = {0.0f, 0.0f}, m_all = m_used, l_all = sees_odd ? NAN : l;
        weight[stream] = 1.0f;
        if (!paired) {
            norm_s[stream * BM + r] = make_float2(m_used, l_all);
            __syncwarp();
            if (lane == 0) mbar_arrive(smem_u32(&norms_there));
            ok = wait_all(&norms_there, 0, 55) && ok;
            if (ok) {
                const float2 a = norm_s[r], b = norm_s[BM + r];
                m_all = fmaxf(a.x, b.x);
                weight[0] = a.x == -INFINITY ? 0.0f : fast_exp2(a.x - m_all);
                weight[1] = b.x == -INFINITY ? 0.0f : fast_exp2(b.x - m_all);
                l_all = a.y * weight[0] + b.y * weight[1];
                if (isnan(a.y) || isnan(b.y)) l_all = NAN;
            }
        }
        const bool has[2] = {paired ? stream == 0 && n_tiles > 0 : n_tiles > 0, paired ? stream == 1 && n_tiles > 0 : n_tiles > 1};
        for (int s = 0; s < 2; ++s)
            if (ok && has[s]) ok = wait_all(&o_full[s], 0, 56);
        if (ok && active) {
            tc_fence_after();
            const float inv = p.shares > 1 ? 1.0f : l_all > 0.0f ? 1.0f / l_all : isnan(l_all) ? NAN : 0.0f;
            const float w0 = weight[0] * inv, w1 = weight[1] * inv;
            const size_t row = (size_t)(token0 + node) * p.heads + head;
            const int c_begin = paired ? 0 : stream * (D / 64), c_end = paired ? D / 32 : c_begin + D / 64;
            const uint32_t tmem_rows = tmem_base + ((uint32_t)(quarter * 32) << 16) + (uint32_t)O_COL;
#pragma unroll 1
            for (int c = c_begin; c < c_end; ++c) {
                float o[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) o[i] = 0.0f;
                uint32_t x[32];
                if (has[0]) {
                    tmem_ld32(tmem_rows + (uint32_t)(c * 32), x);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = w0 == 0.0f ? 0.0f : __uint_as_float(x[i]) * w0;
                }
                if (has[1]) {
                    tmem_ld32(tmem_rows + (uint32_t)(STREAM_COLS + c * 32), x);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 32; ++i) o[i] = w1 == 0.0f ? o[i] : fmaf(__uint_as_float(x[i]), w1, o[i]);
                }
                if (mine && p.shares > 1) {
                    float4* const to = reinterpret_cast<float4*>(p.part_out + ((size_t)share * p.tokens * p.heads + row) * D + c * 32);
#pragma unroll
                    for (int i = 0; i < 8; ++i) to[i] = make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                } else if (mine) {
                    uint4* const to = reinterpret_cast<uint4*>(p.out + row * D + c * 32);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        to[i] = make_uint4(pack_bf16(o[8 * i], o[8 * i + 1]), pack_bf16(o[8 * i + 2], o[8 * i + 3]), pack_bf16(o[8 * i + 4], o[8 * i + 5]),
                                           pack_bf16(o[8 * i + 6], o[8 * i + 7]));
                }
                __syncwarp();
            }
            if (mine && p.shares > 1 && (paired || stream == 0)) p.part_norm[(size_t)share * p.tokens * p.heads + row] = make_float2(m_all, l_all);
        }
        if (!ok) failed_s = 1;
    }

    tc_fence_before();
    __syncthreads();
    if (failed_s && warp == 0 && lane == 0) {
        // give the copies in flight a bounded chance to land before the CTA's memory goes away
        mbar_wait(smem_u32(&q_full), 0, nullptr, 0);
        for (int i = max(0, issued - SLOTS); i < issued; ++i) mbar_wait(smem_u32(&slot_full[i % SLOTS]), (i / SLOTS) & 1, nullptr, 0);
    }
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)TMEM_COLS) : "memory");
    }
}

// The shares of a row in their order: a quarter warp a row, four columns of a span a lane.
constexpr int JOIN_THREADS = 128;
__global__ void __launch_bounds__(JOIN_THREADS) draft_join_tc_kernel(TcParams p) {
    pdl_prologue();
    constexpr int LANES = D / 4, ROWS = JOIN_THREADS / LANES;
    const int seq = blockIdx.y, start = p.starts[seq], n = p.starts[seq + 1] - start, length = p.lengths[seq];
    const int at = blockIdx.x * ROWS + threadIdx.x / LANES, c = (threadIdx.x % LANES) * 4;
    if (at >= min(n, p.max_nodes) * p.heads) return;
    const size_t row = (size_t)start * p.heads + at, all_rows = (size_t)p.tokens * p.heads;
    const int lo = p.window > 0 ? max(0, length - p.window + 1) : 0, per = p.share / BN;
    const int shares = min(p.shares, ((length + n + BN - 1) / BN - lo / BN + per - 1) / per);
    float top = -INFINITY;
    for (int s = 0; s < shares; ++s) top = fmaxf(top, p.part_norm[s * all_rows + row].x);
    float4 acc = make_float4(0, 0, 0, 0);
    float sum = 0.0f;
#pragma unroll 4
    for (int s = 0; s < shares; ++s) {
        const float2 norm = p.part_norm[s * all_rows + row];
        const float4 o = *reinterpret_cast<const float4*>(p.part_out + (s * all_rows + row) * D + c);
        const float w = norm.x == -INFINITY ? 0.0f : exp2f(norm.x - top);
        if (norm.x == -INFINITY && !isnan(norm.y)) continue;
        sum += isnan(norm.y) ? NAN : norm.y * w;
        acc = make_float4(fmaf(w, o.x, acc.x), fmaf(w, o.y, acc.y), fmaf(w, o.z, acc.z), fmaf(w, o.w, acc.w));
    }
    const float inv = sum > 0.0f ? 1.0f / sum : isnan(sum) ? NAN : 0.0f;
    *reinterpret_cast<uint2*>(p.out + row * D + c) = make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
}

// --------------------------------------------------------------------------------- host side
typedef CUresult (*EncodeTiledFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*, const cuuint64_t*,
                                  const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave, CUtensorMapSwizzle,
                                  CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void* sym = nullptr;
        cudaDriverEntryPointQueryResult res;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &sym, cudaEnableDefault, &res) == cudaSuccess &&
            res == cudaDriverEntryPointSuccess)
            fn = (EncodeTiledFn)sym;
    }
    return fn;
}


int encode(CUtensorMap* map, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail(MLB_CUDA_ERROR, "draft_attention_tc: cuTensorMapEncodeTiled is not available from this driver");
    cuuint32_t elem[3] = {1, 1, 1};
    CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, rank, const_cast<void*>(base), dims, strides, box, elem, CU_TENSOR_MAP_INTERLEAVE_NONE,
                    CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(MLB_CUDA_ERROR, "draft_attention_tc: cuTensorMapEncodeTiled failed with %d", (int)r);
    return MLB_OK;
}

}  // namespace

// q and out [T, NH * D] bf16, pages [num_pages, 2, NKV, page_size, D].  scratch: shares > 1: [shares, T * NH, D] fp32, then [shares, T * NH] float2.
MLB_EXPORT int mlb_draft_attention_tc(const void* q, const void* pages, void* out, const int* starts, const int* lengths, const int* positions, const int* masks,
                                      int words, const int* table, int max_blocks, int num_pages, int page_size, int tokens, int sequences, int max_nodes,
                                      int heads, int kv_heads, float scale, int window, int share, int shares, void* scratch, int* error_flag,
                                      cudaStream_t stream) {
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || heads / kv_heads > BM)
        return fail(MLB_UNSUPPORTED_SIZE, "draft_attention_tc: heads %d/%d", heads, kv_heads);
    if (words <= 0 || words > MAX_WORDS || max_nodes <= 0 || max_nodes > words * 32)
        return fail(MLB_UNSUPPORTED_SIZE, "draft_attention_tc: %d nodes in masks of %d words (at most %d)", max_nodes, words, MAX_WORDS);
    if (page_size < 8 || page_size % 8 != 0 || BN % page_size != 0 || BN / page_size > MAX_PAGES_PER_TILE)
        return fail(MLB_UNSUPPORTED_SIZE, "draft_attention_tc: page_size %d must be a multiple of 8 that divides %d", page_size, BN);
    if (!(scale > 0.0f)) return fail(MLB_UNSUPPORTED_SIZE, "draft_attention_tc: the softmax scale must be positive");
    if (num_pages <= 0 || max_blocks <= 0 || tokens < 0 || sequences < 0 || window < 0) return fail(MLB_INVALID_ARGUMENT, "draft_attention_tc: bad sizes");
    if (share <= 0 || share % BN != 0 || shares <= 0 || (shares > 1 && !scratch)) return fail(MLB_INVALID_ARGUMENT, "draft_attention_tc: bad shares");
    if (((uintptr_t)q & 15) || ((uintptr_t)out & 15) || ((uintptr_t)pages & 15) || ((uintptr_t)scratch & 15))
        return fail(MLB_UNSUPPORTED_SIZE, "draft_attention_tc: q, out, the pages and the scratch must be 16-byte aligned");
    const long long kv_rows = (long long)num_pages * 2 * kv_heads * page_size;
    if (kv_rows >= (1ll << 31)) return fail(MLB_UNSUPPORTED_SIZE, "draft_attention_tc: the cache has too many rows (%lld)", kv_rows);
    const int group = heads / kv_heads, tile_nodes = BM / group, pairs = (max_nodes + 2 * tile_nodes - 1) / (2 * tile_nodes);
    if (sequences > 65535 || pairs * kv_heads > 65535) return fail(MLB_UNSUPPORTED_SIZE, "draft_attention_tc: too many sequences or rows");
    if (tokens == 0 || sequences == 0) return MLB_OK;

    CUtensorMap map_q, map_kv;
    {
        const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)tokens}, strides[2] = {(cuuint64_t)D * 2, (cuuint64_t)heads * D * 2};
        const cuuint32_t box[3] = {64u, (cuuint32_t)group, (cuuint32_t)tile_nodes};
        const int status = encode(&map_q, q, 3, dims, strides, box);
        if (status != MLB_OK) return status;
    }
    {
        const cuuint64_t dims[2] = {(cuuint64_t)D, (cuuint64_t)kv_rows}, strides[1] = {(cuuint64_t)D * 2};
        const cuuint32_t box[2] = {64u, (cuuint32_t)page_size};
        const int status = encode(&map_kv, pages, 2, dims, strides, box);
        if (status != MLB_OK) return status;
    }
    TcParams p{(__nv_bfloat16*)out, starts, lengths, positions, masks, table, words, max_blocks, num_pages, page_size, BN / page_size, heads, kv_heads, group,
               tile_nodes, pairs, window, max_nodes, share, shares, tokens, scale * LOG2E, nullptr, nullptr, error_flag};
    p.part_out = (float*)scratch;
    p.part_norm = (float2*)((float*)scratch + (size_t)shares * tokens * heads * D);
    static bool configured_on[MAX_DEVICES] = {false};         // the attribute belongs to the device
    bool& configured = configured_on[device_index()];
    if (!configured) {
        if (cudaFuncSetAttribute(draft_attention_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES) != cudaSuccess)
            return check_launch("draft_attention_tc: shared memory");
        configured = true;
    }
    launch_kernel(draft_attention_tc_kernel, dim3(shares, pairs * kv_heads, sequences), THREADS, SMEM_BYTES, stream, map_q, map_kv, p);
    const int status = check_launch("draft_attention_tc");
    if (status != MLB_OK || shares == 1) return status;
    constexpr int rows = JOIN_THREADS / (D / 4);
    launch_kernel(draft_join_tc_kernel, dim3((max_nodes * heads + rows - 1) / rows, sequences), JOIN_THREADS, 0, stream, p);
    return check_launch("draft_join_tc");
}
