// Attention of drafted trees over the paged bf16 cache on the fifth-generation tensor cores, heads of 64 or 128 (-DHEAD_DIM).  What a
// row sees is csrc/drafts.cu's.  P is rounded to bf16 for the second product, which tensor cores take no wider beside bf16 values: half a step of each weight, both ways
// (outputs are off by 0.0019 to 0.0023 of their norm against 64 bits, of which 0.0017 is the output's own rounding).  The row's sum is of the weights before that.
//
// An item is the rows (node, head of the group) of up to 2 x floor(128 / group) nodes of one sequence and kv head.  It has two streams of work, each
// with four softmax warps (a thread a row), its own scores and its own accumulator in tensor memory:
//     more nodes than one row tile holds:  a stream a row tile, both over every key tile of 128, which is loaded once for the two
//     else: both streams have the same rows; one takes the even key tiles, the other the odd ones, and they meet at the end
// so that one stream's softmax runs beside the other's products.
//
// The work of a call is a line of units (a row tile times a key tile), sequence after sequence, and every CTA takes an equal
// stretch of it: the device counts the units from the lengths and trees as they are, so sequences of all lengths and trees of all sizes
// fill the CTAs evenly.  A CTA's stretch may end in one item and begin in another; an item that lies in several CTAs leaves a partial result in each,
// which a second kernel joins in order.
//
//     warp 0      TMA: key and value tiles page by page into a ring, in the order in which the products need them
//     warp 3      TMA: a piece's queries (a box of heads x nodes, rows in the order node * group + head)
//     warp 1      one thread issues tcgen05.mma: S = Q K^T; O += P V with P in tensor memory.  P overwrites the scores it was made of; the next scores of a stream
//                 are issued behind the product that reads P, so "scores are there" also says that the accumulator is (the tensor pipe runs in order)
//     warps 4-11  softmax of stream (warp - 4) / 4: mask in the tiles that need one, running maximum and sum in fp32 with base-2
//                 exponentials, the accumulator rescaled only when a row's maximum has grown by 2^8
// In tiles that not every row sees alike the value rows are looked through: a number that is not finite is cleared for the product (0 * NaN would reach rows
// that do not see it), and the rows that do see it add it, in its column, where their results go out (this way out costs calls without such values 1 %: 16 ragged sequences
// 77.0 -> 77.9 us for two layers, 4 of 8,192 keys 157.4 -> 158.9); value rows that nobody sees are cleared as a whole.
//
// What bounds it.  Long calls: the products and the softmax beside one another (40 heads of 8, 50 nodes, 4 sequences, for every 16,384 keys of them all: products alone 55 us,
// softmax alone 61, both 70; memory alone 40).  4 sequences of 8,192 keys and 64 nodes take 70 us a layer with the join (73 to 75 in a long series of calls): 43 GFLOP, 0.62 PFLOP/s, of rows that fill 320 of
// 384 tensor-core rows.  Short calls: a chain that nothing fills, from the wait for the kernel in front on: cutting the line 1.4 us, block table, copies and first scores 2.5,
// a turn 1.6, results 2.3, then the join 5 (one sequence of 2,074 keys and 26 nodes, 12 heads of 2: 14.8 us).
//
// Tried and slower: tiles of 64 keys with two score buffers a stream (Q's rows come from shared memory as often for half the keys), two softmax threads a row (159 us against
// 145 for two layers of the long call above), an issuing warp for each stream (92 us a layer against 70: the streams' products alternate in the tensor pipe).
//
// Every wait on an mbarrier is bounded; when a bound is hit the error flag is raised, the CTA waits (bounded) for the products and copies in flight, frees
// its tensor memory and returns.
#include "common.cuh"
#include "packed.cuh"

#include <cuda.h>

#include <algorithm>

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
constexpr int SHARED_BYTES = 3 << 10;          // barriers and what the warps tell one another, behind the tiles
constexpr int SMEM_BYTES = 2 * Q_BYTES + SLOTS * KV_BYTES + SHARED_BYTES;
static_assert(SMEM_BYTES <= 227 * 1024, "a CTA's shared memory");
constexpr int THREADS = 384;
// 384 threads start with 168 registers each; the softmax warps hold a whole row of scores
constexpr int FEW_REGISTERS = 80, MANY_REGISTERS = 208;
static_assert(128 * FEW_REGISTERS + 256 * MANY_REGISTERS <= THREADS * 168, "no more than the launch has");
constexpr int STREAM_COLS = 256;             // tensor memory of a stream: scores (then P as bf16 pairs) [0, 128), accumulator [128, 128 + D)
constexpr int TMEM_COLS = 2 * STREAM_COLS;
constexpr int O_COL = BN;
#ifndef MLB_SPIN_LIMIT                       // (the tests build objects whose waits run out at once)
#define MLB_SPIN_LIMIT (1 << 21)
#endif
constexpr int SPIN_LIMIT = MLB_SPIN_LIMIT;   // polls of up to 2 us each
constexpr int DRAIN_LIMIT = 1 << 14;         // the same for what is in flight when a wait has run out: microseconds, or never
constexpr int MAX_PAGES_PER_TILE = 16;
constexpr int MAX_WORDS = 8;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float RESCALE_STEP = 8.0f;
constexpr int CHUNK = 32;                    // scores that a softmax thread has in registers at a time

struct TcParams {
    __nv_bfloat16* out;             // [T, NH * D]
    const __nv_bfloat16* pages;     // [num_pages, 2, NKV, page_size, D]: what the key and value map describes
    const int* starts;              // [A + 1]
    const int* lengths;             // [A]
    const int* positions;           // [T]
    const int* masks;               // [T, words]
    const int* table;               // [A, max_blocks]
    int words, max_blocks, num_pages, page_size, pages_per_tile;
    int heads, kv_heads, group, tile_nodes, row_tiles, window, max_nodes;      // row_tiles: of a sequence of max_nodes
    int stretch;                    // units of a CTA at least
    int ctas, sequences, tokens;
    int reach;                      // keys that a row of the table has blocks for
    float scale_log2;
    float* part_out;                // [ctas, 2, 2, D, BM]: of the item that a CTA's stretch begins in, and of the one that it ends in; a column's rows together
    float2* part_norm;              // [ctas, 2, 2, BM]
    int* line;                      // [2 + sequences]: units a CTA, units an item begins with, then every sequence's first unit (what the join asks for)
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
__device__ __forceinline__ void mbar_drain(uint32_t bar, uint32_t parity) {
    for (int i = 0; i < DRAIN_LIMIT; ++i)
        if (mbar_try_wait(bar, parity)) return;
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
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t* r) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
                   "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
                 ::"r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
                   "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
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

// The largest of a row's scores, NaN where one is: eight chains of three operands a step.
__device__ __forceinline__ float max_nan(float a, float b, float c) {       // NaN where one of them is
    float r;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
    return r;
}
template <int N>
__device__ __forceinline__ float row_max(const uint32_t (&s)[N]) {
    auto at = [&](int i) { return __uint_as_float(s[i]); };
    float m[8];
#pragma unroll
    for (int k = 0; k < 8; ++k) m[k] = max_nan(at(2 * k), at(2 * k + 1), at(2 * k + 1));
#pragma unroll
    for (int c = 16; c < N; c += 2) m[(c >> 1) & 7] = max_nan(m[(c >> 1) & 7], at(c), at(c + 1));
    return max_nan(max_nan(m[0], m[1], m[2]), max_nan(m[3], m[4], m[5]), max_nan(m[6], m[7], m[7]));
}

typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float lo, float hi) { return ((f32x2)__float_as_uint(hi) << 32) | __float_as_uint(lo); }
__device__ __forceinline__ float low(f32x2 v) { return __uint_as_float((uint32_t)v); }
__device__ __forceinline__ float high(f32x2 v) { return __uint_as_float((uint32_t)(v >> 32)); }
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
    f32x2 r;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
    return r;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
// P = 2^(s * scale + shift) of N of a row's scores, as bf16 pairs in s[0 .. N / 2); returns the sum of the fp32 terms: neighbours first, then four
// chains of them.  Scaling and summing go two to an instruction, each rounded as always.
template <int N>
__device__ __forceinline__ float row_exp2(uint32_t (&s)[N], float scale, float shift) {
    const f32x2 scale2 = pair(scale, scale), shift2 = pair(shift, shift);
    f32x2 chains[2] = {0ull, 0ull};          // chains 0 and 1, 2 and 3
#pragma unroll
    for (int c = 0; c < N; c += 4) {
        float p[4];
#pragma unroll
        for (int i = 0; i < 4; i += 2) {
            const f32x2 x = fma2(pair(__uint_as_float(s[c + i]), __uint_as_float(s[c + i + 1])), scale2, shift2);
            p[i] = fast_exp2(low(x));
            p[i + 1] = fast_exp2(high(x));
        }
        chains[(c >> 2) & 1] = add2(chains[(c >> 2) & 1], add2(pair(p[0], p[2]), pair(p[1], p[3])));
        s[c / 2] = pack_bf16(p[0], p[1]);
        s[c / 2 + 1] = pack_bf16(p[2], p[3]);
    }
    return (low(chains[0]) + high(chains[0])) + (low(chains[1]) + high(chains[1]));
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

// A sequence's part of the line.
struct Sequence {
    int token0, n, length, lo, first, tiles, row_tiles;    // lo: the first key any node may see; first: its tile
    __device__ __forceinline__ int items() const { return (row_tiles + 1) >> 1; }       // of a head
    __device__ __forceinline__ int units(int kv_heads, int lead) const { return kv_heads * (tiles * row_tiles + lead * items()); }
};
__device__ __forceinline__ Sequence sequence_at(const TcParams& p, int a) {
    Sequence s;
    s.token0 = p.starts[a];
    const int end = p.starts[a + 1];
    s.n = s.token0 < 0 || end > p.tokens ? 0 : min(end - s.token0, p.max_nodes);      // (rows that are not there: the flag is raised where the kernel begins)
    s.length = p.lengths[a];
    if (s.length < 0 || s.length > p.reach - s.n) s.length = s.n = 0;                 // (so are keys that are not)
    s.lo = p.window > 0 ? max(0, s.length - p.window + 1) : 0;
    s.first = s.lo / BN;
    s.tiles = s.n > 0 ? (s.length + s.n + BN - 1) / BN - s.first : 0;
    s.row_tiles = s.n > 0 ? (s.n + p.tile_nodes - 1) / p.tile_nodes : 0;
    return s;
}

// How the line is cut, by one whole warp: units a CTA, and for this CTA its stretch, the sequence that it begins in and that one's first unit.  CTA 0
// leaves all sequences' first units for the join.
//
// Every item begins with `lead` units that stand for no work: what it costs a CTA to end one item (results out, accumulators free) and begin another.  CTAs' times in
// eight calls of all kinds are 1.2 us a unit, 4.5 us an item, 1 us more a tile that needs masks, within 1 us; without `lead` the CTAs that hold an item's end and the
// next one's beginning were the last by a fifth of the kernel's time.  4, 5 and 6 units at most: 16 sequences of up to 2,048 keys and 64 nodes 37.8, 37.5, 37.3 us a
// layer, 4 of 8,192 keys 69.8, 70.1, 71.0.  Shorter stretches take less, and the shortest none (a unit more a CTA would be a turn more: one sequence of 2,074 keys and
// 26 nodes, 12 heads of 2, 15.7 us instead of 17.3).
constexpr int MOST_LEAD = 5;
struct Cut {
    int stretch, lead, unit, end, a, base;
};
__device__ __forceinline__ Cut cut_line(const TcParams& p, int lane) {
    auto sequence = [&](int a) {
        if (a < p.sequences) return sequence_at(p, a);
        Sequence none = {};
        return none;
    };
    const Sequence mine = sequence(lane);                 // of the first 32 sequences, most calls' only ones
    int total = mine.units(p.kv_heads, 0), items = mine.items() * p.kv_heads;
    for (int a = lane + 32; a < p.sequences; a += 32) {
        const Sequence s = sequence(a);
        total += s.units(p.kv_heads, 0);
        items += s.items() * p.kv_heads;
    }
    total = __reduce_add_sync(0xffffffffu, total);
    items = __reduce_add_sync(0xffffffffu, items);
    Cut c;
    const int each = (total + p.ctas - 1) / p.ctas;
    c.lead = each <= p.stretch ? 0 : min(MOST_LEAD, each);
    total += items * c.lead;
    c.stretch = max(p.stretch, (total + p.ctas - 1) / p.ctas);
    c.unit = min((int)blockIdx.x * c.stretch, total);
    c.end = min(c.unit + c.stretch, total);
    c.a = p.sequences;
    c.base = 0;
    if (blockIdx.x == 0 && lane == 0 && p.line) {
        p.line[0] = c.stretch;
        p.line[1] = c.lead;
    }
    int base = 0;
    for (int a0 = 0; a0 < p.sequences; a0 += 32) {
        const int units = (a0 ? sequence(a0 + lane) : mine).units(p.kv_heads, c.lead);
        int sum = units;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int other = __shfl_up_sync(0xffffffffu, sum, o);
            if (lane >= o) sum += other;
        }
        if (blockIdx.x == 0 && p.line && a0 + lane < p.sequences) p.line[2 + a0 + lane] = base + sum - units;
        const unsigned hit = __ballot_sync(0xffffffffu, units > 0 && base + sum > c.unit);
        if (hit && c.a == p.sequences) {
            const int at = __ffs(hit) - 1;
            c.a = a0 + at;
            c.base = base + __shfl_sync(0xffffffffu, sum - units, at);
            if (blockIdx.x != 0 || !p.line) break;
        }
        base += __shfl_sync(0xffffffffu, sum, 31);
    }
    return c;
}

// One item of a sequence, and the key tiles of it that the units [from, to) are.
struct Item {
    int kvh, node0, begin, work, end;    // its units: begin .. work stand for no tile
    bool paired;
};
__device__ __forceinline__ Item item_of(const TcParams& p, const Sequence& s, int base, int lead, int kvh, int pair) {
    Item i;
    i.kvh = kvh;
    i.node0 = pair * 2 * p.tile_nodes;
    i.paired = s.row_tiles - 2 * pair >= 2;
    i.begin = base + kvh * s.units(1, lead) + pair * (2 * s.tiles + lead);
    i.work = i.begin + lead;
    i.end = i.work + (i.paired ? 2 : 1) * s.tiles;
    return i;
}
__device__ __forceinline__ Item item_at(const TcParams& p, const Sequence& s, int base, int lead, int unit) {
    const int per_head = s.units(1, lead), at = unit - base, kvh = at / per_head;
    return item_of(p, s, base, lead, kvh, (at - kvh * per_head) / (2 * s.tiles + lead));
}
// a unit of an item as a key tile: a cut between the two units of a paired item's tile counts the tile to the part in front
__device__ __forceinline__ int tile_of(const Item& i, int unit) {
    const int at = max(0, unit - i.work);
    return i.paired ? (at + 1) >> 1 : at;
}

// What a CTA walks through: every role has its own.
struct Walk {
    int unit, end, a, base, known;       // known: the sequence that `s` is of
    Sequence s;
    Item item;
    int tile, n_tiles, part, parts;      // first key tile (from s.first), how many, which part of how many
    __device__ __forceinline__ bool next(const TcParams& p, int stretch, int lead) {
        while (unit < end) {
            while (true) {
                if (a != known) s = sequence_at(p, a);
                known = a;
                const int units = s.units(p.kv_heads, lead);
                if (unit < base + units) break;
                base += units;
                ++a;
            }
            item = item_at(p, s, base, lead, unit);
            const int to = min(end, item.end);
            tile = tile_of(item, unit);
            n_tiles = tile_of(item, to) - tile;
            part = unit / stretch - item.begin / stretch;
            parts = (item.end - 1) / stretch - item.begin / stretch + 1;
            unit = to;
            if (n_tiles > 0) return true;
        }
        return false;
    }
};

struct Shared {
    unsigned long long q_full, q_empty, slot_full[SLOTS], slot_empty[SLOTS], s_full[2], p_full[2], o_full[2], v_checked[3], norms_there, o_read, stopped;
    uint32_t tmem_base;
    int failed, unit, end, a, base, stretch, lead, pieces, issued;      // pieces, issued: whose copies were asked for
    Sequence s;
    unsigned odd[3][2][4];               // [streams, or both][turn & 1]: which of a tile's value rows are not finite
    float2 norm[2 * BM];                 // the rows' maxima and sums, for streams that share the rows
    bool reads_odd[2 * BM];              // and whether they see such a value row
};
static_assert(sizeof(Shared) <= SHARED_BYTES, "what the warps tell one another");

__global__ void __launch_bounds__(THREADS, 1)
draft_attention_tc_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_kv, TcParams p) {
    extern __shared__ __align__(1024) unsigned char smem_dyn[];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const uint32_t base = smem_u32(smem_dyn);
    const uint32_t q_s = base;
    const uint32_t ring_s = q_s + 2 * Q_BYTES;
    Shared& sh = *reinterpret_cast<Shared*>(smem_dyn + 2 * Q_BYTES + SLOTS * KV_BYTES);

    if (warp == 3 && lane < 2) asm volatile("prefetch.tensormap [%0];" ::"l"(lane ? &map_kv : &map_q) : "memory");
    if (threadIdx.x == 0) {
        mbar_init(smem_u32(&sh.q_full), 1);
        mbar_init(smem_u32(&sh.q_empty), 1);
        for (int s = 0; s < SLOTS; ++s) {
            mbar_init(smem_u32(&sh.slot_full[s]), 1);
            mbar_init(smem_u32(&sh.slot_empty[s]), 1);
        }
        for (int s = 0; s < 2; ++s) {
            mbar_init(smem_u32(&sh.s_full[s]), 1);
            mbar_init(smem_u32(&sh.p_full[s]), 4);          // one arrival per softmax warp
            mbar_init(smem_u32(&sh.o_full[s]), 1);
            mbar_init(smem_u32(&sh.v_checked[s]), 4);
        }
        mbar_init(smem_u32(&sh.v_checked[2]), 8);
        mbar_init(smem_u32(&sh.norms_there), 8);
        mbar_init(smem_u32(&sh.o_read), 8);
        mbar_init(smem_u32(&sh.stopped), 1);                // all products that were issued are done
        sh.failed = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    }
    pdl_wait();                  // queries, this step's keys, and the sequences' extents may be the kernel before's
    // The tensor memory is taken between the wait and the next kernel's early start: neither a kernel in front that still needs some nor one
    // behind that already waits for this one can stand in the way, or be stood in the way of.
    if (warp == 1) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;"
                     ::"r"(smem_u32(&sh.tmem_base)), "r"((uint32_t)TMEM_COLS) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    if (warp == 2) {
        const Cut cut = cut_line(p, lane);
        const Sequence s = sequence_at(p, min(cut.a, p.sequences - 1));
        if (lane == 0) {
            sh.s = s;
            sh.unit = cut.unit;
            sh.end = cut.end;
            sh.a = cut.a;
            sh.base = cut.base;
            sh.stretch = cut.stretch;
            sh.lead = cut.lead;
        }
    } else if (warp == 4 && blockIdx.x == 0) {
        for (int a = lane; a < p.sequences; a += 32) {
            const int start = p.starts[a], end = p.starts[a + 1], length = p.lengths[a];
            if (start < 0 || end > p.tokens || end - start > p.max_nodes) {
                if (p.error_flag) atomicExch(p.error_flag, 3);
            } else if (end > start && (length < 0 || length > p.reach - (end - start))) {
                if (p.error_flag) atomicExch(p.error_flag, 2);
            }
        }
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem_base = sh.tmem_base;
    const int stretch = sh.stretch, lead = sh.lead;
    Walk walk;
    const bool misplaced = (base & 1023u) != 0;             // the swizzle pattern wants 1024-byte alignment
    walk.unit = misplaced ? sh.end : sh.unit;
    walk.end = sh.end;
    walk.a = sh.a;
    walk.base = sh.base;
    walk.known = sh.a;
    walk.s = sh.s;
    if (misplaced && threadIdx.x == 0 && p.error_flag) atomicCAS(p.error_flag, 0, 40);

    // Ring items in order of need, piece after piece.  Shared key tiles: K0 K1 V0 K2 V1 K3 ..; a row tile a stream: K0 V0 K1 V1 ..: K(0 .. dt - 1)
    // first, then for every t: V(t), K(t + dt).  A piece of n key tiles is 2 n items.
    if (warp < 4) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(FEW_REGISTERS));
        if (warp == 0) {
            // -------------------------------------------------------------- keys and values (whole warp)
            bool ok = true;
            int issued = 0;
            while (ok && walk.next(p, stretch, lead)) {
                const Sequence& s = walk.s;
                const int dt = walk.item.paired ? 1 : 2, n_tiles = walk.n_tiles;
                const int* table = p.table + (size_t)walk.a * p.max_blocks;
                // lane g: the page of block g of a tile.  Two key tiles' pages are on their way ahead of their use.
                auto lookup = [&](int t) {
                    const int block = (s.first + walk.tile + t) * p.pages_per_tile + lane;
                    return t < n_tiles && lane < p.pages_per_tile && block < p.max_blocks ? __ldg(table + block) : -1;
                };
                auto load = [&](int t, int page, int is_v) {
                    lag_point();
                    const int slot = issued % SLOTS;
                    if (issued >= SLOTS) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.slot_empty[slot]), ((issued / SLOTS) - 1) & 1, p.error_flag, 42)) != 0;
                    if (!ok) return;
                    const uint32_t bar = smem_u32(&sh.slot_full[slot]);
                    if (lane == 0) mbar_expect_tx(bar, KV_BYTES);
                    __syncwarp();
                    if (lane < p.pages_per_tile) {
                        if (page < 0 || page >= p.num_pages) {
                            // a page that holds a key some row may see has to exist; the others are masked
                            const int first_key = ((s.first + walk.tile + t) * p.pages_per_tile + lane) * p.page_size;
                            if (first_key < s.length + s.n && first_key + p.page_size > s.lo && p.error_flag) atomicExch(p.error_flag, 2);
                            page = 0;
                        }
                        const int row = ((page * 2 + is_v) * p.kv_heads + walk.item.kvh) * p.page_size;
                        const uint32_t dst = ring_s + slot * KV_BYTES + lane * p.page_size * ROW_BYTES;
#pragma unroll
                        for (int c = 0; c < SPANS; ++c) tma_load_2d(dst + c * BN * ROW_BYTES, &map_kv, c * 64, row, bar);
                    }
                    ++issued;
                };
                int page = lookup(0), next = lookup(1), after = lookup(2);       // of tiles t, t + 1, t + 2
                load(0, page, 0);
                if (ok && dt == 2 && n_tiles > 1) load(1, next, 0);
                for (int t = 0; t < n_tiles && ok; ++t) {
                    const int third = lookup(t + 3);
                    load(t, page, 1);
                    if (ok && t + dt < n_tiles) load(t + dt, dt == 1 ? next : after, 0);
                    page = next;
                    next = after;
                    after = third;
                }
            }
            if (!ok && lane == 0) sh.failed = 1;
            if (lane == 0) sh.issued = issued;
        } else if (warp == 3) {
            // -------------------------------------------------------------- queries: a piece ahead of the products at most
            bool ok = true;
            int pieces = 0;
            for (; walk.next(p, stretch, lead); ++pieces) {
                lag_point();
                if (pieces > 0) ok = __all_sync(0xffffffffu, mbar_wait(smem_u32(&sh.q_empty), (pieces - 1) & 1, p.error_flag, 41)) != 0;
                if (!ok) break;
                if (lane == 0) {
                    const int boxes = walk.item.paired ? 2 : 1;
                    mbar_expect_tx(smem_u32(&sh.q_full), boxes * SPANS * p.tile_nodes * p.group * ROW_BYTES);
                    for (int b = 0; b < boxes; ++b)
#pragma unroll
                        for (int c = 0; c < SPANS; ++c)
                            tma_load_3d(q_s + b * Q_BYTES + c * BM * ROW_BYTES, &map_q, c * 64, walk.item.kvh * p.group, walk.s.token0 + walk.item.node0 + b * p.tile_nodes,
                                        smem_u32(&sh.q_full));
                }
                __syncwarp();
            }
            if (!ok && lane == 0) sh.failed = 1;
            if (lane == 0) sh.pieces = pieces;
        } else if (warp == 1) {
            // -------------------------------------------------------------- MMA issue: the warp walks converged, one lane issues
            const uint32_t idesc_qk = idesc(BN, false), idesc_pv = idesc(D, true);
            auto wait_warp = [&](unsigned long long* bar, uint32_t parity, int code) {
                return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, p.error_flag, code)) != 0;
            };
            bool ok = true;
            int item = 0, piece = 0;                           // ring items are consumed in the order they were loaded
            int turn[2] = {0, 0};                              // P's of each stream so far
            auto full = [&](int i, int code) { return wait_warp(&sh.slot_full[i % SLOTS], (i / SLOTS) & 1, code); };
            while (ok && walk.next(p, stretch, lead)) {
                const bool paired = walk.item.paired;
                const int n_tiles = walk.n_tiles;
                auto issue_qk = [&](int s, int i, bool last_use, bool last) {       // stream s's scores from ring item i
                    const uint32_t kb = ring_s + (i % SLOTS) * KV_BYTES, qb = q_s + (paired ? s * Q_BYTES : 0);
                    if (elect_one()) {
                        // (a descriptor's address counts 16 bytes, so the next step's is a sum: made anew each time it cost as long as the product ran)
                        const uint64_t qd = desc_k_major(qb), kd = desc_k_major(kb);
#pragma unroll
                        for (int ks = 0; ks < D / 16; ++ks) {
                            const uint32_t off = ((ks / 4) * (BM * ROW_BYTES) + (ks % 4) * 32) >> 4;
                            umma(tmem_base + (uint32_t)(s * STREAM_COLS), qd + off, kd + off, idesc_qk, ks > 0);
                        }
                        if (last_use) umma_commit(smem_u32(&sh.slot_empty[i % SLOTS]));
                        if (last) umma_commit(smem_u32(&sh.q_empty));
                        umma_commit(smem_u32(&sh.s_full[s]));
                    }
                    __syncwarp();
                };
                auto issue_pv = [&](int s, int i, bool first, bool last, bool last_use) {
                    const uint32_t vb = ring_s + (i % SLOTS) * KV_BYTES;
                    if (elect_one()) {
                        const uint64_t vd = desc_mn_major(vb, BN * ROW_BYTES);
#pragma unroll
                        for (int ks = 0; ks < BN / 16; ++ks)           // 16 keys = 8 columns of P
                            umma_ts(tmem_base + (uint32_t)(s * STREAM_COLS + O_COL), tmem_base + (uint32_t)(s * STREAM_COLS + ks * 8),
                                    vd + ((ks * 16 * ROW_BYTES) >> 4), idesc_pv, (!first || ks > 0) ? 1u : 0u);
                        if (last_use) umma_commit(smem_u32(&sh.slot_empty[i % SLOTS]));
                        if (last) umma_commit(smem_u32(&sh.o_full[s]));
                    }
                    __syncwarp();
                };
                ok = wait_warp(&sh.q_full, piece & 1, 43);
                if (!ok) break;
                ++piece;
                const int dt = paired ? 1 : 2;
                for (int t = 0; t < min(dt, n_tiles) && ok; ++t) {
                    ok = full(item, 44);
                    if (!ok) break;
                    if (paired) {
                        issue_qk(0, item, false, false);
                        issue_qk(1, item, true, n_tiles == 1);
                    } else {
                        issue_qk(t, item, true, t + 1 == n_tiles);
                    }
                    ++item;
                }
                for (int t = 0; t < n_tiles && ok; ++t) {
                    lag_point();
                    const bool more = t + dt < n_tiles, last = t + dt >= n_tiles;
                    const int s0 = paired ? 0 : t & 1;
                    // (the tiles first: they are there long before P, and each look at a barrier costs a hundred cycles of the way from P to the next scores)
                    ok = full(item, 46) && (!more || full(item + 1, 47)) && wait_warp(&sh.p_full[s0], turn[s0] & 1, 45);
                    if (!ok) break;
                    ++turn[s0];
                    tc_fence_after();
                    issue_pv(s0, item, t < dt, last, !paired);
                    if (more) issue_qk(s0, item + 1, !paired, !paired && t + dt + 1 == n_tiles);
                    if (paired) {
                        ok = wait_warp(&sh.p_full[1], turn[1] & 1, 48);
                        if (!ok) break;
                        ++turn[1];
                        tc_fence_after();
                        issue_pv(1, item, t == 0, last, true);
                        if (more) issue_qk(1, item + 1, true, t + 2 == n_tiles);
                    }
                    item += more ? 2 : 1;
                }
            }
            if (!ok && lane == 0) sh.failed = 1;
        }
    } else {
        // ------------------------------------------------------------------ softmax, one thread per row
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(MANY_REGISTERS));
        const int stream = (warp - 4) >> 2;
        const int quarter = warp & 3;                     // the tensor-memory lanes this warp may touch
        const int r = quarter * 32 + lane;
        const uint32_t tmem_rows = tmem_base + ((uint32_t)(quarter * 32) << 16);
        const uint32_t tmem = tmem_rows + (uint32_t)(stream * STREAM_COLS);
        auto wait_all = [&](unsigned long long* bar, uint32_t parity, int code) {
            return __all_sync(0xffffffffu, mbar_wait(smem_u32(bar), parity, p.error_flag, code)) != 0;
        };
        bool ok = true;
        int item0 = 0, turn = 0, shared_pieces = 0;       // the piece's first ring item; this stream's tiles; pieces whose rows the streams share
        int looked[2] = {0, 0};                           // tiles looked through by this stream alone, by both
        int results[2] = {0, 0};                          // accumulators finished, of each stream
        while (ok && walk.next(p, stretch, lead)) {
            const Sequence& s = walk.s;
            const bool paired = walk.item.paired;
            const int n_tiles = walk.n_tiles, kvh = walk.item.kvh, total = s.length + s.n, dt = paired ? 1 : 2;
            const int my_node0 = walk.item.node0 + (paired ? stream * p.tile_nodes : 0);
            const int rows = min(p.tile_nodes, s.n - my_node0) * p.group;
            const bool active = quarter * 32 < rows;      // (the warp) else its rows are nobody's
            const bool mine = r < rows;
            const int node = my_node0 + (mine ? r / p.group : 0), head = kvh * p.group + (mine ? r % p.group : 0);
            const int pos = p.positions[s.token0 + node];
            const int lo_r = p.window > 0 ? max(0, pos - p.window + 1) : 0;
            float m_used = -INFINITY, l = 0.0f;
            bool odd_score = false, odd_value = false;        // the row sees a score that is NaN or +inf, a value in an edge tile that is not finite
            // A tile that not every row sees alike holds a node, or a cached key in front of some node's window.  The latest position is at
            // most length + n - 1.
            const int window_end = p.window > 0 ? max(0, total - p.window) : 0;
            auto is_edge = [&](int kbase) { return kbase + BN > s.length || kbase < window_end; };
            auto seen_of = [&](int from) {                    // which of the 32 keys from `from` on the thread's row sees
                unsigned bits = bit_range(lo_r - from, s.length - from);             // cached keys
                const int j = from - s.length;                // the node at the first of them, if any
                if (j + 31 >= 0 && j < s.n) {
                    // the 32 mask bits from bit j on (j may be negative)
                    const int* const row = p.masks + (size_t)(s.token0 + node) * p.words;
                    const int at = j >> 5;                    // rounds down
                    const unsigned low = at >= 0 && at < p.words ? (unsigned)row[at] : 0u, high = at + 1 >= 0 && at + 1 < p.words ? (unsigned)row[at + 1] : 0u;
                    unsigned nodes = __funnelshift_r(low, high, (unsigned)(j & 31)) & bit_range(-j, s.n - j);
                    if (p.window > 0 && lo_r > s.length) {
                        // a window shorter than the tree is deep
                        for (unsigned left = nodes; left; left &= left - 1) {
                            const int b = __ffs(left) - 1;
                            if (p.positions[s.token0 + j + b] < lo_r) nodes &= ~(1u << b);
                        }
                    }
                    bits |= nodes;
                }
                return bits;
            };
            bool first = true;
            for (int t = paired ? 0 : stream; t < n_tiles; t += dt, ++turn, first = false) {
                const int kbase = (s.first + walk.tile + t) * BN;
                const bool edge = is_edge(kbase);
                unsigned seen[4];
                if (edge) {
#pragma unroll 1
                    for (int w = 0; w < 4; ++w) seen[w] = mine ? seen_of(kbase + w * 32) : 0u;
                }
                lag_point();
                ok = wait_all(&sh.s_full[stream], turn & 1, 49);
                if (!ok) break;
                tc_fence_after();
                if (active) {
                    // CHUNK scores at a time, read twice (for the maximum, for the exponentials)
                    float top = -INFINITY;
#pragma unroll 1
                    for (int c = 0; c < BN / CHUNK; ++c) {
                        uint32_t sr[CHUNK];
#pragma unroll
                        for (int i = 0; i < CHUNK / 32; ++i) tmem_ld32(tmem + (uint32_t)(c * CHUNK + i * 32), sr + i * 32);
                        tmem_wait_ld();
                        if (edge) {
#pragma unroll
                            for (int i = 0; i < CHUNK / 32; ++i) {
                                const unsigned bits = seen[c * (CHUNK / 32) + i];
#pragma unroll
                                for (int k = 0; k < 32; ++k)
                                    if (!((bits >> k) & 1u)) sr[i * 32 + k] = __float_as_uint(-INFINITY);
                                tmem_st32(tmem + (uint32_t)(c * CHUNK + i * 32), sr + i * 32);
                            }
                        }
                        top = max_nan(top, row_max(sr), top);
                    }
                    if (edge) tmem_wait_st();
                    // a score that is NaN or +inf: the row becomes NaN (fmaxf passes over a NaN)
                    if (!(top < INFINITY)) { odd_score = true; top = -INFINITY; }
                    const float m_new = fmaxf(m_used, top * p.scale_log2);
                    const bool grow = m_new > m_used + RESCALE_STEP;      // also true for the first finite maximum
                    const float alpha = grow ? (m_used == -INFINITY ? 0.0f : fast_exp2(m_used - m_new)) : 1.0f;
                    if (!first && __any_sync(0xffffffffu, grow)) {
#pragma unroll 1
                        for (int c = 0; c < D / 16; ++c) {
                            uint32_t o[16];
                            tmem_ld16(tmem + (uint32_t)(O_COL + c * 16), o);
                            tmem_wait_ld();
#pragma unroll
                            for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * alpha);
                            tmem_st16(tmem + (uint32_t)(O_COL + c * 16), o);
                        }
                    }
                    if (grow) { l *= alpha; m_used = m_new; }
                    const float shift = m_used == -INFINITY ? 0.0f : -m_used;
                    // (P of a chunk goes where this chunk's or an earlier one's scores were)
#pragma unroll 1
                    for (int c = 0; c < BN / CHUNK; ++c) {
                        uint32_t sr[CHUNK];
#pragma unroll
                        for (int i = 0; i < CHUNK / 32; ++i) tmem_ld32(tmem + (uint32_t)(c * CHUNK + i * 32), sr + i * 32);
                        tmem_wait_ld();
                        l += row_exp2(sr, p.scale_log2, shift);
                        tmem_st16(tmem + (uint32_t)(c * (CHUNK / 2)), sr);
                    }
                    tmem_wait_st();
                }
                if (edge) {
                    // the tile's value rows: warp q of a stream looks through and clears keys 32 q .. 32 q + 31 (where both streams read the tile, stream 0's warps do)
                    const int v_item = item0 + (paired ? 1 + 2 * t : n_tiles == 1 ? 1 : 2 + t + min(t, n_tiles - 2));
                    const int which = paired ? 2 : stream, buffer = looked[paired] & 1, key = kbase + r;
                    const bool nobodys = key >= total || key < s.lo;
                    const uint32_t vrow = ring_s + (v_item % SLOTS) * KV_BYTES + r * ROW_BYTES;
                    if (!paired || stream == 0) {
                        ok = wait_all(&sh.slot_full[v_item % SLOTS], (v_item / SLOTS) & 1, 50);
                        if (!ok) break;
                        bool odd = false;
                        if (!nobodys) {
                            uint32_t worst = 0u;          // an exponent of all ones is the largest there is
#pragma unroll 4
                            for (int i = 0; i < SPANS * 8; ++i) {
                                uint32_t v[4];
                                asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];" : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3])
                                             : "r"(vrow + (i / 8) * (BN * ROW_BYTES) + ((i ^ lane) & 7) * 16));      // neighbouring rows in different banks
#pragma unroll
                                for (int k = 0; k < 4; ++k) worst = __vmaxu2(worst, v[k] & 0x7f807f80u);
                            }
                            odd = (worst & 0x7f80u) == 0x7f80u || (worst >> 16) == 0x7f80u;
                        }
                        const unsigned mark = __ballot_sync(0xffffffffu, odd);
                        if (lane == 0) sh.odd[which][buffer][quarter] = mark;
                        if (nobodys) {
#pragma unroll 1
                            for (int i = 0; i < SPANS * 8; ++i)
                                asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(vrow + (i / 8) * (BN * ROW_BYTES) + ((i ^ lane) & 7) * 16), "r"(0u) : "memory");
                        } else if (odd) {
#pragma unroll 1
                            for (int i = 0; i < SPANS * 32; ++i) {
                                const uint32_t at = vrow + (i / 32) * (BN * ROW_BYTES) + (i % 32) * 4;
                                uint32_t v;
                                asm volatile("ld.shared.b32 %0, [%1];" : "=r"(v) : "r"(at));
                                v &= ((v & 0x7f80u) == 0x7f80u ? 0u : 0xffffu) | ((v >> 16 & 0x7f80u) == 0x7f80u ? 0u : 0xffff0000u);
                                asm volatile("st.shared.b32 [%0], %1;" ::"r"(at), "r"(v) : "memory");
                            }
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");      // for the tensor core
                    }
                    __syncwarp();
                    if (lane == 0) mbar_arrive(smem_u32(&sh.v_checked[which]));
                    ok = wait_all(&sh.v_checked[which], buffer, 51);
                    if (!ok) break;
#pragma unroll
                    for (int w = 0; w < 4; ++w) odd_value |= (seen[w] & *(volatile unsigned*)&sh.odd[which][buffer][w]) != 0u;
                    ++looked[paired];
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.p_full[stream]));
            }
            if (!ok) break;
            item0 += 2 * n_tiles;
            // ---- the rows' results.  Streams that share the rows meet: each takes half of the columns of both accumulators.
            float weight[2] = {0.0f, 0.0f}, m_all = m_used, l_all = odd_score ? NAN : l;
            weight[stream] = 1.0f;
            if (!paired) {
                sh.norm[stream * BM + r] = make_float2(m_used, l_all);
                sh.reads_odd[stream * BM + r] = odd_value;
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.norms_there));
                ok = wait_all(&sh.norms_there, shared_pieces & 1, 52);
                if (!ok) break;
                const float2 a = sh.norm[r], b = sh.norm[BM + r];
                m_all = fmaxf(a.x, b.x);
                weight[0] = a.x == -INFINITY ? 0.0f : fast_exp2(a.x - m_all);
                weight[1] = b.x == -INFINITY ? 0.0f : fast_exp2(b.x - m_all);
                l_all = a.y * weight[0] + b.y * weight[1];
                if (isnan(a.y) || isnan(b.y)) l_all = NAN;
                odd_value = sh.reads_odd[r] || sh.reads_odd[BM + r];
            }
            // whose accumulators this warp reads, and which there are
            const bool made[2] = {true, paired || n_tiles > 1}, has[2] = {!paired || stream == 0, paired ? stream == 1 : n_tiles > 1};
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                if (ok && has[i]) ok = wait_all(&sh.o_full[i], results[i] & 1, 53);
                results[i] += made[i] ? 1 : 0;
            }
            if (!ok) break;
            tc_fence_after();
            if (active) {
                const bool whole = walk.parts == 1;
                const float inv = !whole ? 1.0f : l_all > 0.0f ? 1.0f / l_all : isnan(l_all) ? NAN : 0.0f;
                const float w0 = weight[0] * inv, w1 = weight[1] * inv;
                const size_t row = (size_t)(s.token0 + node) * p.heads + head;
                const size_t part = ((size_t)blockIdx.x * 2 + (walk.part == 0 ? 1 : 0)) * 2 + (paired ? stream : 0);
                const int c_begin = paired ? 0 : stream * (D / 32), c_end = paired ? D / 16 : c_begin + D / 32;
#pragma unroll 1
                for (int c = c_begin; c < c_end; ++c) {
                    float o[16];
                    uint32_t x[2][16];
                    if (has[0]) tmem_ld16(tmem_rows + (uint32_t)(O_COL + c * 16), x[0]);
                    if (has[1]) tmem_ld16(tmem_rows + (uint32_t)(STREAM_COLS + O_COL + c * 16), x[1]);
                    tmem_wait_ld();
#pragma unroll
                    for (int i = 0; i < 16; ++i) {
                        o[i] = has[0] && w0 != 0.0f ? __uint_as_float(x[0][i]) * w0 : 0.0f;
                        if (has[1] && w1 != 0.0f) o[i] = fmaf(__uint_as_float(x[1][i]), w1, o[i]);
                    }
                    if (mine && !whole) {
                        // a column's rows lie together: a warp's store is one line (rows beside one another would be 32, and took 4 us of 50)
                        float* const to = p.part_out + (part * D + c * 16) * BM + r;
#pragma unroll
                        for (int i = 0; i < 16; ++i) to[i * BM] = o[i];
                    } else if (mine) {
                        uint4* const to = reinterpret_cast<uint4*>(p.out + row * D + c * 16);
#pragma unroll
                        for (int i = 0; i < 2; ++i)
                            to[i] = make_uint4(pack_bf16(o[8 * i], o[8 * i + 1]), pack_bf16(o[8 * i + 2], o[8 * i + 3]), pack_bf16(o[8 * i + 4], o[8 * i + 5]),
                                               pack_bf16(o[8 * i + 6], o[8 * i + 7]));
                    }
                    __syncwarp();
                }
                if (mine && !whole && (paired || stream == 0)) p.part_norm[part * BM + r] = make_float2(m_all, l_all);
                if (odd_value && l_all != 0.0f) {
                    // the values that were cleared, once more from the pages: whatever its weight, one that is not finite makes its column so
                    const int* const table = p.table + (size_t)walk.a * p.max_blocks;
#pragma unroll 1
                    for (int w = 0; w < 4 * n_tiles; ++w) {
                        const int from = (s.first + walk.tile) * BN + w * 32;
                        if (!is_edge(from / BN * BN)) continue;
#pragma unroll 1
                        for (unsigned left = seen_of(from); left; left &= left - 1) {
                            const int key = from + __ffs(left) - 1, page = table[key / p.page_size];
                            if (page < 0 || page >= p.num_pages) continue;
                            const __nv_bfloat16* const v = p.pages + ((((size_t)page * 2 + 1) * p.kv_heads + kvh) * p.page_size + key % p.page_size) * D;
#pragma unroll 1
                            for (int col = c_begin * 16; col < c_end * 16; ++col) {
                                const float x = __bfloat162float(v[col]);
                                if (fabsf(x) < INFINITY) continue;
                                if (whole) p.out[row * D + col] = __float2bfloat16(__bfloat162float(p.out[row * D + col]) + x);
                                else p.part_out[(part * D + col) * BM + r] += x;
                            }
                        }
                    }
                }
                __syncwarp();
            }
            tc_fence_before();                            // the accumulators were read before what the next piece's first P releases
            if (!paired) {
                // the other stream's accumulator too: nobody hands over a new P before everybody has read
                __syncwarp();
                if (lane == 0) mbar_arrive(smem_u32(&sh.o_read));
                ok = wait_all(&sh.o_read, shared_pieces & 1, 54);
                ++shared_pieces;
            }
        }
        if (!ok) sh.failed = 1;
    }

    tc_fence_before();
    __syncthreads();
    if (sh.failed) {
        // What is in flight gets a bounded chance to end before the CTA's memory goes away: copies write shared memory, products read it and write tensor
        // memory.  (A CTA that did not fail has waited for all of them.)
        if (warp == 0 && lane == 0) {
            if (sh.pieces > 0) mbar_drain(smem_u32(&sh.q_full), (sh.pieces - 1) & 1);
            for (int i = max(0, sh.issued - SLOTS); i < sh.issued; ++i) mbar_drain(smem_u32(&sh.slot_full[i % SLOTS]), (i / SLOTS) & 1);
        } else if (warp == 1) {
            if (elect_one()) umma_commit(smem_u32(&sh.stopped));
            __syncwarp();
            mbar_drain(smem_u32(&sh.stopped), 0);
        }
        __syncwarp();
    }
    if (warp == 1) {
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem_base), "r"((uint32_t)TMEM_COLS) : "memory");
    }
}

// The parts of the rows of items that lie in several CTAs, in a fixed order.  A CTA takes 32 rows of a row tile, a lane a row.  Its eight warps take
//     SPREAD:  the parts in turn, all for the same 16 columns, and meet in shared memory: a call of few rows has many parts, and waits for one chain
//              of loads, not for the bandwidth
//     else:    an eighth of the columns each, all parts: a call of many rows has few parts a row
constexpr int JOIN_THREADS = 256, JOIN_ROWS = 32, JOIN_WARPS = JOIN_THREADS / 32;
template <bool SPREAD>
__global__ void __launch_bounds__(JOIN_THREADS) draft_join_tc_kernel(TcParams p) {
    pdl_prologue();
    constexpr int COLS = SPREAD ? 16 : D / JOIN_WARPS, CHUNKS = SPREAD ? D / COLS : 1;
    __shared__ float acc_s[SPREAD ? JOIN_WARPS : 1][COLS][JOIN_ROWS];
    __shared__ float2 norm_s[SPREAD ? JOIN_WARPS : 1][JOIN_ROWS];
    const int seq = blockIdx.y, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int stretch = p.line[0], lead = p.line[1], base = p.line[2 + seq];
    const Sequence s = sequence_at(p, seq);
    int at = blockIdx.x;
    const int col0 = SPREAD ? at % CHUNKS * COLS : warp * COLS;
    at /= CHUNKS;
    const int block = at % (BM / JOIN_ROWS);
    at /= BM / JOIN_ROWS;
    const int tile = at % p.row_tiles, kvh = at / p.row_tiles;
    if (tile >= s.row_tiles) return;
    const int node0 = tile * p.tile_nodes, rows = min(p.tile_nodes, s.n - node0) * p.group - block * JOIN_ROWS;      // from this block's first on
    if (rows <= 0) return;
    const Item item = item_of(p, s, base, lead, kvh, tile >> 1);
    const int first = item.begin / stretch, parts = (item.end - 1) / stretch - first + 1;
    if (parts == 1) return;                               // written whole
    const bool mine = lane < rows;
    float top = -INFINITY, sum = 0.0f, acc[COLS] = {};
#pragma unroll 2
    for (int k = SPREAD ? warp : 0; k < parts; k += SPREAD ? JOIN_WARPS : 1) {
        // part k lies with CTA first + k: the first part is of the item that its stretch ends in, the others of the one that it begins in; a part
        // may be no tile's
        const bool there = mine && tile_of(item, min((first + k + 1) * stretch, item.end)) > tile_of(item, max((first + k) * stretch, item.begin));
        const size_t slot = ((size_t)(first + k) * 2 + (k == 0 ? 1 : 0)) * 2 + (tile & 1);
        const float2 norm = there ? p.part_norm[slot * BM + block * JOIN_ROWS + lane] : make_float2(-INFINITY, 0.0f);
        const float* const o = p.part_out + (slot * D + col0) * BM + block * JOIN_ROWS + lane;
        float v[COLS];
#pragma unroll
        for (int i = 0; i < COLS; ++i) v[i] = there ? o[i * BM] : 0.0f;
        const float m = fmaxf(top, norm.x);
        const float keep = top == -INFINITY ? 0.0f : exp2f(top - m), w = norm.x == -INFINITY ? 0.0f : exp2f(norm.x - m);
        sum = sum * keep + (norm.x == -INFINITY && !isnan(norm.y) ? 0.0f : norm.y * w);
#pragma unroll
        for (int i = 0; i < COLS; ++i) acc[i] = w == 0.0f ? acc[i] * keep : fmaf(w, v[i], acc[i] * keep);
        top = m;
    }
    auto row_of = [&](int r) {
        const int in_tile = block * JOIN_ROWS + r;
        return (size_t)(s.token0 + node0 + in_tile / p.group) * p.heads + kvh * p.group + in_tile % p.group;
    };
    auto inverse = [](float sum) { return sum > 0.0f ? 1.0f / sum : isnan(sum) ? NAN : 0.0f; };
    if constexpr (!SPREAD) {
        if (!mine) return;
        const float inv = inverse(sum);
        uint4* const to = reinterpret_cast<uint4*>(p.out + row_of(lane) * D + col0);
#pragma unroll
        for (int i = 0; i < COLS / 8; ++i)
            to[i] = make_uint4(pack_bf16(acc[8 * i] * inv, acc[8 * i + 1] * inv), pack_bf16(acc[8 * i + 2] * inv, acc[8 * i + 3] * inv),
                               pack_bf16(acc[8 * i + 4] * inv, acc[8 * i + 5] * inv), pack_bf16(acc[8 * i + 6] * inv, acc[8 * i + 7] * inv));
    } else {
        norm_s[warp][lane] = make_float2(top, sum);
#pragma unroll
        for (int i = 0; i < COLS; ++i) acc_s[warp][i][lane] = acc[i];
        __syncthreads();
        // a thread two columns of a row
        const int r = threadIdx.x / (COLS / 2), c = threadIdx.x % (COLS / 2) * 2;
        if (r >= rows) return;
        top = -INFINITY;
#pragma unroll
        for (int w = 0; w < JOIN_WARPS; ++w) top = fmaxf(top, norm_s[w][r].x);
        float a = 0.0f, b = 0.0f;
        sum = 0.0f;
#pragma unroll
        for (int w = 0; w < JOIN_WARPS; ++w) {
            const float2 norm = norm_s[w][r];
            const float f = norm.x == -INFINITY ? 0.0f : exp2f(norm.x - top);
            sum += isnan(norm.y) ? NAN : norm.y * f;
            a = f == 0.0f ? a : fmaf(f, acc_s[w][c][r], a);
            b = f == 0.0f ? b : fmaf(f, acc_s[w][c + 1][r], b);
        }
        const float inv = inverse(sum);
        *reinterpret_cast<uint32_t*>(p.out + row_of(r) * D + col0 + c) = pack_bf16(a * inv, b * inv);
    }
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

// q and out [T, NH * D] bf16, pages [num_pages, 2, NKV, page_size, D].  `ctas` CTAs take `stretch` units or more each; scratch, with more than one:
// [ctas, 2, 2, D, 128] fp32, [ctas, 2, 2, 128] float2, [2 + sequences] int.
MLB_EXPORT int mlb_draft_attention_tc(const void* q, const void* pages, void* out, const int* starts, const int* lengths, const int* positions, const int* masks,
                                      int words, const int* table, int max_blocks, int num_pages, int page_size, int tokens, int sequences, int max_nodes,
                                      int heads, int kv_heads, float scale, int window, int stretch, int ctas, void* scratch, int* error_flag,
                                      cudaStream_t stream) {
    if (heads <= 0 || kv_heads <= 0 || heads % kv_heads != 0 || heads / kv_heads > BM)
        return fail(MLB_UNSUPPORTED_SIZE, "draft_attention_tc: heads %d/%d", heads, kv_heads);
    if (words <= 0 || words > MAX_WORDS || max_nodes <= 0 || max_nodes > words * 32)
        return fail(MLB_UNSUPPORTED_SIZE, "draft_attention_tc: %d nodes in masks of %d words (at most %d)", max_nodes, words, MAX_WORDS);
    if (page_size < 8 || page_size % 8 != 0 || BN % page_size != 0 || BN / page_size > MAX_PAGES_PER_TILE)
        return fail(MLB_UNSUPPORTED_SIZE, "draft_attention_tc: page_size %d must be a multiple of 8 that divides %d", page_size, BN);
    if (!(scale > 0.0f)) return fail(MLB_UNSUPPORTED_SIZE, "draft_attention_tc: the softmax scale must be positive");
    if (num_pages <= 0 || max_blocks <= 0 || tokens < 0 || sequences < 0 || window < 0) return fail(MLB_INVALID_ARGUMENT, "draft_attention_tc: bad sizes");
    if (stretch <= 0 || ctas <= 0 || (ctas > 1 && !scratch)) return fail(MLB_INVALID_ARGUMENT, "draft_attention_tc: bad cut");
    if (((uintptr_t)q & 15) || ((uintptr_t)out & 15) || ((uintptr_t)pages & 15) || ((uintptr_t)scratch & 15))
        return fail(MLB_UNSUPPORTED_SIZE, "draft_attention_tc: q, out, the pages and the scratch must be 16-byte aligned");
    const long long kv_rows = (long long)num_pages * 2 * kv_heads * page_size;
    if (kv_rows >= (1ll << 31)) return fail(MLB_UNSUPPORTED_SIZE, "draft_attention_tc: the cache has too many rows (%lld)", kv_rows);
    const int group = heads / kv_heads, tile_nodes = BM / group;
    // every count of units fits 31 bits: a sequence's tiles are at most the table's
    const long long most_tiles = ((long long)max_blocks * page_size + BN - 1) / BN + 1;
    if (most_tiles * ((max_nodes + tile_nodes - 1) / tile_nodes) * (1 + MOST_LEAD) * kv_heads * (sequences > 0 ? sequences : 1) >= (1ll << 30) || sequences > 65535)
        return fail(MLB_UNSUPPORTED_SIZE, "draft_attention_tc: too much work for a call");
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
    TcParams p{(__nv_bfloat16*)out, (const __nv_bfloat16*)pages, starts, lengths, positions, masks, table, words, max_blocks, num_pages, page_size, BN / page_size, heads, kv_heads, group,
               tile_nodes, (max_nodes + tile_nodes - 1) / tile_nodes, window, max_nodes, stretch, ctas, sequences, tokens,
               (int)std::min((long long)max_blocks * page_size, 1ll << 30), scale * LOG2E, nullptr, nullptr, nullptr, error_flag};
    if (ctas > 1) {
        p.part_out = (float*)scratch;
        p.part_norm = (float2*)(p.part_out + (size_t)ctas * 4 * BM * D);
        p.line = (int*)(p.part_norm + (size_t)ctas * 4 * BM);
    }
    static bool configured_on[MAX_DEVICES] = {false};         // the attribute belongs to the device
    bool& configured = configured_on[device_index()];
    if (!configured) {
        if (cudaFuncSetAttribute(draft_attention_tc_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)SMEM_BYTES) != cudaSuccess)
            return check_launch("draft_attention_tc: shared memory");
        configured = true;
    }
    launch_kernel(draft_attention_tc_kernel, ctas, THREADS, SMEM_BYTES, stream, map_q, map_kv, p);
    const int status = check_launch("draft_attention_tc");
    if (status != MLB_OK || ctas == 1) return status;
    const int blocks = kv_heads * p.row_tiles * (BM / JOIN_ROWS);
    if ((long long)blocks * sequences <= sm_count()) launch_kernel(draft_join_tc_kernel<true>, dim3(blocks * (D / 16), sequences), JOIN_THREADS, 0, stream, p);
    else launch_kernel(draft_join_tc_kernel<false>, dim3(blocks, sequences), JOIN_THREADS, 0, stream, p);
    return check_launch("draft_join_tc");
}

MLB_PACKED(mlb_draft_attention_tc)
