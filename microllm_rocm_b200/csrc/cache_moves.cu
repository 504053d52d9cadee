// Moving what a request holds in the cache: beams that continue from their parents' cache, and the branch of a drafted tree
// that was accepted.  Every kernel moves the same columns (pieces of VEC bytes of a token's row, or of a slot's state) of
// many storages (one a layer) in one launch.
//
// In place, without a second copy and without order between threads: a thread owns a column, reads it from every row that
// it takes part in before it writes any, and no other thread touches that column.  So a permutation with repetitions (beams)
// needs neither a scratch copy nor a synchronisation, and what bounds the kernels is memory: each moved destination is written
// once, each source read once from memory (children of one parent read it from the L1 of the same thread).  Measured: slots of 1 MB in 12 layers, 8 requests of 4 beams,
// 402 MB read and written in 62 us (6.5 TB/s, a copy's rate); 40 to 100 tokens of 4 beams in 28 layers (11 MB) 3.9 us.  An accepted branch is a few rows a layer: 16 trees
// of up to 64 nodes in 28 layers 5.5 us, of which the walk down the tree is a warp's and the rest the launch.
#include "common.cuh"
#include "packed.cuh"

using namespace mlb;

MLB_DEFINE_LAST_ERROR()

namespace {

constexpr int THREADS = 256;
constexpr int MAX_STORAGES = 128;
constexpr int MAX_BEAMS = 32;
constexpr int MAX_NODES = 256;

struct Storages {
    char* base[MAX_STORAGES];
};

// One page: `planes` planes of page_size rows of `row` bytes, then `planes2` planes of rows of `row2` bytes (0: none).
struct PageLayout {
    long long num_pages;
    int page_size, planes, row, planes2, row2;
    __host__ __device__ __forceinline__ long long bytes() const { return ((long long)planes * row + (long long)planes2 * row2) * page_size; }
    // the columns of VEC bytes of one token
    __host__ __device__ __forceinline__ int columns(int vec) const { return planes * (row / vec) + planes2 * (row2 / vec); }
};

template <int VEC> struct Piece;
template <> struct Piece<16> { using T = uint4; };
template <> struct Piece<4> { using T = unsigned; };
template <> struct Piece<2> { using T = unsigned short; };

// ------------------------------------------------------------------------------ slots of fixed size
struct SlotParams {
    const int* slots;        // [requests, beams]
    const int* parents;      // [requests, beams]
    int* error_flag;
    long long num_slots, row;      // row: bytes of a slot
    int beams;
};

template <int VEC, int B>
__global__ void __launch_bounds__(THREADS) reorder_slots_kernel(const __grid_constant__ Storages s, SlotParams p) {
    using T = typename Piece<VEC>::T;
    pdl_prologue();
    __shared__ int s_slot[B], s_from[B];          // the slot of each beam, and the slot it continues from (-1: stays as it is)
    const int request = blockIdx.z, tid = threadIdx.x;
    if (tid < B) {
        int slot = -1, from = -1;
        if (tid < p.beams) {
            slot = p.slots[(size_t)request * p.beams + tid];
            const int parent = p.parents[(size_t)request * p.beams + tid];
            if (parent >= 0 && parent < p.beams && parent != tid) from = p.slots[(size_t)request * p.beams + parent];
            const bool bad = slot < 0 || slot >= p.num_slots || parent >= p.beams || (parent >= 0 && parent != tid && (from < 0 || from >= p.num_slots));
            if (bad) {
                if (p.error_flag) atomicExch(p.error_flag, 4);
                from = -1;
            }
        }
        s_slot[tid] = slot;
        s_from[tid] = from;
    }
    __syncthreads();
    char* const base = s.base[blockIdx.y];
    const long long columns = p.row / VEC;
    for (long long c = (long long)blockIdx.x * THREADS + tid; c < columns; c += (long long)gridDim.x * THREADS) {
        T v[B];
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (s_from[b] >= 0) v[b] = *reinterpret_cast<const T*>(base + s_from[b] * p.row + c * VEC);
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (s_from[b] >= 0) *reinterpret_cast<T*>(base + s_slot[b] * p.row + c * VEC) = v[b];
    }
}

// ------------------------------------------------------------------------------ tokens in pages, between beams
struct PageParams {
    PageLayout at;
    const int* table;        // [requests * beams, max_blocks]
    const int* parents;      // [requests, beams]
    const int* first;        // [requests]
    const int* last;         // [requests]
    int* error_flag;
    int max_blocks, beams;
};

// Where column `c` of a token's VEC-byte columns begins in a page, for the page's token 0; and how far two tokens are apart.
__device__ __forceinline__ long long column_offset(const PageLayout& at, int c, int vec, int& row) {
    const int per = at.row / vec, firsts = at.planes * per;
    if (c < firsts) {
        row = at.row;
        return (long long)(c / per) * at.page_size * at.row + (c % per) * vec;
    }
    const int per2 = at.row2 / vec;
    c -= firsts;
    row = at.row2;
    return (long long)at.planes * at.page_size * at.row + (long long)(c / per2) * at.page_size * at.row2 + (c % per2) * vec;
}

template <int VEC, int B>
__global__ void __launch_bounds__(THREADS) reorder_pages_kernel(const __grid_constant__ Storages s, PageParams p) {
    using T = typename Piece<VEC>::T;
    pdl_prologue();
    __shared__ int s_parent[B];
    const int request = blockIdx.z, tid = threadIdx.x;
    if (tid < B) {
        int parent = tid < p.beams ? p.parents[(size_t)request * p.beams + tid] : -1;
        if (parent >= p.beams) {
            if (p.error_flag) atomicExch(p.error_flag, 4);
            parent = -1;
        }
        s_parent[tid] = parent == tid ? -1 : parent;
    }
    __syncthreads();
    const int first = max(0, p.first[request]);
    long long last = p.last[request];
    if (last > (long long)p.max_blocks * p.at.page_size) {                   // a block beyond the table
        if (tid == 0 && p.error_flag) atomicExch(p.error_flag, 2);
        last = (long long)p.max_blocks * p.at.page_size;
    }
    const int tokens = (int)max(last - first, 0ll);
    char* const base = s.base[blockIdx.y];
    const int* const table = p.table + (size_t)request * p.beams * p.max_blocks;
    const long long page_bytes = p.at.bytes();
    // Neighbouring threads take neighbouring pieces of a row, then neighbouring tokens, then the next plane: within a page that is the order
    // of memory.
    const int per = p.at.row / VEC, per2 = p.at.row2 / VEC;
    const long long firsts = (long long)p.at.planes * per * tokens, items = firsts + (long long)p.at.planes2 * per2 * tokens;
    for (long long i = (long long)blockIdx.x * THREADS + tid; i < items; i += (long long)gridDim.x * THREADS) {
        const bool second = i >= firsts;
        const int each = second ? per2 : per, row = second ? p.at.row2 : p.at.row;
        const long long rest = second ? i - firsts : i;
        const int piece = (int)(rest % each), t = (int)((rest / each) % tokens), plane = (int)(rest / each / tokens);
        const int place = first + t, block = place / p.at.page_size;
        const long long inside = (second ? (long long)p.at.planes * p.at.page_size * p.at.row : 0) +
                                 ((long long)plane * p.at.page_size + place % p.at.page_size) * row + piece * VEC;
        T v[B];
        int to[B];
#pragma unroll
        for (int b = 0; b < B; ++b) {
            to[b] = -1;
            if (s_parent[b] < 0) continue;
            const int from = table[(size_t)s_parent[b] * p.max_blocks + block];
            to[b] = table[(size_t)b * p.max_blocks + block];
            if (from < 0) to[b] = -1;              // a block that a window gave back: nobody reads it any more
            else if (from >= p.at.num_pages || to[b] >= p.at.num_pages || to[b] < 0) {
                if (p.error_flag) atomicExch(p.error_flag, 2);
                to[b] = -1;
            }
            if (to[b] >= 0) v[b] = *reinterpret_cast<const T*>(base + from * page_bytes + inside);
        }
#pragma unroll
        for (int b = 0; b < B; ++b)
            if (to[b] >= 0) *reinterpret_cast<T*>(base + to[b] * page_bytes + inside) = v[b];
    }
}

// ------------------------------------------------------------------------------ the accepted branch of a drafted tree
// From the tree's first node down: the next node is the lowest child whose token is the model's choice at its parent.  The
// nodes on the way stay; node path[i]'s row of every storage moves from place length + path[i] to place length + i.  path rises
// strictly, so path[i] >= i: walking i upward a thread never overwrites a row that it still has to read.
struct AcceptParams {
    PageLayout at;
    const int* tokens;       // [T]
    const int* parents;      // [T] within the sequence, -1: none
    const int* choices;      // [T] the model's choice behind each node
    const int* starts;       // [A + 1]
    const int* lengths;      // [A]
    const int* table;        // [A, max_blocks]
    int* path;               // [A, width]
    int* counts;             // [A]
    int* following;          // [A]
    int* error_flag;
    int nodes, width, max_blocks, storages, write;       // nodes: T
};

template <int VEC>
__global__ void __launch_bounds__(THREADS) accept_kernel(const __grid_constant__ Storages s, AcceptParams p) {
    using T = typename Piece<VEC>::T;
    pdl_prologue();
    __shared__ int s_token[MAX_NODES], s_parent[MAX_NODES], s_choice[MAX_NODES], s_path[MAX_NODES];
    __shared__ int s_from[MAX_NODES], s_to[MAX_NODES];       // page * page_size + place in it; -1: nothing to move
    __shared__ int s_count;
    const int a = blockIdx.y, tid = threadIdx.x;
    const int start = p.starts[a];
    int n = p.starts[a + 1] - start;
    if (n < 0 || n > MAX_NODES || n > p.width || start < 0 || start + n > p.nodes) {
        if (tid == 0 && p.error_flag) atomicExch(p.error_flag, 3);
        n = 0;
    }
    for (int i = tid; i < n; i += THREADS) {
        s_token[i] = p.tokens[start + i];
        s_parent[i] = p.parents[start + i];
        s_choice[i] = p.choices[start + i];
    }
    __syncthreads();
    if (tid < 32) {
        int count = 0;
        if (n > 0) {
            int node = 0;
            while (true) {
                if (tid == 0) s_path[count] = node;
                ++count;
                const int want = s_choice[node];
                int next = -1;
                for (int from = (node + 1) & ~31; from < n && next < 0; from += 32) {
                    const int i = from + tid;
                    const unsigned hit = __ballot_sync(0xffffffffu, i > node && i < n && s_parent[i] == node && s_token[i] == want);
                    if (hit) next = from + __ffs(hit) - 1;
                }
                if (next < 0) break;
                node = next;               // rises: at most n nodes
            }
        }
        if (tid == 0) s_count = count;
    }
    __syncthreads();
    const int count = s_count;
    if (p.write && blockIdx.x == 0) {
        for (int i = tid; i < p.width; i += THREADS) p.path[(size_t)a * p.width + i] = i < count ? s_path[i] : -1;
        if (tid == 0) {
            p.counts[a] = count;
            p.following[a] = count ? s_choice[s_path[count - 1]] : -1;
        }
    }
    if (!p.storages) return;
    const int length = p.lengths[a];
    bool any = false;
    for (int i = tid; i < count; i += THREADS) {
        int from = -1, to = -1;
        if (s_path[i] != i) {
            const int* const table = p.table + (size_t)a * p.max_blocks;
            const int of = length + s_path[i], onto = length + i;
            const int fb = of / p.at.page_size, tb = onto / p.at.page_size;
            const int fp = length >= 0 && fb < p.max_blocks ? table[fb] : -1, tp = length >= 0 && tb < p.max_blocks ? table[tb] : -1;
            if (fp < 0 || fp >= p.at.num_pages || tp < 0 || tp >= p.at.num_pages) {
                if (p.error_flag) atomicExch(p.error_flag, 2);
            } else {
                from = fp * p.at.page_size + of % p.at.page_size;
                to = tp * p.at.page_size + onto % p.at.page_size;
                any = true;
            }
        }
        s_from[i] = from;
        s_to[i] = to;
    }
    if (!__syncthreads_or(any)) return;
    const int each = p.at.columns(VEC);
    const long long page_bytes = p.at.bytes(), columns = (long long)each * p.storages;
    for (long long c = (long long)blockIdx.x * THREADS + tid; c < columns; c += (long long)gridDim.x * THREADS) {
        int row;
        char* const base = s.base[c / each] + column_offset(p.at, (int)(c % each), VEC, row);
        constexpr int AHEAD = 8;
        for (int i0 = 1; i0 < count; i0 += AHEAD) {
            T v[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int from = i0 + i < count ? s_from[i0 + i] : -1;
                if (from >= 0) v[i] = *reinterpret_cast<const T*>(base + (from / p.at.page_size) * page_bytes + (long long)(from % p.at.page_size) * row);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                const int to = i0 + i < count ? s_to[i0 + i] : -1;
                if (to >= 0) *reinterpret_cast<T*>(base + (to / p.at.page_size) * page_bytes + (long long)(to % p.at.page_size) * row) = v[i];
            }
        }
    }
}

// ------------------------------------------------------------------------------ host side
int take_storages(Storages& s, const void* const* bases, int count, const char* what) {
    if (count < 0 || count > MAX_STORAGES || (count && !bases)) return fail(MLB_INVALID_ARGUMENT, "%s: %d storages (at most %d a call)", what, count, MAX_STORAGES);
    for (int i = 0; i < count; ++i) s.base[i] = (char*)bases[i];
    return MLB_OK;
}

// the widest pieces that every row starts at a multiple of
int piece_bytes(const Storages& s, int count, long long a, long long b) {
    unsigned long long bits = (unsigned long long)a | (unsigned long long)b;
    for (int i = 0; i < count; ++i) bits |= (unsigned long long)(uintptr_t)s.base[i];
    return bits % 16 == 0 ? 16 : bits % 4 == 0 ? 4 : bits % 2 == 0 ? 2 : 0;
}

int check_layout(const PageLayout& at, const char* what) {
    if (at.num_pages <= 0 || at.page_size <= 0 || at.planes <= 0 || at.row <= 0 || at.planes2 < 0 || at.row2 < 0 || (at.planes2 > 0) != (at.row2 > 0))
        return fail(MLB_INVALID_ARGUMENT, "%s: bad page geometry", what);
    if (at.num_pages * at.page_size >= (1ll << 31)) return fail(MLB_UNSUPPORTED_SIZE, "%s: more than 2^31 tokens in the pool", what);
    return MLB_OK;
}

unsigned blocks_of(long long items, long long others) {
    // a few waves of CTAs and no more: the rest goes round again
    const long long most = (long long)sm_count() * 32 / (others > 0 ? others : 1) + 1, want = (items + THREADS - 1) / THREADS;
    return (unsigned)(want < 1 ? 1 : want < most ? want : most);
}

template <int VEC, int B>
void launch_slots(const Storages& s, const SlotParams& p, int count, int requests, cudaStream_t stream) {
    launch_kernel(reorder_slots_kernel<VEC, B>, dim3(blocks_of(p.row / VEC, (long long)count * requests), count, requests), THREADS, 0, stream, s, p);
}
template <int VEC>
void launch_slots(const Storages& s, const SlotParams& p, int count, int requests, cudaStream_t stream) {
    if (p.beams <= 4) launch_slots<VEC, 4>(s, p, count, requests, stream);
    else if (p.beams <= 8) launch_slots<VEC, 8>(s, p, count, requests, stream);
    else if (p.beams <= 16) launch_slots<VEC, 16>(s, p, count, requests, stream);
    else launch_slots<VEC, 32>(s, p, count, requests, stream);
}

template <int VEC, int B>
void launch_pages(const Storages& s, const PageParams& p, int count, int requests, int max_tokens, cudaStream_t stream) {
    const long long items = (long long)p.at.columns(VEC) * max_tokens;
    launch_kernel(reorder_pages_kernel<VEC, B>, dim3(blocks_of(items, (long long)count * requests), count, requests), THREADS, 0, stream, s, p);
}
template <int VEC>
void launch_pages(const Storages& s, const PageParams& p, int count, int requests, int max_tokens, cudaStream_t stream) {
    if (p.beams <= 4) launch_pages<VEC, 4>(s, p, count, requests, max_tokens, stream);
    else if (p.beams <= 8) launch_pages<VEC, 8>(s, p, count, requests, max_tokens, stream);
    else if (p.beams <= 16) launch_pages<VEC, 16>(s, p, count, requests, max_tokens, stream);
    else launch_pages<VEC, 32>(s, p, count, requests, max_tokens, stream);
}

int check_beams(int requests, int beams, const char* what) {
    if (requests < 0 || requests > 65535 || beams <= 0 || beams > MAX_BEAMS)
        return fail(MLB_UNSUPPORTED_SIZE, "%s: %d requests of %d beams (at most 65535 of %d)", what, requests, beams, MAX_BEAMS);
    return MLB_OK;
}

}  // namespace

// bases: `count` host pointers to [num_slots, row bytes] arrays; every beam's slot takes its parent's.
MLB_EXPORT int mlb_reorder_slots(const void* const* bases, int count, long long num_slots, long long row_bytes, const int* slots,
                                 const int* parents, int requests, int beams, int* error_flag, cudaStream_t stream) {
    Storages s;
    int status = take_storages(s, bases, count, "reorder_slots");
    if (status == MLB_OK) status = check_beams(requests, beams, "reorder_slots");
    if (status != MLB_OK) return status;
    if (num_slots <= 0 || row_bytes <= 0) return fail(MLB_INVALID_ARGUMENT, "reorder_slots: bad sizes");
    if (count == 0 || requests == 0) return MLB_OK;
    SlotParams p{slots, parents, error_flag, num_slots, row_bytes, beams};
    const int vec = piece_bytes(s, count, row_bytes, 0);
    if (vec == 16) launch_slots<16>(s, p, count, requests, stream);
    else if (vec == 4) launch_slots<4>(s, p, count, requests, stream);
    else if (vec == 2) launch_slots<2>(s, p, count, requests, stream);
    else return fail(MLB_UNSUPPORTED_SIZE, "reorder_slots: rows of an odd number of bytes");
    return check_launch("reorder_slots");
}

// bases: `count` host pointers to pools of num_pages pages of the layout (planes, row, planes2, row2); tokens [first, last) of
// every beam's pages take its parent's.
MLB_EXPORT int mlb_reorder_pages(const void* const* bases, int count, long long num_pages, int page_size, int planes, int row, int planes2, int row2,
                                 const int* table, int max_blocks, const int* parents, int requests, int beams, const int* first, const int* last,
                                 int max_tokens, int* error_flag, cudaStream_t stream) {
    Storages s;
    int status = take_storages(s, bases, count, "reorder_pages");
    if (status == MLB_OK) status = check_beams(requests, beams, "reorder_pages");
    PageParams p{PageLayout{num_pages, page_size, planes, row, planes2, row2}, table, parents, first, last, error_flag, max_blocks, beams};
    if (status == MLB_OK) status = check_layout(p.at, "reorder_pages");
    if (status != MLB_OK) return status;
    if (max_blocks <= 0 || max_tokens < 0) return fail(MLB_INVALID_ARGUMENT, "reorder_pages: bad sizes");
    if (count == 0 || requests == 0 || max_tokens == 0) return MLB_OK;
    const int vec = piece_bytes(s, count, row, row2);
    if (vec == 16) launch_pages<16>(s, p, count, requests, max_tokens, stream);
    else if (vec == 4) launch_pages<4>(s, p, count, requests, max_tokens, stream);
    else if (vec == 2) launch_pages<2>(s, p, count, requests, max_tokens, stream);
    else return fail(MLB_UNSUPPORTED_SIZE, "reorder_pages: rows of an odd number of bytes");
    return check_launch("reorder_pages");
}

MLB_EXPORT int mlb_accept_drafts(const void* const* bases, int count, long long num_pages, int page_size, int planes, int row, int planes2, int row2,
                                 const int* tokens, const int* parents, const int* choices, const int* starts, const int* lengths, int nodes, int sequences,
                                 const int* table, int max_blocks, int* path, int width, int* counts, int* following, int write, int* error_flag,
                                 cudaStream_t stream) {
    Storages s;
    int status = take_storages(s, bases, count, "accept_drafts");
    if (status != MLB_OK) return status;
    AcceptParams p{PageLayout{num_pages, page_size, planes, row, planes2, row2}, tokens, parents, choices, starts, lengths, table, path, counts,
                   following, error_flag, nodes, width, max_blocks, count, write};
    if (count && (status = check_layout(p.at, "accept_drafts")) != MLB_OK) return status;
    if (sequences < 0 || sequences > 65535 || width <= 0 || (count && max_blocks <= 0)) return fail(MLB_INVALID_ARGUMENT, "accept_drafts: bad sizes");
    if (sequences == 0) return MLB_OK;
    const int vec = count ? piece_bytes(s, count, row, row2) : 16;
    if (vec == 0) return fail(MLB_UNSUPPORTED_SIZE, "accept_drafts: rows of an odd number of bytes");
    const dim3 grid(count ? blocks_of((long long)p.at.columns(vec) * count, sequences) : 1, sequences);
    if (vec == 16) launch_kernel(accept_kernel<16>, grid, THREADS, 0, stream, s, p);
    else if (vec == 4) launch_kernel(accept_kernel<4>, grid, THREADS, 0, stream, s, p);
    else launch_kernel(accept_kernel<2>, grid, THREADS, 0, stream, s, p);
    return check_launch("accept_drafts");
}

MLB_PACKED(mlb_reorder_slots)
MLB_PACKED(mlb_reorder_pages)
MLB_PACKED(mlb_accept_drafts)
