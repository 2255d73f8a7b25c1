// kv_pages.cu - the blocks of the cache handed out, shared, moved and taken back on the device, for all layers that share a table.
//
//   refs[b]  how many entries of the table hold block b; 0: it is free.  Whoever needs blocks gets the free ones of the lowest numbers, in the order of
//            asking, so that a call's outcome does not depend on how its threads run.
//   reserve  entries for the new tokens of a batch; a block that others hold too and that new tokens would be written to is replaced by a copy
//   fork     sequences go on from others (a beam search's step): full blocks are shared, the one in the middle of which the child stands is copied
//   free     sequences give up their blocks
//   compact  the live blocks take the lowest numbers: the i-th live block behind the border moves into the i-th hole in front of it, or only the first so many
//   copy     blocks to blocks
//
// Two launches a call (free and copy: one).  What is counted and ranked - a few thousand numbers - is one thread block's work, since every rank depends on all in
// front of it; its time is the latency of four to six look-ups, one behind the other.  What moves is copied by as many thread blocks as fit, who find the list
// and its length in the scratch.  Sources and destinations are disjoint: blocks are handed out that were free when the call began, and a compaction moves across its
// border.  Reference counts change by atomic additions of whole numbers alone, in any order the same.
#include "maya_kv.cuh"
#include "maya_scan.cuh"

namespace maya {
namespace {

constexpr int kRefsEach = 16;                  // blocks a thread looks at in a round
constexpr int kPieceBytes = 16384;             // of keys or values that a thread block copies at a time
constexpr int kCopyThreads = 256;

struct Pages {
    const maya_kv_layer* layers;
    int* table;
    int* refs;
    int n_seq, table_ld, n_blocks, n_layers, n_kv, head_dim, sums;
    int* words;                                // [0] error, [1] blocks to move, [2] live blocks (compact)
    int* src;                                  // [n_blocks] the list of moves
    int* dst;
    int* list;                                 // [n_blocks] free blocks; compact: where a block went
    int* owner;                                // [n_seq] fork: the pair that a child belongs to; reserve: items in front of a sequence
    int* fresh;                                // [n_seq] fork: a pair's new block; -1: none, -2: nothing to do
    int* rows;                                 // [n_seq][table_ld] fork: the children's rows; reserve: ranks
};
constexpr int kPageWords = 64;

size_t pages_carve(const maya_kv_pages* p, Pages* v) {
    size_t at = kPageWords;
    auto take = [&](size_t n) { const size_t a = at; at += (n + 63) & ~(size_t) 63; return a; };
    const size_t nb = (size_t) p->n_blocks, ns = (size_t) p->n_seq, moves = nb > ns ? nb : ns;
    const size_t o[6] = {take(moves), take(moves), take(nb), take(ns + 1), take(ns), take(ns * p->table_ld)};
    if (v) {
        int* w = (int*) p->scratch;
        *v = Pages{p->layers, p->table, p->refs, p->n_seq, p->table_ld, p->n_blocks, p->n_layers, p->n_kv, p->head_dim, p->has_sums,
                   w, w + o[0], w + o[1], w + o[2], w + o[3], w + o[4], w + o[5]};
    }
    return at * sizeof(int);
}

int pages_check(const maya_kv_pages* p) {
    if (!p || !p->layers || !p->table || !p->refs || p->n_seq <= 0 || p->table_ld <= 0 || p->n_blocks <= 0 || p->n_layers <= 0 || p->n_kv <= 0) return MAYA_ERR_ARG;
    if (p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 192 && p->head_dim != 256) return MAYA_ERR_LIMIT;
    if (p->n_blocks > MAYA_MAX_PAGES || p->n_seq > 65535 || (int64_t) p->n_seq * p->table_ld > (1 << 28) || p->n_layers > 1024 || p->n_kv > 65535) return MAYA_ERR_LIMIT;
    if ((int64_t) p->table_ld * kKvBlock > 0x7FFFFFFF) return MAYA_ERR_LIMIT;        // (tokens of a row are counted in an int)
    return MAYA_OK;
}
int pages_ready(const maya_kv_pages* p, Pages* v) {
    const int st = pages_check(p);
    if (st != MAYA_OK) return st;
    if (!p->scratch || (((uintptr_t) p->scratch) & 255u) || !aligned16(p->refs) || !aligned16(p->layers)) return MAYA_ERR_ARG;
    if (p->scratch_bytes < pages_carve(p, v)) return MAYA_ERR_LIMIT;
    return MAYA_OK;
}

// ---------------------------------------------------------------- counting and ranking, by one thread block
// Bit i: block b0 + i is held by the table (blocks from n on: `beyond`).
__device__ __forceinline__ unsigned live_bits(const Pages& P, int b0, bool beyond) {
    unsigned m = 0u;
    if (b0 + kRefsEach <= P.n_blocks) {
        int4 r[kRefsEach / 4];
#pragma unroll
        for (int i = 0; i < kRefsEach / 4; ++i) r[i] = __ldcg((const int4*) (P.refs + b0) + i);
#pragma unroll
        for (int i = 0; i < kRefsEach / 4; ++i)
            m |= (unsigned) ((r[i].x > 0) | (r[i].y > 0) << 1 | (r[i].z > 0) << 2 | (r[i].w > 0) << 3) << (4 * i);
    } else {
        for (int i = 0; i < kRefsEach; ++i) m |= (unsigned) (b0 + i < P.n_blocks ? __ldcg(P.refs + b0 + i) > 0 : beyond) << i;
    }
    return m;
}
// list[0 .. need) = the free blocks of the lowest numbers; returns how many there are.  bits: live_bits of the first round, asked for while something else was
// waited for.  Ends with the block synchronised.
__device__ __forceinline__ int take_free(const Pages& P, int need, unsigned bits, PlanShared& sh) {
    int found = 0;
    for (int c0 = 0; c0 < P.n_blocks && found < need; c0 += kPlan * kRefsEach) {
        const int b0 = c0 + threadIdx.x * kRefsEach;
        if (c0 > 0) bits = live_bits(P, b0, true);
        unsigned open = ~bits & 0xffffu;
        int total, r = found + rank_of(__popc(open), sh, total);
        while (open != 0u && r < need) {
            P.list[r++] = b0 + __ffs(open) - 1;
            open &= open - 1u;
        }
        found += total;
    }
    __syncthreads();
    return min(found, need);
}
// Numbers of sequences in shared memory where they fit (a look-up there takes a tenth of one in the scratch).
constexpr int kSeqShared = 4096;
__device__ __forceinline__ bool is_block(const Pages& P, int b) { return b >= 0 && b < P.n_blocks; }

// ---------------------------------------------------------------- reserve
// Items: the (sequence, block) that new tokens fall into, in that order.
__global__ void __launch_bounds__(kPlan) pages_reserve_kernel(const Pages P, const BatchView B) {
    __shared__ PlanShared sh;
    __shared__ int s_moves, s_first[kSeqShared];
    const int tid = threadIdx.x;
    grid_launch_dependents();
    grid_dependency_wait();
    int* first = B.n_seq <= kSeqShared ? s_first : P.owner;   // items in front of every sequence
    const unsigned bits = live_bits(P, tid * kRefsEach, true);
    if (tid == 0) s_moves = 0;
    int items = 0;
    for (int s0 = 0; s0 < B.n_seq; s0 += kPlan) {
        const int s = s0 + tid;
        int n = 0;
        if (s < B.n_seq) {
            const Seq q = seq_of(B, s);
            if (q.n_new > 0 && q.len > 0) n = min((q.len - 1) / kKvBlock, P.table_ld - 1) - max(0, q.len - q.n_new) / kKvBlock + 1;
        }
        int total;
        const int r = rank_of(n, sh, total);
        if (s < B.n_seq) first[s] = items + r;
        items += total;
    }
    __syncthreads();
    auto find = [&](int i, int& at, bool& held) {             // item i: its place in the table, and whether the block holds tokens from before
        int lo = 0, hi = B.n_seq - 1;
        while (lo < hi) {
            const int mid = (lo + hi + 1) >> 1;
            if (first[mid] <= i) lo = mid; else hi = mid - 1;
        }
        const Seq q = seq_of(B, lo);
        const int old = max(0, q.len - q.n_new), b = old / kKvBlock + i - first[lo];
        at = lo * P.table_ld + b;                             // (n_seq * table_ld is held below 2^28)
        held = b * kKvBlock < old;
    };
    // what each needs, by the counts as they are before anything changes
    int need = 0, at = 0, e = -1, r = -1;
    bool held = false;
    for (int i0 = 0; i0 < items; i0 += kPlan) {
        const int i = i0 + tid;
        int want = 0;
        if (i < items) {
            find(i, at, held);
            e = P.table[at];
            want = !is_block(P, e) || __ldcg(P.refs + e) > 1;
        }
        int total;
        r = rank_of(want, sh, total);
        r = want ? need + r : -1;
        if (i < items && items > kPlan) P.rows[at] = r;       // (one round: it stays in registers)
        need += total;
    }
    const int got = take_free(P, need, bits, sh);
    if (tid == 0 && got < need) P.words[0] = 1;
    for (int i = tid; i < items; i += kPlan) {
        if (items > kPlan) {
            find(i, at, held);
            r = P.rows[at];
            e = P.table[at];
        }
        if (r < 0) continue;
        const int fresh = r < got ? P.list[r] : -1;
        if (fresh >= 0) P.refs[fresh] = 1;
        if (is_block(P, e)) {
            atomicSub(P.refs + e, 1);                         // (also without a fresh one: new tokens must not go into a block that others hold)
            if (held && fresh >= 0) {
                const int m = atomicAdd(&s_moves, 1);
                P.src[m] = e;
                P.dst[m] = fresh;
            }
        }
        P.table[at] = fresh;
    }
    __syncthreads();
    if (tid == 0) P.words[1] = s_moves;
}

// ---------------------------------------------------------------- fork
// A pair's new row, and what it and the old one change of the counts, by `nt` threads.  The table itself stays: other pairs still read it.
__device__ __forceinline__ void fork_row(const Pages& P, int i, int parent, int child, int len, int fresh, int t, int nt) {
    const int* from = P.table + (size_t) parent * P.table_ld;
    const int* old = P.table + (size_t) child * P.table_ld;
    const int full = min(max(len, 0), P.table_ld * kKvBlock) / kKvBlock;
    for (int b = t; b < P.table_ld; b += nt) {
        const int gone = old[b];
        int e = -1;
        if (b < full) {
            e = from[b];
            if (is_block(P, e)) atomicAdd(P.refs + e, 1);
            else e = -1;
        } else if (b == full) {
            e = fresh;
        }
        if (is_block(P, gone)) atomicSub(P.refs + gone, 1);
        P.rows[(size_t) i * P.table_ld + b] = e;
    }
}
__global__ void __launch_bounds__(256) pages_fork_rows_kernel(const Pages P, const int* __restrict__ parents, const int* __restrict__ children,
                                                              const int* __restrict__ lens) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int i = blockIdx.x, fresh = P.fresh[i];
    if (fresh != -2) fork_row(P, i, parents[i], children[i], lens[i], fresh, threadIdx.x, 256);
}

// rows_too: a warp a pair makes the rows as well and puts them into the table: few of them are done before another launch would have begun.
__global__ void __launch_bounds__(kPlan) pages_fork_kernel(const Pages P, const int* __restrict__ parents, const int* __restrict__ children,
                                                           const int* __restrict__ lens, int n, int rows_too) {
    __shared__ PlanShared sh;
    __shared__ int s_owner[kSeqShared];
    const int tid = threadIdx.x;
    grid_launch_dependents();
    grid_dependency_wait();
    int* owner = P.n_seq <= kSeqShared ? s_owner : P.owner;
    const unsigned bits = live_bits(P, tid * kRefsEach, true);
    // the first pair of a child counts
    for (int i = tid; i < n; i += kPlan) {
        const int c = children[i];
        if (c >= 0 && c < P.n_seq) owner[c] = 0x7fffffff;
    }
    __syncthreads();
    for (int i = tid; i < n; i += kPlan) {
        const int c = children[i];
        if (c >= 0 && c < P.n_seq) atomicMin(owner + c, i);
    }
    __syncthreads();
    int need = 0;
    for (int i0 = 0; i0 < n; i0 += kPlan) {
        const int i = i0 + tid;
        int want = 0, from = -1;
        bool moves = false;
        if (i < n) {
            const int p = parents[i], c = children[i];
            moves = p >= 0 && p < P.n_seq && c >= 0 && c < P.n_seq && p != c && *(volatile int*) (owner + c) == i;
            const int len = min(max(lens[i], 0), P.table_ld * kKvBlock);
            if (moves && len % kKvBlock != 0) from = P.table[(size_t) p * P.table_ld + len / kKvBlock];
            want = is_block(P, from);
        }
        int total;
        const int r = need + rank_of(want, sh, total);
        if (want) P.src[r] = from;                        // (the list of moves is the list of wants)
        if (i < n) P.fresh[i] = want ? r : moves ? -1 : -2;
        need += total;
    }
    const int got = take_free(P, need, bits, sh);
    for (int i = tid; i < n; i += kPlan) {
        const int r = P.fresh[i];
        if (r < 0) continue;
        const int b = r < got ? P.list[r] : -1;
        P.fresh[i] = b;
        if (b >= 0) { P.refs[b] = 1; P.dst[r] = b; }
    }
    if (tid == 0) {
        P.words[1] = got;
        if (got < need) P.words[0] = 1;
    }
    if (!rows_too) return;
    __syncthreads();
    const int lane = tid & 31;
    for (int i = tid >> 5; i < n; i += kPlan / 32)
        if (P.fresh[i] != -2) fork_row(P, i, parents[i], children[i], lens[i], P.fresh[i], lane, 32);
    __syncthreads();
    for (int i = tid >> 5; i < n; i += kPlan / 32)
        if (P.fresh[i] != -2)
            for (int b = lane; b < P.table_ld; b += 32) P.table[(size_t) children[i] * P.table_ld + b] = P.rows[(size_t) i * P.table_ld + b];
}

// ---------------------------------------------------------------- free
__global__ void __launch_bounds__(256) pages_free_kernel(const Pages P, const int* __restrict__ seqs) {
    grid_launch_dependents();
    grid_dependency_wait();
    const int s = seqs[blockIdx.x];
    if (s < 0 || s >= P.n_seq) return;
    int* row = P.table + (size_t) s * P.table_ld;
    for (int b = threadIdx.x; b < P.table_ld; b += 256) {
        if (__ldcg(row + b) == -1) continue;
        const int e = atomicExch(row + b, -1);             // (a sequence that is named twice gives its blocks up once)
        if (is_block(P, e)) atomicSub(P.refs + e, 1);
    }
}

// ---------------------------------------------------------------- compact
__global__ void __launch_bounds__(kPlan) pages_compact_kernel(const Pages P, int most) {
    __shared__ PlanShared sh;
    const int tid = threadIdx.x;
    grid_launch_dependents();
    grid_dependency_wait();
    // holes of a thread's blocks (bits `open`), the first of which is hole number r; live ones behind the border (bits m) likewise
    auto take_holes = [&](int b0, unsigned open, int r) {
        while (open != 0u && r < most) {
            P.dst[r++] = b0 + __ffs(open) - 1;
            open &= open - 1u;
        }
    };
    auto move_tails = [&](int b0, unsigned m, int live, int r) {
        for (int i = 0; i < kRefsEach; ++i) {
            const int b = b0 + i;
            if (b < live || b >= P.n_blocks) continue;
            if (((m >> i) & 1u) && r < most) {
                const int to = P.dst[r];
                P.src[r++] = b;
                P.list[b] = to;
                P.refs[to] = P.refs[b];
                P.refs[b] = 0;
            } else {
                P.list[b] = b;
            }
        }
    };
    // bits of a thread's blocks in front of block `end`
    auto below = [](int b0, int end) { return end <= b0 ? 0u : end - b0 >= kRefsEach ? 0xffffu : (1u << (end - b0)) - 1u; };
    const int b0 = tid * kRefsEach;
    const unsigned bits = live_bits(P, b0, false);
    int live, tails;
    if (P.n_blocks <= kPlan * kRefsEach) {                // one look: every rank follows from the live blocks in front
        __shared__ int s_low;
        const int front = rank_of(__popc(bits), sh, live);
        if (tid == 0) s_low = live;                       // live blocks in front of the border
        __syncthreads();
        if (b0 <= live && live < b0 + kRefsEach) s_low = front + __popc(bits & below(b0, live));
        if (b0 < live) take_holes(b0, ~bits & below(b0, live), b0 - front);
        __syncthreads();
        tails = live - s_low;
        if (b0 + kRefsEach > live) move_tails(b0, bits & ~below(b0, live), live, front + __popc(bits & below(b0, live)) - s_low);
    } else {
        int mine = __popc(bits);
        for (int c = b0 + kPlan * kRefsEach; c - b0 < P.n_blocks; c += kPlan * kRefsEach) mine += __popc(live_bits(P, c, false));
        rank_of(mine, sh, live);
        int holes = 0;
        for (int c0 = 0; c0 < live && holes < most; c0 += kPlan * kRefsEach) {
            const int c = c0 + b0;
            const unsigned open = c < live ? ~live_bits(P, c, true) & below(c, live) : 0u;
            int total;
            const int r = holes + rank_of(__popc(open), sh, total);
            take_holes(c, open, r);
            holes += total;
        }
        __syncthreads();
        tails = 0;
        for (int c0 = live & ~(kRefsEach - 1); c0 < P.n_blocks; c0 += kPlan * kRefsEach) {
            const int c = c0 + b0;
            const unsigned m = c < P.n_blocks ? live_bits(P, c, false) & ~below(c, live) : 0u;
            int total;
            const int r = tails + rank_of(__popc(m), sh, total);
            move_tails(c, m, live, r);
            tails += total;
        }
    }
    if (tid == 0) { P.words[1] = min(tails, most); P.words[2] = live; }
}

// ---------------------------------------------------------------- what moves
// mode 0: nothing but the moves; 1 (fork): the children's rows into the table; 2 (compact): the table's entries behind the border.
enum { kMoves = 0, kForkRows = 1, kRemap = 2 };

__device__ __forceinline__ void copy_bytes(const uint8_t* from, uint8_t* to, int n, int tid) {
#pragma unroll
    for (int a = 0; a < kPieceBytes; a += kCopyThreads * 16 * 4) {
        uint4 v[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = a + (i * kCopyThreads + tid) * 16;
            if (at < n) v[i] = __ldcs((const uint4*) (from + at));
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int at = a + (i * kCopyThreads + tid) * 16;
            if (at < n) __stcs((uint4*) (to + at), v[i]);
        }
    }
}

__global__ void __launch_bounds__(kCopyThreads) pages_move_kernel(const Pages P, const int* __restrict__ src, const int* __restrict__ dst, int n_given, int mode,
                                                                  const int* __restrict__ children, int n_pairs) {
    const int tid = threadIdx.x;
    grid_launch_dependents();
    grid_dependency_wait();
    if (mode == kForkRows) {
        for (int i = blockIdx.x; i < n_pairs; i += gridDim.x) {
            if (P.fresh[i] == -2) continue;
            int* row = P.table + (size_t) children[i] * P.table_ld;
            for (int b = tid; b < P.table_ld; b += kCopyThreads) row[b] = P.rows[(size_t) i * P.table_ld + b];
        }
    } else if (mode == kRemap) {
        const int live = P.words[2];
        const int64_t n = (int64_t) P.n_seq * P.table_ld;
        for (int64_t i = (int64_t) blockIdx.x * kCopyThreads + tid; i < n; i += (int64_t) gridDim.x * kCopyThreads) {
            const int e = P.table[i];
            if (e >= live && e < P.n_blocks) P.table[i] = P.list[e];
        }
    }
    const int n = n_given >= 0 ? n_given : P.words[1];
    const int bytes = P.n_kv * kKvBlock * P.head_dim, pieces = (bytes + kPieceBytes - 1) / kPieceBytes;
    const int64_t units = (int64_t) n * P.n_layers * 2 * pieces;
    for (int64_t u = blockIdx.x; u < units; u += gridDim.x) {
        const int piece = (int) (u % pieces);
        const int64_t w = u / pieces;
        const bool values = w & 1;
        const int layer = (int) ((w >> 1) % P.n_layers), m = (int) ((w >> 1) / P.n_layers);
        const int from = src[m], to = dst[m];
        if (!is_block(P, from) || !is_block(P, to) || from == to) continue;
        const maya_kv_layer L = P.layers[layer];
        uint8_t* base = (uint8_t*) (values ? L.v : L.k);
        const int at = piece * kPieceBytes;
        copy_bytes(base + (size_t) from * bytes + at, base + (size_t) to * bytes + at, min(kPieceBytes, bytes - at), tid);
        if (piece == 0) {                                  // the block's scales, with the keys its sums
            float* s = values ? L.v_scale : L.k_scale;
            for (int i = tid; i < P.n_kv; i += kCopyThreads) s[(size_t) to * P.n_kv + i] = s[(size_t) from * P.n_kv + i];
            if (!values && P.sums) {
                const int words = P.n_kv * P.head_dim / 8;
                const uint4* a = (const uint4*) (L.k_sum + (size_t) from * P.n_kv * P.head_dim);
                uint4* b = (uint4*) (L.k_sum + (size_t) to * P.n_kv * P.head_dim);
                for (int i = tid; i < words; i += kCopyThreads) b[i] = a[i];
            }
        }
    }
}

// A thread block a piece where the host knows how many there are (500 blocks of four layers 85 us, 96 with eight thread blocks an SM that go through the
// pieces); where the count is in the scratch, as many as the most there can be to do, 16 an SM at most, since those that find nothing cost too.
int launch_moves(const Pages& P, const int* src, const int* dst, int n_given, int64_t most, int mode, const int* children, int n_pairs, cudaStream_t s) {
    const int64_t pieces = ((int64_t) P.n_kv * kKvBlock * P.head_dim + kPieceBytes - 1) / kPieceBytes;
    int64_t blocks = most * P.n_layers * 2 * pieces;
    if (mode == kForkRows && blocks < n_pairs) blocks = n_pairs;
    if (mode == kRemap && blocks * kCopyThreads < (int64_t) P.n_seq * P.table_ld) blocks = ((int64_t) P.n_seq * P.table_ld + kCopyThreads - 1) / kCopyThreads;
    const int64_t cap = n_given >= 0 ? 1 << 30 : (int64_t) sm_count() * 16;
    if (blocks > cap) blocks = cap;
    if (blocks < 1) blocks = 1;
    launch_dependent(pages_move_kernel, dim3((unsigned) blocks), dim3(kCopyThreads), 0, s, P, src, dst, n_given, mode, children, n_pairs);
    return note_launch("kv_pages move");
}

}  // namespace
}  // namespace maya

using namespace maya;

extern "C" size_t maya_pages_scratch_bytes(const maya_kv_pages* p) { return pages_check(p) == MAYA_OK ? pages_carve(p, nullptr) : 0; }

extern "C" int maya_pages_error(const maya_kv_pages* p, void* stream) {
    if (pages_check(p) != MAYA_OK || !p->scratch) return refuse(MAYA_ERR_ARG);
    int word = 0;
    cudaStream_t s = as_stream(stream);
    if (cudaMemcpyAsync(&word, p->scratch, sizeof(word), cudaMemcpyDeviceToHost, s) != cudaSuccess || cudaStreamSynchronize(s) != cudaSuccess) return note_launch("kv_pages error");
    return word;
}

extern "C" int maya_pages_reserve(const maya_kv_pages* p, const maya_attn_batch* b, void* stream) {
    Pages P;
    const int st = pages_ready(p, &P);
    if (st != MAYA_OK) return refuse(st);
    if (!b || !b->start || !b->kv_len || b->n_seq < 0 || b->n_tokens < 0 || b->max_new < 0 || b->max_len < 0 || b->n_seq > p->n_seq) return refuse(MAYA_ERR_ARG);
    if (b->n_tokens > 0 && (b->n_seq == 0 || b->max_new == 0)) return refuse(MAYA_ERR_ARG);
    if (b->max_len > (long long) p->table_ld * kKvBlock) return refuse(MAYA_ERR_ARG);
    if (b->n_tokens > (1 << 24)) return refuse(MAYA_ERR_LIMIT);
    if (b->n_tokens == 0 || b->max_len == 0) return MAYA_OK;
    cudaStream_t s = as_stream(stream);
    launch_dependent(pages_reserve_kernel, dim3(1), dim3(kPlan), 0, s, P, batch_view(*b));
    const int launched = note_launch("kv_pages reserve");
    if (launched != MAYA_OK) return launched;
    return launch_moves(P, P.src, P.dst, -1, b->n_seq, kMoves, nullptr, 0, s);
}

extern "C" int maya_pages_fork(const maya_kv_pages* p, const int* parents, const int* children, const int* lens, int n, void* stream) {
    Pages P;
    const int st = pages_ready(p, &P);
    if (st != MAYA_OK) return refuse(st);
    if (n == 0) return MAYA_OK;
    if (n < 0 || !parents || !children || !lens) return refuse(MAYA_ERR_ARG);
    if (n > p->n_seq) return refuse(MAYA_ERR_LIMIT);              // more pairs than children there are
    cudaStream_t s = as_stream(stream);
    // A warp a row in the plan's launch while there is one for each and a row is three looks long, otherwise a launch with a thread block a row.  Both ways, plan's / own (the fork alone, us): 32
    // rows of 64 blocks 9.3 / 9.3, one 8.3 / 8.6; 64 rows of 64 11.0 / 9.3; one row of 256 10.9 / 9.0, of 16384 222 / 45.
    const bool rows_too = n <= kPlan / 32 && p->table_ld <= 96;
    launch_dependent(pages_fork_kernel, dim3(1), dim3(kPlan), 0, s, P, parents, children, lens, n, (int) rows_too);
    int launched = note_launch("kv_pages fork");
    if (launched != MAYA_OK) return launched;
    if (!rows_too) {
        launch_dependent(pages_fork_rows_kernel, dim3((unsigned) n), dim3(256), 0, s, P, parents, children, lens);
        launched = note_launch("kv_pages fork rows");
        if (launched != MAYA_OK) return launched;
    }
    return launch_moves(P, P.src, P.dst, -1, n, rows_too ? kMoves : kForkRows, children, n, s);
}

extern "C" int maya_pages_free(const maya_kv_pages* p, const int* seqs, int n, void* stream) {
    Pages P;
    const int st = pages_ready(p, &P);
    if (st != MAYA_OK) return refuse(st);
    if (n == 0) return MAYA_OK;
    if (n < 0 || !seqs) return refuse(MAYA_ERR_ARG);
    launch_dependent(pages_free_kernel, dim3((unsigned) n), dim3(256), 0, as_stream(stream), P, seqs);
    return note_launch("kv_pages free");
}

extern "C" int maya_pages_compact(const maya_kv_pages* p, int most, void* stream) {
    Pages P;
    const int st = pages_ready(p, &P);
    if (st != MAYA_OK) return refuse(st);
    if (most < 0) return refuse(MAYA_ERR_ARG);
    if (most > p->n_blocks / 2) most = p->n_blocks / 2;
    cudaStream_t s = as_stream(stream);
    launch_dependent(pages_compact_kernel, dim3(1), dim3(kPlan), 0, s, P, most);
    const int launched = note_launch("kv_pages compact");
    if (launched != MAYA_OK) return launched;
    return launch_moves(P, P.src, P.dst, -1, most, kRemap, nullptr, 0, s);
}

extern "C" int maya_pages_copy(const maya_kv_pages* p, const int* src, const int* dst, int n, void* stream) {
    Pages P;
    const int st = pages_ready(p, &P);
    if (st != MAYA_OK) return refuse(st);
    if (n == 0) return MAYA_OK;
    if (n < 0 || !src || !dst) return refuse(MAYA_ERR_ARG);
    if (n > p->n_blocks) return refuse(MAYA_ERR_LIMIT);
    return launch_moves(P, src, dst, n, n, kMoves, nullptr, 0, as_stream(stream));
}
