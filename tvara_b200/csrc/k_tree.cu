// Bookkeeping and commit of drafted-token trees (tvara_tree_plan,
// tvara_tree_commit of include/tvara_kernels.h).
#include <algorithm>
#include <climits>

#include "tree.cuh"

namespace tvara {
namespace {

// ------------------------------------------------------------------- plan
// Sequence s needs need(s) = max(0, ceil((L + n) / bt) - held) new blocks;
// first(s) is the exclusive prefix sum of need, and new block e of sequence s
// is free_blocks[count - 1 - (first(s) + e)].  Every CTA computes the whole
// prefix sum itself (at most 8192 sequences, 12 bytes each, from L2) instead
// of waiting for another one's, so the step is one launch; then rows and new
// table entries are spread over the grid and find their sequence by a binary
// search in shared memory.  All sequences are checked before anything is
// written, by every CTA alike, so a refused plan writes nothing.
//
// Bound by latency, not bytes: a launch, one read of the lengths, the scan, a
// search and, for trees, the walk up in shared memory.  One tree of 26 nodes
// 7.5 us a call, 500 trees of up to 63 nodes 7.8 us, 511 prompts of up to 2,047
// rows (6.3 MB) 10.2 us.  Counts in place (held_out = held or free_left =
// free_count) take a second launch of one CTA, once no CTA reads them any more:
// 10.4 and 11.7 us for the first two.  (Summing all needs with one contended shared-memory
// atomic cost 12 us; a thread per prompt row instead of four, another 8 us.)
constexpr int kPlanThreads = 512;
constexpr int kPlanRun = 4;  // consecutive rows a thread takes when there are no trees
enum { kPlanRows = 1, kPlanCounts = 2 };

__device__ __forceinline__ int last_at_most(const int* sorted, int n, int x) {
    int lo = 0, hi = n;  // sorted[lo] <= x < sorted[hi] (sorted[n] counts as infinite)
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (sorted[mid] <= x)
            lo = mid;
        else
            hi = mid;
    }
    return lo;
}

__global__ void __launch_bounds__(kPlanThreads) tree_plan_kernel(TreePlan a, int mode) {
    extern __shared__ int plan_smem[];
    int* cu_s = plan_smem;                      // [n_seq + 1]
    int* first_s = plan_smem + a.n_seq + 1;     // [n_seq + 1]
    int* parents_s = first_s + a.n_seq + 1;     // trees: parents of this CTA's rows, from their first sequence's start
    __shared__ int warp_sum[kPlanThreads / 32];
    __shared__ long long warp_need[kPlanThreads / 32];
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int free_count = *a.free_count;
    int bad = 0, carry = 0;
    long long mine = 0;
    if (free_count < 0 || free_count > a.free_capacity) bad = kTreeBadLengths;
    for (int base = 0; base < a.n_seq; base += kPlanThreads) {
        const int i = base + tid;
        int need = 0, c0 = 0;
        if (i < a.n_seq) {
            c0 = a.cu[i];
            const int c1 = a.cu[i + 1], len = a.lengths[i], held = a.held[i];
            const long long n = (long long)c1 - c0, end = (long long)len + n;
            const long long blocks = (end + a.bt - 1) / a.bt;
            if (n < 0 || c1 > a.capacity || (i == 0 && c0 != 0) || len < 0 || held < 0 || held > a.stride ||
                (long long)held * a.bt < len || end > INT_MAX || blocks > a.stride || (a.ancestors && n > a.max_nodes))
                bad |= kTreeBadLengths;
            else
                need = int(max(0ll, blocks - held));
        }
        mine += need;
        int scan = need;
        for (int d = 1; d < 32; d <<= 1) {
            const int up = __shfl_up_sync(0xffffffffu, scan, d);
            if (lane >= d) scan += up;
        }
        if (lane == 31) warp_sum[warp] = scan;
        __syncthreads();
        int before = carry, all = 0;
        for (int w = 0; w < kPlanThreads / 32; ++w) {
            if (w < warp) before += warp_sum[w];
            all += warp_sum[w];
        }
        if (i < a.n_seq) {
            cu_s[i] = c0;
            first_s[i] = before + scan - need;
        }
        carry += all;
        __syncthreads();
    }
    for (int d = 16; d; d >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, d);
    if (lane == 0) warp_need[warp] = mine;
    const int refused = __syncthreads_or(bad);
    long long need_total = 0;
    for (int w = 0; w < kPlanThreads / 32; ++w) need_total += warp_need[w];
    if (refused || need_total > free_count) {
        if (blockIdx.x == 0 && tid == 0) atomicOr(a.status, refused ? kTreeBadLengths : kTreeNoBlocks);
        return;
    }
    if (tid == 0) {
        cu_s[a.n_seq] = a.cu[a.n_seq];
        first_s[a.n_seq] = int(need_total);
    }
    __syncthreads();
    const int total = cu_s[a.n_seq], fresh = first_s[a.n_seq];
    const int step = int(gridDim.x) * kPlanThreads, at = int(blockIdx.x) * kPlanThreads + tid;
    if (mode & kPlanCounts) {
        for (int i = at; i < a.n_seq; i += step) a.held_out[i] = a.held[i] + first_s[i + 1] - first_s[i];
        if (at == 0) *a.free_left = free_count - fresh;
    }
    if (!(mode & kPlanRows)) return;
    int flags = 0;
    for (long long at_new = at; at_new < fresh; at_new += step) {  // (fresh may be near 2^31, as total below)
        const int j = int(at_new);
        // first_s repeats over sequences that need nothing: the last of equal
        // entries is the one that takes block j
        const int s = last_at_most(first_s, a.n_seq, j);
        const int block = a.free_blocks[free_count - 1 - j];
        if (unsigned(block) >= unsigned(a.max_blocks)) flags |= kTreeBadBlock;
        a.tables[(long long)s * a.stride + a.held[s] + j - first_s[s]] = block;
    }
    // the slot and position of row t of sequence s
    const auto place = [&](int t, int s, int len, int held) {
        const int p = len + t - cu_s[s], entry = unsigned(p) / unsigned(a.bt);
        const int block = entry < held ? a.tables[(long long)s * a.stride + entry]
                                       : a.free_blocks[free_count - 1 - (first_s[s] + entry - held)];
        const bool good = unsigned(block) < unsigned(a.max_blocks);
        if (!good) flags |= kTreeBadBlock;
        a.slots[t] = good ? (long long)block * a.bt + (p - entry * a.bt) : -1;
        return p;
    };
    if (!a.parents) {
        for (long long t0 = at * kPlanRun; t0 < total; t0 += step * kPlanRun) {
            int s = last_at_most(cu_s, a.n_seq, int(t0)), len = a.lengths[s], held = a.held[s];
            const int behind = int(min(t0 + kPlanRun, (long long)total));
            for (int t = int(t0); t < behind; ++t) {
                while (t >= cu_s[s + 1]) {
                    ++s;
                    len = a.lengths[s];
                    held = a.held[s];
                }
                a.positions[t] = place(t, s, len, held);
            }
        }
    } else {
        for (int tile = int(blockIdx.x) * kPlanThreads; tile < total; tile += step) {
            // the tile's rows and those before them back to their sequence's first
            const int from = cu_s[last_at_most(cu_s, a.n_seq, tile)], to = min(tile + kPlanThreads, total);
            __syncthreads();
            for (int i = from + tid; i < to; i += kPlanThreads) parents_s[i - from] = a.parents[i];
            __syncthreads();
            const int t = tile + tid;
            if (t >= to) continue;
            const int s = last_at_most(cu_s, a.n_seq, t), len = a.lengths[s];
            place(t, s, len, a.held[s]);
            // Up the tree: indices only fall, so each word of the mask is
            // complete when the walk leaves it.
            const int* parents = parents_s + (cu_s[s] - from);
            unsigned long long* row = a.ancestors + (long long)t * a.words;
            const int i = t - cu_s[s];
            int word = i >> 6, depth = 0, node = i;
            for (int w = a.words - 1; w > word; --w) row[w] = 0;
            unsigned long long bits = 1ull << (i & 63);
            for (;;) {
                const int up = parents[node];
                if (up < 0 || up >= node) {
                    if (up != -1) flags |= kTreeBadParent;
                    break;
                }
                node = up;
                ++depth;
                while (word > (node >> 6)) {
                    row[word--] = bits;
                    bits = 0;
                }
                bits |= 1ull << (node & 63);
            }
            while (word >= 0) {
                row[word--] = bits;
                bits = 0;
            }
            a.positions[t] = len + depth;
        }
    }
    if (flags) atomicOr(a.status, flags);
}

// ----------------------------------------------------------------- commit
// Each CTA takes one sequence and a slice of its K/V columns.  It first walks
// the tree: every node whose token equals the choice at its parent offers
// itself to the parent (atomicMin on shared memory: the lowest index wins), so
// the walk itself is one chain of shared-memory reads; CTAs of the same
// sequence repeat it rather than wait for one another.  Then thread u copies
// column u (a 16-byte piece of one layer's K or V of one head) of every
// accepted row, kCommitRows rows in flight at a time.  In place, path[k] > k
// or the rows coincide, and a batch is read before it is written, so
// ascending batches never read a row that was overwritten.
//
// 48 sequences, 32 layers of 8 heads of 128 F16: 34 MB in 14.3 us (5.3 us at
// the copy bandwidth; in a loop over two inputs 12.2, and 10.3 in place); one
// sequence 7.2 us, a launch and four dependent fetches.  next over first with several slices takes a second launch
// for the answers: 2 to 3.5 us more.  Slices of one sequence beyond those that run at the same time only
// repeat the walk (1,536 instead of 864 CTAs: 16.4 us).
constexpr int kCommitThreads = 256;
constexpr int kCommitRows = 8;

// Columns of `units` = runs x row_units pieces, a run being the bt rows of one
// (layer, kind, head) in a block; from / to are row indexes of the first run.
template <typename U>
__device__ __forceinline__ void move_columns(U* base, int units, int row_units, int bt, const long long* from,
                                             const long long* to, int rows) {
    for (int u = int(blockIdx.y) * kCommitThreads + int(threadIdx.x); u < units; u += int(gridDim.y) * kCommitThreads) {
        const int run = u / row_units;
        U* mine = base + (long long)run * bt * row_units + (u - run * row_units);
        for (int k0 = 0; k0 < rows; k0 += kCommitRows) {
            U v[kCommitRows];
#pragma unroll
            for (int k = 0; k < kCommitRows; ++k)
                if (k0 + k < rows && from[k0 + k] >= 0) v[k] = mine[from[k0 + k] * row_units];
#pragma unroll
            for (int k = 0; k < kCommitRows; ++k)
                if (k0 + k < rows && from[k0 + k] >= 0) mine[to[k0 + k] * row_units] = v[k];
        }
    }
}

// parts: kCommitMove, kCommitAnswers, or both in one launch (the answers by
// slice 0, which is safe as long as no other slice still reads what they overwrite).
enum { kCommitMove = 1, kCommitAnswers = 2 };

template <typename U>
__global__ void __launch_bounds__(kCommitThreads) tree_commit_kernel(TreeCommit a, int parts) {
    extern __shared__ long long commit_smem[];
    long long* from = commit_smem;           // [max_nodes] source row of accepted node k, -1: not moved
    long long* to = from + a.max_nodes;      // [max_nodes]
    int* best = reinterpret_cast<int*>(to + a.max_nodes);  // [max_nodes + 1] first matching child of node - 1
    int* path = best + a.max_nodes + 1;      // [max_nodes]
    unsigned* choice = reinterpret_cast<unsigned*>(path + a.max_nodes);  // [max_nodes]
    __shared__ int count_s;
    const int s = blockIdx.x, tid = threadIdx.x;
    const bool answers = (parts & kCommitAnswers) && blockIdx.y == 0;
    // (lengths_out may be lengths: other slices see either value, and only ask whether it is negative)
    const int c0 = a.cu[s], c1 = a.cu[s + 1], len = a.lengths[s];
    const long long n64 = (long long)c1 - c0;
    if (c0 < 0 || n64 < 0 || n64 > a.max_nodes || c1 > a.capacity || c1 > a.cu[a.n_seq] || len < 0) {
        if (blockIdx.y == 0 && tid == 0) atomicOr(a.status, kTreeBadLengths);
        return;
    }
    const int n = int(n64);
    const unsigned none = 0xffffffffu;
    // everything that is known before the walk is fetched at once
    const unsigned first = a.first ? a.first[s] : none;
    const long long* dest = a.dest ? a.dest : a.slots;
    for (int i = tid; i < n; i += kCommitThreads) {
        best[i] = INT_MAX;
        choice[i] = a.choices[c0 + i];
        if (a.pool) {
            from[i] = a.slots[c0 + i];
            to[i] = dest[c0 + i];
        }
    }
    if (tid == 0) best[n] = INT_MAX;
    const int parent0 = tid < n ? a.parents[c0 + tid] : 0;
    const unsigned token0 = tid < n ? a.tokens[c0 + tid] : 0;
    __syncthreads();
    int flags = s == 0 && c0 != 0 ? kTreeBadLengths : 0;
    for (int i = tid; i < n; i += kCommitThreads) {
        const int p = i == tid ? parent0 : a.parents[c0 + i];
        if (p < -1 || p >= i) {
            flags |= kTreeBadParent;
            continue;
        }
        const unsigned want = p >= 0 ? choice[p] : first;
        const bool match = !a.first && i == 0 ? true : want != none && (i == tid ? token0 : a.tokens[c0 + i]) == want;
        if (match) atomicMin(&best[p + 1], i);
    }
    __syncthreads();
    if (tid == 0) {
        int k = 0, at = -1;
        while (best[at + 1] != INT_MAX) path[k++] = at = best[at + 1];
        count_s = k;
        if (answers) {
            a.accepted[s] = k;
            a.next[s] = at >= 0 ? choice[at] : first;
            a.lengths_out[s] = len + k;
        }
    }
    __syncthreads();
    const int rows = count_s;
    if (answers)
        for (int i = tid; i < n; i += kCommitThreads) a.path[c0 + i] = i < rows ? path[i] : -1;
    if (a.pool && rows && (parts & kCommitMove)) {
        const long long limit = (long long)a.max_blocks * a.bt;
        const int runs = a.layers * 2 * a.hkv;
        const long long block_rows = (long long)runs * a.bt;
        for (int k0 = 0; k0 < rows; k0 += kCommitThreads) {  // path[k] >= k: a pass reads before it writes
            const int k = k0 + tid;
            long long f = -1, t = -1;
            if (k < rows) {
                f = from[path[k]];
                t = to[k];
                const bool good = f >= 0 && f < limit && t >= 0 && t < limit;
                if (!good) flags |= kTreeBadBlock;
                const bool moves = good && f != t;
                f = moves ? f / a.bt * block_rows + f % a.bt : -1;
                t = moves ? t / a.bt * block_rows + t % a.bt : -1;
            }
            __syncthreads();
            if (k < rows) {
                from[k] = f;
                to[k] = t;
            }
        }
        __syncthreads();
        const int row_units = a.dim * a.elem / int(sizeof(U));
        move_columns(static_cast<U*>(a.pool), runs * row_units, row_units, a.bt, from, to, rows);
        if (a.scales) move_columns(a.scales, runs, 1, a.bt, from, to, rows);
    }
    if (flags && blockIdx.y == 0) atomicOr(a.status, flags);
}

template <typename U>
void run_commit(const TreeCommit& a, cudaStream_t s) {
    const std::size_t smem = std::size_t(a.max_nodes) * 28 + 8;
    const long long units = (long long)a.layers * 2 * a.hkv * a.dim * a.elem / (long long)sizeof(U);
    // every slice repeats the walk: no more of them than run at the same time
    const long long room = std::max<long long>(1, 148 * 6 / a.n_seq);
    const long long slices = a.pool ? std::min<long long>((units + kCommitThreads - 1) / kCommitThreads, room) : 1;
    // next written over first waits until no slice reads first any more
    const bool apart = a.first && a.next == a.first && slices > 1;
    tree_commit_kernel<U><<<dim3(unsigned(a.n_seq), unsigned(slices)), kCommitThreads, smem, s>>>(
        a, apart ? kCommitMove : kCommitMove | kCommitAnswers);
    TVARA_LAUNCHED();
    if (apart) {
        tree_commit_kernel<U><<<dim3(unsigned(a.n_seq), 1), kCommitThreads, smem, s>>>(a, kCommitAnswers);
        TVARA_LAUNCHED();
    }
}

}  // namespace

void launch_tree_plan(const TreePlan& a, cudaStream_t s) {
    const std::size_t smem = std::size_t(a.n_seq + 1) * 8 + (a.parents ? (kPlanThreads + kTreeMaxNodes) * 4 : 0);
    if (smem > 48 * 1024)
        TVARA_CUDA(cudaFuncSetAttribute(tree_plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, int(smem)));
    const long long most = std::max<long long>(a.parents ? a.capacity : (a.capacity + kPlanRun - 1ll) / kPlanRun, a.n_seq);
    const int grid = int(std::clamp<long long>((most + kPlanThreads - 1) / kPlanThreads, 1, 296));
    // counts written over their own inputs wait until no CTA reads these
    const bool in_place = a.held_out == a.held || a.free_left == a.free_count;
    tree_plan_kernel<<<grid, kPlanThreads, smem, s>>>(a, in_place ? kPlanRows : kPlanRows | kPlanCounts);
    TVARA_LAUNCHED();
    if (in_place) {
        tree_plan_kernel<<<1, kPlanThreads, smem, s>>>(a, kPlanCounts);
        TVARA_LAUNCHED();
    }
}

void launch_tree_commit(const TreeCommit& a, cudaStream_t s) {
    const std::size_t row = std::size_t(a.dim) * a.elem;
    const auto base = reinterpret_cast<std::uintptr_t>(a.pool);
    if (row % 16 == 0 && base % 16 == 0)
        run_commit<uint4>(a, s);
    else if (row % 4 == 0 && base % 4 == 0)
        run_commit<unsigned>(a, s);
    else if (row % 2 == 0 && base % 2 == 0)
        run_commit<unsigned short>(a, s);
    else
        run_commit<unsigned char>(a, s);
}

}  // namespace tvara
