// Attention of drafted-token trees over the paged KV cache
// (tvara_tree_attention of include/tvara_kernels.h).
//
// Row i of sequence s, query head h:  o = sum_j w_j v_j,  w = softmax over
// the visible j of q.k_j / sqrt(d),  j running over the L cached positions
// (block table) and the nodes whose bit is set in the row's mask (slots).
#include <algorithm>
#include <cmath>

#include <cuda_fp16.h>

#include "tma.cuh"
#include "tree.cuh"

namespace tvara {
namespace {

// Rows, node count and length of sequence s; false when they are invalid.
__device__ __forceinline__ bool tree_sequence_ok(const TreeAttn& a, int s, int& c0, int& n, int& len) {
    c0 = a.cu[s];
    const int c1 = a.cu[s + 1], end = a.cu[a.n_seq];  // rows from `end` on are no sequence's
    len = a.lengths[s];
    const long long rows = (long long)c1 - c0;
    n = int(rows);
    return c0 >= 0 && rows >= 0 && rows <= a.max_nodes && c1 <= a.capacity && c1 <= end && len >= 0 &&
           len <= (long long)a.stride * a.bt && len <= 0x7fffffff - 2 * kTreeMaxNodes;
}

// What every form reports about sequence s, rows or not.
__device__ __forceinline__ bool tree_reported(const TreeAttn& a, int s) {
    int c0, n, len;
    return !tree_sequence_ok(a, s, c0, n, len) || (s == 0 && c0 != 0);
}

// x / bt for x < 2^44 by the reciprocal 2^64 / bt rounded up (0 stands for
// bt 1), which is too large by less than 2^-64: the product by less than
// 2^-20, and the fraction of x / bt is at most 1 - 2^-20 (bt <= 2^20).
__device__ __forceinline__ long long div_bt(const TreeAttn& a, long long x) {
    return a.bt_inverse ? (long long)__umul64hi((unsigned long long)x, a.bt_inverse) : x;
}
// Row (of dim elements) in the pool that holds K of head 0 of the layer for
// index p of a sequence (cached positions, then nodes), or -1 with the status
// bit for a block or slot outside the pool.
__device__ __forceinline__ long long tree_row(const TreeAttn& a, int s, int c0, int len, int p, int& flags) {
    long long block, off;
    if (p < len) {
        const int e = int(div_bt(a, p));
        block = a.tables[(long long)s * a.stride + e];
        off = p - e * a.bt;
    } else {
        const long long slot = a.slots[c0 + p - len];
        const bool in = slot >= 0 && slot < (long long)a.max_blocks * a.bt;
        block = in ? div_bt(a, slot) : -1;
        off = slot - block * a.bt;
    }
    if (block < 0 || block >= a.max_blocks) {
        flags |= kTreeBadBlock;
        return -1;
    }
    return block * a.block_rows + a.layer_rows + off;
}

// ---------------------------------------------------------- any shape
// One CTA of four warps per (row, query head), positions dealt to the warps,
// online softmax in F32, merged through shared memory.  Each position's K is
// reduced across the warp, so this form is bound by those shuffles (a few
// percent of memory bandwidth), and every row and head reads K and V again; it
// serves the shapes that the tensor-core form does not take
// (launch_tree_attention).  26 nodes on 1,900 positions: 16/4 heads of 256 F16
// 522 us, int8 823, F32 668 (16 such sequences 4.2, 6.1, 6.6 ms); 32/8 heads of
// 128 F16 with query rows off 16 bytes 447 us, where aligned ones take 29.
constexpr int kAnyWarps = 4;

__device__ __forceinline__ float kv_value(const TreeAttn& a, long long at) {
    if (a.kv_kind == 0) return static_cast<const float*>(a.kv)[at];
    if (a.kv_kind == 1) return __half2float(static_cast<const __half*>(a.kv)[at]);
    return float(static_cast<const signed char*>(a.kv)[at]);
}

template <int E>  // elements of a row per lane
__global__ void __launch_bounds__(kAnyWarps * 32) tree_any_kernel(TreeAttn a) {
    __shared__ float sm_m[kAnyWarps], sm_l[kAnyWarps];
    __shared__ float sm_acc[kAnyWarps][E * 32];
    const int t = blockIdx.x, h = blockIdx.y, warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (t == 0 && h == 0) {  // sizes are reported by sequence: an empty one has no row here
        bool bad = false;
        for (int s = threadIdx.x; s < a.n_seq; s += kAnyWarps * 32) bad |= tree_reported(a, s);
        if (__syncthreads_or(bad) && threadIdx.x == 0) atomicOr(a.status, kTreeBadLengths);
    }
    if (t >= a.cu[a.n_seq]) return;
    int lo = 0, hi = a.n_seq;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a.cu[mid] <= t)
            lo = mid;
        else
            hi = mid;
    }
    int c0, n, len, flags = 0;
    const auto holds = [&](int s) { return tree_sequence_ok(a, s, c0, n, len) && t >= c0 && t - c0 < n; };
    if (!holds(lo)) {
        // a row of no sequence, or one that the search missed among sizes that
        // do not ascend: of the valid sequences that hold it, the last
        __shared__ int holder;
        if (threadIdx.x == 0) holder = -1;
        __syncthreads();
        int mine = -1;
        for (int s = threadIdx.x; s < a.n_seq; s += kAnyWarps * 32)
            if (holds(s)) mine = s;
        if (mine >= 0) atomicMax(&holder, mine);
        __syncthreads();
        lo = holder;
        if (lo < 0) return;
        holds(lo);
    }
    const int node = t - c0, g = h / a.group;
    const unsigned long long* mask = a.ancestors ? a.ancestors + (long long)t * a.words : nullptr;
    const float* q = a.q + (long long)t * a.ldq + (long long)h * a.dim;
    float qv[E], acc[E];
#pragma unroll
    for (int e = 0; e < E; ++e) {
        qv[e] = lane + 32 * e < a.dim ? q[lane + 32 * e] : 0.f;
        acc[e] = 0.f;
    }
    const float scale = 1.f / sqrtf(float(a.dim));
    float m = -INFINITY, l = 0.f;
    const long long end = (long long)len + n;
    for (long long p = warp; p < end; p += kAnyWarps) {
        if (p >= len) {
            const int j = int(p) - len;
            if (mask ? !((mask[j >> 6] >> (j & 63)) & 1) : j > node) continue;
        }
        const long long base = tree_row(a, lo, c0, len, int(p), flags);
        if (base < 0) continue;
        const long long k_row = base + (long long)g * a.bt, k = k_row * a.dim, v = k + a.kind_rows * a.dim;
        float dot = 0.f;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane + 32 * e < a.dim) dot = fmaf(qv[e], kv_value(a, k + lane + 32 * e), dot);
#pragma unroll
        for (int d = 16; d; d >>= 1) dot += __shfl_xor_sync(0xffffffffu, dot, d);
        float s = dot * scale, sv = 1.f;
        if (a.scales) {
            s *= a.scales[k_row];
            sv = a.scales[k_row + a.kind_rows];
        }
        const float mn = fmaxf(m, s);
        const float ref = mn == -INFINITY ? 0.f : mn;
        const float keep = expf(m - ref), w = expf(s - ref);
        m = mn;
        l = l * keep + w;
#pragma unroll
        for (int e = 0; e < E; ++e)
            if (lane + 32 * e < a.dim) acc[e] = fmaf(w * sv, kv_value(a, v + lane + 32 * e), acc[e] * keep);
    }
    if (lane == 0) {
        sm_m[warp] = m;
        sm_l[warp] = l;
    }
#pragma unroll
    for (int e = 0; e < E; ++e) sm_acc[warp][lane + 32 * e] = acc[e];
    __syncthreads();
    float top = -INFINITY;
    for (int w = 0; w < kAnyWarps; ++w) top = fmaxf(top, sm_m[w]);
    const float ref = top == -INFINITY ? 0.f : top;
    float total = 0.f;
    for (int w = 0; w < kAnyWarps; ++w) total += sm_l[w] * expf(sm_m[w] - ref);
    for (int d = threadIdx.x; d < a.dim; d += kAnyWarps * 32) {
        float sum = 0.f;
        for (int w = 0; w < kAnyWarps; ++w) sum += sm_acc[w][d] * expf(sm_m[w] - ref);
        // NaN sums (non-finite inputs) stay NaN; a row that attends to nothing is zero
        a.out[(long long)t * a.ldo + (long long)h * a.dim + d] = total == 0.f && top == -INFINITY ? 0.f : sum / total;
    }
    if (flags && lane == 0) atomicOr(a.status, flags);
}

// ------------------------------------------------------- tensor cores
// head_dim up to 128 (rows of a multiple of 16 bytes), any block size.
//
// A work item is (sequence, KV head, group of query vectors): its n drafted
// rows times the G query heads that share the KV head, up to 128 vectors on
// the M dimension of a tcgen05.mma (256 as two M tiles for F16 pools).  The
// L + n keys are walked in tiles of kBn positions; a tile may hold cached
// positions and nodes, since every row of it is fetched by its own address
// (block table or slot map), so any block size and slot order costs the same.
//   S  = Q K^T   per tile into tensor memory,
//   P  = 2^(S c - m + 11) by the softmax warps, one thread per query vector
//        (no shuffles), written back over S as the A operand,
//   Ot = P V     per tile into tensor memory, added to the thread's F32 row
//        O = O 2^(m_old - m) + Ot in registers.
// The tensor core's own F32 accumulation truncates, so it is kept to one
// tile (the small lo products first) and the long sum over tiles is rounded
// to nearest in registers; that costs one fused multiply-add per element.
// F32 results from F16 operands: Q, P (and K, V of F32 pools) enter as hi +
// lo F16 pairs that carry 2^-23 of each value, int8 codes are exact in F16; the
// scales of int8 rows, and the powers of two that bring F32 rows below 2^15,
// are applied to the columns of S and to P.  With such scales O has a reference
// of its own, 2^(m + m_v), m_v from the V scales that a row sees.
//
// Two softmax warpgroups ("streams") keep the tensor core busy: with one M
// tile they take the even and the odd tiles of the same item, each with its
// own O, m and l, merged through tensor memory at the end; with two M tiles
// each owns one and every K/V tile is used twice.
//
// Work is dealt to one CTA per SM in equal runs of tiles over all items
// (each CTA scans the lengths and cuts out its run), so ragged batches and a
// single long sequence fill the device alike; an item cut by a run boundary
// leaves partial (O, m, l, m_v) in the workspace for tree_combine_kernel.
//
// What bounds it.  A tile of 128 positions costs a stream 32 MMAs of 64
// cycles (hi and lo of Q, and of P), of which the Q K^T half reads shared
// memory at its full rate (8 KB in 64 cycles); softmax, acc and the waits in
// between are hidden by the other stream.  F16 with two M tiles: 6,700 cycles
// a tile for 4,096 of MMA (4 trees of up to 255 nodes over 8,000-30,000
// positions: 560 us sustained, tensor pipe 65% busy).  F16 with one M tile:
// about 3,200 cycles a tile, 2,835 of HBM; a ragged batch adds some 17,000 to
// 25,000 cycles an item for Q, the pipeline's ends and the output (64 trees
// over 200-4,000 positions: 262 us, 36% of the copy bandwidth, tensor pipe
// 49%).  int8 and F32 pools: the conversion warps, whose loads wait behind the
// MMAs' reads of shared memory (24 sequences int8: 205 us; F32: 31 of the small
// heads 91 us, 32 of 128 values 146 us).  Small calls: instruction fetch; code
// executed once costs about a nanosecond per three instructions, so loops here
// stay rolled unless registers force them open (unrolling everything was 181 KB
// and 3 times slower on the batch).  Register shares of 200/64/48 or 184/96/48 for softmax,
// loads and the rest were 2 to 10% slower than 192/72/56.
constexpr int kTreeThreads = 512;   // WG0, WG1 softmax; WG2 loads; warp 12 issues the MMAs, warp 13 deals
                                    // the pieces, warp 14 fetches the rows that WG2 converts (F32, int8)
constexpr int kTreeMmaWarp = 12;
constexpr int kTreePieceWarp = 13;
constexpr int kTreeRawWarp = 14;
constexpr int kTreeLoadWarp = 8;
constexpr unsigned kTreeNap = 2000;                       // ns a wait may sleep at a time
constexpr unsigned long long kTreeLimit = 4000000000ull;  // ns after which a wait gives up
constexpr int kTreeRows = 256;      // query vectors of a partial slot
constexpr int kTreeState = 3;       // and values beside O: m, l, m_v
constexpr int kPieceRing = 4;
constexpr int kMetaRing = 8;        // tiles of column masks and int8 scales kept

constexpr int kTreeMetaBytes = 1024;

template <int KV, int DP>
struct TreeForm {  // KV: 0 F32, 1 F16, 2 int8
    static constexpr bool kPairs = KV == 1;              // two M tiles per item
    static constexpr int kBn = KV == 0 ? 64 : 128;       // positions per tile
    static constexpr int kParts = KV == 0 ? 2 : 1;       // hi, lo planes of K and V
    static constexpr int kHalves = DP / 64;              // 128-byte wide column halves
    static constexpr int kQPart = kHalves * 128 * 128;   // bytes of one Q plane
    static constexpr int kQTile = 2 * kQPart;
    static constexpr int kSlotPart = kHalves * kBn * 128;
    static constexpr int kSlot = kParts * kSlotPart;     // one K or V tile
    // an item's own cost (Q, merge, output) in tiles, chosen on ragged batches
    // of each type before F32 and int8 weights had their present reference, which
    // cost 2 to 3% (64 trees F16 with 4, 6, 8, 11: 248, 244, 231, 233 us; F32
    // heads of 128 with 4, 7, 9: 32 sequences 152, 141, 139 us, 8 sequences 68,
    // 64, 75; F32 heads of 64 with 3, 4, 7: 31 sequences 88, 86, 93 us, 12
    // sequences 74, 77, 79; int8 with 5, 6, 7: 24 sequences 197, 195, 199 us,
    // 64 sequences 62, 66, 68, 16 sequences 63, 66, 63)
    static constexpr int kItemWeight = KV == 0 ? (DP == 64 ? 3 : 7) : KV == 1 ? 8 : 5;
    static constexpr int kElem = KV == 0 ? 4 : KV == 1 ? 2 : 1;
    static constexpr int kRaw = KV == 1 ? 0 : kBn * DP * kElem;  // one unconverted tile
    static constexpr int kRawPitch = DP * kElem < 128 ? DP * kElem : 128;  // its rows lie in parts of this many bytes,
    static constexpr int kRawParts = DP * kElem / kRawPitch;               // part after part
    static constexpr int kRawDepth = KV == 1 ? 0 : DP == 64 ? 4 : KV == 0 ? 2 : 3;
    static constexpr int kBase = KV == 1 ? (DP == 64 ? 6 : 3) : (DP == 64 ? 4 : 3);  // ring slots
    static constexpr int kExtra = kPairs ? 2 : 0;        // more of them in the second Q tile when it is not used
    static constexpr int kScaleRing = KV == 1 ? 0 : KV == 2 ? kMetaRing : 4;
    static constexpr int kOffSlots = kQTile * (kPairs ? 2 : 1);
    static constexpr int kOffRaw = kOffSlots + kBase * kSlot;
    static constexpr int kOffScale = kOffRaw + kRawDepth * kRaw;
    static constexpr int kOffMeta = kOffScale + kScaleRing * 2 * kBn * 4;
    static constexpr int kSmem = kOffMeta + kTreeMetaBytes;
    static_assert(kExtra * kSlot <= kQTile || !kPairs);
    static_assert(kSmem <= 232448);
};

// One piece of an item: tiles [t0, t1) of it run in this CTA.
struct TreePiece {
    int s, c0, n, len;
    int t0, t1, whole;            // whole: the item begins and ends here
    int head, row0, rows, split;  // split: vectors of the first M tile; rows 0 ends the list
    int pair;
    unsigned tile_base, count;    // tiles and pieces before this one

    // Entry e of the piece's 2 (t1 - t0) loads, in the order of their use:
    // K runs two tiles (one with two M tiles) ahead of V.
    __device__ __forceinline__ int entry(int e, bool& is_v) const {
        const int c = t1 - t0, ahead = min(pair ? 1 : 2, c);
        if (e < ahead) {
            is_v = false;
            return e;
        }
        const int f = e - ahead;
        if (f < 2 * (c - ahead)) {
            is_v = !(f & 1);
            return is_v ? f >> 1 : (f >> 1) + ahead;
        }
        is_v = true;
        return c - ahead + (f - 2 * (c - ahead));
    }
};

struct TreeMeta {  // at kOffMeta
    std::uint64_t full[8], empty[8];
    std::uint64_t v_ready[kMetaRing];  // a tile's V scales and vbad are in place
    std::uint64_t raw_full[4], raw_empty[4], piece_full[kPieceRing], piece_empty[kPieceRing];
    std::uint64_t s_full[2], p_full[2], o_full[2];
    std::uint64_t q_full, merge_ready, merge_read, drain;
    union {
        TreePiece piece[kPieceRing];
        long long warp_sum[16];  // while the run is cut out
    };
    alignas(16) unsigned valid[kMetaRing][4];   // columns of a tile that hold a row
    alignas(16) unsigned vspan[kMetaRing][4];   // per load warp: the largest V scale (upper half of its bits, rounded
                                                // up) and the smallest one (rounded down; rows that do not exist apart)
    union {
        unsigned vbad[kMetaRing][4];  // nodes whose V (kept out of the products: 0 * inf) is not finite
        struct {                      // while the run is cut out
            long long excl0, excl1;
            int seq0, seq1, bad;
        };
    };
    unsigned tmem;
    int abort_flag;
};
constexpr int kTreeBars = 50;
static_assert(kMetaRing == 8 && kPieceRing == 4 && offsetof(TreeMeta, drain) == (kTreeBars - 1) * 8);
static_assert(sizeof(TreeMeta) <= kTreeMetaBytes);

struct TreeRec {  // an item that continues in the next CTAs, by the CTA it starts in
    int c0, row0, rows, split, head, pieces;
    int streams;  // slot halves that hold parts of the same vectors (1: of different ones)
};

__device__ __forceinline__ unsigned sm_addr(const void* p) { return unsigned(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void bar_init(std::uint64_t* b, unsigned n) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(sm_addr(b)), "r"(n));
}
__device__ __forceinline__ void bar_arrive(std::uint64_t* b) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(sm_addr(b)) : "memory");
}
__device__ __forceinline__ bool bar_test(std::uint64_t* b, unsigned parity) {
    unsigned ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(sm_addr(b)), "r"(parity), "r"(kTreeNap)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ bool bar_done(std::uint64_t* b, unsigned parity) {  // without waiting
    unsigned ok;
    asm volatile(
        "{\n .reg .pred p;\n mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n selp.u32 %0, 1, 0, p;\n}\n"
        : "=r"(ok)
        : "r"(sm_addr(b)), "r"(parity)
        : "memory");
    return ok != 0;
}
__device__ __forceinline__ unsigned long long now_ns() {
    unsigned long long t;
    asm volatile("mov.u64 %0, %globaltimer;" : "=l"(t));
    return t;
}
// On the way out: copies in flight land within microseconds.
__device__ __forceinline__ void bar_land(std::uint64_t* b, unsigned parity) {
    const unsigned long long since = now_ns();
#pragma unroll 1
    while (!bar_test(b, parity) && now_ns() - since < 20000000ull) {
    }
}
// Bounded; false after the limit or when another role gave up.
__device__ __forceinline__ bool bar_wait(std::uint64_t* b, unsigned parity, volatile int* abort_flag, int* status) {
    if (bar_test(b, parity)) return true;
    const unsigned long long since = now_ns();
#pragma unroll 1
    while (!bar_test(b, parity)) {
        if (*abort_flag) return false;
        if (now_ns() - since > kTreeLimit) {
            *abort_flag = 1;
            atomicOr(status, kTreeTimeout);
            return false;
        }
    }
    return true;
}
__device__ __forceinline__ bool elect_one() {
    unsigned p;
    asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(p));
    return p != 0;
}
__device__ __forceinline__ void tree_commit_to(std::uint64_t* b) {
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(sm_addr(b))
                 : "memory");
}
__device__ __forceinline__ void mma_ss(unsigned d, std::uint64_t a, std::uint64_t b, unsigned idesc, int acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n}\n" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(acc));
}
__device__ __forceinline__ void mma_ts(unsigned d, unsigned a, std::uint64_t b, unsigned idesc, int acc) {
    asm volatile(
        "{\n .reg .pred p;\n setp.ne.b32 p, %4, 0;\n tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n}\n" ::"r"(d),
        "r"(a), "l"(b), "r"(idesc), "r"(acc));
}
// 128-byte swizzled operand: 8-row atoms of 1024 bytes (SBO); lbo is the
// distance of 64-column halves for an operand with the MMA's N contiguous.
__device__ __forceinline__ std::uint64_t sw128_desc(unsigned addr, unsigned lbo) {
    return ((addr >> 4) & 0x3FFFull) | (std::uint64_t((lbo >> 4) & 0x3FFF) << 16) | (64ull << 32) | (1ull << 46) |
           (2ull << 61);
}
__device__ __forceinline__ void tm_ld32(unsigned addr, unsigned (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
        "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]),
          "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]),
          "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tm_ld16(unsigned addr, unsigned (&r)[16]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(addr));
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tm_st16(unsigned addr, const unsigned (&r)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(
            addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
        : "memory");
}
__device__ __forceinline__ void tm_st32(unsigned addr, const unsigned (&r)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(addr),
        "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]),
        "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]),
        "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
        "r"(r[30]), "r"(r[31])
        : "memory");
}
__device__ __forceinline__ void tm_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tm_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tm_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void proxy_fence() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
__device__ __forceinline__ void cp16(unsigned dst, const void* src, unsigned bytes) {  // bytes 16, or 0: zero fill
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp4(unsigned dst, const void* src, unsigned bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void bulk_load(unsigned dst, const void* src, unsigned bytes, unsigned bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst), "l"(src),
                 "r"(bytes), "r"(bar)
                 : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float max3(float x, float y, float z) {
    float r;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(x), "f"(y), "f"(z));
    return r;
}
__device__ __forceinline__ float two_to(int e) { return __uint_as_float(unsigned(127 + e) << 23); }  // -126 <= e <= 127
// The power of two that brings a largest |value| into [2^14, 2^15).
__device__ __forceinline__ int lift(float top) {
    const int e = int((__float_as_uint(top) >> 23) & 255) - 127;
    return top > 0.f && e < 128 ? max(-113, min(112, 14 - e)) : 0;
}
// Packed pairs of F32.
using f32x2 = unsigned long long;
__device__ __forceinline__ f32x2 pair_of(float x, float y) {
    f32x2 r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
    return r;
}
__device__ __forceinline__ void halves_of(f32x2 r, float& x, float& y) { asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(r)); }
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
__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
    f32x2 r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}
__device__ __forceinline__ void mul2_in(unsigned& x, unsigned& y, f32x2 f) {
    float u, v;
    halves_of(mul2(pair_of(__uint_as_float(x), __uint_as_float(y)), f), u, v);
    x = __float_as_uint(u);
    y = __float_as_uint(v);
}
// A pair of values below 2^16 as hi + lo, F16 each: hi is the value rounded to
// 11 bits and lo what is left, so hi + lo carries 2^-23 of each value (not of
// the largest: small softmax weights, and the other channels of a K or V row
// with a large one, keep their digits), down to 2^-25 absolute.  (A split in
// packed additions alone, lo in steps of the row's largest, is no faster: F32
// heads of 64 89.8 and 89.6 us, of 128 140.8 and 142.3.)
__device__ __forceinline__ void split_pair(float x, float y, unsigned& hi, unsigned& lo) {
    const __half2 h = __floats2half2_rn(x, y);
    const float2 f = __half22float2(h);
    const __half2 l = __floats2half2_rn(x - f.x, y - f.y);
    hi = *reinterpret_cast<const unsigned*>(&h);
    lo = *reinterpret_cast<const unsigned*>(&l);
}
__device__ __forceinline__ void split_packed(f32x2 p, unsigned& hi, unsigned& lo) {
    float x, y;
    halves_of(p, x, y);
    split_pair(x, y, hi, lo);
}

// Quotients of non-negative numbers, mostly below 2^32.
__device__ __forceinline__ long long quotient(long long x, long long y) {
    return (x | y) >> 32 ? x / y : (long long)(unsigned(x) / unsigned(y));
}

// What every role knows of a sequence, and its tiles in the global order
// (KV heads outermost, then groups of query vectors, then tiles).
struct TreeSeq {
    int s, c0, n, len, groups, weight;
    long long tiles;   // per item
    long long total;   // hkv * groups * tiles
    bool pair;
};
template <class F>
__device__ __forceinline__ bool tree_seq(const TreeAttn& a, int s, TreeSeq& q) {
    q.s = s;
    const bool ok = tree_sequence_ok(a, s, q.c0, q.n, q.len);
    if (!ok || q.n == 0) {
        q.total = 0;
        return ok && !(s == 0 && q.c0 != 0);
    }
    const int vectors = q.n * a.group;
    const int most = F::kPairs ? 256 : 128;
    q.groups = unsigned(vectors + most - 1) / most;
    q.pair = F::kPairs && vectors > 128;
    q.weight = q.pair ? 2 : 1;
    q.tiles = (unsigned(q.len) + unsigned(q.n) + F::kBn - 1) / F::kBn;
    q.total = q.tiles * q.groups * a.hkv;
    return !(s == 0 && q.c0 != 0);
}

// Bits [j0, j0 + 32) of the mask row of node `node` (negative j0: cached
// positions, visible), columns behind the last node cleared.
__device__ __forceinline__ unsigned node_bits(const TreeAttn& a, int c0, int n, int node, long long j0) {
    if (j0 >= n) return 0;
    if (j0 + 32 <= 0) return 0xffffffffu;
    const int j = int(j0);
    const int from = max(j, 0), shift = from & 31;  // bits [from, from + 32) of the nodes, moved up by from - j
    unsigned w;
    if (a.ancestors) {
        const unsigned* row = reinterpret_cast<const unsigned*>(a.ancestors + (long long)(c0 + node) * a.words);
        const int i = from >> 5;
        w = row[i] >> shift;
        if (shift && i + 1 < 2 * a.words) w |= row[i + 1] << (32 - shift);
    } else {
        const int left = node + 1 - from;  // a chain sees nodes up to its own
        w = left <= 0 ? 0u : left >= 32 ? 0xffffffffu : (1u << left) - 1;
    }
    const int have = n - from;
    if (have < 32) w &= (1u << have) - 1;
    if (j < 0) w = (w << -j) | ((1u << -j) - 1);
    return w;
}

template <int KV, int DP>
__global__ void __launch_bounds__(kTreeThreads, 1) tree_mma_kernel(const __grid_constant__ CUtensorMap kv_map,
                                                                   const __grid_constant__ TreeAttn a, float* partial,
                                                                   TreeRec* recs, int min_weight) {
    using F = TreeForm<KV, DP>;
    extern __shared__ __align__(1024) unsigned char tree_smem[];
    TreeMeta& M = *reinterpret_cast<TreeMeta*>(tree_smem + F::kOffMeta);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int group = a.group;

    if (tid < kTreeBars) {  // TreeMeta begins with its barriers
        const int i = tid;
        bar_init(&M.full[0] + i, i < 8    ? 4                   // full: load warps
                                 : i < 16 ? 1                   // empty: MMA commits
                                 : i < 24 ? 4                   // v_ready: load warps
                                 : i < 32 ? (i & 4 ? 4 : 33)          // raw_full: the row fetch warp and its copies; raw_empty
                                 : i < 40 ? (i & 4 ? (KV == 1 ? 13 : 14) : 1)  // piece_full, piece_empty: 8 softmax
                                                                               // warps, 4 load warps, MMA, row fetch
                                 : i < 42 ? 1                   // s_full
                                 : i < 44 ? 4                   // p_full
                                 : i < 46 ? 1                   // o_full
                                 : i < 47 ? 8                   // q_full
                                 : i < 49 ? 4                   // merge_ready, merge_read
                                          : 1);                 // drain
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (tid == 64) {
        M.abort_flag = 0;
        M.bad = 0;
        M.seq0 = M.seq1 = a.n_seq;
        M.excl0 = M.excl1 = 0;
    }
    __syncthreads();
    // The run of tiles: weights are scanned in sequence order by every CTA
    // (twice if they are more than the threads: for the sum, then for the cuts).
    const int cta = blockIdx.x;
    long long total = 0, w0 = 0, w1 = 0;
    int ctas = 1;
    const bool once = a.n_seq <= kTreeThreads;
#pragma unroll 1
    for (int pass = once ? 1 : 0; pass < 2; ++pass) {
        long long carry = 0;
#pragma unroll 1
        for (int base = 0; base < a.n_seq; base += kTreeThreads) {
            TreeSeq q;
            q.total = 0;
            if (base + tid < a.n_seq && !tree_seq<F>(a, base + tid, q)) M.bad = 1;
            const long long w = q.total ? q.total * q.weight + (long long)q.groups * a.hkv * F::kItemWeight : 0;
            long long scan = w;
#pragma unroll 1
            for (int d = 1; d < 32; d <<= 1) {
                const long long up = __shfl_up_sync(0xffffffffu, scan, d);
                if (lane >= d) scan += up;
            }
            if (lane == 31) M.warp_sum[warp] = scan;
            __syncthreads();
            long long before = carry, all = 0;
#pragma unroll 4
            for (int i = 0; i < kTreeThreads / 32; ++i) {
                const long long x = M.warp_sum[i];
                before += i < warp ? x : 0;
                all += x;
            }
            carry += all;
            if (once) total = carry;
            if (pass) {
                if (once || base == 0) {
                    ctas = int(max(1ll, min((long long)gridDim.x, quotient(total, min_weight))));
                    w0 = quotient(total * cta, ctas);
                    w1 = quotient(total * (cta + 1), ctas);
                }
                const long long excl = before + scan - w;
                if (w && excl <= w0 && w0 < excl + w) {
                    M.seq0 = base + tid;
                    M.excl0 = excl;
                }
                if (w && excl < w1 && w1 <= excl + w) {
                    M.seq1 = base + tid;
                    M.excl1 = excl;
                }
            }
            __syncthreads();
        }
        total = carry;
    }
    if (cta == 0 && tid == 0 && M.bad) atomicOr(a.status, kTreeBadLengths);
    if (tid == 0) recs[cta].pieces = 0;
    if (cta >= ctas || total == 0) return;
    if (warp == kTreeMmaWarp) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(sm_addr(&M.tmem)), "r"(512));
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
    }
    tm_before();
    __syncthreads();
    tm_after();
    const unsigned tmem = M.tmem;
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    volatile int* abort_flag = &M.abort_flag;
    if (warp >= kTreeMmaWarp) asm volatile("setmaxnreg.dec.sync.aligned.u32 56;");
    if (warp == kTreePieceWarp) {
        // --------------------------------------------------------- pieces
        if (lane == 0) {
            const int seq1 = M.seq1, seq0 = M.seq0;  // read before the first piece: their place is used again
            const long long excl1 = M.excl1, excl0 = M.excl0;
            TreeSeq q;
            tree_seq<F>(a, seq1, q);
            // Item i of a sequence takes the weights from i (tiles weight + kItemWeight)
            // on, its tile t starts at t weight of them; a tile belongs to the
            // CTA whose run holds its start.
            const auto tile_at = [&](long long w) {
                const long long each = q.tiles * q.weight + F::kItemWeight, i = quotient(w, each), left = w - i * each;
                return i * q.tiles + min(q.tiles, q.weight == 2 ? (left + 1) >> 1 : left);
            };
            const long long u1 = min(q.total, tile_at(w1 - excl1));
            tree_seq<F>(a, seq0, q);
            long long u = tile_at(w0 - excl0);
            unsigned count = 0, tile_base = 0;
            bool go = true;
#pragma unroll 1
            for (int seq = seq0; go; ++count) {
                long long end = seq == seq1 ? u1 : q.total;
#pragma unroll 1
                while (u >= end && seq < seq1) {
                    u = 0;
                    tree_seq<F>(a, ++seq, q);
                    end = seq == seq1 ? u1 : q.total;
                }
                const int ring = count % kPieceRing;
                go = bar_wait(&M.piece_empty[ring], (count / kPieceRing & 1) ^ 1, abort_flag, a.status);
                if (!go) break;
                TreePiece& p = M.piece[ring];
                if (u >= end) {
                    p.rows = 0;
                    bar_arrive(&M.piece_full[ring]);
                    break;
                }
                const long long item = quotient(u, q.tiles);
                const int t0 = int(u - item * q.tiles), t1 = int(min(q.tiles, t0 + (end - u)));
                u += t1 - t0;
                const int head = int(unsigned(item) / unsigned(q.groups)), grp = int(item - (long long)head * q.groups);
                // groups of nearly equal size, and M tiles of nearly equal size
                const int vectors = q.n * group, per = unsigned(vectors + q.groups - 1) / unsigned(q.groups);
                const int row0 = grp * per, rows = min(per, vectors - row0);
                p.s = seq;
                p.c0 = q.c0;
                p.n = q.n;
                p.len = q.len;
                p.t0 = t0;
                p.t1 = t1;
                p.whole = t0 == 0 && t1 == q.tiles;
                p.head = head;
                p.row0 = row0;
                p.rows = rows;
                p.split = q.pair ? (rows + 1) / 2 : rows;
                p.pair = q.pair;
                p.tile_base = tile_base;
                p.count = count;
                bar_arrive(&M.piece_full[ring]);
                tile_base += unsigned(t1 - t0);
                if (t0 == 0 && t1 < q.tiles) {  // continues in other CTAs: up to the one its last tile starts in
                    const long long last = excl1 + item * (q.tiles * q.weight + F::kItemWeight) + (q.tiles - 1) * q.weight;
                    TreeRec rec;
                    rec.c0 = q.c0;
                    rec.row0 = row0;
                    rec.rows = rows;
                    rec.split = p.split;
                    rec.head = head;
                    rec.pieces = int(quotient((last + 1) * ctas + total - 1, total) - 1) - cta + 1;
                    rec.streams = q.pair ? 1 : 2;
                    recs[cta] = rec;
                }
            }
        }
        __syncwarp();
    }
    const unsigned smem = sm_addr(tree_smem);
    const auto slot_at = [&](int slot) -> unsigned {
        return slot < F::kBase ? F::kOffSlots + slot * F::kSlot : F::kQTile + (slot - F::kBase) * F::kSlot;
    };

    // Piece i of the run is in M.piece[i % kPieceRing] until every role has released it; rows 0 ends the run.
    const auto get_piece = [&](unsigned i) -> bool {
        return bar_wait(&M.piece_full[i % kPieceRing], (i / kPieceRing) & 1, abort_flag, a.status) &&
               M.piece[i % kPieceRing].rows != 0;
    };
    const auto release_piece = [&](unsigned i) { bar_arrive(&M.piece_empty[i % kPieceRing]); };

    const int row_bytes = a.dim * F::kElem, chunks = row_bytes >> 4;
    const unsigned char* pool = static_cast<const unsigned char*>(a.kv);
    // Index p of a piece's sequence (cached positions, then nodes): its K row in the pool (-1: none).
    const auto row_of = [&](const TreePiece& w, int p, int& flags) -> long long {
        if (p >= w.len + w.n) return -1;
        const long long at = tree_row(a, w.s, w.c0, w.len, p, flags);
        return at < 0 ? -1 : at + (long long)w.head * a.bt;
    };

    if (warp < kTreeLoadWarp) {
        // ------------------------------------------------ softmax warpgroups
        asm volatile("setmaxnreg.inc.sync.aligned.u32 192;");
        const int stream = warp >> 2, wq = warp & 3, r = tid & 127;
        const unsigned lane_base = tmem + (unsigned(wq * 32) << 16);
        const unsigned s_at = lane_base + stream * 128, o_at = lane_base + 256 + stream * 128;
        const float score_unit = 1.4426950408889634f / sqrtf(float(a.dim));
        unsigned n_s = 0;  // tiles of this stream so far
        bool go = true;
        float o[DP];
        for (unsigned piece = 0;; ++piece) {
            go = __all_sync(0xffffffffu, get_piece(piece));
            if (!go) break;
            const TreePiece& q = M.piece[piece % kPieceRing];
            const int tile_rows = q.pair ? (stream ? q.rows - q.split : q.split) : q.rows;
            const int first_row = q.row0 + (q.pair && stream ? q.split : 0);  // this stream's rows within the sequence
            const int node = unsigned(first_row + r) / unsigned(group);
            const int first_node = unsigned(first_row + wq * 32) / unsigned(group);  // of the warp's vectors
            const int first_g = first_row + wq * 32 - first_node * group;
            const bool live = r < tile_rows, warp_live = wq * 32 < tile_rows;
            // The warp's query vectors, scaled below 2^15 and split, into this
            // stream's Q tile; lane i keeps the score factor of vector i.
            float c = 0.f;
            if (warp_live) {
                // raw rows first, all in flight, each in the 512 (256) bytes its two halves will take
                const int quads = a.dim >> 2, most = min(32, tile_rows - wq * 32);
                const bool writes = stream == 0 || q.pair;
                unsigned char* tile = tree_smem + (q.pair && stream ? F::kQTile : 0) + wq * 4096;
                int g = first_g;
                const float* src = a.q + (long long)(q.c0 + first_node) * a.ldq + (long long)(q.head * group + g) * a.dim + lane * 4;
                const long long turn = a.ldq - (long long)(group - 1) * a.dim;  // to the next node's first head
                if (writes) {
                    const unsigned to = sm_addr(tile) + (lane >> 3) * 16384;
#pragma unroll 1
                    for (int i = 0; i < most; ++i) {
                        if (lane < DP / 4)
                            cp16(to + i * 128 + (((lane & 7) ^ (i & 7)) << 4), lane < quads ? src : a.q, lane < quads ? 16u : 0u);
                        const bool last = g + 1 == group;
                        src += last ? turn : a.dim;
                        g = last ? 0 : g + 1;
                    }
                    cp_commit();
                    cp_wait<0>();
                    __syncwarp();
                    // then lane i takes row i (the accumulators' registers are free yet)
                    unsigned char* mine = tile + lane * 128;
                    float tops[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int i = 0; i < DP / 4; ++i) {
                        const float4 x = *reinterpret_cast<const float4*>(mine + (i >> 3) * 16384 + (((i & 7) ^ (lane & 7)) << 4));
                        o[4 * i] = x.x;
                        o[4 * i + 1] = x.y;
                        o[4 * i + 2] = x.z;
                        o[4 * i + 3] = x.w;
                        tops[i & 3] = max3(tops[i & 3], fmaxf(fabsf(x.x), fabsf(x.y)), fmaxf(fabsf(x.z), fabsf(x.w)));
                    }
                    const int up = lift(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])));
                    // (K scales of F32 rows are 2^14 lower: their product with S must not overflow)
                    c = live ? score_unit * two_to((KV == 0 ? 14 : 0) - up) : 0.f;
                    const float f = two_to(up);
#pragma unroll
                    for (int i = 0; i < DP / 8; ++i) {
                        uint4 hi, lo;
                        split_pair(o[8 * i] * f, o[8 * i + 1] * f, hi.x, lo.x);
                        split_pair(o[8 * i + 2] * f, o[8 * i + 3] * f, hi.y, lo.y);
                        split_pair(o[8 * i + 4] * f, o[8 * i + 5] * f, hi.z, lo.z);
                        split_pair(o[8 * i + 6] * f, o[8 * i + 7] * f, hi.w, lo.w);
                        unsigned char* at = mine + (i >> 3) * 16384 + (((i & 7) ^ (lane & 7)) << 4);
                        *reinterpret_cast<uint4*>(at) = hi;
                        *reinterpret_cast<uint4*>(at + F::kQPart) = lo;
                    }
                    if (!q.pair) {
                        // For the other stream, in its accumulator's place: free once that
                        // stream is done with the piece before (which is known already,
                        // unless that one had two M tiles).
                        if (piece) {
                            go = __all_sync(0xffffffffu, bar_wait(&M.merge_ready, (piece - 1) & 1, abort_flag, a.status));
                            if (!go) break;
                            tm_after();
                        }
                        asm volatile("tcgen05.st.sync.aligned.32x32b.x1.b32 [%0], {%1};" ::"r"(lane_base + 384),
                                     "r"(__float_as_uint(c))
                                     : "memory");
                        tm_wait_st();
                        tm_before();
                    }
                }
            }
            proxy_fence();
            __syncwarp();
            if (lane == 0) bar_arrive(&M.q_full);
            if (!q.pair && stream) {
                go = __all_sync(0xffffffffu, bar_wait(&M.q_full, piece & 1, abort_flag, a.status));
                if (!go) break;
                if (warp_live) {
                    unsigned x;
                    tm_after();
                    asm volatile("tcgen05.ld.sync.aligned.32x32b.x1.b32 {%0}, [%1];" : "=r"(x) : "r"(lane_base + 384));
                    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
                    c = __uint_as_float(x);
                }
            }
            float m = -INFINITY, l = 0.f;
            float m_v = 0.f;  // l is in units of 2^m, O of 2^(m + m_v)
#pragma unroll
            for (int i = 0; i < DP; ++i) o[i] = 0.f;
            const int tiles = q.t1 - q.t0;
            for (int j = q.pair ? 0 : stream; j < tiles && go; j += q.pair ? 1 : 2, ++n_s) {
                const unsigned t = q.tile_base + j;
                go = bar_wait(&M.s_full[stream], n_s & 1, abort_flag, a.status);
                go = __all_sync(0xffffffffu, go);
                if (!go) break;
                tm_after();
                float keep = 1.f;
                if (warp_live) {
                    const int ring = t % kMetaRing;
                    const long long p0 = (long long)(q.t0 + j) * F::kBn;
                    const bool nodes = p0 + F::kBn > q.len;
                    bool all = !nodes;
#pragma unroll
                    for (int k = 0; k < F::kBn / 32; ++k) all &= M.valid[ring][k] == 0xffffffffu;
                    unsigned seen[F::kBn / 32] = {};  // columns 32 k .. that this vector sees, when not all
                    const auto see_of = [&](int k) -> unsigned {
                        unsigned w = seen[0];
#pragma unroll
                        for (int i = 1; i < F::kBn / 32; ++i) w = k == i ? seen[i] : w;
                        return w;
                    };
                    const float* k_scale = reinterpret_cast<const float*>(tree_smem + F::kOffScale) +
                                           t % (F::kScaleRing ? F::kScaleRing : 1) * 2 * F::kBn;
                    const float* v_scale = k_scale + F::kBn;
                    float tops[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll 1
                    for (int k = 0; k < F::kBn / 32; ++k) {
                        unsigned x[32];
                        tm_ld32(s_at + 32 * k, x);
                        if constexpr (KV != 1) {
#pragma unroll
                            for (int i = 0; i < 32; i += 4) {
                                const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(k_scale + 32 * k + i);
                                mul2_in(x[i], x[i + 1], f.x);
                                mul2_in(x[i + 2], x[i + 3], f.y);
                            }
                        }
                        if (!all) {
                            unsigned see = M.valid[ring][k];
                            if (nodes) see &= node_bits(a, q.c0, q.n, live ? node : 0, p0 + 32 * k - q.len);
#pragma unroll
                            for (int i = 0; i < F::kBn / 32; ++i) seen[i] = k == i ? see : seen[i];
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (!(see >> i & 1)) x[i] = 0xff800000u;
                        }
                        if constexpr (KV != 1) tm_st32(s_at + 32 * k, x);
#pragma unroll
                        for (int i = 0; i < 32; i += 2)
                            tops[(i >> 1) & 3] = max3(tops[(i >> 1) & 3], __uint_as_float(x[i]), __uint_as_float(x[i + 1]));
                    }
                    const float top = fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3]));
                    if (KV != 1 || nodes) {  // scales of V, nodes with a non-finite V
                        go = __all_sync(0xffffffffu, bar_wait(&M.v_ready[t % kMetaRing], (t / kMetaRing) & 1, abort_flag, a.status));
                        if (!go) break;
                        if (nodes) {
#pragma unroll
                            for (int k = 0; k < F::kBn / 32; ++k)
                                if (seen[k] & M.vbad[ring][k]) l = NAN;  // the row's result is not finite
                        }
                    }
                    // The reference of the weights.  F16: the largest score so far.
                    // With V scales it has a second part, so that weight times
                    // scale stays below 2^11 and a row keeps the digits of what
                    // it sees, whatever the V of others are: the largest score -
                    // m + log2(V scale).  Where a tile's scales lie within 2^6 of
                    // one another its largest score and its largest scale together
                    // stand for that; elsewhere (a masked node's or a single
                    // position's V far above the rest, a row of zeros with all the
                    // weight) every column is looked at.  The weights themselves
                    // stay below 2^119, so that a tile's sum does not overflow; l
                    // has the first part alone as its reference.  Both are whole,
                    // so that a change of reference costs no digit.
                    const float score = top * c;
                    const float mn = fmaxf(m, KV == 1 ? score : ceilf(score));
                    const bool none = mn == -INFINITY;
                    // Beyond 2^22 the reference is so coarse that the exact product
                    // less it could reach past F16's range: scores rounded to F32,
                    // less their maximum, go back into S.
                    const bool far = fabsf(mn) >= 4194304.f && !none;
                    bool look = far;
                    float mv = -108.f, big = 0.f;
                    if constexpr (KV != 1) {
                        const uint4 span = *reinterpret_cast<const uint4*>(M.vspan[ring]);
                        big = __uint_as_float(max(max(span.x, span.y), max(span.z, span.w)) & 0xffff0000u);
                        const float low = __uint_as_float(
                            min(min(span.x & 0xffffu, span.y & 0xffffu), min(span.z & 0xffffu, span.w & 0xffffu)) << 16);
                        look |= big > 64.f * low;
                        mv = fmaxf(mv, __log2f(big));
                        tm_wait_st();
                    }
                    if (__any_sync(0xffffffffu, look)) {
                        const float back = 1.f / c;
                        mv = -108.f;
                        float most = -INFINITY;
#pragma unroll 1
                        for (int k = 0; k < F::kBn / 16; ++k) {
                            unsigned x[16];
                            tm_ld16(s_at + 16 * k, x);
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const float y = __fsub_rn(__fmul_rn(__uint_as_float(x[i]), c), mn);
                                if constexpr (KV != 1) most = fmaxf(most, y + __log2f(fabsf(v_scale[16 * k + i])));
                                if (far) x[i] = __float_as_uint(y * back);
                            }
                            tm_st16(s_at + 16 * k, x);
                        }
                        mv = fmaxf(mv, most - (score - mn));
                        tm_wait_st();
                    }
                    float off = none ? 11.f : far ? 11.f : 11.f - mn;
                    keep = none ? 1.f : ex2(m - mn);
                    if constexpr (KV != 1) {
                        if (!none) {
                            mv = fmaxf(m_v + (m - mn), ceilf(mv + (score - mn)));
                            off -= mv;
                            l *= keep;
                            keep = ex2((m - mn) + (m_v - mv));
                            m_v = mv;
                        }
                    } else {
                        l *= keep;
                    }
                    m = mn;
                    // P over S, sixteen positions (one K step of the MMA) at a
                    // time: hi in their first eight columns, lo in the others.
                    f32x2 sums[2] = {0, 0};
                    const f32x2 c2 = pair_of(c, c), off2 = pair_of(off, off);
#pragma unroll 1
                    for (int k = 0; k < F::kBn / 32; ++k) {
                        unsigned x[32];
                        tm_ld32(s_at + 32 * k, x);
                        if (KV == 1 && !all) {
                            const unsigned see = see_of(k);
#pragma unroll
                            for (int i = 0; i < 32; ++i)
                                if (!(see >> i & 1)) x[i] = 0xff800000u;  // weight 0
                        }
#pragma unroll
                        for (int g = 0; g < 2; ++g) {
                            unsigned y[16];
#pragma unroll
                            for (int i = 0; i < 8; i += 2) {
                                const int at = 16 * g + 2 * i;
                                float p0, p1, p2, p3;
                                halves_of(fma2(pair_of(__uint_as_float(x[at]), __uint_as_float(x[at + 1])), c2, off2), p0, p1);
                                halves_of(fma2(pair_of(__uint_as_float(x[at + 2]), __uint_as_float(x[at + 3])), c2, off2), p2, p3);
                                f32x2 p = pair_of(ex2(p0), ex2(p1)), r2 = pair_of(ex2(p2), ex2(p3));
                                sums[0] = add2(sums[0], p);
                                sums[1] = add2(sums[1], r2);
                                if constexpr (KV != 1) {
                                    const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(v_scale + 32 * k + at);
                                    p = mul2(p, f.x);
                                    r2 = mul2(r2, f.y);
                                }
                                split_packed(p, y[i], y[8 + i]);
                                split_packed(r2, y[i + 1], y[9 + i]);
                            }
                            tm_st16(s_at + 32 * k + 16 * g, y);
                        }
                    }
                    float sum0, sum1;
                    halves_of(add2(sums[0], sums[1]), sum0, sum1);
                    l += KV == 1 ? sum0 + sum1 : (sum0 + sum1) * ex2(m_v);
                    tm_wait_st();
                }
                tm_before();
                __syncwarp();
                if (lane == 0) bar_arrive(&M.p_full[stream]);
                go = __all_sync(0xffffffffu, bar_wait(&M.o_full[stream], n_s & 1, abort_flag, a.status));
                if (!go) break;
                tm_after();
                if (warp_live) {
                    const f32x2 keep2 = pair_of(keep, keep);
#pragma unroll
                    for (int k = 0; k < DP / 32; ++k) {
                        unsigned x[32];
                        tm_ld32(o_at + 32 * k, x);
#pragma unroll
                        for (int i = 0; i < 32; i += 2)
                            halves_of(fma2(pair_of(o[32 * k + i], o[32 * k + i + 1]), keep2,
                                           pair_of(__uint_as_float(x[i]), __uint_as_float(x[i + 1]))),
                                      o[32 * k + i], o[32 * k + i + 1]);
                    }
                }
            }
            if (!go) break;
            // The part of an item that other CTAs continue: (O, m, l, m_v) of each
            // stream into the workspace, one thread a row, rows side by side.
            // The CTA's slot 1 holds an item that begins here, slot 0 one that
            // began earlier; stream 1 uses the upper half of a slot.
            if (!q.whole && live) {
                float* slot = partial + (long long)(2 * cta + (q.t0 == 0)) * kTreeRows * (DP + kTreeState);
                const int pr = stream * 128 + r;
#pragma unroll
                for (int i = 0; i < DP / 4; ++i)
                    *reinterpret_cast<float4*>(slot + (i * kTreeRows + pr) * 4) =
                        make_float4(o[4 * i], o[4 * i + 1], o[4 * i + 2], o[4 * i + 3]);
                slot[kTreeRows * DP + pr] = m;
                slot[kTreeRows * DP + kTreeRows + pr] = l;
                if constexpr (KV != 1) slot[kTreeRows * DP + 2 * kTreeRows + pr] = m_v;
            }
            if (!q.pair) {
                // A whole item: the odd tiles' (O, m, l) through stream 1's tensor
                // memory.  Either way each stream learns that the other is done
                // with the shared Q tile.
                const bool merge = q.whole && warp_live && tiles > 1;
                const unsigned b_o = lane_base + 256 + 128, b_ml = lane_base + 128;
                if (stream) {
                    if (merge) {
#pragma unroll
                        for (int k = 0; k < DP / 16; ++k) {
                            unsigned x[16];
#pragma unroll
                            for (int i = 0; i < 16; ++i) x[i] = __float_as_uint(o[16 * k + i]);
                            tm_st16(b_o + 16 * k, x);
                        }
                        unsigned x[16] = {__float_as_uint(m), __float_as_uint(l), __float_as_uint(m_v)};
                        tm_st16(b_ml, x);
                        tm_wait_st();
                    }
                    tm_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&M.merge_ready);
                    go = __all_sync(0xffffffffu, bar_wait(&M.merge_read, q.count & 1, abort_flag, a.status));
                    tm_after();
                } else {
                    go = __all_sync(0xffffffffu, bar_wait(&M.merge_ready, q.count & 1, abort_flag, a.status));
                    tm_after();
                    if (go && merge) {
                        unsigned ml[16];
                        tm_ld16(b_ml, ml);
                        const float m2 = __uint_as_float(ml[0]), l2 = __uint_as_float(ml[1]);
                        const float mn = fmaxf(m, m2);
                        float ka = mn == -INFINITY ? 0.f : ex2(m - mn), kb = mn == -INFINITY ? 0.f : ex2(m2 - mn);
                        l = l * ka + l2 * kb;
                        if (KV != 1 && mn != -INFINITY) {
                            const float va = (m - mn) + m_v, vb = (m2 - mn) + __uint_as_float(ml[2]);
                            m_v = fmaxf(va, vb);
                            ka = ex2(va - m_v);
                            kb = ex2(vb - m_v);
                        }
                        m = mn;
                        const f32x2 ka2 = pair_of(ka, ka), kb2 = pair_of(kb, kb);
#pragma unroll
                        for (int k = 0; k < DP / 32; ++k) {
                            unsigned x[32];
                            tm_ld32(b_o + 32 * k, x);
#pragma unroll
                            for (int i = 0; i < 32; i += 2)
                                halves_of(fma2(pair_of(o[32 * k + i], o[32 * k + i + 1]), ka2,
                                               mul2(pair_of(__uint_as_float(x[i]), __uint_as_float(x[i + 1])), kb2)),
                                          o[32 * k + i], o[32 * k + i + 1]);
                        }
                    }
                    tm_before();
                    __syncwarp();
                    if (lane == 0) bar_arrive(&M.merge_read);
                }
            } else {  // both barriers count every piece
                tm_before();
                __syncwarp();
                if (lane == 0) bar_arrive(stream ? &M.merge_ready : &M.merge_read);
            }
            if (!go) break;
            if (q.whole && warp_live && (q.pair || stream == 0)) {
                // Rows through the Q tile, whose MMAs are done (the places of this
                // warp's own vectors), so that each is written by a whole warp.
                unsigned char* tile = tree_smem + (q.pair && stream ? F::kQTile : 0) + wq * 4096;
                const auto stage = [&](int row, int ch) {
                    return reinterpret_cast<float4*>(tile + (ch >> 3) * 16384 + row * 128 + (((ch & 7) ^ (row & 7)) << 4));
                };
                const float f = m == -INFINITY && l == 0.f ? 0.f : KV == 1 ? 1.f / l : ex2(m_v) / l;
#pragma unroll
                for (int i = 0; i < DP / 4; ++i)  // lane is the row
                    *stage(lane, i) = make_float4(o[4 * i] * f, o[4 * i + 1] * f, o[4 * i + 2] * f, o[4 * i + 3] * f);
                __syncwarp();
                const int most = min(32, tile_rows - wq * 32), width = a.dim >> 2;
                int g = first_g;
                float* dst = a.out + (long long)(q.c0 + first_node) * a.ldo + (long long)(q.head * group + g) * a.dim + lane * 4;
                const long long turn = a.ldo - (long long)(group - 1) * a.dim;
#pragma unroll 4
                for (int i = 0; i < most; ++i) {
                    if (lane < width) *reinterpret_cast<float4*>(dst) = *stage(i, lane);
                    const bool last = g + 1 == group;
                    dst += last ? turn : a.dim;
                    g = last ? 0 : g + 1;
                }
            }
            proxy_fence();  // the Q tile's next readers and writers
            __syncwarp();
            if (lane == 0) release_piece(piece);
        }
    } else if (warp < kTreeMmaWarp) {
        // ------------------------------------------------------------ loads
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        const int lw = warp - kTreeLoadWarp;

        unsigned empty_phase = 0xffffffffu;
        int slot = 0, flags = 0;
        if constexpr (KV == 1) {
            bool go = true;
            // The extra slots lie in the second Q tile, which a piece with two M
            // tiles uses until its last output row has been staged there.  `tail` is
            // the latest such piece that this warp has not seen released yet: it
            // stays set over any number of pieces that fit the other slots.
            constexpr unsigned kNoPiece = 0xffffffffu;
            unsigned tail = kNoPiece;
            int pend[2], n_pend = 0;
            const auto signal = [&](int s) {
                proxy_fence();
                __syncwarp();
                if (lane == 0) bar_arrive(&M.full[s]);
            };
            const auto drain = [&]() {
                cp_wait<0>();
                for (int i = 0; i < n_pend; ++i) signal(pend[i]);
                n_pend = 0;
            };
            for (unsigned piece = 0; go; ++piece) {
                if (!__all_sync(0xffffffffu, get_piece(piece))) break;
                const TreePiece& walk = M.piece[piece % kPieceRing];
                const bool pair = walk.pair;
                const int ns = pair ? F::kBase : F::kBase + F::kExtra;
                if (slot >= ns) slot = 0;
                const int loads = 2 * (walk.t1 - walk.t0);
                long long row_cur = -1, row_prev = -1;
                int k_last = -1;
                for (int e = 0; e < loads && go; ++e) {
                    bool is_v;
                    const int j = walk.entry(e, is_v);
                    if (!is_v) {
                        row_prev = row_cur;
                        row_cur = row_of(walk, (walk.t0 + j) * F::kBn + lw * 32 + lane, flags);
                        k_last = j;
                    }
                    // V of a tile uses the row that K left behind: by the order of the
                    // entries it is the last or the last but one
                    const long long k_row = j == k_last ? row_cur : row_prev;
                    const unsigned have = __ballot_sync(0xffffffffu, k_row >= 0);
                    if (slot >= F::kBase && tail != kNoPiece) {
                        // Piece `tail` released by every role.  Its phase of the ring's
                        // barrier is the present or the last one, so the parity says
                        // which: piece tail - kPieceRing was released before `tail` was
                        // dealt, and once tail + kPieceRing has been dealt, as this
                        // warp then knows, nothing is left to wait for.
                        if (piece - tail < unsigned(kPieceRing)) {
                            drain();
                            go = __all_sync(0xffffffffu, bar_wait(&M.piece_empty[tail % kPieceRing], (tail / kPieceRing) & 1,
                                                                  abort_flag, a.status));
                            if (!go) break;
                        }
                        tail = kNoPiece;
                    }
                    const unsigned parity = (empty_phase >> slot) & 1;
                    if (!__all_sync(0xffffffffu, bar_done(&M.empty[slot], parity))) {
                        drain();  // nothing can be issued: hand over what has landed meanwhile
                        go = __all_sync(0xffffffffu, bar_wait(&M.empty[slot], parity, abort_flag, a.status));
                        if (!go) break;
                    }
                    empty_phase ^= 1u << slot;
                    if (!is_v && lane == 0) M.valid[(walk.tile_base + j) % kMetaRing][lw] = have;
                    const unsigned dst = smem + slot_at(slot);
                    const long long shift = is_v ? a.kind_rows : 0;
                    constexpr int kLanes = DP / 8, kStep = 32 / kLanes;  // lanes per row, rows per instruction
                    const int ch = lane % kLanes;
                    // a slab of 32 cached positions, all in the pool: by TMA,
                    // box_rows rows x 64 columns at a time
                    if (a.box_rows && have == 0xffffffffu && (walk.t0 + j) * F::kBn + lw * 32 + 32 <= walk.len) {
                        if (lane == 0) {
                            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(sm_addr(&M.full[slot])),
                                         "r"(32 * DP * 2)
                                         : "memory");
                            if (is_v) {
                                M.vbad[(walk.tile_base + j) % kMetaRing][lw] = 0;
                                bar_arrive(&M.v_ready[(walk.tile_base + j) % kMetaRing]);
                            }
                        }
                        __syncwarp();
                        if ((lane & (a.box_rows - 1)) == 0) {
#pragma unroll
                            for (int half = 0; half < F::kHalves; ++half)
                                tma_load_2d(dst + half * (F::kBn * 128) + (lw * 32 + lane) * 128, &kv_map, half * 64,
                                            int(k_row + shift), sm_addr(&M.full[slot]));
                        }
                        __syncwarp();
                        slot = slot + 1 == ns ? 0 : slot + 1;
                        continue;
                    }
#pragma unroll 4
                    for (int i = 0; i < 32 / kStep; ++i) {
                        const int rr = i * kStep + lane / kLanes;
                        const long long at = __shfl_sync(0xffffffffu, k_row, rr);
                        const bool ok = at >= 0 && ch < chunks;
                        const int rt = lw * 32 + rr;
                        cp16(dst + (ch >> 3) * (F::kBn * 128) + rt * 128 + (((ch & 7) ^ (rt & 7)) << 4),
                             ok ? pool + (at + shift) * row_bytes + ch * 16 : pool, ok ? 16u : 0u);
                    }
                    cp_commit();
                    if (is_v && (walk.t0 + j + 1) * F::kBn > walk.len) {
                        // a tile with nodes: non-finite V must not meet a weight of zero in the products
                        drain();
                        __syncwarp();
                        unsigned bad_rows = 0;
                        const int rt = lw * 32 + lane;
                        bool bad = false;
                        if ((walk.t0 + j) * F::kBn + rt >= walk.len && k_row >= 0) {
                            const auto chunk = [&](int k) {
                                return reinterpret_cast<uint4*>(tree_smem + slot_at(slot) + (k >> 3) * (F::kBn * 128) + rt * 128 +
                                                                (((k & 7) ^ (rt & 7)) << 4));
                            };
                            // an exponent of all ones carries into the sign bit
                            const auto full = [](unsigned w) { return ((w & 0x7c007c00u) + 0x04000400u) & 0x80008000u; };
                            unsigned any = 0;
#pragma unroll 8
                            for (int k = 0; k < kLanes; ++k) {
                                const uint4 w = *chunk(k);
                                any |= full(w.x) | full(w.y) | full(w.z) | full(w.w);
                            }
                            if (any) {
                                bad = true;
#pragma unroll 1
                                for (int k = 0; k < kLanes; ++k) *chunk(k) = make_uint4(0, 0, 0, 0);
                            }
                        }
                        bad_rows = __ballot_sync(0xffffffffu, bad);
                        if (lane == 0) {
                            M.vbad[(walk.tile_base + j) % kMetaRing][lw] = bad_rows;
                            bar_arrive(&M.v_ready[(walk.tile_base + j) % kMetaRing]);
                        }
                        signal(slot);
                    } else {
                        if (is_v && lane == 0) bar_arrive(&M.v_ready[(walk.tile_base + j) % kMetaRing]);  // nothing to report
                        if (n_pend == 2) {
                            cp_wait<2>();
                            signal(pend[0]);
                            pend[0] = pend[1];
                            n_pend = 1;
                        }
                        pend[n_pend++] = slot;
                    }
                    slot = slot + 1 == ns ? 0 : slot + 1;
                }
                if (pair) tail = piece;
                if (lane == 0) release_piece(piece);
            }
            drain();
            // on the way out after an error: the slots' own copies first
#pragma unroll 1
            for (int i = 0; i < F::kBase + F::kExtra && *abort_flag; ++i)
                bar_land(&M.full[i], empty_phase >> i & 1);
        } else {
            // Rows that the row fetch warp (below) has put into the raw ring
            // become F16 operands.
            bool go = true;
            int raw = 0;
            unsigned raw_phase = 0;
            // int8: a lane per row; F32: a lane per 128 bytes of a row.  With the
            // swizzle of the TMA boxes a warp reads and writes without bank conflicts.
            constexpr int kRound = 32 / F::kRawParts;  // rows a warp takes at a time
            const int row = lw * (F::kBn / 4) + lane % kRound;
            const int f16_swizzle = row & 7;
            for (unsigned piece = 0; go; ++piece) {
                if (!__all_sync(0xffffffffu, get_piece(piece))) break;
                const TreePiece& walk = M.piece[piece % kPieceRing];
                const int first_p = walk.t0 * F::kBn, len = walk.len, tiles = walk.t1 - walk.t0, ahead = min(2, tiles);
                const unsigned tile_base = walk.tile_base;
                const int loads = 2 * tiles;
                for (int e = 0; e < loads && go; ++e) {
                    // the order of TreePiece::entry, with one M tile
                    const int f = e - ahead, both = 2 * (tiles - ahead);
                    const bool is_v = f >= 0 && (f >= both || !(f & 1));
                    const int j = f < 0 ? e : f < both ? (f >> 1) + (f & 1 ? ahead : 0) : f - (tiles - ahead);
                    go = __all_sync(0xffffffffu, bar_wait(&M.raw_full[raw], (raw_phase >> raw) & 1, abort_flag, a.status));
                    raw_phase ^= 1u << raw;
                    if (!go) break;
                    const unsigned parity = (empty_phase >> slot) & 1;
                    go = __all_sync(0xffffffffu, bar_wait(&M.empty[slot], parity, abort_flag, a.status));
                    if (!go) break;
                    empty_phase ^= 1u << slot;
                    const int meta = int((tile_base + j) % kMetaRing);
                    const int p0 = first_p + j * F::kBn;
                    const bool node_values = is_v && p0 + F::kBn > len;  // V of nodes may be masked: finite in the products
                    float* scale_col = reinterpret_cast<float*>(tree_smem + F::kOffScale) +
                                       (int((tile_base + j) % F::kScaleRing) * 2 + is_v) * F::kBn;
                    unsigned char* out = tree_smem + slot_at(slot);
                    unsigned char* src = tree_smem + F::kOffRaw + raw * F::kRaw + row * F::kRawPitch;
                    const int swizzle = F::kRawPitch == 128 ? row & 7 : row >> 1 & 3;
                    float big = 0.f, low = INFINITY;
                    unsigned bad_rows = 0;
                    unsigned char* dst = out + row * 128;
                    if constexpr (KV == 2) {
                        uint4 row_codes[DP / 16];  // all read before any is written: no load waits behind a store
#pragma unroll
                        for (int i = 0; i < DP / 16; ++i)
                            row_codes[i] = i < chunks ? *reinterpret_cast<const uint4*>(src + ((i ^ swizzle) << 4)) : make_uint4(0, 0, 0, 0);
                        if (is_v) {
                            float sc = scale_col[row];
                            const bool bad = node_values && p0 + row >= len && !isfinite(sc);
                            bad_rows = __ballot_sync(0xffffffffu, bad);
                            unsigned any = 0;
#pragma unroll
                            for (int i = 0; i < DP / 16; ++i) any |= row_codes[i].x | row_codes[i].y | row_codes[i].z | row_codes[i].w;
                            // a row of zeros may have any scale (the encoder gives 1): it adds nothing, and is not to be
                            // what the others' digits are measured by
                            if (bad || (!any && isfinite(sc))) scale_col[row] = sc = 0.f;
                            big = fabsf(sc);
                            if (M.valid[meta][lw] >> lane & 1) low = big;
                        }
#pragma unroll
                        for (int i = 0; i < DP / 16; ++i) {
                            const unsigned w[4] = {row_codes[i].x, row_codes[i].y, row_codes[i].z, row_codes[i].w};
                            unsigned h[8];
#pragma unroll
                            for (int x = 0; x < 4; ++x) {
                                // code + 128 beside 0x64: 1024 + 128 + code, exact in F16
                                const unsigned b = w[x] ^ 0x80808080u;
                                const __half2 off = __half2half2(__ushort_as_half(0x6480));
                                const unsigned l0 = __byte_perm(b, 0x64646464u, 0x4140), l1 = __byte_perm(b, 0x64646464u, 0x4342);
                                const __half2 a0 = __hsub2(*reinterpret_cast<const __half2*>(&l0), off);
                                const __half2 a1 = __hsub2(*reinterpret_cast<const __half2*>(&l1), off);
                                h[2 * x] = *reinterpret_cast<const unsigned*>(&a0);
                                h[2 * x + 1] = *reinterpret_cast<const unsigned*>(&a1);
                            }
#pragma unroll
                            for (int x = 0; x < 2; ++x)
                                *reinterpret_cast<uint4*>(dst + (i >> 2) * (F::kBn * 128) + ((((2 * i + x) & 7) ^ f16_swizzle) << 4)) =
                                    make_uint4(h[4 * x], h[4 * x + 1], h[4 * x + 2], h[4 * x + 3]);
                        }
                    } else {
                        const int part = lane / kRound;
#pragma unroll 1
                        for (int round = 0; round < F::kBn / 4; round += kRound) {
                            const unsigned char* mine = src + part * (F::kBn * 128) + round * 128;  // (rounds of 8 or 16 rows
                            uint4 quads[8];                                                         // keep the swizzle)
#pragma unroll
                            for (int i = 0; i < 8; ++i)
                                quads[i] = part * 8 + i < chunks ? *reinterpret_cast<const uint4*>(mine + ((i ^ swizzle) << 4)) : make_uint4(0, 0, 0, 0);
                            if (node_values) {
                                unsigned most = 0;  // magnitudes as bits: infinity and NaN are the largest
#pragma unroll
                                for (int i = 0; i < 8; ++i)
                                    most = max(max(most, max(quads[i].x & 0x7fffffffu, quads[i].y & 0x7fffffffu)),
                                               max(quads[i].z & 0x7fffffffu, quads[i].w & 0x7fffffffu));
#pragma unroll
                                for (int d = kRound; d < 32; d <<= 1) most = max(most, __shfl_xor_sync(0xffffffffu, most, d));
                                const bool bad = p0 + row + round >= len && most >= 0x7f800000u;
                                bad_rows |= (__ballot_sync(0xffffffffu, bad) & ((1u << kRound) - 1)) << round;
                                if (bad)
#pragma unroll
                                    for (int i = 0; i < 8; ++i) quads[i] = make_uint4(0, 0, 0, 0);
                            }
                            float tops[2] = {0.f, 0.f};
#pragma unroll
                            for (int i = 0; i < 8; ++i) {
                                tops[0] = max3(tops[0], fabsf(__uint_as_float(quads[i].x)), fabsf(__uint_as_float(quads[i].y)));
                                tops[1] = max3(tops[1], fabsf(__uint_as_float(quads[i].z)), fabsf(__uint_as_float(quads[i].w)));
                            }
                            float top = fmaxf(tops[0], tops[1]);
#pragma unroll
                            for (int d = kRound; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                            const int up = lift(top);
                            // a row of zeros has scale 0: with 1 its weight, which is in units of the
                            // other rows' scales, overflows F16, and inf * 0 is NaN
                            const float f = two_to(up), back = top > 0.f ? two_to(-up) : 0.f;
                            if (lane < kRound) scale_col[row + round] = is_v ? back : back * two_to(-14);
                            big = fmaxf(big, back);
                            low = fminf(low, back > 0.f || (M.valid[meta][(row + round) >> 5] >> ((row + round) & 31) & 1) ? back : INFINITY);
                            const f32x2 f2 = pair_of(f, f);
#pragma unroll
                            for (int i = 0; i < 8; i += 2) {
                                uint4 hi, lo;
                                split_packed(mul2(pair_of(__uint_as_float(quads[i].x), __uint_as_float(quads[i].y)), f2), hi.x, lo.x);
                                split_packed(mul2(pair_of(__uint_as_float(quads[i].z), __uint_as_float(quads[i].w)), f2), hi.y, lo.y);
                                split_packed(mul2(pair_of(__uint_as_float(quads[i + 1].x), __uint_as_float(quads[i + 1].y)), f2), hi.z, lo.z);
                                split_packed(mul2(pair_of(__uint_as_float(quads[i + 1].z), __uint_as_float(quads[i + 1].w)), f2), hi.w, lo.w);
                                const int hc = part * 4 + i / 2;  // 16-byte chunk of the F16 row
                                unsigned char* at = dst + round * 128 + (hc >> 3) * (F::kBn * 128) + (((hc & 7) ^ f16_swizzle) << 4);
                                *reinterpret_cast<uint4*>(at) = hi;
                                *reinterpret_cast<uint4*>(at + F::kSlotPart) = lo;
                            }
                        }
                    }
                    if (is_v) {
                        if (lane == 0) {
                            if constexpr (KV == 2)
                                M.vbad[meta][lw] = bad_rows;
                            else
                                reinterpret_cast<unsigned short*>(M.vbad[meta])[lw] = (unsigned short)bad_rows;
                        }
#pragma unroll
                        for (int d = 16; d; d >>= 1) {
                            big = fmaxf(big, __shfl_xor_sync(0xffffffffu, big, d));
                            low = fminf(low, __shfl_xor_sync(0xffffffffu, low, d));
                        }
                        if (lane == 0)
                            M.vspan[meta][lw] = ((__float_as_uint(big) + 0xffffu) & 0xffff0000u) | __float_as_uint(low) >> 16;
                    }
                    proxy_fence();
                    __syncwarp();
                    if (lane == 0) {
                        bar_arrive(&M.raw_empty[raw]);
                        if (is_v) bar_arrive(&M.v_ready[meta]);
                        bar_arrive(&M.full[slot]);
                    }
                    raw = raw + 1 == F::kRawDepth ? 0 : raw + 1;
                    slot = slot + 1 == F::kBase ? 0 : slot + 1;
                }
                if (lane == 0) release_piece(piece);
            }
        }
        if (flags) atomicOr(a.status, flags);
    } else if (warp == kTreeMmaWarp) {
        {
            // -------------------------------------------------- MMA issue
            constexpr unsigned kIdescS = (1u << 4) | (unsigned(F::kBn >> 3) << 17) | (8u << 24);
            constexpr unsigned kIdescO = (1u << 4) | (1u << 16) | (unsigned(DP >> 3) << 17) | (8u << 24);
            unsigned full_phase = 0, n_p = 0;  // phase bits per slot and stream
            int slot = 0;
            bool go = true;
            const auto at128 = [&](unsigned addr) { return sw128_desc(addr, 16); };
            const std::uint64_t q_desc = at128(smem), v_desc = sw128_desc(smem, F::kBn * 128);
            const auto take = [&](int ns) -> int {  // next ring slot, filled
                const int s = slot;
                go = __all_sync(0xffffffffu, bar_wait(&M.full[s], (full_phase >> s) & 1, abort_flag, a.status));
                full_phase ^= 1u << s;
                slot = s + 1 == ns ? 0 : s + 1;
                tm_after();
                return s;
            };
            for (unsigned piece = 0; go; ++piece) {
                if (!__all_sync(0xffffffffu, get_piece(piece))) break;
                const TreePiece& walk = M.piece[piece % kPieceRing];
                const bool pair = __shfl_sync(0xffffffffu, walk.pair, 0);
                const int ns = pair ? F::kBase : F::kBase + F::kExtra, tiles = __shfl_sync(0xffffffffu, walk.t1 - walk.t0, 0);
                if (slot >= ns) slot = 0;
                go = __all_sync(0xffffffffu, bar_wait(&M.q_full, piece & 1, abort_flag, a.status));
                if (!go) break;
                tm_after();
                // Products i of S = Q K^T and of P V, stream i & 1: one K and V
                // tile each, or one for the two streams of a pair.  S of
                // product i + 2 follows P V of product i, whose P it overwrites.
                const int steps = pair ? 2 * tiles : tiles;
                int s_k = 0, s_v = 0;
#pragma unroll 1
                for (int i = -2; i < steps && go; ++i) {
                    const int st = i & 1;
                    if (i >= 0) {
                        if (!pair || !st) s_v = take(ns);
                        go = go && __all_sync(0xffffffffu, bar_wait(&M.p_full[st], (n_p >> st) & 1, abort_flag, a.status));
                        n_p ^= 1u << st;
                        if (!go) break;
                        tm_after();
                        const unsigned d = tmem + 256 + st * 128;
                        const std::uint64_t v = v_desc + (slot_at(s_v) >> 4);
                        int acc = 0;
                        if (elect_one()) {
#pragma unroll 1
                        for (int part = 0; part <= F::kParts; ++part) {  // small products first: P lo (and V lo)
                            const unsigned pa = tmem + st * 128 + (part == 0 ? 8 : 0);
                            const std::uint64_t vb = v + (F::kParts == 2 && part == 1 ? F::kSlotPart >> 4 : 0);
#pragma unroll 4
                            for (int kk = 0; kk < F::kBn / 16; ++kk) {
                                mma_ts(d, pa + kk * 16, vb + kk * (2048 >> 4), kIdescO, acc);
                                acc = 1;
                            }
                        }
                        if (!pair || st) tree_commit_to(&M.empty[s_v]);
                        tree_commit_to(&M.o_full[st]);
                        }
                        __syncwarp();
                    }
                    if (i + 2 < steps) {
                        if (!pair || !st) s_k = take(ns);
                        if (!go) break;
                        const unsigned d = tmem + st * 128;
                        const std::uint64_t q = q_desc + (pair && st ? F::kQTile >> 4 : 0), k = q_desc + (slot_at(s_k) >> 4);
                        int acc = 0;
                        if (elect_one()) {
#pragma unroll 1
                        for (int part = 0; part <= F::kParts; ++part) {  // lo Q, (lo K,) hi hi
                            const std::uint64_t qa = q + (part == 0 ? F::kQPart >> 4 : 0);
                            const std::uint64_t kb = k + (F::kParts == 2 && part == 1 ? F::kSlotPart >> 4 : 0);
#pragma unroll 1
                            for (int half = 0; half < F::kHalves; ++half)
#pragma unroll
                                for (int kk = 0; kk < 4; ++kk) {
                                    mma_ss(d, qa + half * (16384 >> 4) + kk * 2, kb + half * ((F::kBn * 128) >> 4) + kk * 2,
                                           kIdescS, acc);
                                    acc = 1;
                                }
                        }
                        if (!pair || st) tree_commit_to(&M.empty[s_k]);
                        tree_commit_to(&M.s_full[st]);
                        }
                        __syncwarp();
                    }
                }
                if (!go) break;
                if (lane == 0) release_piece(piece);
            }
            // nothing of this CTA's may be in flight when its memory is given back
            if (lane == 0) tree_commit_to(&M.drain);
            bar_land(&M.drain, 0);
        }
        __syncwarp();
    }
    if (KV != 1 && warp == kTreeRawWarp) {
        // --------------------------------------- rows of F32 and int8 pools
        // Tiles of cached positions by TMA, a lane per box; others in pieces of
        // 16 bytes, whole rows to an instruction, into the same swizzle (rows
        // that hold nothing are zero).  Bulk copies of 128 bytes a lane, which
        // issue one after another and land without the swizzle, were slower (one
        // tree of 60 nodes on 300 positions, 32/8 heads of 128: F32 53.5 -> 41.2 us,
        // int8 33.0 -> 30.8; 24 sequences int8 205 -> 196).
        constexpr int kSlabs = F::kBn / 32, kPitch = F::kRawPitch;
        constexpr int kLanes = F::kRawParts * kPitch / 16, kStep = 32 / kLanes;  // lanes per row, rows per instruction
        bool go = true;
        int raw = 0, flags = 0;
        unsigned empty_phase = 0xffffffffu;
        for (unsigned piece = 0; go; ++piece) {
            if (!__all_sync(0xffffffffu, get_piece(piece))) break;
            const TreePiece& walk = M.piece[piece % kPieceRing];
            const int loads = 2 * (walk.t1 - walk.t0);
            long long cur[kSlabs], prev[kSlabs];
            long long box_cur = 0, box_prev = 0;
            int k_last = -1, ahead = 0, ahead_j = -1;  // ahead: the table entry of this lane's box in tile ahead_j
            int k_box = -1;
            const int boxes = a.box_rows ? F::kBn / a.box_rows : 0;
            const auto entry_of = [&](int j) -> int {
                const int p = (walk.t0 + j) * F::kBn + lane * a.box_rows;
                return a.tables[(long long)walk.s * a.stride + div_bt(a, p)];
            };
#pragma unroll
            for (int i = 0; i < kSlabs; ++i) cur[i] = prev[i] = -1;
#pragma unroll 1
            for (int e = 0; e < loads; ++e) {
                bool is_v;
                const int j = walk.entry(e, is_v);
                const unsigned tile = walk.tile_base + j;
                if (boxes && (walk.t0 + j + 1) * F::kBn <= walk.len) {
                    if (!is_v) {
                        box_prev = box_cur;
                        box_cur = -1;
                        if (lane < boxes) {
                            const int block = ahead_j == j ? ahead : entry_of(j);
                            const int p = (walk.t0 + j) * F::kBn + lane * a.box_rows;
                            if (unsigned(block) < unsigned(a.max_blocks))
                                box_cur = block * a.block_rows + a.layer_rows + (long long)walk.head * a.bt + (p - int(div_bt(a, p)) * a.bt);
                            ahead_j = j + 1;
                            if ((walk.t0 + j + 2) * F::kBn <= walk.len && walk.t0 + j + 1 < walk.t1) ahead = entry_of(j + 1);
                            else ahead_j = -1;
                        }
                    }
                    const long long at = is_v && j != k_box ? box_prev : box_cur;
                    if (!is_v) k_box = j;
                    if (__all_sync(0xffffffffu, lane >= boxes || at >= 0)) {
                        go = __all_sync(0xffffffffu, bar_wait(&M.raw_empty[raw], (empty_phase >> raw) & 1, abort_flag, a.status));
                        if (!go) break;
                        empty_phase ^= 1u << raw;
                        if (!is_v && lane < 4) M.valid[tile % kMetaRing][lane] = 0xffffffffu;
                        __syncwarp();
                        const unsigned full = sm_addr(&M.raw_full[raw]);
                        if (lane == 0)
                            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(full),
                                         "r"(F::kBn * (DP * F::kElem + (KV == 2 ? 4 : 0)))
                                         : "memory");
                        __syncwarp();
                        if (lane < boxes) {
                            const long long row = at + (is_v ? a.kind_rows : 0);
#pragma unroll
                            for (int part = 0; part < F::kRawParts; ++part)
                                tma_load_2d(smem + F::kOffRaw + raw * F::kRaw + (part * F::kBn + lane * a.box_rows) * kPitch, &kv_map,
                                            part * (kPitch / F::kElem), int(row), full);
                            if constexpr (KV == 2)
                                bulk_load(smem + F::kOffScale + ((tile % F::kScaleRing * 2 + is_v) * F::kBn + lane * a.box_rows) * 4,
                                          a.scales + row, a.box_rows * 4, full);
                        }
                        bar_arrive(&M.raw_full[raw]);
                        raw = raw + 1 == F::kRawDepth ? 0 : raw + 1;
                        continue;
                    }
                }
                if (j != k_last && (!is_v || j != k_last - 1)) {
#pragma unroll
                    for (int i = 0; i < kSlabs; ++i) {
                        prev[i] = cur[i];
                        cur[i] = row_of(walk, (walk.t0 + j) * F::kBn + 32 * i + lane, flags);
                    }
                    k_last = j;
                }
                go = __all_sync(0xffffffffu, bar_wait(&M.raw_empty[raw], (empty_phase >> raw) & 1, abort_flag, a.status));
                if (!go) break;
                empty_phase ^= 1u << raw;
                const unsigned dst = smem + F::kOffRaw + raw * F::kRaw, full = sm_addr(&M.raw_full[raw]);
                const int ch = lane % kLanes, column = ch % (kPitch / 16);
#pragma unroll
                for (int i = 0; i < kSlabs; ++i) {
                    const long long at = j == k_last ? cur[i] : prev[i], row = at + (is_v ? a.kind_rows : 0);
                    const unsigned have = __ballot_sync(0xffffffffu, at >= 0);
                    if (!is_v && lane == 0) M.valid[tile % kMetaRing][i] = have;
                    if constexpr (KV == 2)  // the row's scale, straight into its column
                        cp4(smem + F::kOffScale + ((tile % F::kScaleRing * 2 + is_v) * F::kBn + 32 * i + lane) * 4,
                            at >= 0 ? a.scales + row : a.scales, at >= 0 ? 4u : 0u);
#pragma unroll 4
                    for (int r0 = 0; r0 < 32; r0 += kStep) {
                        const int rr = r0 + lane / kLanes, rt = 32 * i + rr;
                        const long long from = __shfl_sync(0xffffffffu, row, rr);
                        const bool ok = (have >> rr & 1) && ch < chunks;
                        const int swizzle = kPitch == 128 ? rt & 7 : rt >> 1 & 3;
                        cp16(dst + (ch / (kPitch / 16) * F::kBn + rt) * kPitch + ((column ^ swizzle) << 4),
                             ok ? pool + from * row_bytes + ch * 16 : pool, ok ? 16u : 0u);
                    }
                }
                asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(full) : "memory");
                if (lane == 0) bar_arrive(&M.raw_full[raw]);
                __syncwarp();
                raw = raw + 1 == F::kRawDepth ? 0 : raw + 1;
            }
            if (lane == 0 && go) release_piece(piece);
        }
        // every copy of this warp has landed before the memory is given back
#pragma unroll 1
        for (int i = 0; i < F::kRawDepth; ++i)
            bar_land(&M.raw_full[i], empty_phase >> i & 1);
        cp_wait<0>();
        if (flags) atomicOr(a.status, flags);
    }
    tm_before();
    __syncthreads();
    if (warp == kTreeMmaWarp) {
        tm_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512));
    }
}

// Items cut by run boundaries: out = sum_i O_i 2^(m_i - M) / sum_i l_i 2^(m_i - M)
// over the pieces in order (a fixed order, so results repeat bit for bit).
// Block (b, y) takes rows 32 y .. 32 y + 31 of the item that starts in CTA b:
// columns 32 z .. 32 z + 31: lanes are rows, warps groups of four columns.
// With V scales (kScaled) O_i is in units of 2^(m_i + v_i), l_i of 2^m_i.
template <int DP, bool kScaled>
__global__ void __launch_bounds__(256) tree_combine_kernel(TreeAttn a, const float* partial, const TreeRec* recs) {
    __shared__ float4 stage[32][9];
    asm volatile("griddepcontrol.wait;" ::: "memory");  // launched while the tiles are still being worked on
    const TreeRec rec = recs[blockIdx.x];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, row = blockIdx.y * 32 + lane;
    if (rec.pieces < 2 || int(blockIdx.y) * 32 >= rec.rows) return;
    const int mine = min(row, rec.rows - 1);  // idle lanes repeat the last row
    const int pr = mine < rec.split ? mine : 128 + mine - rec.split, parts = rec.pieces * rec.streams;
    const int group4 = blockIdx.z * 8 + warp;
    const auto slot_of = [&](int i, int& at) {  // part i: its slot, and the row's place in it
        const int piece = rec.streams == 2 ? i >> 1 : i;
        at = rec.streams == 2 ? (i & 1) * 128 + pr : pr;
        return partial + (2ll * (int(blockIdx.x) + piece) + (piece == 0)) * kTreeRows * (DP + kTreeState);
    };
    float top = -INFINITY, top_v = -INFINITY;
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
        int at;
        const float* slot = slot_of(i, at);
        const float m = slot[kTreeRows * DP + at];
        top = fmaxf(top, m);
        if constexpr (kScaled) top_v = fmaxf(top_v, m + slot[kTreeRows * DP + 2 * kTreeRows + at]);
    }
    if (kScaled && top != -INFINITY) top_v -= top;  // O's reference beyond l's: any near the largest will do
    float l = 0.f;
    float4 o = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
    for (int i = 0; i < parts; ++i) {
        int at;
        const float* slot = slot_of(i, at);
        // nothing seen (or nothing but NaN scores): the sums decide
        const float down = slot[kTreeRows * DP + at] - top;
        float f = top == -INFINITY ? 1.f : ex2(down);
        const float4 x = *reinterpret_cast<const float4*>(slot + (group4 * kTreeRows + at) * 4);
        l += slot[kTreeRows * DP + kTreeRows + at] * f;
        if (kScaled && top != -INFINITY) f = ex2(down + slot[kTreeRows * DP + 2 * kTreeRows + at] - top_v);
        o.x += x.x * f;
        o.y += x.y * f;
        o.z += x.z * f;
        o.w += x.w * f;
    }
    float f = l == 0.f && top == -INFINITY ? 0.f : 1.f / l;
    if (kScaled && top != -INFINITY) f = ex2(top_v) / l;
    stage[lane][warp] = make_float4(o.x * f, o.y * f, o.z * f, o.w * f);
    __syncthreads();
    // eight lanes write a row's 32 columns
    const int i = threadIdx.x >> 3, col = threadIdx.x & 7;
    if (int(blockIdx.y) * 32 + i < rec.rows && (int(blockIdx.z) * 8 + col) * 4 < a.dim) {
        const int vec = rec.row0 + blockIdx.y * 32 + i, node = unsigned(vec) / unsigned(a.group);
        const int head = rec.head * a.group + vec - node * a.group;
        float* dst = a.out + (long long)(rec.c0 + node) * a.ldo + (long long)head * a.dim;
        reinterpret_cast<float4*>(dst)[blockIdx.z * 8 + col] = stage[i][col];
    }
}

int tree_ctas() {
    int device = 0, sms = 0;
    TVARA_CUDA(cudaGetDevice(&device));
    TVARA_CUDA(cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device));
    return sms;
}

constexpr int kTreeMaxCtas = 148, kTreeRecBytes = 8192;
// Weight of the shortest run: one tree of 26 nodes on 1,900 positions with 2, 3,
// 4, 6, 10: 28.9, 28.9, 30.5, 30.4, 39.2 us; alike for other small calls.
constexpr int kTreeMinRun = 2;

template <int KV, int DP>
void run_tree_mma(const TreeAttn& a, void* workspace, cudaStream_t s) {
    using F = TreeForm<KV, DP>;
    const int ctas = std::min(tree_ctas(), kTreeMaxCtas);
    auto* recs = static_cast<TreeRec*>(workspace);
    auto* partial = reinterpret_cast<float*>(static_cast<unsigned char*>(workspace) + kTreeRecBytes);
    TVARA_CUDA(cudaFuncSetAttribute(tree_mma_kernel<KV, DP>, cudaFuncAttributeMaxDynamicSharedMemorySize, F::kSmem));
    // head_dim 64 or 128 and blocks of a multiple of 8 positions: cached
    // positions come by TMA, whose boxes never cross a block
    CUtensorMap map{};
    TreeAttn job = a;
    job.box_rows = 0;
    const unsigned long long rows = (unsigned long long)a.max_blocks * a.block_rows;
    if (a.dim % 64 == 0 && a.bt % 8 == 0 && rows < 0x7fffffffull && reinterpret_cast<std::uintptr_t>(a.scales) % 16 == 0) {
        job.box_rows = a.bt % 32 == 0 ? 32 : a.bt % 16 == 0 ? 16 : 8;
        const cuuint64_t dims[2] = {cuuint64_t(a.dim), cuuint64_t(rows)};
        const cuuint64_t strides[1] = {cuuint64_t(a.dim) * F::kElem};
        const cuuint32_t box[2] = {cuuint32_t(KV == 1 ? 64 : F::kRawPitch / F::kElem), cuuint32_t(job.box_rows)}, ones[2] = {1, 1};
        const auto type = KV == 0 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32 : KV == 1 ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16 : CU_TENSOR_MAP_DATA_TYPE_UINT8;
        if (tensor_map_encoder()(&map, type, 2, const_cast<void*>(a.kv), dims, strides, box, ones,
                                 CU_TENSOR_MAP_INTERLEAVE_NONE, KV != 1 && F::kRawPitch == 64 ? CU_TENSOR_MAP_SWIZZLE_64B : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                                 CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) != CUDA_SUCCESS)
            throw std::runtime_error("cuTensorMapEncodeTiled failed for the KV pool");
    }
    tree_mma_kernel<KV, DP><<<ctas, kTreeThreads, F::kSmem, s>>>(map, job, partial, recs, kTreeMinRun);
    TVARA_LAUNCHED();
    // launched early; its blocks wait for the first kernel's end (one token F32:
    // 18.5 us in place of 19.7, one tree of 26 nodes F16: 28.9 in place of 31.0)
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(unsigned(ctas), kTreeRows / 32, DP / 32);
    config.blockDim = dim3(256);
    config.stream = s;
    cudaLaunchAttribute early{};
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    config.attrs = &early;
    config.numAttrs = 1;
    TVARA_CUDA(cudaLaunchKernelEx(&config, tree_combine_kernel<DP, KV != 1>, a, static_cast<const float*>(partial),
                                  static_cast<const TreeRec*>(recs)));
    TVARA_LAUNCHED();
}

// The tensor-core form reads rows in 16-byte pieces.
bool tree_mma_takes(const TreeAttn& a) {
    const auto at = [](const void* p) { return reinterpret_cast<std::uintptr_t>(p); };
    const int elem = a.kv_kind == 0 ? 4 : a.kv_kind == 1 ? 2 : 1;
    return a.dim <= 128 && a.dim * elem % 16 == 0 && a.dim % 4 == 0 && at(a.kv) % 16 == 0 && at(a.q) % 16 == 0 &&
           at(a.out) % 16 == 0 && a.ldq % 4 == 0 && a.ldo % 4 == 0;
}

}  // namespace

std::size_t tree_attention_workspace(const TreeAttn& a) {
    static_assert(sizeof(TreeRec) * kTreeMaxCtas <= kTreeRecBytes);
    const int dp = a.dim <= 64 ? 64 : 128;
    return a.dim <= 128 ? kTreeRecBytes + std::size_t(2) * kTreeMaxCtas * kTreeRows * (dp + kTreeState) * 4 : 256;
}

void launch_tree_attention(const TreeAttn& a, void* workspace, cudaStream_t s) {
    if (tree_mma_takes(a)) {
        if (a.dim <= 64) {
            if (a.kv_kind == 0) return run_tree_mma<0, 64>(a, workspace, s);
            if (a.kv_kind == 1) return run_tree_mma<1, 64>(a, workspace, s);
            return run_tree_mma<2, 64>(a, workspace, s);
        }
        if (a.kv_kind == 0) return run_tree_mma<0, 128>(a, workspace, s);
        if (a.kv_kind == 1) return run_tree_mma<1, 128>(a, workspace, s);
        return run_tree_mma<2, 128>(a, workspace, s);
    }
    const dim3 grid(unsigned(a.capacity), unsigned(a.hq));
    if (a.dim <= 32)
        tree_any_kernel<1><<<grid, kAnyWarps * 32, 0, s>>>(a);
    else if (a.dim <= 64)
        tree_any_kernel<2><<<grid, kAnyWarps * 32, 0, s>>>(a);
    else if (a.dim <= 128)
        tree_any_kernel<4><<<grid, kAnyWarps * 32, 0, s>>>(a);
    else
        tree_any_kernel<8><<<grid, kAnyWarps * 32, 0, s>>>(a);
    TVARA_LAUNCHED();
}

}  // namespace tvara
