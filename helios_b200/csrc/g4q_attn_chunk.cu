// g4q_attn_chunk.cu -- attention of a prompt's chunk over a paged cache, on the 5th-generation tensor cores (sm_100a): the
// sequences of more query rows per key head than the kernel of few rows takes, which are 64 (32 at head_dim 512), and in a
// step that mixes both 16 (or the rows of one token, where those are more).
//
//   out = softmax(scale * q k^T + mask) v, masked to the positions j <= t (and j > t - window)
//
// A tile is 256 query rows of a CTA pair (cta_group::2), 128 to a CTA: floor(128 / group) tokens times the query
// heads of one key head, so every K and V tile serves the whole group. Each CTA fetches half of a K tile's keys
// and half of a V tile's columns, and the pair's MMAs read both halves: on single CTAs, which fetch twice as much,
// one producer's page look-ups and boxes took 2600-4000 cycles a tile where the products are 2048 (head_dim 256).
// The pair walks the 128-key tiles that its rows see, warp-specialised in each CTA:
//   warps 0, 10 fill a ring of K and a ring of V stages (up to 32 KB each) by TMA: boxes of one page x 64 elements,
//               SWIZZLE_128B. A warp issues a box in about 90 cycles, and pages of 16 slots make 16 boxes a stage: one
//               warp for both took 3200 cycles a tile. Warp 0 also loads Q and finds the work for all warps.
//   warp 1      of the first CTA: one thread issues the MMAs: S = Q K^T (both operands K-major in shared memory,
//               M = 256, N = 128) into one of two TMEM buffers, and O += P V (P from TMEM, V as it lies, MN-major)
//               into up to 256 TMEM columns. S of tile j+1 is computed before P V of tile j, so the tensor cores
//               have work while the softmax of tile j runs.
//   warps 2-9   the softmax, two threads to a row: S from TMEM, row maximum, 2^(s - m) rounded to bf16 back over S.
//               The maximum used, m, is only raised when a row exceeds it by more than 2^8: the weights stay below
//               256 (bf16 keeps its relative precision), and the output, which would have to be rescaled in TMEM, is
//               touched in the first few tiles only. Then O / sum to global memory. With one thread to a row a tile's
//               softmax was 1550 cycles of one warp per scheduler: 2530 cycles a tile at head_dim 256, now 2050.
//
// Bound by the tensor cores for a long context: a key tile takes its products' cycles (2050 measured of 2048 at head_dim
// 256, three times 1024 at 512). 2048 tokens of 16 heads of 512 over 16384 keys: 1040 us a call, at the 1.4 GHz that the
// power limit leaves (1.49 PFLOP/s of products; the first ten calls from idle take 910 us each, 1.70). 2048 tokens of 16
// heads of 256 with a window of 1024, 9 or 10 key tiles a row tile: 43 us a call with new inputs, 39 with the same ones at
// 1.8 GHz, of which the start (finding the work 2 us, Q and K, the first softmax: 5 us) and each tile's epilogue (2 us) are
// latency. head_dim 128 and 64: the exponentials, 1024 cycles of a tile, and 1750 a tile.
//
// head_dim 64: a pair would leave each CTA 32 columns of V, less than a swizzle row, and its tiles' bytes are few
// for the softmax they take: single CTAs (cta_group::1) run the same code.
// head_dim 512: O would take all of TMEM, so a CTA computes half of the output columns and the scores whole
// (1.5 times the products of a single pass; a row tile of 64 would halve the tensor cores' rate instead).
// The row tiles (x key heads x halves) that fill the GPU in whole waves are computed whole, the longest of a causal
// chunk first. The rest, which would leave SMs idle for a wave (or all of them, for a drafted block or a small chunk
// over a long context), have their keys cut into as many pieces as there are CTAs for them; a join kernel adds the fp32
// partials in piece order. The pairs are as many as fit the GPU, and each walks the list back and forth (the first
// wave's order, then the reverse, so that a long tile is followed by a short one).
#include <cuda_runtime.h>

#include <algorithm>

#include "g4q_attn.cuh"
#include "g4q_common.cuh"
#include "g4q_internal.h"

namespace g4q {
namespace {

constexpr int kTile = 128;             // query rows and keys of a tile
constexpr int kThreads = 352;
constexpr int kSoftWarps = 8;          // of the softmax: warps 2..9
constexpr int kVWarp = 10;
constexpr int kItems = 4;              // of work, between the warp that finds them and the others
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRaise = 8.0f;         // how far (log2) a score may exceed the maximum in use
constexpr uint32_t kTmemCols = 512;
constexpr int kMaxSplits = 32;         // pieces of a tile's keys
// Key tiles of a piece, at least. Where all the work is one wave, pieces always shorten it (300 tokens over 2000 keys:
// 29.4 us with 6, 28.5 with 3; 12 tokens of two sequences at head_dim 512: 32.7 and 28.0). After a wave of whole tiles
// more pieces also land behind the long ones (4 prompts beside 2 tokens: 59.7 us with 6, 69.9 with 3).
constexpr int kMinPiece = 6, kMinPieceAlone = 3;

template <int D>
struct ChunkCfg {
    static constexpr int kCtas = D == 64 ? 1 : 2;            // CTAs that share a K / V tile
    static constexpr int kDv = D < 256 ? D : 256;            // output columns computed
    static constexpr int kHalves = D / kDv;
    static constexpr int kKeysHeld = kTile / kCtas;          // K stage: kKeysHeld keys x kKCols elements
    static constexpr int kKCols = D < 256 ? D : 256;
    static constexpr int kKSt = D / kKCols;                  // stages of a K tile
    static constexpr int kVCols = kDv / kCtas;               // V stage: 128 keys x kVCols elements
    static constexpr int kStageBytes = kTile * kVCols * 2;
    static constexpr int kQBytes = kTile * D * 2;
    // barriers, items of work, and the row maxima of two halves and two tiles
    static constexpr int kTail = 256 + kItems * 64 + 2 * 2 * kTile * 4;
    static constexpr int kFit = (227 * 1024 - kTail - kQBytes) / kStageBytes;
    static constexpr int kStages = kFit > 8 ? 8 : kFit;
    static constexpr int kVStages = kStages / 2 < 1 ? 1 : (kStages - (kKSt - 1)) / 2;   // of the ring of V tiles
    static constexpr int kKStages = kStages - kVStages;                                 // of the ring of K tiles
    static constexpr int kSmem = kQBytes + kStages * kStageBytes + kTail;
    static_assert(kKeysHeld / 16 * (kKCols / 64) <= 32 && kTile / 16 * (kVCols / 64) <= 32, "a lane issues one box of a stage");
    static_assert(kKeysHeld * kKCols == kTile * kVCols && kVCols % 64 == 0, "stages hold either operand");
    static_assert(kVStages >= 1 && kKStages >= kKSt, "a tile of each fits");
};

// n / d for 0 <= n < 2^31 as a product: with 2^(l-1) < d <= 2^l and mul = floor(2^(31+l) / d) + 1, mul d exceeds
// 2^(31+l) by e in (0, 2^l], and n e < 2^(31+l) leaves the quotient as it is.
struct Divisor {
    uint32_t mul;
    int shift;
    explicit Divisor(uint32_t d = 1) {
        int l = 0;
        while ((1ull << l) < d) ++l;
        mul = (uint32_t)((1ull << (31 + l)) / d + 1);
        shift = 31 + l;
    }
    __device__ __forceinline__ int of(int n) const { return (int)(((uint64_t)(uint32_t)n * mul) >> shift); }
};

struct ChunkCall {
    AttnCall a;
    int group;
    int few_rows;        // sequences of at most so many rows belong to the other kernel
    int tokens;          // tokens of a CTA's 128 rows: 128 / group
    int tile_tokens;     // tokens of a tile: of all the CTAs that share it
    int box, box_shift;
    int wave;            // tiles that the GPU computes at once
    int clusters;        // CTAs or CTA pairs of the launch
    int max_pieces;      // of a tile's keys
    Divisor by_tile_tokens, by_wave, by_per_tile;    // per_tile: key heads x halves
    float* part_o;       // [pieces, at most a wave][CTAs of a tile][output columns of a CTA / 4][128 rows][4]
    float* part_ml;      // [pieces][CTAs of a tile * 128][2]
    int* err;
};

// A tile of work: rows of sequence b, key head, half of the output columns, and the piece of its keys.
struct Work {
    SeqGeom g;
    int b, tile, h, half;
    int piece, pieces;   // of the keys
    int slot;            // place of the piece's partial
    int count;           // of all the work of the launch
};

struct TileWork {
    SeqGeom g;
    int t0;              // first token of the tile in its sequence
    int lo, n;           // first key of the first key tile, and their number
    int any_lo, any_hi;  // keys that some row of the tile sees
};

__device__ __forceinline__ int tiles_of(const ChunkCall& c, const SeqGeom& g) {
    return g.q_len * c.group > c.few_rows ? c.by_tile_tokens.of(g.q_len + c.tile_tokens - 1) : 0;
}

__device__ __forceinline__ TileWork tile_work(const ChunkCall& c, const SeqGeom& g, int tile) {
    TileWork w;
    w.g = g;
    w.t0 = tile * c.tile_tokens;
    const int last = w.g.first + min(w.t0 + c.tile_tokens, w.g.q_len) - 1;
    w.any_hi = min(max(last + 1, 0), w.g.kv_len);
    w.any_lo = c.a.window > 0 ? max(0, w.g.first + w.t0 - c.a.window + 1) : 0;
    w.lo = min(w.any_lo, w.any_hi) & ~(c.box - 1);
    w.n = max(1, (w.any_hi - w.lo + kTile - 1) / kTile);    // rows that see nothing still become zeros
    return w;
}

// A piece of work as the warps of a CTA share it.
struct alignas(16) Item {
    int q0, q_len, first, kv_len;      // its sequence
    int b, h, half, t0;                // t0: first token of this CTA's rows
    int lo, n, any_lo, any_hi;         // first key of the first key tile, their number (0: no more work)
    int pieces, slot, unused[2];
};
static_assert(sizeof(Item) == 64, "items lie in kTail");

// The index-th piece of work of the launch, or the index-th tile of the last wave (kLast); b < 0: none. One warp.
// Tiles of the whole waves come first, each one piece; then the rest's first pieces, second pieces and so on.
// The longest tiles come first: a sequence's last one, and up to 32 sequences by their lengths (more: the batch's last
// first).
template <int D, bool kLast>
__device__ __noinline__ Work find_work(const ChunkCall& c, int index, int lane) {
    constexpr int kHalves = ChunkCfg<D>::kHalves;
    const int n_seqs = c.a.pv.n_seqs;
    auto geom_of = [&](int b) {
        SeqGeom g;
        g.q0 = g.q_len = g.first = g.kv_len = 0;
        return b < n_seqs ? seq_geom(c.a.pv, b) : g;
    };
    Work w;
    w.b = -1;
    SeqGeom g = geom_of(lane);                   // the first 32 sequences stay in registers
    int nt = tiles_of(c, g), total = nt;
    for (int b = lane + 32; b < n_seqs; b += 32) total += tiles_of(c, seq_geom(c.a.pv, b));
    total = __reduce_add_sync(0xFFFFFFFFu, total);
    const int per_tile = c.a.hk * kHalves, items = max(0, total * per_tile);
    const int whole = c.by_wave.of(items) * c.wave, rest = items - whole;
    const int cuts = rest > 0 && c.max_pieces > 1 ? min(c.max_pieces, c.wave / rest) : 1;
    w.count = whole + rest * cuts;
    int item = index, piece = 0;
    if (kLast) {
        if (index >= rest) return w;
        item = whole + index;
    } else if (index >= whole && rest > 0) {
        piece = cuts > 1 ? (index - whole) / rest : 0;
        item = index - piece * rest;
    }
    if (item >= items || piece >= cuts) return w;
    int t = c.by_per_tile.of(item), at = 0;
    const int unit = item - t * per_tile;        // of the row tile's
    if (n_seqs <= 32) {
        int before = 0;                          // tiles of the sequences that come before this lane's
        for (int o = 0; o < n_seqs; ++o) {
            const int kv_o = __shfl_sync(0xFFFFFFFFu, g.kv_len, o), nt_o = __shfl_sync(0xFFFFFFFFu, nt, o);
            if (kv_o > g.kv_len || (kv_o == g.kv_len && o < lane)) before += nt_o;
        }
        at = __ffs(__ballot_sync(0xFFFFFFFFu, t >= before && t < before + nt)) - 1;
        t -= __shfl_sync(0xFFFFFFFFu, before, at);
        w.tile = __shfl_sync(0xFFFFFFFFu, nt, at) - 1 - t;
        w.b = at;
    } else {
        t = total - 1 - t;
        int before = 0;
        for (int b0 = 0;; b0 += 32) {            // t < total: ends
            g = geom_of(b0 + lane);
            nt = tiles_of(c, g);
            int inc = nt;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int v = __shfl_up_sync(0xFFFFFFFFu, inc, o);
                if (lane >= o) inc += v;
            }
            const unsigned past = __ballot_sync(0xFFFFFFFFu, before + inc > t);
            if (past != 0) {
                at = __ffs(past) - 1;
                w.tile = t - (before + __shfl_sync(0xFFFFFFFFu, inc - nt, at));
                w.b = b0 + at;
                break;
            }
            before += __shfl_sync(0xFFFFFFFFu, inc, 31);
            if (b0 + 32 >= n_seqs) return w;     // the lengths changed while they were read
        }
    }
    w.g.q0 = __shfl_sync(0xFFFFFFFFu, g.q0, at);
    w.g.q_len = __shfl_sync(0xFFFFFFFFu, g.q_len, at);
    w.g.first = __shfl_sync(0xFFFFFFFFu, g.first, at);
    w.g.kv_len = __shfl_sync(0xFFFFFFFFu, g.kv_len, at);
    w.h = unit / kHalves;
    w.half = unit % kHalves;
    const int least = whole > 0 ? kMinPiece : kMinPieceAlone;
    w.pieces = cuts == 1 || item < whole ? 1 : max(1, min(cuts, tile_work(c, w.g, w.tile).n / least));
    w.piece = piece;
    w.slot = (item - whole) * cuts + piece;
    if (piece >= w.pieces) w.b = -1;
    return w;
}

// Shared-memory descriptor of a SWIZZLE_128B operand. K-major: rows of 128 bytes, 8-row groups 1024 bytes
// apart (lbo unused). MN-major: 64 elements of the MN dimension per 128-byte row, one row per k, 8 k's 1024
// bytes apart, the next 64 elements lbo bytes on.
// The upper word is the same for all of them; the lower one is the address in units of 16 bytes, below lbo, so a step
// of a tile is one addition.
constexpr uint32_t kDescHigh = (1024u >> 4) | (1u << 14) | (2u << 29);
__device__ __forceinline__ uint32_t desc_low(uint32_t saddr, uint32_t lbo) {
    return ((saddr & 0x3FFFFu) >> 4) | ((lbo >> 4) << 16);
}

// kind::f16 instruction descriptor: D f32, A and B bf16; b_mn: B is MN-major.
constexpr uint32_t instr_desc(int m, int n, bool b_mn) {
    return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | ((uint32_t)(n >> 3) << 17) | ((uint32_t)(m >> 4) << 24);
}

// D += A B with A in shared memory (mma_ss) or TMEM (mma_ts). On a CTA pair each CTA holds its 128 rows of A and
// D, and half of B's columns.
template <int kCtas>
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
    if constexpr (kCtas == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
            "setp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
            "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kDescHigh)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 a, b;\n\t"
            "setp.ne.b32 p, %4, 0;\n\tmov.b64 a, {%1, %5};\n\tmov.b64 b, {%2, %5};\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], a, b, %3, p;\n\t}" ::"r"(d),
            "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kDescHigh)
            : "memory");
}

template <int kCtas>
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool accumulate) {
    if constexpr (kCtas == 2)
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
            "setp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
            "tcgen05.mma.cta_group::2.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
            "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kDescHigh)
            : "memory");
    else
        asm volatile(
            "{\n\t.reg .pred p;\n\t.reg .b64 b;\n\t"
            "setp.ne.b32 p, %4, 0;\n\tmov.b64 b, {%2, %5};\n\t"
            "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], b, %3, p;\n\t}" ::"r"(d),
            "r"(a), "r"(b), "r"(idesc), "r"((uint32_t)accumulate), "r"(kDescHigh)
            : "memory");
}

// Arrives on the barrier (of every CTA of the pair) when the MMAs issued so far are done.
template <int kCtas>
__device__ __forceinline__ void mma_commit(uint32_t bar) {
    if constexpr (kCtas == 2)
        asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
                         bar),
                     "h"((uint16_t)3)
                     : "memory");
    else
        asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}

// True for one thread of a converged warp. The compiler knows that the code behind it is one thread's, and keeps the
// operands of the MMAs in uniform registers: with a test of the lane it moved them there before every MMA, 65 to 85
// cycles each (2048 tokens, 16384 keys of head_dim 512, ten calls from idle: 970 us against 900).
__device__ __forceinline__ bool elect() {
    uint32_t one;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xFFFFFFFF;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(one));
    return one != 0;
}

// The address of the same shared-memory object in the first CTA of the cluster.
__device__ __forceinline__ uint32_t in_first_cta(uint32_t addr) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(addr));
    return r;
}

// Arrivals on a barrier of the cluster. They order nothing beyond this CTA (a cluster-wide release costs 900
// cycles): what they announce are TMA bytes, which the barrier counts itself, or TMEM contents, ordered by the
// tcgen05 fences on both sides.
__device__ __forceinline__ void bar_arrive_cluster(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(bar) : "memory");
}

__device__ __forceinline__ void bar_expect_tx_cluster(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cluster.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

// The two steps of a barrier of the pair.
__device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release;" ::: "memory"); }
__device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire;" ::: "memory"); }

__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t* v) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]),
          "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]),
          "=r"(v[16]), "=r"(v[17]), "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]),
          "=r"(v[24]), "=r"(v[25]), "=r"(v[26]), "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr));
}

__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t* v) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(v[0]),
        "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]),
        "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]),
        "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]),
        "r"(v[29]), "r"(v[30]), "r"(v[31]), "r"(taddr)
        : "memory");
}

// Waits for this thread's TMEM loads. The values are then passed through an empty statement, so that no use of
// them can be moved before the wait.
__device__ __forceinline__ void tmem_wait_ld(uint32_t* v, int n) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < n; ++i) asm volatile("" : "+r"(v[i]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }

// TMA loads into this CTA's shared memory; on a pair their bytes count on the barrier of the pair's first CTA.
template <int kCtas>
__device__ __forceinline__ void tma_rows(uint32_t dst, const CUtensorMap* map, int x, int head, int token, uint32_t bar) {
    if constexpr (kCtas == 2)
        asm volatile(
            "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
                dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(token), "r"(bar)
            : "memory");
    else
        asm volatile(
            "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(head), "r"(token), "r"(bar)
            : "memory");
}

template <int kCtas>
__device__ __forceinline__ void tma_page(uint32_t dst, const CUtensorMap* map, int x, int slot, int head, int page, uint32_t bar) {
    if constexpr (kCtas == 2)
        asm volatile(
            "cp.async.bulk.tensor.4d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
                dst),
            "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(bar)
            : "memory");
    else
        tma_load_page(dst, map, x, slot, head, page, bar);
}

// Four lanes with four 16-byte chunks each, of a row of their own: afterwards lane i has chunk i of all four rows.
__device__ __forceinline__ void quad_transpose(uint32_t (&ch)[4][4], int lane) {
#pragma unroll
    for (int bit = 1; bit < 4; bit <<= 1) {
        const bool upper = (lane & bit) != 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if ((i & bit) != 0) continue;
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t got = __shfl_xor_sync(0xFFFFFFFFu, upper ? ch[i][e] : ch[i + bit][e], bit);
                if (upper)
                    ch[i][e] = got;
                else
                    ch[i + bit][e] = got;
            }
        }
    }
}

template <int D>
__global__ void __launch_bounds__(kThreads, 1)
    attn_chunk_kernel(const __grid_constant__ CUtensorMap tm_q, const __grid_constant__ CUtensorMap tm_k,
                      const __grid_constant__ CUtensorMap tm_v, const __grid_constant__ ChunkCall c) {
    using C = ChunkCfg<D>;
    constexpr int kCtas = C::kCtas;
    extern __shared__ __align__(1024) uint8_t gen[];     // SWIZZLE_128B repeats every 1024 bytes
    const uint32_t base = smem_addr(gen);
    const uint32_t s_q = base, s_ring = s_q + C::kQBytes, s_bar = s_ring + C::kStages * C::kStageBytes;
    auto full = [&](int s) { return s_bar + 8u * s; };
    auto empty = [&](int s) { return s_bar + 8u * (C::kStages + s); };
    auto s_full = [&](int b) { return s_bar + 8u * (2 * C::kStages + b); };
    auto p_full = [&](int b) { return s_bar + 8u * (2 * C::kStages + 2 + b); };
    const uint32_t q_full = s_bar + 8u * (2 * C::kStages + 4);
    auto o_done = [&](int b) { return q_full + 8u + 8u * b; };    // products of the even and the odd tiles
    const uint32_t edge_full = q_full + 24, q_free = q_full + 32;
    uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(gen + (s_bar - base) + 8u * (2 * C::kStages + 9));
    auto work_full = [&](uint32_t i) { return s_bar + 8u * (2 * C::kStages + 10 + i % kItems); };
    Item* s_item = reinterpret_cast<Item*>(gen + (s_bar - base) + 256);
    float* s_max = reinterpret_cast<float*>(s_item + kItems);                // [parity of the exchange][half][row]

    bool gave_up = false;
    auto wait = [&](uint32_t bar, uint32_t parity, int code) {
        if (!bar_wait(bar, parity, c.err, code)) gave_up = true;
    };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = blockIdx.x % kCtas;                 // place in the pair
    const int cluster = blockIdx.x / kCtas;
    if (warp == 1) {
        if constexpr (kCtas == 2) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                         "r"(kTmemCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;");
        } else {
            asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_addr(tmem_slot)),
                         "r"(kTmemCols));
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
        }
    } else if (threadIdx.x == 64) {
        for (int s = 0; s < C::kStages; ++s) {
            bar_init(full(s), kCtas);             // one arrival of each producer, with its bytes
            bar_init(empty(s), 1);
        }
        for (int b = 0; b < 2; ++b) {
            bar_init(s_full(b), 1);
            bar_init(p_full(b), kSoftWarps * kCtas);     // every softmax warp of the pair
            bar_init(o_done(b), 1);
        }
        bar_init(q_full, kCtas);
        bar_init(q_free, 1);
        bar_init(edge_full, 1);
        for (int i = 0; i < kItems; ++i) {
            bar_init(work_full(i), 1);
            s_item[i].n = 0;
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        for (const CUtensorMap* map : {&tm_q, &tm_k, &tm_v})
            asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(map)) : "memory");
    }
    tc_fence_before();
    __syncthreads();
    if constexpr (kCtas == 2) cluster_arrive();
    wait_for_predecessor();
    release_successor();

    if constexpr (kCtas == 2) cluster_wait();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    const uint32_t t_o = tmem, t_s = tmem + 256;     // output, two score buffers of 128 columns
    uint32_t done = 0;     // items done, and their key tiles: the phases of the barriers go on
    uint32_t g = 0;
    Item w;                // the one at hand
    // Warp 0 finds the work: a search takes 2000 to 4000 cycles, which every warp would wait for. It is at most three
    // items ahead of the others, as Q of an item is only loaded when the scores of the one before are done.
    auto take = [&] {
        wait(work_full(done), done / kItems & 1, 90);
        w = s_item[done % kItems];
        return w.n > 0;
    };
    if (warp == 0 || warp == kVWarp) {
        // ---------------- producers: Q and K tiles (warp 0), V tiles (kVWarp)
        const int first_stage = warp == 0 ? 0 : C::kKStages, last_stage = warp == 0 ? C::kKStages : C::kStages;
        int stage = first_stage;
        uint32_t round = 0, edge_round = 0;
        const PagedView& pv = c.a.pv;
        const int page_mask = (1 << pv.page_shift) - 1;
        const uint32_t box_bytes = (uint32_t)c.box * 128u;
        const int boxes = kTile / c.box;             // of a tile of keys; box i is lane i's
        // The page of this lane's box of tile j, looked up two tiles ahead of its use (the look-up takes as long
        // as half a tile's products) and checked when it is used, so that nothing waits for it before.
        constexpr int kNoBox = INT32_MIN;
        auto look_up = [&](int j) {
            const int key = w.lo + j * kTile + lane * c.box;
            return j < w.n && lane < boxes && key < w.any_hi ? pv.table[w.b * pv.table_ld + (key >> pv.page_shift)] : kNoBox;
        };
        auto checked = [&](int page) {
            if (page >= 0 && page < pv.n_pages) return page;
            if (page != kNoBox) record_input_error(pv.err, kErrPage);
            return pv.n_pages;                        // outside the map: reads zeros
        };
        // Fills the next stage with boxes [b0, b1) of its keys k0.. (`keys` of them, the first one box `first` of
        // its tile), columns [col0, col0 + 64 * blocks): at most one box a lane. All of it is worked out before the
        // stage is free: with two or three stages, what happens between its release and the copies is waited for.
        auto fill = [&](const CUtensorMap* map, bool edge, int pages, int k0, int keys, int first, int b0, int b1, int col0,
                        int blocks) {
            const int box = b0 + lane / blocks, cb = lane % blocks;
            const int page = __shfl_sync(0xFFFFFFFFu, pages, (first + box) & 31);
            const uint32_t dst = s_ring + stage * C::kStageBytes + cb * (keys * 128) + box * box_bytes;
            const int slot = (k0 + box * c.box) & page_mask, count = (b1 - b0) * blocks;
            const uint32_t bar = edge ? edge_full : in_first_cta(full(stage));
            if (round > 0) wait(empty(stage), (round - 1) & 1, 80);
            if (lane == 0) bar_expect_tx_cluster(bar, (uint32_t)count * box_bytes);
            __syncwarp();
            if (lane < count) tma_page<kCtas>(dst, map, col0 + cb * 64, slot, w.h, page, bar);
        };
        auto load_k = [&](int j, int raw_pages) {
            const int pages = checked(raw_pages);
            const int k0 = w.lo + j * kTile + rank * C::kKeysHeld;
            // a box without a key that some row sees is left out: its scores are masked
            const int nb = max(0, min(C::kKeysHeld / c.box, (w.any_hi - k0 + c.box - 1) >> c.box_shift));
            for (int p = 0; p < C::kKSt; ++p) {
                fill(&tm_k, false, pages, k0, C::kKeysHeld, rank * C::kKeysHeld / c.box, 0, nb, p * C::kKCols, C::kKCols / 64);
                if (++stage == last_stage) stage = first_stage, ++round;
            }
        };
        auto load_v = [&](int j, int raw_pages) {
            const int pages = checked(raw_pages);
            const int k0 = w.lo + j * kTile, col0 = w.half * C::kDv + rank * C::kVCols;
            const int b1 = max(0, min(boxes, (w.any_hi - k0 + c.box - 1) >> c.box_shift));
            if (k0 >= w.any_lo && k0 + kTile <= w.any_hi) {
                fill(&tm_v, false, pages, k0, kTile, 0, 0, boxes, col0, C::kVCols / 64);
            } else {
                // Keys that no row of the tile sees hold anything, and a zero weight times NaN is NaN: the stage
                // is filled on a barrier of this CTA's own, their rows are zeroed, and it is handed over then.
                const int b0 = max(0, w.any_lo - k0) >> c.box_shift;
                fill(&tm_v, true, pages, k0, kTile, 0, min(b0, b1), b1, col0, C::kVCols / 64);
                wait(edge_full, edge_round++ & 1, 88);
                const int lo = min(kTile, max(0, w.any_lo - k0)), hi = min(kTile, max(lo, w.any_hi - k0));
                for (int i = lane; i < (lo + kTile - hi) * (C::kVCols / 8); i += 32) {
                    const int ch = i & 7, x = i >> 3, cb = x % (C::kVCols / 64);
                    int row = x / (C::kVCols / 64);
                    if (row >= lo) row += hi - lo;
                    *reinterpret_cast<uint4*>(gen + (s_ring - base) + stage * C::kStageBytes + cb * (kTile * 128) + row * 128 +
                                              ch * 16) = make_uint4(0, 0, 0, 0);
                }
                asm volatile("fence.proxy.async.shared::cta;\n\tfence.acq_rel.cluster;" ::: "memory");
                __syncwarp();
                if (lane == 0) bar_expect_tx_cluster(in_first_cta(full(stage)), 0);
            }
            if (++stage == last_stage) stage = first_stage, ++round;
        };
        auto load_v_tiles = [&] {
            int pages = look_up(0), pages1 = look_up(1);
            for (int j = 0; j < w.n; ++j) {
                const int pages2 = look_up(j + 2);
                load_v(j, pages);
                pages = pages1;
                pages1 = pages2;
            }
        };
        if (warp == kVWarp) {
            for (; take(); ++done) load_v_tiles();
        } else {
            // The work of this cluster: the way back and forth over the clusters, so that who had a long tile in one
            // round has a short one in the next.
            int r = 0, count = 1;                        // of the list: known after the first search
            auto find = [&] {
                Item it = {};
                for (; it.n == 0 && r * c.clusters < count; ++r) {
                    const Work at =
                        find_work<D, false>(c, r * c.clusters + ((r & 1) ? c.clusters - 1 - cluster : cluster), lane);
                    count = at.count;
                    if (at.b < 0) continue;
                    const TileWork t = tile_work(c, at.g, at.tile);
                    int j0 = 0, n = t.n;                                 // this piece's key tiles
                    if (at.pieces > 1) {
                        j0 = t.n * at.piece / at.pieces;
                        n = t.n * (at.piece + 1) / at.pieces - j0;
                    }
                    it = {at.g.q0, at.g.q_len, at.g.first, at.g.kv_len, at.b, at.h, at.half, t.t0 + rank * c.tokens,
                          t.lo + j0 * kTile, n, t.any_lo, t.any_hi, at.pieces, at.slot};
                }
                return it;
            };
            uint32_t made = 0;
            auto hand_out = [&](const Item& it) {
                if (lane == 0) {
                    s_item[made % kItems] = it;
                    bar_arrive(work_full(made));
                }
                __syncwarp();
                ++made;
            };
            w = find();
            hand_out(w);
            while (w.n > 0) {
                int pages = look_up(0), pages1 = look_up(1);
                if (done > 0) wait(q_free, (done - 1) & 1, 89);
                if (lane == 0) {
                    const uint32_t qb = in_first_cta(q_full);
                    bar_expect_tx_cluster(qb, (uint32_t)(c.tokens * c.group) * 128u * (D / 64));
                    for (int x = 0; x < D / 64; ++x)
                        tma_rows<kCtas>(s_q + x * (kTile * 128), &tm_q, x * 64, w.h * c.group, w.q0 + w.t0, qb);
                }
                __syncwarp();
                Item next;
                const int ahead = min(w.n, C::kKStages / C::kKSt) - 1;
                for (int j = 0; j < w.n; ++j) {
                    const int pages2 = look_up(j + 2);
                    load_k(j, pages);
                    pages = pages1;
                    pages1 = pages2;
                    if (j == ahead) {                    // while these tiles arrive
                        next = find();
                        hand_out(next);
                    }
                }
                w = next;
                ++done;
            }
        }
    } else if (warp == 1) {
        // ---------------- MMA issuer (of the pair's first CTA)
        if (rank == 0) {
            int stage = 0, v_stage = C::kKStages;
            uint32_t round = 0, v_round = 0;
            auto scores = [&](int j) {
                for (int p = 0; p < C::kKSt; ++p) {
                    wait(full(stage), round & 1, 81);
                    tc_fence_after();
                    if (elect()) {
                        const uint32_t q = desc_low(s_q + p * (C::kKCols / 64) * (kTile * 128), 16);
                        const uint32_t k = desc_low(s_ring + stage * C::kStageBytes, 16);
                        const uint32_t d = t_s + ((g + j) & 1) * kTile;
#pragma unroll
                        for (int kk = 0; kk < C::kKCols / 16; ++kk)
                            mma_ss<kCtas>(d, q + ((kk >> 2) * (kTile * 128) + (kk & 3) * 32) / 16,
                                          k + ((kk >> 2) * (C::kKeysHeld * 128) + (kk & 3) * 32) / 16,
                                          instr_desc(kTile * kCtas, kTile, false), (p | kk) != 0);
                        mma_commit<kCtas>(empty(stage));
                    }
                    __syncwarp();
                    if (++stage == C::kKStages) stage = 0, ++round;
                }
                if (elect()) {
                    mma_commit<kCtas>(s_full((g + j) & 1));
                    if (j + 1 == w.n) mma_commit<kCtas>(q_free);   // Q has been read
                }
                __syncwarp();
            };
            while (take()) {
                const int n = w.n;
                wait(q_full, done & 1, 82);
                scores(0);
                for (int j = 0; j < n; ++j) {
                    if (j + 1 < n) scores(j + 1);
                    const uint32_t b = (g + j) & 1;
                    wait(p_full(b), ((g + j) >> 1) & 1, 83);
                    wait(full(v_stage), v_round & 1, 84);
                    tc_fence_after();
                    if (elect()) {
                        const uint32_t v = desc_low(s_ring + v_stage * C::kStageBytes, kTile * 128);
#pragma unroll
                        for (int kk = 0; kk < kTile / 16; ++kk)
                            mma_ts<kCtas>(t_o, t_s + b * kTile + kk * 8, v + kk * (2048 / 16),
                                          instr_desc(kTile * kCtas, C::kDv, true), (j | kk) != 0);
                        mma_commit<kCtas>(empty(v_stage));
                        mma_commit<kCtas>(o_done(b));
                    }
                    __syncwarp();
                    if (++v_stage == C::kStages) v_stage = C::kKStages, ++v_round;
                }
                g += n;
                ++done;
            }
        }
    } else {
        // ---------------- softmax: two threads to a row, in warps w and w + 4, which reach the same TMEM lanes; each
        // has 64 of a tile's keys and half of the output columns
        const int quarter = warp & 3, side = (warp - 2) >> 2;
        const int row_in = quarter * 32 + lane;
        constexpr int kKeys = kTile / 2, kCols = C::kDv / 2;
        uint32_t swaps = 0;
        // The other thread's value. Two places in turn: the next write to one comes after the barrier that its reader
        // has to reach first.
        auto swap = [&](float v) {
            float* at = s_max + (swaps++ & 1) * (2 * kTile) + row_in;
            at[side * kTile] = v;
            tc_fence_before();
            asm volatile("bar.sync %0, 64;" ::"r"(1 + quarter) : "memory");
            tc_fence_after();
            return at[(side ^ 1) * kTile];
        };
        const uint32_t lanes = (uint32_t)(quarter * 32) << 16;
        const int tok = row_in / c.group;
        const float scale2 = c.a.scale * kLog2e;
        for (;;) {
            // Both warps take the same number of steps, whatever they have read (a wait that gave up leaves an old item):
            // the barrier between the two has no limit of its own.
            const int steps = take() ? w.n : 0;
            const int n = min(steps, __float_as_int(swap(__int_as_float(steps))));
            if (n == 0) break;
            const bool mine = tok < c.tokens && w.t0 + tok < w.q_len;
            int vis_lo = 0, vis_hi = 0;
            if (mine) {
                const int pos = w.first + w.t0 + tok;
                vis_hi = min(max(pos + 1, 0), w.kv_len);
                if (c.a.window > 0) vis_lo = max(0, pos - c.a.window + 1);
            }
            // keys that every row of this CTA sees (rows beyond the sequence do not matter)
            const int all_hi = min(max(w.first + w.t0 + 1, 0), w.kv_len);
            const int all_lo = c.a.window > 0 ? max(0, w.first + min(w.t0 + c.tokens, w.q_len) - c.a.window) : 0;
            float m = -INFINITY, l = 0.0f;
            for (int j = 0; j < n; ++j) {
                const int k0 = w.lo + j * kTile + side * kKeys;
                const uint32_t b = (g + j) & 1, ts = t_s + b * kTile + lanes;
                wait(s_full(b), ((g + j) >> 1) & 1, 85);
                tc_fence_after();
                uint32_t s[kKeys];
#pragma unroll
                for (int i = 0; i < kKeys; i += 32) tmem_ld32(ts + side * kKeys + i, s + i);
                tmem_wait_ld(s, kKeys);
                if (k0 < all_lo || k0 + kKeys > all_hi) {
#pragma unroll
                    for (int x = 0; x < kKeys; x += 32) {
                        // bit i: key k0 + x + i is seen
                        const int lo = min(max(vis_lo - k0 - x, 0), 32), hi = min(max(vis_hi - k0 - x, 0), 32);
                        const uint32_t seen = (hi == 32 ? 0xFFFFFFFFu : (1u << hi) - 1u) & ~(lo == 32 ? 0xFFFFFFFFu : (1u << lo) - 1u);
#pragma unroll
                        for (int i = 0; i < 32; ++i)
                            if ((seen & (1u << i)) == 0) s[x + i] = 0xFF800000u;       // -inf
                    }
                }
                float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                for (int i = 0; i < kKeys; i += 4)
#pragma unroll
                    for (int e = 0; e < 4; ++e) top[e] = fmaxf(top[e], __uint_as_float(s[i + e]));
                float tile_max = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3])) * scale2;
                // after this the other thread has read its scores too, over which this one's weights will lie
                tile_max = fmaxf(tile_max, swap(tile_max));
                // rows of no token hold anything: they have no say, or the others' last bits would depend on it
                if (__any_sync(0xFFFFFFFFu, mine && tile_max > m + kRaise)) {
                    const float m_new = fmaxf(m, tile_max);
                    const float f = fast_exp2(m - (m_new == -INFINITY ? 0.0f : m_new));
                    if (j > 0) {
                        wait(o_done(b ^ 1), ((g + j - 1) >> 1) & 1, 86);
                        tc_fence_after();
#pragma unroll 1
                        for (int x = 0; x < kCols; x += 32) {
                            const uint32_t to = t_o + lanes + side * kCols + x;
                            uint32_t o[32];
                            tmem_ld32(to, o);
                            tmem_wait_ld(o, 32);
#pragma unroll
                            for (int i = 0; i < 32; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                            tmem_st32(to, o);
                        }
                    }
                    l *= f;
                    m = m_new;
                }
                const float ref = m == -INFINITY ? 0.0f : m;           // a row that has seen nothing yet
                float sum[2] = {0.0f, 0.0f};
                uint32_t pk[32];
#pragma unroll
                for (int i = 0; i < 32; ++i) {
                    const float e0 = fast_exp2(fmaf(__uint_as_float(s[2 * i]), scale2, -ref));
                    const float e1 = fast_exp2(fmaf(__uint_as_float(s[2 * i + 1]), scale2, -ref));
                    sum[0] += e0;
                    sum[1] += e1;
                    pk[i] = pack_bf16(e0, e1);
                }
                tmem_st32(ts + 32 * side, pk);
                l += sum[0] + sum[1];
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) bar_arrive_cluster(in_first_cta(p_full(b)));
            }
            l += swap(l);
            // ---------------- epilogue (before the next work's first weights, so its products do not start yet)
            wait(o_done((g + n - 1) & 1), ((g + n - 1) >> 1) & 1, 87);
            tc_fence_after();
            const bool last = w.pieces == 1;
            const float inv = l == 0.0f ? 0.0f : 1.0f / l;
            if (last) {
                // A thread's own row, 16 bytes at a time, would touch 32 lines a store: four lanes exchange the chunks
                // of their rows, and each store has 64 bytes of eight rows.
                uint16_t* dst = c.a.out + (int64_t)(w.q0 + w.t0 + tok) * c.a.o_t +
                                (int64_t)(w.h * c.group + row_in % c.group) * c.a.o_h + w.half * C::kDv;
                uint16_t* dst4[4];
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    dst4[i] = reinterpret_cast<uint16_t*>(
                                  __shfl_sync(0xFFFFFFFFu, mine ? reinterpret_cast<uintptr_t>(dst) : 0, (lane & ~3) + i));
#pragma unroll 1
                for (int x = side * kCols; x < (side + 1) * kCols; x += 32) {
                    uint32_t o[32];
                    tmem_ld32(t_o + lanes + x, o);
                    tmem_wait_ld(o, 32);
                    uint32_t ch[4][4];
#pragma unroll
                    for (int i = 0; i < 16; ++i)
                        ch[i >> 2][i & 3] = pack_bf16(__uint_as_float(o[2 * i]) * inv, __uint_as_float(o[2 * i + 1]) * inv);
                    quad_transpose(ch, lane);
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (dst4[i] != nullptr)
                            *reinterpret_cast<uint4*>(dst4[i] + x + (lane & 3) * 8) = make_uint4(ch[i][0], ch[i][1], ch[i][2], ch[i][3]);
                }
            } else {
                // partials lie as [4 columns][row], so that a store of 32 rows is contiguous
                const int64_t cta = (int64_t)w.slot * kCtas + rank;
                float* part = c.part_o + cta * kTile * C::kDv + row_in * 4;
#pragma unroll 1
                for (int x = side * kCols; x < (side + 1) * kCols; x += 32) {
                    uint32_t o[32];
                    tmem_ld32(t_o + lanes + x, o);
                    tmem_wait_ld(o, 32);
#pragma unroll
                    for (int i = 0; i < 32; i += 4)
                        *reinterpret_cast<uint4*>(part + (x + i) * kTile) = make_uint4(o[i], o[i + 1], o[i + 2], o[i + 3]);
                }
                if (side == 0) *reinterpret_cast<float2*>(c.part_ml + (cta * kTile + row_in) * 2) = make_float2(m, l);
            }
            tc_fence_before();      // the next first weights say that the output has been read
            g += n;
            ++done;
        }
    }
    if (gave_up) let_copies_land();
    // The pair's MMAs read both CTAs' shared memory and signal both: neither leaves before the other is done.
    tc_fence_before();
    __syncthreads();
    if constexpr (kCtas == 2) {
        cluster_arrive();
        cluster_wait();
    }
    if (warp == 1) {
        tc_fence_after();
        if constexpr (kCtas == 2)
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
        else
            asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(kTmemCols));
    }
}

// Joins the pieces of the last wave's tiles (blockIdx.y), the partials added in piece order. A warp has 32 rows, one a
// lane, and 16 columns.
constexpr int kJoinCols = 16, kJoinWarps = 8;

template <int D>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_chunk_join_kernel(const __grid_constant__ ChunkCall c) {
    using C = ChunkCfg<D>;
    constexpr int kGroups = C::kCtas * kTile / 32;                   // of rows
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    wait_for_predecessor();
    release_successor();
    const Work at = find_work<D, true>(c, blockIdx.y, lane);
    if (at.b < 0 || at.pieces == 1) return;
    const TileWork w = tile_work(c, at.g, at.tile);
    const int unit = blockIdx.x * kJoinWarps + warp, row = unit % kGroups * 32 + lane, col = unit / kGroups * kJoinCols;
    const int r = row % kTile, tok = row / kTile * c.tokens + r / c.group;
    if (r >= c.tokens * c.group || w.t0 + tok >= w.g.q_len) return;
    const int64_t cta = (int64_t)at.slot * C::kCtas + row / kTile;   // of the first piece
    const float* part = c.part_o + cta * kTile * C::kDv + (col * kTile + r * 4);
    const float* ml = c.part_ml + (cta * kTile + r) * 2;
    constexpr int kBatch = 4;
    float acc[kJoinCols];
#pragma unroll
    for (int e = 0; e < kJoinCols; ++e) acc[e] = 0.0f;
    float top = -INFINITY, sum = 0.0f;
    for (int z0 = 0; z0 < at.pieces; z0 += kBatch) {
        float2 s[kBatch];
        float4 v[kBatch][kJoinCols / 4];
#pragma unroll
        for (int z = 0; z < kBatch; ++z) {
            s[z] = make_float2(-INFINITY, 0.0f);
#pragma unroll
            for (int e = 0; e < kJoinCols / 4; ++e) v[z][e] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (z0 + z < at.pieces) {
                s[z] = *reinterpret_cast<const float2*>(ml + (int64_t)(z0 + z) * C::kCtas * kTile * 2);
#pragma unroll
                for (int e = 0; e < kJoinCols / 4; ++e)
                    v[z][e] = *reinterpret_cast<const float4*>(part + (int64_t)(z0 + z) * C::kCtas * kTile * C::kDv + e * 4 * kTile);
            }
        }
        float now = top;
#pragma unroll
        for (int z = 0; z < kBatch; ++z) now = fmaxf(now, s[z].x);
        const float ref = now == -INFINITY ? 0.0f : now, back = fast_exp2(top - ref);
        top = now;
        sum *= back;
#pragma unroll
        for (int e = 0; e < kJoinCols; ++e) acc[e] *= back;
#pragma unroll
        for (int z = 0; z < kBatch; ++z) {
            const float f = fast_exp2(s[z].x - ref);
            sum += f * s[z].y;
#pragma unroll
            for (int e = 0; e < kJoinCols / 4; ++e) {
                acc[4 * e] += f * v[z][e].x;
                acc[4 * e + 1] += f * v[z][e].y;
                acc[4 * e + 2] += f * v[z][e].z;
                acc[4 * e + 3] += f * v[z][e].w;
            }
        }
    }
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    uint16_t* dst = c.a.out + (int64_t)(w.g.q0 + w.t0 + tok) * c.a.o_t + (int64_t)(at.h * c.group + r % c.group) * c.a.o_h +
                    at.half * C::kDv + col;
#pragma unroll
    for (int e = 0; e < kJoinCols; e += 8) {
        uint32_t pk[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) pk[i] = pack_bf16(acc[e + 2 * i] * inv, acc[e + 2 * i + 1] * inv);
        *reinterpret_cast<uint4*>(dst + e) = make_uint4(pk[0], pk[1], pk[2], pk[3]);
    }
}

template <int D>
void launch_chunk_dim(const Attn& hd, const AttnCall& a, int few_rows, cudaStream_t st) {
    using C = ChunkCfg<D>;
    static bool attr_set[64] = {false};
    const int dev = current_device();
    if (!attr_set[dev & 63]) {
        check_cuda(cudaFuncSetAttribute(attn_chunk_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem),
                   "cudaFuncSetAttribute(attn_chunk)");
        attr_set[dev & 63] = true;
    }
    ChunkCall c;
    c.a = a;
    c.group = a.hq / a.hk;
    c.few_rows = few_rows;
    c.tokens = kTile / c.group;
    c.tile_tokens = c.tokens * C::kCtas;
    c.box = std::min(1 << a.pv.page_shift, 64);
    c.box_shift = std::min(a.pv.page_shift, 6);
    c.wave = device_sm_count() / C::kCtas;
    c.by_tile_tokens = Divisor(c.tile_tokens);
    c.by_wave = Divisor(c.wave);
    c.by_per_tile = Divisor(a.hk * C::kHalves);
    // a sequence has at most one tile that is not full
    const int64_t tiles = std::min<int64_t>((int64_t)a.pv.rows / c.tile_tokens + a.pv.n_seqs,
                                            (int64_t)a.pv.n_seqs * ((a.pv.max_q + c.tile_tokens - 1) / c.tile_tokens));
    if ((tiles * a.hk * C::kHalves + c.wave) * kMaxSplits > 0x7FFFFFFF)
        throw Error(G4Q_ERR_INVALID_ARGUMENT, "too many rows for one call");
    // as many as run at once, unless there can be less work
    int64_t cap = (int64_t)a.pv.max_pages << a.pv.page_shift;
    if (a.window > 0) cap = std::min<int64_t>(cap, (int64_t)a.window + c.tile_tokens + c.box);
    const int64_t key_tiles = (cap + kTile - 1) / kTile, items = tiles * a.hk * C::kHalves, rest = items % c.wave;
    c.max_pieces = (int)std::min<int64_t>(kMaxSplits, std::max<int64_t>(1, key_tiles / kMinPieceAlone));
    // Sequences of one length: the tiles are known here, and where none will be cut there is nothing to join (an empty
    // join costs 6 us).
    const bool known = (int64_t)a.pv.n_seqs * a.pv.max_q == a.pv.rows;
    if (known && (rest * 2 > c.wave || rest == 0 || (items > c.wave && key_tiles / kMinPiece < 2))) c.max_pieces = 1;
    c.clusters = (int)std::min<int64_t>(c.wave, items * c.max_pieces);
    c.part_o = hd.part_o;
    c.part_ml = hd.part_ml;
    c.err = device_scratch().err;
    const CUtensorMap tq = rows_map(a.q, a.q_t, a.q_h, a.hq, a.pv.rows, D, c.group, c.tokens);
    const CUtensorMap tk = paged_map(a, a.k, D, c.box), tv = paged_map(a, a.v, D, c.box);
    launch_dependent<C::kCtas>(attn_chunk_kernel<D>, dim3((unsigned)(c.clusters * C::kCtas)), dim3(kThreads), C::kSmem, st, tq,
                               tk, tv, c);
    const int cut = (int)std::min<int64_t>(c.wave / 2, items);   // a wave holds two pieces of each
    if (c.max_pieces > 1 && cut > 0)   // else no tile is long enough for two pieces
        launch_dependent(attn_chunk_join_kernel<D>,
                         dim3(C::kCtas * kTile / 32 * (C::kDv / kJoinCols) / kJoinWarps, (unsigned)cut), dim3(kJoinWarps * 32), 0,
                         st, c);
}

}  // namespace

size_t chunk_part_rows() { return (size_t)device_sm_count() * kTile; }   // split launches have at most one CTA per SM

void launch_chunk(const Attn& h, const AttnCall& a, int few_rows, cudaStream_t st) {
    switch (h.head_dim) {
        case 64: return launch_chunk_dim<64>(h, a, few_rows, st);
        case 128: return launch_chunk_dim<128>(h, a, few_rows, st);
        case 256: return launch_chunk_dim<256>(h, a, few_rows, st);
        case 512: return launch_chunk_dim<512>(h, a, few_rows, st);
    }
}

}  // namespace g4q
