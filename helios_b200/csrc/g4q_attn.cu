// g4q_attn.cu -- attention of a few new tokens per sequence over a paged cache (sm_100a): one decoded token
// each, or a block of drafted ones, up to 64 query rows (tokens x query heads of a key head) per key head (32 at
// head_dim 512; in a step that has longer sequences too 16, or the rows of one token).
//
//   out = softmax(scale * q k^T + mask) v, masked to the positions j <= t (and j > t - window)
//
// Bound by HBM: K and V are read once, for all the query heads of the group, and everything else is small.
// The work is a list of (sequence, key head, 64-key tile), cut into equal contiguous ranges of tiles, one per
// CTA: every SM streams the same number of bytes whatever the lengths are, and the TMA ring runs on from one
// sequence to the next without a pause. A range that ends inside a sequence leaves its fp32 partial
// (unnormalized output, running maximum and sum per row) in the handle's scratch, at most two per CTA, and a
// second kernel, launched while the first one drains, joins a sequence's partials in CTA order, so results do not
// depend on timing. (Having the CTA that comes last join them instead was slower: one token over a window of 1024,
// 10.4 us against 8.8; the last CTA waits for its stores, its ticket and the others' partials one after another.)
//
// In a CTA one warp feeds the ring (SWIZZLE_128B boxes of one page x 64 elements) and eight compute warps
// share each tile: for the scores, warp w takes keys 8w..8w+7 against all query rows (mma.sync, rows padded
// to 16); the running softmax is in fp32 over 16-key slices per thread; for the output, warp w takes head_dim/8
// columns over the 64 keys. mma.sync is enough here: at 64 rows a tile's products take less time than its bytes.
//
// Measured, with the join, a call with new inputs (in brackets: with the same ones in a graph): 16 tokens over 69,823 keys
// in all (8 key heads of 256) 98 us (96), 5.8 TB/s of keys and values; one token over a window of 1024 8.7 us (8.0) and
// over 16384 keys of head_dim 512 16.1 us (12.4), latencies of a tile or two in sequence and of the join.
#include <cuda_runtime.h>

#include <algorithm>

#include "g4q_attn.cuh"
#include "g4q_common.cuh"
#include "g4q_internal.h"

namespace g4q {
namespace {

// Rows per key head that this kernel takes. At head_dim 512 the registers end at 32: blocks of 4 tokens x 16 heads of two
// sequences of 16000 keys take 56 us here with spills, 41 in the chunk kernel (of 2049 and 4000 keys 25.7 and 26.6).
constexpr int few_rows(int head_dim) { return head_dim == 512 ? 32 : 64; }
constexpr int kKeys = 64;            // keys per tile
constexpr int kComputeWarps = 8;
constexpr int kThreads = (kComputeWarps + 1) * 32;
constexpr float kLog2e = 1.4426950408889634f;
// Few units (sequence x key head) of few tiles, 16 rows at most and head_dim up to 256: a cluster of 8 CTAs has a unit to
// itself and joins its partials in shared memory; there is no second launch. A CTA may have up to 3 tiles, and one more
// than an even split over the GPU gives. One token over 300 keys, four sequences: 6.0 us against 8.4; four over a window of
// 1024: 9.6 and 12.1; blocks of 8, of four sequences: 11.2 and 13.3. One token over a window of 1024 has one tile a CTA in
// the even split and three here: 9.6 us and 8.7, its keys coming from memory. With more rows or at head_dim 512, where a
// tile takes longer and one CTA fits an SM, fewer CTAs a unit cost more than the launch (15 tokens of two sequences, window
// of 1024: 20.7 and 13.7; 1500 keys of head_dim 512, four sequences: 12.7 and 10.1).
constexpr int kUnitCtas = 8, kUnitTiles = 3;
template <int D, int MT>
constexpr bool kUnitClusters = MT == 1 && D <= 256;
constexpr float kNoTiles = -1.0f;    // in the place of a CTA's sums, which are not negative

template <int D, int MT>
struct FewCfg {
    static constexpr int kRows = 16 * MT;
    static constexpr int kCols = D < 256 ? D : 256;          // elements of a ring stage's rows
    static constexpr int kParts = D / kCols;                 // stages of one K (or V) tile
    static constexpr int kStageBytes = kKeys * kCols * 2;
    static constexpr int kQBytes = kRows * D * 2;
    static constexpr int kSLd = kKeys + 8;                   // fp32 row stride of the scores: conflict free
    static constexpr int kSBytes = kRows * kSLd * 4;
    static constexpr int kPBytes = kRows * kKeys * 2;
    static constexpr int kFixed = kQBytes + kSBytes + kPBytes + kRows * 12 + 256 + 1024;
    // two CTAs per SM where three stages each fit (one CTA's prologue and combine then hide behind the other);
    // else one CTA with the ring as deep as fits
    static constexpr bool kTwo = kFixed + 3 * kParts * kStageBytes <= 113 * 1024 && kParts == 1;
    static constexpr int kFit = ((kTwo ? 113 : 226) * 1024 - kFixed) / kStageBytes;
    static constexpr int kStages = kFit > 8 ? 8 : kFit;
    static constexpr int kSmem = kFixed + kStages * kStageBytes;
    static_assert(kStages >= 2 * kParts && kSmem <= 227 * 1024, "ring does not fit");
    static_assert(kRows * D * 4 <= kStages * kStageBytes, "a partial takes the ring's place");
};

struct FewCall {
    AttnCall a;
    int group;          // query heads per key head
    int max_rows;       // sequences of more rows (tokens x group) belong to the chunk kernel
    int box;            // keys per TMA box: min(page_size, 64)
    int ctas;
    int part_rows;      // rows of a partial
    float* part_o;      // [2 * ctas][part_rows][D]
    float* part_ml;     // [2 * ctas][part_rows][2]
    int* err;           // wait-error word
};

struct SeqWork {
    SeqGeom g;
    int lo;             // first key of the first tile
    int nt;             // 64-key tiles, 0: nothing for this kernel
};

__device__ __forceinline__ SeqWork seq_work(const FewCall& c, int b) {
    SeqWork w;
    w.g = seq_geom(c.a.pv, b);
    w.lo = 0;
    w.nt = 0;
    if (w.g.q_len == 0 || w.g.q_len * c.group > c.max_rows) return w;
    if (c.a.window > 0) w.lo = min(max(0, w.g.first - c.a.window + 1), w.g.kv_len) & ~(c.box - 1);
    w.nt = max(1, (w.g.kv_len - w.lo + kKeys - 1) / kKeys);   // a sequence without keys still writes zeros
    return w;
}

// The list of tiles cut into equal contiguous ranges: the first `more` CTAs have base + 1 tiles, the others base.
struct Ranges {
    uint32_t base, more;
    __device__ __forceinline__ Ranges(uint32_t total, int ctas) : base(total / ctas), more(total % ctas) {}
    __device__ __forceinline__ uint32_t first(uint32_t cta) const { return cta * base + min(cta, more); }
    __device__ __forceinline__ uint32_t owner(uint32_t tile) const {
        const uint32_t cut = more * (base + 1);
        return tile < cut ? tile / (base + 1) : more + (tile - cut) / base;
    }
};

__device__ __forceinline__ uint32_t warp_scan(uint32_t v, int lane) {   // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const uint32_t t = __shfl_up_sync(0xFFFFFFFFu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}

// A position in the list of tiles.
struct Cursor {
    int b, h, t;        // sequence, key head, tile
    SeqWork w;
    __device__ __forceinline__ void next_unit(const FewCall& c) {
        t = 0;
        if (++h < c.a.hk) return;
        h = 0;
        do {
            ++b;
            if (b < c.a.pv.n_seqs) w = seq_work(c, b);
        } while (b < c.a.pv.n_seqs && w.nt == 0);
    }
};

// This CTA's first tile, and how many it has. Every warp finds it by itself: handing it over through shared memory
// costs a barrier and another round of loads at the start, where nothing else can run.
__device__ __forceinline__ Cursor first_place(const FewCall& c, int lane, int& left) {
    auto work_of = [&](int b) {
        SeqWork w;
        w.g.q0 = w.g.q_len = w.g.first = w.g.kv_len = w.lo = w.nt = 0;
        if (b < c.a.pv.n_seqs) w = seq_work(c, b);
        return w;
    };
    SeqWork w = work_of(lane);                       // the first 32 sequences stay in registers
    uint32_t inc = warp_scan(w.nt * c.a.hk, lane), total = __shfl_sync(0xFFFFFFFFu, inc, 31);
    for (int b0 = 32; b0 < c.a.pv.n_seqs; b0 += 32)
        total += __shfl_sync(0xFFFFFFFFu, warp_scan(work_of(b0 + lane).nt * c.a.hk, lane), 31);
    const Ranges ranges(total, c.ctas);
    const uint32_t t0 = ranges.first(blockIdx.x);
    Cursor cur;
    cur.b = cur.h = cur.t = 0;
    left = (int)(ranges.first(blockIdx.x + 1) - t0);
    uint32_t before = 0;
    for (int b0 = 0; b0 < c.a.pv.n_seqs && left > 0; b0 += 32) {
        if (b0 > 0) {
            w = work_of(b0 + lane);
            inc = warp_scan(w.nt * c.a.hk, lane);
        }
        const unsigned past = __ballot_sync(0xFFFFFFFFu, before + inc > t0);
        if (past != 0) {
            const int at = __ffs(past) - 1;
            cur.b = b0 + at;
            cur.w.g.q0 = __shfl_sync(0xFFFFFFFFu, w.g.q0, at);
            cur.w.g.q_len = __shfl_sync(0xFFFFFFFFu, w.g.q_len, at);
            cur.w.g.first = __shfl_sync(0xFFFFFFFFu, w.g.first, at);
            cur.w.g.kv_len = __shfl_sync(0xFFFFFFFFu, w.g.kv_len, at);
            cur.w.lo = __shfl_sync(0xFFFFFFFFu, w.lo, at);
            cur.w.nt = __shfl_sync(0xFFFFFFFFu, w.nt, at);
            const uint32_t rest = t0 - (before + __shfl_sync(0xFFFFFFFFu, inc, at) - (uint32_t)cur.w.nt * c.a.hk);
            cur.h = (int)(rest / (uint32_t)cur.w.nt);
            cur.t = (int)(rest % (uint32_t)cur.w.nt);
            break;
        }
        before += __shfl_sync(0xFFFFFFFFu, inc, 31);
    }
    return cur;
}

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(addr) : "memory");
}

__device__ __forceinline__ void ldmatrix4t(uint32_t addr, uint32_t& a, uint32_t& b, uint32_t& c, uint32_t& d) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a), "=r"(b), "=r"(c), "=r"(d) : "r"(addr) : "memory");
}

__device__ __forceinline__ void compute_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

// Clusters: a unit's tiles belong to the kUnitCtas CTAs of a cluster, whose partials stay in shared memory and are
// joined there.
__device__ __forceinline__ uint32_t in_cta(uint32_t addr, int rank) {
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ float ld_cluster(uint32_t addr) {
    float v;
    asm volatile("ld.shared::cluster.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ float4 ld_cluster4(uint32_t addr) {
    float4 v;
    asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
                 : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

template <int D, int MT, bool kCluster>
__global__ void __launch_bounds__(kThreads, FewCfg<D, MT>::kTwo ? 2 : 1)
    attn_few_kernel(const __grid_constant__ CUtensorMap tm_k, const __grid_constant__ CUtensorMap tm_v,
                    const __grid_constant__ FewCall c) {
    using C = FewCfg<D, MT>;
    extern __shared__ uint8_t smem_raw[];
    const uint32_t base = (smem_addr(smem_raw) + 1023u) & ~1023u;
    uint8_t* gen = smem_raw + (base - smem_addr(smem_raw));
    const uint32_t s_ring = base;
    const uint32_t s_q = s_ring + C::kStages * C::kStageBytes;
    const uint32_t s_p = s_q + C::kQBytes;
    const uint32_t s_bar = s_p + C::kPBytes;
    float* s_s = reinterpret_cast<float*>(gen + (s_bar - base) + 256);
    float* s_alpha = s_s + C::kRows * C::kSLd;       // rescaling factor of a row's output
    float* s_sum = s_alpha + C::kRows;
    float* s_max = s_sum + C::kRows;
    auto full = [&](int s) { return s_bar + 8u * s; };
    auto empty = [&](int s) { return s_bar + 8u * (C::kStages + s); };

    bool gave_up = false;
    auto wait = [&](uint32_t bar, uint32_t parity, int code) {
        if (!bar_wait(bar, parity, c.err, code)) gave_up = true;
    };

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == kComputeWarps * 32) {
        for (int s = 0; s < C::kStages; ++s) {
            bar_init(full(s), 1);
            bar_init(empty(s), 1);
        }
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_k)) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(reinterpret_cast<uint64_t>(&tm_v)) : "memory");
    }
    __syncthreads();
    wait_for_predecessor();
    release_successor();
    int left;
    Cursor cur;
    if constexpr (kCluster) {
        const int unit = blockIdx.x / kUnitCtas, rank = blockIdx.x % kUnitCtas;
        cur.b = unit / c.a.hk;
        cur.h = unit % c.a.hk;
        cur.w = seq_work(c, cur.b);
        cur.t = cur.w.nt * rank / kUnitCtas;
        left = cur.w.nt * (rank + 1) / kUnitCtas - cur.t;
        if (left == 0 && threadIdx.x < C::kRows) {
            s_max[threadIdx.x] = -INFINITY;
            s_sum[threadIdx.x] = kNoTiles;
        }
    } else {
        cur = first_place(c, lane, left);
    }
    if (left > 0) {
        if (warp == kComputeWarps) {
            // ---------------- producer: K then V of every tile, in ring order
            int stage = 0;
            uint32_t round = 0;
            const int boxes = kKeys / c.box;
            const PagedView& pv = c.a.pv;
            const int page_mask = (1 << pv.page_shift) - 1;
            const uint32_t box_bytes = (uint32_t)c.box * 128u;
            while (left > 0) {
                const int k0 = cur.w.lo + cur.t * kKeys;
                // the boxes that hold a key of the sequence; the others are zeroed (V) or masked (K)
                const int nb = min(boxes, (cur.w.g.kv_len - k0 + c.box - 1) / c.box);
#pragma unroll 1
                for (int part = 0; part < 2 * C::kParts; ++part) {
                    if (round > 0) wait(empty(stage), (round - 1) & 1, 70);
                    const CUtensorMap* map = part < C::kParts ? &tm_k : &tm_v;
                    const int col0 = (part % C::kParts) * C::kCols;
                    if (lane == 0) bar_expect_tx(full(stage), (uint32_t)max(nb, 0) * box_bytes * (C::kCols / 64));
                    __syncwarp();
                    for (int i = lane; i < nb * (C::kCols / 64); i += 32) {
                        const int box = i / (C::kCols / 64), cb = i % (C::kCols / 64);
                        const int key = k0 + box * c.box;
                        int page = pv.table[cur.b * pv.table_ld + (key >> pv.page_shift)];
                        if (page < 0 || page >= pv.n_pages) {
                            record_input_error(pv.err, kErrPage);
                            page = pv.n_pages;                 // outside the map: reads zeros
                        }
                        tma_load_page(s_ring + stage * C::kStageBytes + cb * (kKeys * 128) + box * box_bytes, map,
                                      col0 + cb * 64, key & page_mask, cur.h, page, full(stage));
                    }
                    if (++stage == C::kStages) stage = 0, ++round;
                }
                --left;
                if (++cur.t == cur.w.nt && left > 0) cur.next_unit(c);
            }
        } else {
            // ---------------- compute
            constexpr int kTpr = 256 / C::kRows;             // threads per row in the softmax
            constexpr int kKpt = kKeys / kTpr;               // keys per thread
            constexpr int kNt = D / 64;                      // 8-column tiles per warp in the output
            const int gi = lane >> 2, t4 = lane & 3;
            const int srow = threadIdx.x / kTpr, sj = threadIdx.x % kTpr;
            const float scale2 = c.a.scale * kLog2e;
            int stage = 0, v_held = -1;      // v_held: V stage(s) not handed back yet
            uint32_t round = 0;
            while (left > 0) {
                // one unit: the tiles of (b, h) in this CTA's range
                const SeqGeom g = cur.w.g;
                const int rows = g.q_len * c.group;
                const int n = min(left, cur.w.nt - cur.t);
                const bool whole = n == cur.w.nt, first_part = cur.t > 0;
                constexpr int kPieces = C::kRows * (D / 8), kLoads = (kPieces + 255) / 256;
                uint4 qv[kLoads];
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const int r = (threadIdx.x + i * 256) / (D / 8), ch = (threadIdx.x + i * 256) % (D / 8);
                    qv[i] = make_uint4(0, 0, 0, 0);
                    if (r < rows) {      // rows <= kRows
                        const int tok = r / c.group, hd = cur.h * c.group + r % c.group;
                        qv[i] = *reinterpret_cast<const uint4*>(c.a.q + (int64_t)(g.q0 + tok) * c.a.q_t + (int64_t)hd * c.a.q_h + ch * 8);
                    }
                }
#pragma unroll
                for (int i = 0; i < kLoads; ++i) {
                    const int r = (threadIdx.x + i * 256) / (D / 8), ch = (threadIdx.x + i * 256) % (D / 8);
                    if (kPieces % 256 == 0 || r < C::kRows)
                        *reinterpret_cast<uint4*>(gen + (s_q - base) + (ch >> 3) * (C::kRows * 128) + r * 128 +
                                                  (((ch & 7) ^ (r & 7)) << 4)) = qv[i];
                }
                // keys a row sees: [vis_lo, vis_hi)
                int vis_lo = 0, vis_hi = 0;
                if (srow < rows) {
                    const int pos = g.first + srow / c.group;
                    vis_hi = min(max(0, pos + 1), g.kv_len);
                    if (c.a.window > 0) vis_lo = max(0, pos - c.a.window + 1);
                }
                // keys some row of the unit sees: V outside of them is not looked at (it may hold anything)
                const int any_lo = c.a.window > 0 ? max(0, g.first - c.a.window + 1) : 0;
                float m = -INFINITY, l = 0.0f;
                float o[MT][kNt][4];
#pragma unroll
                for (int a = 0; a < MT; ++a)
#pragma unroll
                    for (int b = 0; b < kNt; ++b)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[a][b][e] = 0.0f;
                compute_sync();
                for (int it = 0; it < n; ++it) {
                    const int k0 = cur.w.lo + (cur.t + it) * kKeys;
                    // ---- scores of keys 8w..8w+7
                    // two sums per score, of the even and the odd products: half the chain of dependent MMAs
                    float s[MT][2][4];
#pragma unroll
                    for (int a = 0; a < MT; ++a)
#pragma unroll
                        for (int e = 0; e < 8; ++e) s[a][e >> 2][e & 3] = 0.0f;
                    int st = stage;
                    uint32_t rd = round;
#pragma unroll
                    for (int part = 0; part < C::kParts; ++part) {
                        wait(full(st), rd & 1, 71);
                        const uint32_t kb = s_ring + st * C::kStageBytes + (8 * warp + (lane & 7)) * 128;
#pragma unroll(MT == 1 ? 8 : 2)
                        for (int kk = 0; kk < C::kCols / 32; ++kk) {
                            const int dc = kk * 4 + (lane >> 3);             // 16-byte chunk of this lane's row
                            uint32_t b0, b1, b2, b3;
                            ldmatrix4(kb + (dc >> 3) * (kKeys * 128) + (((dc & 7) ^ (lane & 7)) << 4), b0, b1, b2, b3);
#pragma unroll
                            for (int a = 0; a < MT; ++a) {
#pragma unroll
                                for (int half = 0; half < 2; ++half) {
                                    const int qc = part * (C::kCols / 8) + kk * 4 + half * 2 + (lane >> 4);
                                    const int qr = 16 * a + (lane & 15);
                                    uint32_t a0, a1, a2, a3;
                                    ldmatrix4(s_q + (qc >> 3) * (C::kRows * 128) + qr * 128 + (((qc & 7) ^ (qr & 7)) << 4),
                                              a0, a1, a2, a3);
                                    mma_bf16_16816(s[a][half], a0, a1, a2, a3, half ? b2 : b0, half ? b3 : b1);
                                }
                            }
                        }
                        if (++st == C::kStages) st = 0, ++rd;
                    }
#pragma unroll
                    for (int a = 0; a < MT; ++a) {
                        float* sr = s_s + (16 * a + gi) * C::kSLd + 8 * warp + 2 * t4;
                        *reinterpret_cast<float2*>(sr) = make_float2(s[a][0][0] + s[a][1][0], s[a][0][1] + s[a][1][1]);
                        *reinterpret_cast<float2*>(sr + 8 * C::kSLd) =
                            make_float2(s[a][0][2] + s[a][1][2], s[a][0][3] + s[a][1][3]);
                    }
                    compute_sync();
                    // every warp is past this tile's K and the previous tile's V
                    if (threadIdx.x == 0) {
#pragma unroll
                        for (int part = 0; part < C::kParts; ++part) {
                            bar_arrive(empty((stage + part) % C::kStages));
                            if (v_held >= 0) bar_arrive(empty((v_held + part) % C::kStages));
                        }
                    }
                    stage = st;
                    round = rd;
                    v_held = st;
                    // ---- running softmax: thread (srow, sj) has keys sj * kKpt ..
                    {
                        float x[kKpt];
                        float top = -INFINITY;
#pragma unroll
                        for (int i = 0; i < kKpt; i += 4) {
                            const float4 v = *reinterpret_cast<const float4*>(s_s + srow * C::kSLd + sj * kKpt + i);
                            x[i] = v.x, x[i + 1] = v.y, x[i + 2] = v.z, x[i + 3] = v.w;
                        }
#pragma unroll
                        for (int i = 0; i < kKpt; ++i) {
                            const int key = k0 + sj * kKpt + i;
                            x[i] = key >= vis_lo && key < vis_hi ? x[i] * scale2 : -INFINITY;
                            top = fmaxf(top, x[i]);
                        }
#pragma unroll
                        for (int w = kTpr / 2; w > 0; w >>= 1) top = fmaxf(top, __shfl_xor_sync(0xFFFFFFFFu, top, w));
                        const float m_new = fmaxf(m, top);
                        const float ref = m_new == -INFINITY ? 0.0f : m_new;      // a row that sees nothing yet
                        const float alpha = fast_exp2(m - ref);
                        m = m_new;
                        float sum = 0.0f;
                        uint32_t pk[kKpt / 2];
#pragma unroll
                        for (int i = 0; i < kKpt; i += 2) {
                            const float e0 = fast_exp2(x[i] - ref), e1 = fast_exp2(x[i + 1] - ref);
                            pk[i / 2] = pack_bf16(e0, e1);
                            // the sum takes the weights as the product will: their bf16 rounding cancels in part
                            sum += bf16_bits_to_f32(pk[i / 2] & 0xFFFFu) + __uint_as_float(pk[i / 2] & 0xFFFF0000u);
                        }
#pragma unroll
                        for (int w = kTpr / 2; w > 0; w >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, w);
                        l = l * alpha + sum;
                        if (sj == 0) s_alpha[srow] = alpha;
                        uint8_t* pr = gen + (s_p - base) + srow * 128;
#pragma unroll
                        for (int i = 0; i < kKpt / 2; i += 2) {
                            const int byte = sj * kKpt * 2 + i * 4;
                            *reinterpret_cast<uint2*>(pr + (((byte >> 4) ^ (srow & 7)) << 4) + (byte & 15)) =
                                make_uint2(pk[i], pk[i + 1]);
                        }
                    }
                    // ---- V rows that no row of the unit sees become zeros (a zero weight times NaN is NaN)
                    if (k0 < any_lo || k0 + kKeys > g.kv_len) {
                        int vs = stage;
                        uint32_t vr = round;
#pragma unroll
                        for (int part = 0; part < C::kParts; ++part) {
                            wait(full(vs), vr & 1, 72);
                            uint8_t* vb = gen + (s_ring - base) + vs * C::kStageBytes;
                            for (int i = threadIdx.x; i < kKeys * (C::kCols / 8); i += 256) {
                                const int key = (i >> 3) & (kKeys - 1);
                                if (k0 + key < any_lo || k0 + key >= g.kv_len)
                                    *reinterpret_cast<uint4*>(vb + i * 16) = make_uint4(0, 0, 0, 0);
                            }
                            if (++vs == C::kStages) vs = 0, ++vr;
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");   // before the stage's next copy
                    }
                    compute_sync();
                    // ---- output columns of this warp
                    {
                        constexpr int kWarpCols = D / kComputeWarps;
                        const int col = warp * kWarpCols;                     // first column of this warp
                        const int part = col / C::kCols, pc = col % C::kCols;
                        int vs = stage + part;
                        uint32_t vr = round;
                        if (vs >= C::kStages) vs -= C::kStages, ++vr;
                        wait(full(vs), vr & 1, 73);
                        const uint32_t vb = s_ring + vs * C::kStageBytes;
#pragma unroll
                        for (int a = 0; a < MT; ++a) {
                            const float f0 = s_alpha[16 * a + gi], f1 = s_alpha[16 * a + gi + 8];
#pragma unroll
                            for (int b = 0; b < kNt; ++b) {
                                o[a][b][0] *= f0, o[a][b][1] *= f0;
                                o[a][b][2] *= f1, o[a][b][3] *= f1;
                            }
                        }
#pragma unroll(MT == 1 ? 4 : 1)
                        for (int kk = 0; kk < kKeys / 16; ++kk) {
                            uint32_t pa[MT][4];
#pragma unroll
                            for (int a = 0; a < MT; ++a) {
                                const int pr = 16 * a + (lane & 15), ch = kk * 2 + (lane >> 4);
                                ldmatrix4(s_p + pr * 128 + ((ch ^ (pr & 7)) << 4), pa[a][0], pa[a][1], pa[a][2], pa[a][3]);
                            }
                            const int key = kk * 16 + (lane & 15);
#pragma unroll
                            for (int b = 0; b < kNt; b += 2) {
                                uint32_t v0, v1, v2 = 0, v3 = 0;
                                // D = 64 has one 8-column tile per warp: the upper half re-reads the same chunk
                                const int ch = (pc >> 3) + b + (kNt > 1 ? (lane >> 4) : 0);
                                ldmatrix4t(vb + (ch >> 3) * (kKeys * 128) + key * 128 + (((ch & 7) ^ (key & 7)) << 4), v0, v1,
                                           v2, v3);
#pragma unroll
                                for (int a = 0; a < MT; ++a) {
                                    mma_bf16_16816(o[a][b], pa[a][0], pa[a][1], pa[a][2], pa[a][3], v0, v1);
                                    if constexpr (kNt > 1)
                                        mma_bf16_16816(o[a][b + 1], pa[a][0], pa[a][1], pa[a][2], pa[a][3], v2, v3);
                                }
                            }
                        }
                    }
                    stage += C::kParts;
                    if (stage >= C::kStages) stage -= C::kStages, ++round;
                }
                // ---- the unit's rows: final, or this CTA's partial
                if (sj == 0) {
                    s_sum[srow] = l;
                    s_max[srow] = m;
                }
                compute_sync();
                const int64_t slot = (int64_t)blockIdx.x * 2 + (first_part ? 0 : 1);
#pragma unroll
                for (int a = 0; a < MT; ++a) {
#pragma unroll
                    for (int half = 0; half < 2; ++half) {
                        const int r = 16 * a + gi + 8 * half;
                        if (r >= rows) continue;
                        const float sum = s_sum[r];
                        const int col = warp * (D / kComputeWarps) + 2 * t4;
                        if constexpr (kCluster) {
                            float* dst = reinterpret_cast<float*>(gen) + r * D + col;    // the ring has been read
#pragma unroll
                            for (int b = 0; b < kNt; ++b)
                                *reinterpret_cast<float2*>(dst + 8 * b) = make_float2(o[a][b][2 * half], o[a][b][2 * half + 1]);
                        } else if (whole) {
                            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;   // a row that sees nothing is zero
                            const int tok = r / c.group, hd = cur.h * c.group + r % c.group;
                            uint16_t* dst = c.a.out + (int64_t)(g.q0 + tok) * c.a.o_t + (int64_t)hd * c.a.o_h + col;
#pragma unroll
                            for (int b = 0; b < kNt; ++b)
                                *reinterpret_cast<uint32_t*>(dst + 8 * b) =
                                    pack_bf16(o[a][b][2 * half] * inv, o[a][b][2 * half + 1] * inv);
                        } else {
                            float* dst = c.part_o + (slot * c.part_rows + r) * D + col;
#pragma unroll
                            for (int b = 0; b < kNt; ++b)
                                *reinterpret_cast<float2*>(dst + 8 * b) = make_float2(o[a][b][2 * half], o[a][b][2 * half + 1]);
                            if (warp == 0 && t4 == 0)
                                *reinterpret_cast<float2*>(c.part_ml + (slot * c.part_rows + r) * 2) = make_float2(s_max[r], sum);
                        }
                    }
                }
                left -= n;
                cur.t += n;
                if (left > 0) cur.next_unit(c);
            }
        }
    }
    if (gave_up) let_copies_land();
    if constexpr (kCluster) {
        __syncwarp();
        cluster_sync();      // no CTA leaves before the second one: the others read its shared memory
        // each CTA joins its share of the unit's rows and columns, four columns a thread, in rank order
        const SeqGeom g = cur.w.g;
        const int rank = blockIdx.x % kUnitCtas, rows = cur.w.nt > 0 ? g.q_len * c.group : 0, items = rows * (D / 4);
        const int end = items * (rank + 1) / kUnitCtas;
        for (int i = items * rank / kUnitCtas + (int)threadIdx.x; i < end; i += kThreads) {
            const int r = i / (D / 4), col = i % (D / 4) * 4;
            float top = -INFINITY, m[kUnitCtas], l[kUnitCtas];
#pragma unroll
            for (int k = 0; k < kUnitCtas; ++k) {
                m[k] = ld_cluster(in_cta(smem_addr(s_max + r), k));
                l[k] = ld_cluster(in_cta(smem_addr(s_sum + r), k));
                top = fmaxf(top, m[k]);
            }
            const float ref = top == -INFINITY ? 0.0f : top;
            float sum = 0.0f;
            float4 acc = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < kUnitCtas; ++k) {
                if (l[k] == kNoTiles) continue;      // its shared memory may hold anything
                const float f = fast_exp2(m[k] - ref);
                const float4 v = ld_cluster4(in_cta(base + (r * D + col) * 4, k));
                sum += f * l[k];
                acc.x += f * v.x, acc.y += f * v.y, acc.z += f * v.z, acc.w += f * v.w;
            }
            const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
            const int tok = r / c.group, hd = cur.h * c.group + r % c.group;
            *reinterpret_cast<uint2*>(c.a.out + (int64_t)(g.q0 + tok) * c.a.o_t + (int64_t)hd * c.a.o_h + col) =
                make_uint2(pack_bf16(acc.x * inv, acc.y * inv), pack_bf16(acc.z * inv, acc.w * inv));
        }
        cluster_sync();
    }
}

// Joins the partials of the units that CTA ranges cut. An item is 128 columns of one row of a unit; kWpi warps of
// a block share it: they take the unit's partials in turn, in CTA order, and their sums are added in warp order.
constexpr int kJoinBatch = 10;

template <int D, int kWpi, int kJoinWarps>
__global__ void __launch_bounds__(kJoinWarps * 32) attn_join_kernel(const __grid_constant__ FewCall c) {
    constexpr int kW = D < 128 ? D : 128;        // columns of an item
    constexpr int kV = kW / 32;                  // per lane
    constexpr int kItems = kJoinWarps / kWpi;    // of a block: consecutive rows
    __shared__ float s_top[kJoinWarps], s_sum[kJoinWarps];
    __shared__ float s_o[kJoinWarps][kW];
    wait_for_predecessor();
    release_successor();
    const int item = threadIdx.x / (32 * kWpi), warp = (threadIdx.x >> 5) % kWpi, lane = threadIdx.x & 31;
    const int groups = (c.part_rows + kItems - 1) / kItems;
    const int b = blockIdx.y, h = blockIdx.x / groups, r = blockIdx.x % groups * kItems + item;
    const SeqWork w = seq_work(c, b);
    const int rows = w.g.q_len * c.group;
    if (w.nt <= 1 || blockIdx.x % groups * kItems >= rows) return;
    // the unit's tiles in the list, and the CTAs whose ranges hold its first and its last one
    uint32_t total = 0, u0 = 0;
    for (int b0 = 0; b0 < c.a.pv.n_seqs; b0 += 32) {
        const int nt = b0 + lane < c.a.pv.n_seqs ? seq_work(c, b0 + lane).nt : 0;
        const uint32_t inc = warp_scan(nt * c.a.hk, lane);
        if (b >= b0 && b < b0 + 32) u0 = total + __shfl_sync(0xFFFFFFFFu, inc - nt * c.a.hk, b - b0);
        total += __shfl_sync(0xFFFFFFFFu, inc, 31);
    }
    u0 += (uint32_t)h * w.nt;
    const Ranges ranges(total, c.ctas);
    const int c0 = (int)ranges.owner(u0), parts = (int)ranges.owner(u0 + w.nt - 1) - c0 + 1;
    if (parts == 1) return;                      // one CTA had all of it and wrote the result
    float acc[kV];
#pragma unroll
    for (int e = 0; e < kV; ++e) acc[e] = 0.0f;
    float top = -INFINITY, sum = 0.0f;           // of this warp's partials so far
    if (r < rows) {
        // The CTA that has the unit's first tile left its partial in slot 1, the ones whose ranges start inside the
        // unit in slot 0. This warp's partials are warp, warp + kWpi, ...: lane k has the k-th one's numbers.
        auto row_of = [&](int i) { return ((int64_t)(c0 + i) * 2 + (i == 0 ? 1 : 0)) * c.part_rows + r; };
        for (int i0 = warp; i0 < parts; i0 += kJoinBatch * kWpi) {
            const int mine = i0 + lane * kWpi;
            float2 ml = make_float2(-INFINITY, 0.0f);
            if (lane < kJoinBatch && mine < parts) ml = *reinterpret_cast<const float2*>(c.part_ml + row_of(mine) * 2);
            float v[kJoinBatch][kV];
#pragma unroll
            for (int k = 0; k < kJoinBatch; ++k) {
                const int i = i0 + k * kWpi;
                if (i < parts) {
                    const float* p = c.part_o + row_of(i) * D + blockIdx.z * kW + lane * kV;
                    if constexpr (kV == 4) {
                        const float4 t = *reinterpret_cast<const float4*>(p);
                        v[k][0] = t.x, v[k][1] = t.y, v[k][2] = t.z, v[k][3] = t.w;
                    } else {
                        const float2 t = *reinterpret_cast<const float2*>(p);
                        v[k][0] = t.x, v[k][1] = t.y;
                    }
                } else {
#pragma unroll
                    for (int e = 0; e < kV; ++e) v[k][e] = 0.0f;
                }
            }
            float now = fmaxf(top, ml.x);
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) now = fmaxf(now, __shfl_xor_sync(0xFFFFFFFFu, now, o));
            const float ref = now == -INFINITY ? 0.0f : now, back = fast_exp2(top - ref), f = fast_exp2(ml.x - ref);
            top = now;
            sum = sum * back + f * ml.y;
#pragma unroll
            for (int e = 0; e < kV; ++e) acc[e] *= back;
#pragma unroll
            for (int k = 0; k < kJoinBatch; ++k) {
                const float g = __shfl_sync(0xFFFFFFFFu, f, k);
#pragma unroll
                for (int e = 0; e < kV; ++e) acc[e] += g * v[k][e];
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xFFFFFFFFu, sum, o);
    }
    if constexpr (kWpi > 1) {   // the item's warps, each relative to its own maximum
        if (lane == 0) s_top[item * kWpi + warp] = top;
        __syncthreads();
        float all = s_top[item * kWpi + lane % kWpi];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) all = fmaxf(all, __shfl_xor_sync(0xFFFFFFFFu, all, o));
        const float scale = top == -INFINITY ? 0.0f : fast_exp2(top - all);
#pragma unroll
        for (int e = 0; e < kV; ++e) s_o[item * kWpi + warp][lane * kV + e] = acc[e] * scale;
        if (lane == 0) s_sum[item * kWpi + warp] = sum * scale;
        __syncthreads();
        if (warp != 0) return;
        sum = 0.0f;
#pragma unroll
        for (int e = 0; e < kV; ++e) acc[e] = 0.0f;
#pragma unroll
        for (int i = 0; i < kWpi; ++i) {
            sum += s_sum[item * kWpi + i];
#pragma unroll
            for (int e = 0; e < kV; ++e) acc[e] += s_o[item * kWpi + i][lane * kV + e];
        }
    }
    if (r >= rows) return;
    const float inv = sum == 0.0f ? 0.0f : 1.0f / sum;
    const int tok = r / c.group, hd = h * c.group + r % c.group;
    uint16_t* dst = c.a.out + (int64_t)(w.g.q0 + tok) * c.a.o_t + (int64_t)hd * c.a.o_h + blockIdx.z * kW + lane * kV;
#pragma unroll
    for (int e = 0; e < kV; e += 2) *reinterpret_cast<uint32_t*>(dst + e) = pack_bf16(acc[e] * inv, acc[e + 1] * inv);
}

template <int D, int kWpi, int kJoinWarps>
void launch_join(const FewCall& c, cudaStream_t st) {
    constexpr int kItems = kJoinWarps / kWpi;
    const dim3 grid((unsigned)((c.part_rows + kItems - 1) / kItems * c.a.hk), (unsigned)c.a.pv.n_seqs, D < 128 ? 1 : D / 128);
    launch_dependent(attn_join_kernel<D, kWpi, kJoinWarps>, grid, dim3(kJoinWarps * 32), 0, st, c);
}

using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

template <int D, int MT>
int few_ctas() { return device_sm_count() * (FewCfg<D, MT>::kTwo ? 2 : 1); }

template <int D, int MT>
void launch_few(const Attn& h, const AttnCall& a, cudaStream_t st) {
    using C = FewCfg<D, MT>;
    static bool attr_set[64] = {false};
    const int dev = current_device();
    if (!attr_set[dev & 63]) {
        check_cuda(cudaFuncSetAttribute(attn_few_kernel<D, MT, false>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem),
                   "cudaFuncSetAttribute(attn_few)");
        if constexpr (kUnitClusters<D, MT>)
            check_cuda(cudaFuncSetAttribute(attn_few_kernel<D, MT, true>, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem),
                       "cudaFuncSetAttribute(attn_few)");
        attr_set[dev & 63] = true;
    }
    const int page_size = 1 << a.pv.page_shift;
    FewCall c;
    c.a = a;
    c.group = a.hq / a.hk;
    c.max_rows = C::kRows;
    c.box = std::min(page_size, kKeys);
    c.part_rows = std::min<int64_t>((int64_t)a.pv.max_q * c.group, C::kRows);
    c.part_o = h.part_o;
    c.part_ml = h.part_ml;
    c.err = device_scratch().err;
    // no more CTAs than there can be tiles: by the table's capacity, or the window
    int64_t cap = (int64_t)a.pv.max_pages << a.pv.page_shift;
    if (a.window > 0) cap = std::min<int64_t>(cap, (int64_t)a.window + c.max_rows / c.group + c.box);
    const int64_t per_unit = std::max<int64_t>(1, (cap + kKeys - 1) / kKeys);
    if (per_unit * a.hk * a.pv.n_seqs > 0x7FFFFFFF) throw Error(G4Q_ERR_UNSUPPORTED_CONFIG, "too many key tiles for one call");
    const int64_t units = (int64_t)a.hk * a.pv.n_seqs;
    c.ctas = (int)std::min<int64_t>(few_ctas<D, MT>(), per_unit * units);
    const CUtensorMap tk = paged_map(a, a.k, D, c.box), tv = paged_map(a, a.v, D, c.box);
    if constexpr (kUnitClusters<D, MT>) {
        const int64_t mine = (per_unit + kUnitCtas - 1) / kUnitCtas, even = (per_unit * units + c.ctas - 1) / c.ctas;
        if (per_unit > 1 && mine <= std::min<int64_t>(kUnitTiles, even + 1) && units * kUnitCtas <= few_ctas<D, MT>()) {
            launch_dependent<kUnitCtas>(attn_few_kernel<D, MT, true>, dim3((unsigned)(units * kUnitCtas)), dim3(kThreads),
                                        C::kSmem, st, tk, tv, c);
            return;
        }
    }
    launch_dependent(attn_few_kernel<D, MT, false>, dim3((unsigned)c.ctas), dim3(kThreads), C::kSmem, st, tk, tv, c);
    if (per_unit > 1) {   // a unit of one tile is never cut
        // Few items with possibly many partials each: a block to an item. Else two warps: the blocks are few then,
        // and a unit has about as many partials as CTAs there are to a unit.
        const int64_t items = (int64_t)c.part_rows * a.hk * a.pv.n_seqs * (D < 128 ? 1 : D / 128);
        if (per_unit > 64 && items <= 256)
            launch_join<D, 16, 16>(c, st);
        else
            launch_join<D, 2, 4>(c, st);
    }
}

template <int D>
void launch_few_rows(const Attn& h, const AttnCall& a, int64_t rows, cudaStream_t st) {
    if (rows <= 16)
        launch_few<D, 1>(h, a, st);
    else if (rows <= 32)
        launch_few<D, 2>(h, a, st);
    else if constexpr (few_rows(D) == 64)
        launch_few<D, 4>(h, a, st);
}

template <int D>
size_t few_part_rows() {
    size_t rows = std::max((size_t)few_ctas<D, 1>() * 16, (size_t)few_ctas<D, 2>() * 32);
    if constexpr (few_rows(D) == 64) rows = std::max(rows, (size_t)few_ctas<D, 4>() * 64);
    return 2 * rows;
}

}  // namespace

namespace {
CUtensorMap bf16_map(int rank, const uint16_t* base, const cuuint64_t* dims, const cuuint64_t* strides, const cuuint32_t* box) {
    static const EncodeTiledFn encode = [] {
        void* p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) != cudaSuccess ||
            q != cudaDriverEntryPointSuccess)
            p = nullptr;
        return reinterpret_cast<EncodeTiledFn>(p);
    }();
    if (encode == nullptr) throw Error(G4Q_ERR_RUNTIME, "cuTensorMapEncodeTiled is unavailable");
    const cuuint32_t es[4] = {1, 1, 1, 1};
    CUtensorMap m;
    const CUresult r = encode(&m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, (cuuint32_t)rank, const_cast<uint16_t*>(base), dims, strides,
                              box, es, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                              CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) throw Error(G4Q_ERR_RUNTIME, "cuTensorMapEncodeTiled failed (" + std::to_string((int)r) + ")");
    return m;
}
}  // namespace

CUtensorMap paged_map(const AttnCall& a, const uint16_t* base, int D, int box) {
    const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)1 << a.pv.page_shift, (cuuint64_t)a.hk, (cuuint64_t)a.pv.n_pages};
    const cuuint64_t strides[3] = {(cuuint64_t)a.slot_stride * 2, (cuuint64_t)a.head_stride * 2, (cuuint64_t)a.page_stride * 2};
    const cuuint32_t shape[4] = {64, (cuuint32_t)box, 1, 1};
    return bf16_map(4, base, dims, strides, shape);
}

CUtensorMap rows_map(const uint16_t* base, int64_t token_stride, int64_t head_stride, int heads, int rows, int D, int box_heads,
                     int box_tokens) {
    const cuuint64_t dims[3] = {(cuuint64_t)D, (cuuint64_t)heads, (cuuint64_t)rows};
    // the stride of a single head, or of a single token, is never used, but has to be a legal one (16 bytes to 2^40)
    const cuuint64_t strides[2] = {(cuuint64_t)(heads == 1 ? D : head_stride) * 2, (cuuint64_t)(rows == 1 ? D : token_stride) * 2};
    const cuuint32_t shape[3] = {64, (cuuint32_t)box_heads, (cuuint32_t)box_tokens};
    return bf16_map(3, base, dims, strides, shape);
}

size_t attn_part_rows(int head_dim) {
    const size_t few = head_dim == 64 ? few_part_rows<64>() : head_dim == 128 ? few_part_rows<128>()
                       : head_dim == 256 ? few_part_rows<256>() : few_part_rows<512>();
    return std::max(few, chunk_part_rows());
}

void launch_few_any(const Attn& h, const AttnCall& a, int64_t rows, cudaStream_t st) {
    switch (h.head_dim) {
        case 64: return launch_few_rows<64>(h, a, rows, st);
        case 128: return launch_few_rows<128>(h, a, rows, st);
        case 256: return launch_few_rows<256>(h, a, rows, st);
        case 512: return launch_few_rows<512>(h, a, rows, st);
    }
}

void launch_attention(const Attn& h, const AttnCall& a, cudaStream_t st) {
    // A sequence goes by its own rows (new tokens x group): few to the kernel above, which shares the keys evenly over
    // the SMs, more to the chunk kernel. Only the lengths on the device say which are there; where every row belongs
    // to a sequence of max_q tokens, or there is one sequence only, the host knows. In a mixed step the few are the
    // single tokens (16 rows unless the group is larger): with 64 rows the kernel's products outweigh the bytes
    // (two tokens beside four prompts, head_dim 256: 20.8 us against 8).
    const int group = a.hq / a.hk;
    const int64_t rows = (int64_t)a.pv.max_q * group;
    if (rows <= few_rows(h.head_dim)) return launch_few_any(h, a, rows, st);
    const int few = group <= 16 ? 16 : group <= 32 ? 32 : 64;
    if ((int64_t)a.pv.n_seqs * a.pv.max_q == a.pv.rows || few > few_rows(h.head_dim)) return launch_chunk(h, a, 0, st);
    launch_few_any(h, a, few, st);
    launch_chunk(h, a, few, st);
}

}  // namespace g4q
