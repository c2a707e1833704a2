// g4q_attn.cuh -- what the attention kernels share: the paged batch's geometry on the device, and the
// mbarrier, TMA and matrix-load wrappers.
//
// A batch of n_seqs sequences: sequence b owns the rows [q_offsets[b], q_offsets[b+1]) of the new tokens,
// which are the LAST ones of its kv_lens[b] tokens in the cache (row i is at position kv_len - q_len + i);
// position j lives in page block_table[b][j / page_size] at slot j % page_size. All of that is read on the
// device, so a captured graph replays with the lengths and tables of the moment. What those arrays say is
// checked there too: whatever they hold, no access leaves the cache, the table or the rows. What is refused
// is recorded in the device's input-error word (read with g4q_device_error):
//   60  a page id outside [0, n_pages): nothing is stored there, and it reads as zeros
//   61  a sequence longer than its row of the block table
//   62  offsets that decrease or leave the rows, a negative length, more new tokens than kv_len or max_q
#pragma once

#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "g4q_internal.h"

namespace g4q {

constexpr int kErrPage = 60, kErrTable = 61, kErrLens = 62;

struct PagedView {
    const int32_t* q_offsets;
    const int32_t* kv_lens;
    const int32_t* table;
    int64_t table_ld;
    int n_seqs, max_pages, n_pages, page_shift;
    int rows;        // rows of the new tokens' tensors
    int max_q;
    int* err;        // input-error word
};

// The call of the norm-and-rotate kernel: q, k and v heads of `rows` tokens (element strides per token and
// head), and where they go. Append: the keys and values go to the pages of pv (k_out / v_out: the cache,
// ko_h its head stride); otherwise the keys go to k_out and there are no values.
struct HeadRowsCall {
    const uint16_t *q, *k, *v;
    int64_t q_t, q_h, k_t, k_h, v_t, v_h;
    int hq, hk, hv;
    int rotary;
    int raw_v;                  // store the values as they are
    float eps;
    int64_t rows;
    const uint64_t* turns;      // [rotary / 2] inv_freq / 2 pi, in units of 2^-64 turn
    const int32_t* positions;   // [rows]; append: from pv
    const uint16_t *q_weight, *k_weight;
    uint16_t *q_out, *k_out, *v_out;
    int64_t qo_t, qo_h, ko_t, ko_h;
    int64_t page_stride, slot_stride;
    PagedView pv;
};
void launch_head_rows(const HeadRowsCall& c, int head_dim, bool append, cudaStream_t st);

// The call of the paged attention kernels. The cache's strides are in elements and hold for k and v alike.
struct AttnCall {
    const uint16_t* q;
    uint16_t* out;
    int64_t q_t, q_h, o_t, o_h;
    const uint16_t *k, *v;
    int64_t page_stride, head_stride, slot_stride;
    int hq, hk;
    float scale;
    int window;                 // 0: none
    PagedView pv;
};

CUtensorMap paged_map(const AttnCall& a, const uint16_t* base, int head_dim, int box);   // box: slots x 64 elements
// boxes of 64 elements x box_heads heads x box_tokens tokens of head rows
CUtensorMap rows_map(const uint16_t* base, int64_t token_stride, int64_t head_stride, int heads, int rows, int head_dim,
                     int box_heads, int box_tokens);
size_t attn_part_rows(int head_dim);    // rows of scratch that the two kernels' partials need at most
size_t chunk_part_rows();
void launch_chunk(const Attn& h, const AttnCall& a, int few_rows, cudaStream_t st);
void launch_attention(const Attn& h, const AttnCall& a, cudaStream_t st);

struct SeqGeom {
    int q0, q_len;
    int first;       // position of the first new token
    int kv_len;      // keys that the table reaches
};

__device__ __forceinline__ void record_input_error(int* err, int code) { atomicCAS(err, 0, code); }

// Sequence b with its lengths made safe: 0 <= q0, q0 + q_len <= rows, q_len <= max_q and
// 0 <= kv_len <= max_pages * page_size. first may be negative (rows before position 0 see no key).
__device__ __forceinline__ SeqGeom seq_geom(const PagedView& p, int b) {
    SeqGeom g;
    const int q0 = p.q_offsets[b], q1 = p.q_offsets[b + 1], kv = p.kv_lens[b];
    const int64_t cap = (int64_t)p.max_pages << p.page_shift;
    g.q0 = q0;
    g.q_len = q1 - q0;
    g.first = kv - g.q_len;
    g.kv_len = kv;
    if (q0 < 0 || q1 < q0 || q1 > p.rows || q1 - q0 > p.max_q || kv < 0) {
        record_input_error(p.err, kErrLens);
        g.q0 = g.q_len = g.first = g.kv_len = 0;
    } else if (kv > cap) {
        record_input_error(p.err, kErrTable);
        g.kv_len = (int)cap;
    } else if (kv < g.q_len) {
        record_input_error(p.err, kErrLens);
    }
    return g;
}

// Launch as a programmatic dependent of the stream's previous kernel (the kernel waits for it itself).
template <int kCluster = 1, typename Arg, typename... Rest>
void launch_dependent(void (*kernel)(Arg, Rest...), dim3 grid, dim3 block, size_t smem, cudaStream_t st, const Arg& a,
                      const Rest&... rest) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = block;
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    attr[1].id = cudaLaunchAttributeClusterDimension;
    attr[1].val.clusterDim.x = kCluster;
    attr[1].val.clusterDim.y = attr[1].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = kCluster > 1 ? 2 : 1;
    check_cuda(cudaLaunchKernelEx(&cfg, kernel, a, rest...), "attention kernel launch");
}

__device__ __forceinline__ uint32_t smem_addr(const void* p) {
    return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}

__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
    asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count));
}

__device__ __forceinline__ void bar_expect_tx(uint32_t bar, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}

__device__ __forceinline__ void bar_arrive(uint32_t bar) {
    asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}

constexpr long long kAttnWaitCycles = 4000000000ll;   // ~2 s at 2 GHz

// Bounded wait on an mbarrier phase; false: it gave up. Such a wait records `code` in the device error word; every
// other wait on the device then returns at once, so the kernel runs to its end.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, int* err, int code) {
    long long t0 = 0;
    for (uint32_t it = 0;; ++it) {
        uint32_t done;
        asm volatile(
            "{\n\t.reg .pred p;\n\t"
            "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
            "selp.u32 %0, 1, 0, p;\n\t}"
            : "=r"(done)
            : "r"(bar), "r"(parity)
            : "memory");
        if (done) return true;
        if (it == 0) {
            t0 = clock64();
        } else if ((it & 255u) == 255u) {
            if (*reinterpret_cast<volatile int*>(err) != 0) return false;
            if (clock64() - t0 > kAttnWaitCycles) {
                atomicCAS(err, 0, code);
                return false;
            }
        }
    }
}

// What a warp does at its end after a wait that gave up: it keeps the CTA's shared memory for about a millisecond, in
// which the copies that were issued have long landed.
__device__ __forceinline__ void let_copies_land() {
    const long long t0 = clock64();
    while (clock64() - t0 < 2000000ll) {
    }
}

// One box of a paged tensor: coordinates (element, slot, head, page).
__device__ __forceinline__ void tma_load_page(uint32_t dst, const CUtensorMap* map, int x, int slot, int head, int page,
                                              uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(
            dst),
        "l"(reinterpret_cast<uint64_t>(map)), "r"(x), "r"(slot), "r"(head), "r"(page), "r"(bar)
        : "memory");
}

__device__ __forceinline__ float fast_exp2(float x) {   // 2^x; 0 for -inf
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

__device__ __forceinline__ uint32_t pack_bf16(float lo, float hi) {
    uint32_t r;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
    return r;
}

// Programmatic dependent launch: the kernel may be scheduled while its predecessor on the stream drains;
// nothing global is touched before this wait, which returns when the predecessor's writes are visible.
__device__ __forceinline__ void wait_for_predecessor() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void release_successor() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

}  // namespace g4q
