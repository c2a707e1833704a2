// g4q_rope.cu -- what a decoder layer does to its query and key heads between the q|k|v matmul and the
// attention: RMSNorm of every head, the norm weight, the position rotation, and for a paged cache the
// store of the keys and of the normalized values into their pages (sm_100a).
//
// For one head x of D elements at position t, with r = rotary_dim and h = r / 2:
//   y_i = w_i * x_i / sqrt(mean(x^2) + eps)
//   out_i     = y_i cos(t f_i) - y_{i+h} sin(t f_i)      (i < h)
//   out_{i+h} = y_{i+h} cos(t f_i) + y_i sin(t f_i)      (i < h);   out_i = y_i for i >= r
// All of it in fp32 with one rounding to bf16 at the end (the separate kernels round the normalized value,
// its product with the weight and the rotated value).
//
// The angle: t * f_i reaches 10^5 radians, where an fp32 product is off by 0.01. The table holds
// F_i = f_i / 2 pi, in turns, as a 64-bit fixed-point fraction; the integer product t * F_i wraps modulo 2^64,
// which is modulo one turn, so the fraction of a turn is exact to t * 2^-65. Its upper 32 bits, as a signed
// fraction, go to sincospi.
//
// Bound by HBM: every element is read and written once. One warp takes the heads of one token, a 16-byte
// chunk of 8 elements per lane (two at D = 512, two or four heads side by side at D = 128, 64), so one head is
// one shuffle reduction and the partner element a shuffle away; the sines of the token are computed once for
// all the warp's heads.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "g4q_attn.cuh"
#include "g4q_common.cuh"
#include "g4q_internal.h"

namespace g4q {
namespace {

constexpr int kWarps = 4;

template <int D, int IPW, bool kAppend>
__global__ void __launch_bounds__(kWarps * 32) head_rows_kernel(const __grid_constant__ HeadRowsCall p) {
    constexpr int NV = D > 256 ? D / 256 : 1;       // chunks per lane
    constexpr int LPH = D / 8 / NV;                 // lanes per head
    constexpr int HPP = 32 / LPH;                   // heads a warp takes at once
    wait_for_predecessor();
    release_successor();
    const int lane = threadIdx.x & 31, l = lane % LPH, sub = lane / LPH;
    const int heads = p.hq + p.hk + p.hv;
    const int per_token = (heads + HPP * IPW - 1) / (HPP * IPW);
    const int64_t wid = (int64_t)blockIdx.x * kWarps + (threadIdx.x >> 5);
    const int64_t m = wid / per_token;
    const int s0 = (int)(wid - m * per_token) * IPW;
    if (m >= p.rows) return;

    // the heads' data first: everything below can run while it arrives
    uint4 raw[IPW][NV];
#pragma unroll
    for (int i = 0; i < IPW; ++i) {
        const int hd = (s0 + i) * HPP + sub;
        const uint16_t* src = nullptr;
        if (hd < p.hq)
            src = p.q + m * p.q_t + hd * p.q_h;
        else if (hd < p.hq + p.hk)
            src = p.k + m * p.k_t + (hd - p.hq) * p.k_h;
        else if (hd < heads)
            src = p.v + m * p.v_t + (hd - p.hq - p.hk) * p.v_h;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            raw[i][j] = src != nullptr ? *reinterpret_cast<const uint4*>(src + (l + j * LPH) * 8) : make_uint4(0, 0, 0, 0);
    }

    int pos;
    int64_t slot_off = -1;   // element offset of the token's slot (head 0) in the cache, -1: not stored
    if constexpr (kAppend) {
        // the token's sequence: the number of ends q_offsets[1..n] that are <= m (they do not decrease)
        int seq = 0;
        for (int b0 = 0; b0 < p.pv.n_seqs; b0 += 32) {
            const bool before = b0 + lane < p.pv.n_seqs && p.pv.q_offsets[b0 + lane + 1] <= m;
            const int c = __popc(__ballot_sync(0xFFFFFFFFu, before));
            seq += c;
            if (c < 32) break;
        }
        if (seq >= p.pv.n_seqs) return;   // a row behind the last sequence
        const SeqGeom g = seq_geom(p.pv, seq);
        if (m < g.q0 || m - g.q0 >= g.q_len) return;
        pos = g.first + (int)(m - g.q0);
        if (pos >= 0 && pos < g.kv_len) {
            const int page = p.pv.table[seq * p.pv.table_ld + (pos >> p.pv.page_shift)];
            if (page < 0 || page >= p.pv.n_pages)
                record_input_error(p.pv.err, kErrPage);
            else
                slot_off = page * p.page_stride + (pos & ((1 << p.pv.page_shift) - 1)) * p.slot_stride;
        }
    } else {
        pos = p.positions[m];
    }

    // cos and sin of this lane's pairs; chunk c of a head holds elements 8c..8c+7, pairs with chunk c +- off
    const int off = p.rotary / 16;
    float cs[NV][8], sn[NV][8];
    if (s0 * HPP < p.hq + p.hk) {
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int c = l + j * LPH;
            if (c < 2 * off) {
                const int pair = 8 * (c < off ? c : c - off);
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const uint64_t turn = (uint64_t)(int64_t)pos * p.turns[pair + e];
                    sincospif((float)(int32_t)(turn >> 32) * 0x1p-31f, &sn[j][e], &cs[j][e]);
                    if (c < off) sn[j][e] = -sn[j][e];
                }
            } else {
#pragma unroll
                for (int e = 0; e < 8; ++e) cs[j][e] = 1.0f, sn[j][e] = 0.0f;
            }
        }
    }

#pragma unroll
    for (int i = 0; i < IPW; ++i) {
        const int hd = (s0 + i) * HPP + sub;
        const bool is_q = hd < p.hq, is_v = hd >= p.hq + p.hk;
        float y[NV][8];
        float ss = 0.0f;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const uint32_t w[4] = {raw[i][j].x, raw[i][j].y, raw[i][j].z, raw[i][j].w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[j][2 * e] = bf16_bits_to_f32(w[e] & 0xFFFFu);
                y[j][2 * e + 1] = bf16_bits_to_f32(w[e] >> 16);
                ss = fmaf(y[j][2 * e], y[j][2 * e], ss);
                ss = fmaf(y[j][2 * e + 1], y[j][2 * e + 1], ss);
            }
        }
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
        const float inv = __frsqrt_rn(ss * (1.0f / D) + p.eps);
        const uint16_t* wt = is_v ? nullptr : is_q ? p.q_weight : p.k_weight;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            uint4 wv = make_uint4(0x3F803F80u, 0x3F803F80u, 0x3F803F80u, 0x3F803F80u);   // bf16 1.0 pairs
            if (wt != nullptr) wv = *reinterpret_cast<const uint4*>(wt + (l + j * LPH) * 8);
            const uint32_t w[4] = {wv.x, wv.y, wv.z, wv.w};
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                y[j][2 * e] *= inv * bf16_bits_to_f32(w[e] & 0xFFFFu);
                y[j][2 * e + 1] *= inv * bf16_bits_to_f32(w[e] >> 16);
            }
        }
        if ((s0 + i) * HPP < p.hq + p.hk) {   // some head of this pass is rotated (all lanes shuffle)
            float other[NV][8];
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                const int c = l + j * LPH;
                const int pc = c < off ? c + off : c < 2 * off ? c - off : c;
                const int src = sub * LPH + pc % LPH;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    float o = __shfl_sync(0xFFFFFFFFu, y[0][e], src);
#pragma unroll
                    for (int jj = 1; jj < NV; ++jj) {
                        const float t = __shfl_sync(0xFFFFFFFFu, y[jj][e], src);
                        o = pc / LPH == jj ? t : o;
                    }
                    other[j][e] = o;
                }
            }
            if (!is_v) {
#pragma unroll
                for (int j = 0; j < NV; ++j)
#pragma unroll
                    for (int e = 0; e < 8; ++e) y[j][e] = fmaf(other[j][e], sn[j][e], y[j][e] * cs[j][e]);
            }
        }
        uint16_t* dst = nullptr;
        if (is_q) {
            dst = p.q_out + m * p.qo_t + hd * p.qo_h;
        } else if (hd < heads) {
            const int kh = is_v ? hd - p.hq - p.hk : hd - p.hq;
            if constexpr (kAppend) {
                if (slot_off >= 0) dst = (is_v ? p.v_out : p.k_out) + slot_off + kh * p.ko_h;
            } else {
                dst = p.k_out + m * p.ko_t + kh * p.ko_h;
            }
        }
        if (dst == nullptr) continue;
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            uint4 o;
            if (is_v && p.raw_v)
                o = raw[i][j];
            else
                o = make_uint4(pack_bf16(y[j][0], y[j][1]), pack_bf16(y[j][2], y[j][3]), pack_bf16(y[j][4], y[j][5]),
                               pack_bf16(y[j][6], y[j][7]));
            *reinterpret_cast<uint4*>(dst + (l + j * LPH) * 8) = o;
        }
    }
}

template <int D, int IPW, bool kAppend>
void launch_one(const HeadRowsCall& c, cudaStream_t st) {
    constexpr int HPP = D >= 256 ? 1 : 256 / D;
    const int heads = c.hq + c.hk + c.hv;
    const int64_t per_token = (heads + HPP * IPW - 1) / (HPP * IPW);
    const int64_t blocks = (c.rows * per_token + kWarps - 1) / kWarps;
    if (blocks > 0x7FFFFFFF) throw Error(G4Q_ERR_INVALID_ARGUMENT, "too many rows");
    launch_dependent(head_rows_kernel<D, IPW, kAppend>, dim3((unsigned)blocks), dim3(kWarps * 32), 0, st, c);
}

template <int D>
void launch_dim(const HeadRowsCall& c, bool append, cudaStream_t st) {
    // One head per warp keeps a single token's latency low; with more rows than fill the GPU a warp takes
    // several heads of its token, so the sines are computed once for all of them.
    const int heads = c.hq + c.hk + c.hv;
    const bool wide = c.rows * heads >= (int64_t)device_sm_count() * 64;
    if (append)
        wide ? launch_one<D, 4, true>(c, st) : launch_one<D, 1, true>(c, st);
    else
        wide ? launch_one<D, 4, false>(c, st) : launch_one<D, 1, false>(c, st);
}

}  // namespace

void launch_head_rows(const HeadRowsCall& c, int head_dim, bool append, cudaStream_t st) {
    switch (head_dim) {
        case 64: return launch_dim<64>(c, append, st);
        case 128: return launch_dim<128>(c, append, st);
        case 256: return launch_dim<256>(c, append, st);
        case 512: return launch_dim<512>(c, append, st);
    }
    throw Error(G4Q_ERR_UNSUPPORTED_CONFIG, "head_dim must be 64, 128, 256 or 512");
}

}  // namespace g4q
