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
// fraction of a turn, are an angle in [-pi, pi), where the hardware sine and cosine are off by about 2^-21 at most
// (absolute), beside a rounding to bf16 of 2^-8 of the value.
//
// Bound by HBM for a prompt's chunk: every element is read and written once (16 query and 8 key heads of 256,
// 2048 tokens: 50 MB, 11.0 us with the rows in L2, 13.7 us with new ones each call, where a plain copy of as many
// bytes takes 12.4). The instructions come close: with the library's sincospi for every head,
// and weight, norm and rotation applied one after the other, a head took 305 warp instructions and the kernel
// 18.7 us, issue-bound at 13 % of DRAM. So a block takes one token, and what the token's heads share is folded
// into two factors per element before the heads are looked at:
//   out_i = inv * (x_i * A_i + x_partner * B_i),   A = w_i cos, B = -+ w_partner sin,   inv = 1 / rms(x)
// A warp takes heads of one kind (queries, keys or values); a lane has a 16-byte chunk of 8 elements of a head (two at
// D = 512; two or four heads side by side at D = 128, 64), and the partner chunk comes from another lane as it was
// read, four shuffles.
#include <cuda_bf16.h>
#include <cuda_runtime.h>

#include <cstdint>

#include "g4q_attn.cuh"
#include "g4q_common.cuh"
#include "g4q_internal.h"

namespace g4q {
namespace {

constexpr int kWarps = 16;      // of a block, at most: the heads of one token

__device__ __forceinline__ void unpack8(const uint4& v, float* f) {
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        f[2 * e] = __uint_as_float(w[e] << 16);
        f[2 * e + 1] = __uint_as_float(w[e] & 0xFFFF0000u);
    }
}

// Two fp32 operations in one instruction.
struct F2 {
    float x, y;
};
__device__ __forceinline__ F2 fma2(F2 a, F2 b, F2 c) {
    F2 d;
    asm("{\n\t.reg .b64 p, q, r;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\tmov.b64 r, {%6, %7};\n\t"
        "fma.rn.f32x2 p, p, q, r;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
    return d;
}
__device__ __forceinline__ F2 mul2(F2 a, F2 b) {
    F2 d;
    asm("{\n\t.reg .b64 p, q;\n\tmov.b64 p, {%2, %3};\n\tmov.b64 q, {%4, %5};\n\t"
        "mul.rn.f32x2 p, p, q;\n\tmov.b64 {%0, %1}, p;\n\t}"
        : "=f"(d.x), "=f"(d.y) : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
    return d;
}

__device__ __forceinline__ uint4 shfl4(const uint4& v, int src) {
    return make_uint4(__shfl_sync(0xFFFFFFFFu, v.x, src), __shfl_sync(0xFFFFFFFFu, v.y, src),
                      __shfl_sync(0xFFFFFFFFu, v.z, src), __shfl_sync(0xFFFFFFFFu, v.w, src));
}

template <int D, int IPW, bool kAppend>
__global__ void __launch_bounds__(kWarps * 32) head_rows_kernel(const __grid_constant__ HeadRowsCall p) {
    constexpr int NV = D > 256 ? D / 256 : 1;       // chunks per lane
    constexpr int LPH = D / 8 / NV;                 // lanes per head
    constexpr int HPP = 32 / LPH;                   // heads a warp takes at once
    constexpr int kGroup = HPP * IPW;               // heads of a warp
    wait_for_predecessor();
    release_successor();
    const int lane = threadIdx.x & 31, l = lane % LPH, sub = lane / LPH;
    const int gq = (p.hq + kGroup - 1) / kGroup, gk = (p.hk + kGroup - 1) / kGroup, gv = (p.hv + kGroup - 1) / kGroup;
    // A and B of a query head and of a key head: [kind][A, B][which four of a chunk's eight][chunk][4], so that a
    // warp's 16-byte reads do not conflict
    __shared__ float s_f[2][2][2][D / 8][4];
    const int64_t m = blockIdx.x;
    int g = (int)(blockIdx.y * (blockDim.x >> 5) + (threadIdx.x >> 5));
    const bool in_range = g < gq + gk + gv;
    const bool is_q = g < gq, is_v = g >= gq + gk;
    g -= is_q ? 0 : is_v ? gq + gk : gq;
    const int heads = is_q ? p.hq : is_v ? p.hv : p.hk;
    const int64_t in_h = is_q ? p.q_h : is_v ? p.v_h : p.k_h;
    const uint16_t* src = is_q ? p.q + m * p.q_t : is_v ? p.v + m * p.v_t : p.k + m * p.k_t;

    // the heads' data first: everything below can run while it arrives
    uint4 raw[IPW][NV];
#pragma unroll
    for (int i = 0; i < IPW; ++i) {
        const int hd = g * kGroup + i * HPP + sub;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            raw[i][j] = in_range && hd < heads ? *reinterpret_cast<const uint4*>(src + hd * in_h + (l + j * LPH) * 8) : make_uint4(0, 0, 0, 0);
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
        const SeqGeom sg = seq_geom(p.pv, seq);
        if (m < sg.q0 || m - sg.q0 >= sg.q_len) return;
        pos = sg.first + (int)(m - sg.q0);
        if (!is_q && pos >= 0 && pos < sg.kv_len) {
            const int page = p.pv.table[seq * p.pv.table_ld + (pos >> p.pv.page_shift)];
            if (page < 0 || page >= p.pv.n_pages)
                record_input_error(p.pv.err, kErrPage);
            else
                slot_off = page * p.page_stride + (pos & ((1 << p.pv.page_shift) - 1)) * p.slot_stride;
        }
    } else {
        pos = p.positions[m];
    }

    // four consecutive elements of a kind per thread: pairs (i, i + half), and the elements that are not rotated
    const int half = p.rotary / 2, pairs4 = half / 4, units = pairs4 + (D - p.rotary) / 4;
    for (int u = threadIdx.x; u < 2 * units; u += blockDim.x) {
        const int kd = u >= units ? 1 : 0, v = u - kd * units;
        const uint16_t* wt = kd == 0 ? p.q_weight : p.k_weight;
        auto weights = [&](int i) {
            const uint2 w = wt != nullptr ? *reinterpret_cast<const uint2*>(wt + i) : make_uint2(0x3F803F80u, 0x3F803F80u);   // bf16 1.0
            return make_float4(__uint_as_float(w.x << 16), __uint_as_float(w.x & 0xFFFF0000u), __uint_as_float(w.y << 16),
                               __uint_as_float(w.y & 0xFFFF0000u));
        };
        auto put = [&](int ab, int i, float4 f) { *reinterpret_cast<float4*>(s_f[kd][ab][(i >> 2) & 1][i >> 3]) = f; };
        if (v < pairs4) {
            const int i = 4 * v;
            float cs[4], sn[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint64_t turn = (uint64_t)(int64_t)pos * p.turns[i + e];
                const float angle = (float)(int32_t)(turn >> 32) * 1.4629180792671596e-9f;   // 2 pi * 2^-32
                cs[e] = __cosf(angle);
                sn[e] = __sinf(angle);
            }
            const float4 w0 = weights(i), w1 = weights(i + half);
            put(0, i, make_float4(w0.x * cs[0], w0.y * cs[1], w0.z * cs[2], w0.w * cs[3]));
            put(1, i, make_float4(-w1.x * sn[0], -w1.y * sn[1], -w1.z * sn[2], -w1.w * sn[3]));
            put(0, i + half, make_float4(w1.x * cs[0], w1.y * cs[1], w1.z * cs[2], w1.w * cs[3]));
            put(1, i + half, make_float4(w0.x * sn[0], w0.y * sn[1], w0.z * sn[2], w0.w * sn[3]));
        } else {
            const int i = p.rotary + 4 * (v - pairs4);
            put(0, i, weights(i));
            put(1, i, make_float4(0.0f, 0.0f, 0.0f, 0.0f));
        }
    }
    __syncthreads();
    if (!in_range) return;
    const int off = p.rotary / 16, kind = is_q ? 0 : 1;   // chunk c of a head holds 8c..8c+7, its partner is chunk c +- off

#pragma unroll
    for (int i = 0; i < IPW; ++i) {
        const int hd = g * kGroup + i * HPP + sub;
        if (g * kGroup + i * HPP >= heads) break;        // the whole warp is past the last head
        float x[NV][8];
        F2 sq = {0.0f, 0.0f};
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            unpack8(raw[i][j], x[j]);
#pragma unroll
            for (int e = 0; e < 8; e += 2) sq = fma2({x[j][e], x[j][e + 1]}, {x[j][e], x[j][e + 1]}, sq);
        }
        float ss = sq.x + sq.y;
#pragma unroll
        for (int o = LPH / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
        const float inv = rsqrtf(ss * (1.0f / D) + p.eps);
        if (!is_v) {
            uint4 other[NV];
            if (NV == 1 || 2 * off <= 32) {              // partners within the first 32 chunks
                const int c = l, pc = c < off ? c + off : c < 2 * off ? c - off : c;
                other[0] = shfl4(raw[i][0], sub * LPH + pc);
#pragma unroll
                for (int j = 1; j < NV; ++j) other[j] = raw[i][j];
            } else if (off == 32) {                      // the lane's own other chunk
#pragma unroll
                for (int j = 0; j < NV; ++j) other[j] = raw[i][NV - 1 - j];
            } else {
#pragma unroll
                for (int j = 0; j < NV; ++j) {
                    const int c = l + j * LPH, pc = c < off ? c + off : c < 2 * off ? c - off : c;
#pragma unroll
                    for (int jj = 0; jj < NV; ++jj) {
                        const uint4 t = shfl4(raw[i][jj], pc % LPH);
                        if (pc / LPH == jj) other[j] = t;
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < NV; ++j) {
                if (j > 0 && 2 * off <= 32) {            // none of these chunks is rotated
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        const float4 fa = *reinterpret_cast<const float4*>(s_f[kind][0][q][l + j * LPH]);
                        x[j][4 * q] *= fa.x, x[j][4 * q + 1] *= fa.y, x[j][4 * q + 2] *= fa.z, x[j][4 * q + 3] *= fa.w;
                    }
                    continue;
                }
                float y[8];
                unpack8(other[j], y);
#pragma unroll
                for (int q = 0; q < 2; ++q) {
                    const float4 fa = *reinterpret_cast<const float4*>(s_f[kind][0][q][l + j * LPH]);
                    const float4 fb = *reinterpret_cast<const float4*>(s_f[kind][1][q][l + j * LPH]);
                    const F2 r0 = fma2({y[4 * q], y[4 * q + 1]}, {fb.x, fb.y}, mul2({x[j][4 * q], x[j][4 * q + 1]}, {fa.x, fa.y}));
                    const F2 r1 = fma2({y[4 * q + 2], y[4 * q + 3]}, {fb.z, fb.w}, mul2({x[j][4 * q + 2], x[j][4 * q + 3]}, {fa.z, fa.w}));
                    x[j][4 * q] = r0.x, x[j][4 * q + 1] = r0.y, x[j][4 * q + 2] = r1.x, x[j][4 * q + 3] = r1.y;
                }
            }
        }
        if (hd >= heads) continue;
        uint16_t* dst;
        if (is_q) {
            dst = p.q_out + m * p.qo_t + hd * p.qo_h;
        } else if constexpr (kAppend) {
            if (slot_off < 0) continue;
            dst = (is_v ? p.v_out : p.k_out) + slot_off + hd * p.ko_h;
        } else {
            dst = p.k_out + m * p.ko_t + hd * p.ko_h;
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            uint32_t o[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const F2 r = mul2({x[j][2 * e], x[j][2 * e + 1]}, {inv, inv});
                o[e] = pack_bf16(r.x, r.y);
            }
            *reinterpret_cast<uint4*>(dst + (l + j * LPH) * 8) = is_v && p.raw_v ? raw[i][j] : make_uint4(o[0], o[1], o[2], o[3]);
        }
    }
}

template <int D, int IPW, bool kAppend>
void launch_one(const HeadRowsCall& c, cudaStream_t st) {
    constexpr int kGroup = (D >= 256 ? 1 : 256 / D) * IPW;
    const int64_t groups = (c.hq + kGroup - 1) / kGroup + (c.hk + kGroup - 1) / kGroup + (c.hv + kGroup - 1) / kGroup;
    const int blocks = (int)((groups + kWarps - 1) / kWarps), warps = (int)((groups + blocks - 1) / blocks);
    launch_dependent(head_rows_kernel<D, IPW, kAppend>, dim3((unsigned)c.rows, (unsigned)blocks), dim3(warps * 32), 0, st, c);
}

template <int D>
void launch_dim(const HeadRowsCall& c, bool append, cudaStream_t st) {
    // One head per warp keeps a single token's latency low; with more rows than fill the GPU a warp takes several, so
    // fewer warps pass through (24 heads of 256, 2048 tokens: one head 13.7 us, two 11.9, four 11.0; 18 heads of 512:
    // one 21.2, two 17.7, four 27.3, whose registers leave too few warps to cover the loads).
    constexpr int kWide = D > 256 ? 2 : 4;
    const int heads = c.hq + c.hk + c.hv;
    const bool wide = c.rows * heads >= (int64_t)device_sm_count() * 64;
    if (append)
        wide ? launch_one<D, kWide, true>(c, st) : launch_one<D, 1, true>(c, st);
    else
        wide ? launch_one<D, kWide, false>(c, st) : launch_one<D, 1, false>(c, st);
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
