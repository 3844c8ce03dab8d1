// Attention of few rows per sequence over the paged cache: decoding, and short chunks.
//
// With at most 64 rows (new tokens x group) per key/value head, every cached key and value is
// used for few rows, and the time is that of reading them once: 2 * 2 * head_dim bytes per key
// and head. The arithmetic (4 * head_dim operations per row and key) stays far below what the
// warp-level tensor instructions (m16n8k16) deliver, so the kernel is built for a steady stream:
// 4 warps take 64-key tiles from a ring of shared-memory stages that 16-byte asynchronous copies
// fill ahead; each thread finds its rows' pages one tile ahead. Copies of keys outside the unit's
// range are zero-filled, so nothing that lies in unused slots reaches the products. A row of 128
// (or 64) elements is stored with its 16-byte pieces permuted by the row's low three bits, which
// keeps the matrix loads free of bank conflicts.
//
// The 4 warps split a tile by rows (16 per warp) and, where the rows are fewer, by keys: with at
// most 16 rows each warp takes 16 keys of the tile and keeps running maxima, sums and outputs of
// its own, joined in shared memory at the end of the unit. No warp waits for another inside a
// tile. Scores, maxima, sums and outputs are fp32; the weights are rounded to the cache's type
// for the second product, as the instruction takes both operands in one type.
#pragma once

#include "paged_plan.cuh"

namespace zc {
namespace paged {

constexpr int kStreamThreads = 128;
constexpr int kStreamKeys = 64;  // keys per tile
constexpr int kStreamExtra = 1;  // a unit's fill and end, in tiles

template <int DP>
constexpr int stream_stage_bytes() {
    return 2 * kStreamKeys * DP * 2;
}
template <int DP>
constexpr int stream_stages() {
    return DP == 128 ? 3 : 4;
}

template <int DP>
constexpr int stream_ctas_per_sm() {
    return DP == 128 ? 2 : 3;
}

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

__device__ __forceinline__ void ldmatrix4(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t (&r)[4], uint32_t addr) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                 : "r"(addr));
}

template <typename T>
__device__ __forceinline__ void mma16816(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__half>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}

__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// WM warps over the rows (R = 16 WM), 4 / WM over the keys of a tile.
template <typename T, int DP, int WM>
__global__ void __launch_bounds__(kStreamThreads, stream_ctas_per_sm<DP>()) stream_kernel(const AttnParams p) {
    constexpr int R = 16 * WM;
    constexpr int WK = 4 / WM;
    constexpr int KW = kStreamKeys / WK;  // keys of a tile per warp
    constexpr int kStages = stream_stages<DP>();
    constexpr int kPieces = DP / 8;              // 16-byte pieces of a row
    constexpr int kRowsPerStep = kStreamThreads / kPieces;
    constexpr int kSteps = kStreamKeys / kRowsPerStep;
    constexpr int kLine = DP + 8;  // floats per row of the joining buffer
    extern __shared__ __align__(1024) uint8_t smem[];
    __shared__ PlanShared<kStreamThreads> plan_shared;
    __shared__ int s_last;
    __shared__ float s_ml[WK][R][2];

    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int wr = warp % WM, wk = warp / WM;
    const View& view = p.view;
    const int d_pieces = view.head_dim / 8;

    Planner<R, kStreamKeys, kStreamThreads, 1, kStreamExtra> plan(p, plan_shared);
    if (!plan.start(1)) return;
    Segment g = plan_shared.segment;

    const int my_piece = tid % kPieces, my_row = tid / kPieces;
    const bool my_piece_valid = my_piece < d_pieces;
    const uint32_t smem_base = smem_u32(smem);

    for (;;) {
        const int rows = g.seq.n * p.group;
        const int cap = static_cast<int>(min(static_cast<long long>(g.seq.length), static_cast<long long>(view.table_cols) * view.page_size));
        const uint8_t* kbase = view.keys + 2 * g.head * view.head_stride;
        const uint8_t* vbase = view.values + 2 * g.head * view.head_stride;

        // Slots of this thread's rows of a tile, found one tile ahead of their copies.
        long long slots[kSteps];
        auto find = [&](int tile) {
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int pos = (g.range.first + tile) * kStreamKeys + my_row + i * kRowsPerStep;
                slots[i] = pos >= g.range.lo && pos < g.range.hi ? slot_offset(view, g.s, pos) : -1;
            }
        };
        auto copy = [&](int stage) {
            const uint32_t dst = smem_base + stage * stream_stage_bytes<DP>();
#pragma unroll
            for (int i = 0; i < kSteps; ++i) {
                const int row = my_row + i * kRowsPerStep;
                const bool valid = slots[i] >= 0 && my_piece_valid;
                const long long at = valid ? 2 * (slots[i] + my_piece * 8) : 0;
                const uint32_t off = static_cast<uint32_t>(row * DP * 2 + ((my_piece ^ (row & 7)) << 4));
                cp_async16(dst + off, kbase + at, valid);
                cp_async16(dst + kStreamKeys * DP * 2 + off, vbase + at, valid);
            }
        };

        const int tiles = g.end - g.begin;
        find(g.begin);
#pragma unroll
        for (int i = 0; i < kStages - 1; ++i) {
            if (i < tiles) {
                copy(i);
                if (i + 1 < tiles) find(g.begin + i + 1);
            }
            cp_async_commit();
        }

        // Queries, as the first product's left fragments: rows lane / 4 and lane / 4 + 8 of the
        // warp's 16, elements 2 (lane % 4) + {0, 1} and + 8 of each 16.
        uint32_t qf[DP / 16][4];
        int lo[2], hi[2];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            const int row = g.rt * R + wr * 16 + (lane >> 2) + 8 * h;
            const bool live = row < rows;
            row_range(p, g.seq, row, cap, lo[h], hi[h]);
            if (!live) hi[h] = 0;
            const int j = p.by_group.quotient(row);
            const long long token = g.seq.begin + j;
            const int head = g.head * p.group + row - j * p.group;
            const uint8_t* src = p.q + 2 * (token * p.q_token + head * p.q_head);
#pragma unroll
            for (int kk = 0; kk < DP / 16; ++kk) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int d = kk * 16 + e * 8 + 2 * (lane & 3);
                    qf[kk][h + 2 * e] = live && d < view.head_dim ? *reinterpret_cast<const uint32_t*>(src + 2 * d) : 0u;
                }
            }
        }
        // A tile inside every row's range needs no mask.
        int all_lo = 0, all_hi = INT_MAX;
        {
            const int r0 = g.rt * R, r1 = min(rows, r0 + R) - 1;
            int a, b;
            row_range(p, g.seq, r0, cap, a, all_hi);
            row_range(p, g.seq, r1, cap, all_lo, b);
        }

        float o[DP / 8][4];
#pragma unroll
        for (int i = 0; i < DP / 8; ++i) {
#pragma unroll
            for (int j = 0; j < 4; ++j) o[i][j] = 0.0f;
        }
        float top[2] = {-INFINITY, -INFINITY}, sum[2] = {0.0f, 0.0f};

        int stage = 0;
#pragma unroll 1
        for (int t = 0; t < tiles; ++t) {
            cp_async_wait<kStages - 2>();
            __syncthreads();
            {
                int ahead = stage + kStages - 1;
                if (ahead >= kStages) ahead -= kStages;
                if (t + kStages - 1 < tiles) {
                    copy(ahead);
                    if (t + kStages < tiles) find(g.begin + t + kStages);
                }
                cp_async_commit();
            }
            const uint32_t kt = smem_base + stage * stream_stage_bytes<DP>();
            const uint32_t vt = kt + kStreamKeys * DP * 2;
            const int key0 = wk * KW;

            float s[KW / 8][4];
#pragma unroll
            for (int n = 0; n < KW / 8; ++n) {
#pragma unroll
                for (int j = 0; j < 4; ++j) s[n][j] = 0.0f;
            }
#pragma unroll
            for (int n = 0; n < KW / 16; ++n) {
#pragma unroll
                for (int kk = 0; kk < DP / 16; ++kk) {
                    uint32_t b[4];
                    const int row = key0 + n * 16 + (lane & 7) + ((lane >> 4) << 3);
                    const int piece = kk * 2 + ((lane >> 3) & 1);
                    ldmatrix4(b, kt + row * DP * 2 + ((piece ^ (row & 7)) << 4));
                    mma16816<T>(s[2 * n], qf[kk], b[0], b[1]);
                    mma16816<T>(s[2 * n + 1], qf[kk], b[2], b[3]);
                }
            }

            const int pos0 = (g.range.first + g.begin + t) * kStreamKeys;
            const bool whole = pos0 >= all_lo && pos0 + kStreamKeys <= all_hi;
            float best[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int n = 0; n < KW / 8; ++n) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    float x = s[n][j] * p.scale_log2;
                    if (!whole) {
                        const int pos = pos0 + key0 + n * 8 + 2 * (lane & 3) + (j & 1);
                        if (pos < lo[j >> 1] || pos >= hi[j >> 1]) x = -INFINITY;
                    }
                    s[n][j] = x;
                    best[j >> 1] = fmaxf(best[j >> 1], x);
                }
            }
            float base[2], shrink[2];
#pragma unroll
            for (int h = 0; h < 2; ++h) {
                best[h] = fmaxf(best[h], __shfl_xor_sync(0xffffffffu, best[h], 1));
                best[h] = fmaxf(best[h], __shfl_xor_sync(0xffffffffu, best[h], 2));
                const float now = fmaxf(top[h], best[h]);
                base[h] = now == -INFINITY ? 0.0f : now;
                shrink[h] = exp2_approx(top[h] - base[h]);
                top[h] = now;
                sum[h] *= shrink[h];
            }
            if (__any_sync(0xffffffffu, shrink[0] != 1.0f || shrink[1] != 1.0f)) {
#pragma unroll
                for (int i = 0; i < DP / 8; ++i) {
                    o[i][0] *= shrink[0];
                    o[i][1] *= shrink[0];
                    o[i][2] *= shrink[1];
                    o[i][3] *= shrink[1];
                }
            }
#pragma unroll
            for (int n = 0; n < KW / 8; ++n) {
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    s[n][j] = exp2_approx(s[n][j] - base[j >> 1]);
                    sum[j >> 1] += s[n][j];
                }
            }
#pragma unroll
            for (int n = 0; n < KW / 16; ++n) {
                const uint32_t a[4] = {pack2<T>(s[2 * n][0], s[2 * n][1]), pack2<T>(s[2 * n][2], s[2 * n][3]),
                                       pack2<T>(s[2 * n + 1][0], s[2 * n + 1][1]), pack2<T>(s[2 * n + 1][2], s[2 * n + 1][3])};
#pragma unroll
                for (int i = 0; i < DP / 16; ++i) {
                    uint32_t b[4];
                    const int row = key0 + n * 16 + (lane & 15);
                    const int piece = i * 2 + (lane >> 4);
                    ldmatrix4_trans(b, vt + row * DP * 2 + ((piece ^ (row & 7)) << 4));
                    mma16816<T>(o[2 * i], a, b[0], b[1]);
                    mma16816<T>(o[2 * i + 1], a, b[2], b[3]);
                }
            }
            if (++stage == kStages) stage = 0;
        }

        // Join the warps that shared the rows, and write the unit's rows or its partial result.
        cp_async_wait<0>();
        __syncthreads();
        float* buffer = reinterpret_cast<float*>(smem);  // [WK][R][kLine]
#pragma unroll
        for (int h = 0; h < 2; ++h) {
            sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 1);
            sum[h] += __shfl_xor_sync(0xffffffffu, sum[h], 2);
            const int r = wr * 16 + (lane >> 2) + 8 * h;
            if ((lane & 3) == 0) {
                s_ml[wk][r][0] = top[h];
                s_ml[wk][r][1] = sum[h];
            }
#pragma unroll
            for (int i = 0; i < DP / 8; ++i) {
                *reinterpret_cast<float2*>(buffer + (wk * R + r) * kLine + i * 8 + 2 * (lane & 3)) = make_float2(o[i][2 * h], o[i][2 * h + 1]);
            }
        }
        __syncthreads();
        const bool whole_unit = g.begin == 0 && g.end == g.range.count;
        const int live_rows = min(R, rows - g.rt * R);
        const long long cta = blockIdx.x;
        const long long slot = plan.slot(cta, g.unit_start);
        for (int i = tid; i < live_rows * (DP / 4); i += kStreamThreads) {
            const int r = i / (DP / 4), d = (i % (DP / 4)) * 4;
            float m = s_ml[0][r][0];
#pragma unroll
            for (int w = 1; w < WK; ++w) m = fmaxf(m, s_ml[w][r][0]);
            const float base = m == -INFINITY ? 0.0f : m;
            float l = 0.0f;
            float4 y = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int w = 0; w < WK; ++w) {
                const float f = exp2_approx(s_ml[w][r][0] - base);
                const float4 part = *reinterpret_cast<const float4*>(buffer + (w * R + r) * kLine + d);
                l += f * s_ml[w][r][1];
                y.x += f * part.x;
                y.y += f * part.y;
                y.z += f * part.z;
                y.w += f * part.w;
            }
            if (whole_unit) {
                const int row = g.rt * R + r;
                const int j = p.by_group.quotient(row);
                const long long token = g.seq.begin + j;
                const int head = g.head * p.group + row - j * p.group;
                const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);
                if (d < view.head_dim) {
                    *reinterpret_cast<uint2*>(p.out + 2 * (token * p.out_token + head * p.out_head + d)) =
                        make_uint2(pack2<T>(y.x * inv, y.y * inv), pack2<T>(y.z * inv, y.w * inv));
                }
                if (d == 0 && p.lse != nullptr) {
                    p.lse[token * p.q_heads + head] = l > 0.0f ? (base + log2f(l)) * 0.69314718056f : (l == 0.0f ? -INFINITY : l);
                }
            } else {
                *reinterpret_cast<float4*>(p.part_o + (slot * R + r) * DP + d) = y;
                if (d == 0) *reinterpret_cast<float2*>(p.part_ml + (slot * R + r) * 2) = make_float2(m, l);
            }
        }
        if (!whole_unit) {
            __threadfence();
            __syncthreads();
            if (tid == 0) {
                const long long c_first = g.unit_start / plan.quota, c_last = (g.unit_start + g.range.count - 1) / plan.quota;
                s_last = arrive_last(p.tickets + c_first, p.epoch, static_cast<uint32_t>(c_last - c_first + 1)) ? 1 : 0;
            }
            __syncthreads();
            if (s_last) {
                __threadfence();
                join_partials<T, R, DP, kStreamThreads>(p, plan, g);
            }
        }
        __syncthreads();  // the buffer is free again
        Segment following;
        if (!plan.next(g, following)) break;
        g = following;
    }
}

}  // namespace paged
}  // namespace zc
