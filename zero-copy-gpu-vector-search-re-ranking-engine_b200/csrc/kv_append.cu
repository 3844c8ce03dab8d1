// zcgvs_kv_append: per-head RMS norm and position rotation of a step's queries and keys, and the
// store of its keys and values into the paged cache, in one pass over the projections' rows.
//
//   y = x * rsqrt(sum(x^2) / d + eps) * w            (queries and keys, where weights are given)
//   (a, b) -> (a cos - b sin, b cos + a sin)          (pairs of the first rotary_dim elements)
//
// Bound by memory: every value is read once and written once, 2 * 2 bytes per value, and the
// rotation table's row once per token. A head's row is held by 8 lanes (head_dim <= 64) or 16,
// 16 bytes each, so all loads and stores are 16 bytes wide and a head's sum of squares is three or
// four shuffles. A pair of the split form lies rotary_dim / 16 lanes apart (rotary_dim is a
// multiple of 16), so it is exchanged by shuffles too; a pair of the interleaved form lies within
// a lane. A block takes up to 8 tokens, one after the other: its warps find a token's sequence,
// position and slot each while the first values are on their way, and every token's values and
// cosines are loaded while the one before is worked on. (A token per block left the search, the
// rotation row and the stores one behind the other: 18,293 tokens of 48 heads took 163 us.)
#include <algorithm>

#include "common.cuh"
#include "paged.h"

namespace zc {
namespace paged {

namespace {

constexpr int kThreads = 256;
constexpr int kHeadsPerLane = 4;  // loads in flight per thread
constexpr int kMaxTokens = kThreads / 32;  // of a block: a warp finds the place of each

struct AppendParams {
    View view;
    const uint8_t* q;
    const uint8_t* k;
    const uint8_t* v;
    long long q_token, q_head, k_token, k_head, v_token, v_head;  // strides, elements
    const uint8_t* q_norm;
    const uint8_t* k_norm;
    float eps;
    const float* rotary;
    long long rotary_rows;
    int rotary_dim;
    int interleaved;
    const int* positions;
    uint8_t* q_out;
    long long q_out_token, q_out_head;
    int q_heads;
    int heads;   // of all three: q_heads + 2 * kv_heads, without the ones not given
    int chunks;  // blocks per token
    int tokens_per_block;
};

// Number of entries of starts[1 .. sequences] that are <= token: the token's sequence, or
// `sequences` for a padding token. The whole warp searches: each round probes 32 places.
__device__ __forceinline__ int sequence_of(const View& v, int token, int lane) {
    int lo = 0, hi = v.sequences;  // the answer is in [lo, hi]
    while (lo < hi) {
        const int step = (hi - lo + 31) >> 5;
        const int probe = lo + (lane + 1) * step;  // starts[probe] <= token: the answer is >= probe
        const bool below = probe <= hi && __ldg(v.starts + probe) <= token;
        const int n = __popc(__ballot_sync(0xffffffffu, below));
        lo += n * step;
        hi = min(hi, lo + step - 1);
    }
    return lo;
}

// Where a token goes.
struct Place {
    long long slot;  // element offset in keys and values; -1: not stored
    int row;         // rotation row; -1: outside the table, -2: a padding token
};

template <typename T, int LANES>
__global__ void __launch_bounds__(kThreads, 2) append_kernel(const AppendParams p) {
    constexpr int kSegments = kThreads / LANES;
    __shared__ Place s_place[kMaxTokens];
    const View& view = p.view;
    const int tid = threadIdx.x;
    const int lane = tid & (LANES - 1);
    const int segment = tid / LANES;
    const int token0 = static_cast<int>(blockIdx.x / static_cast<unsigned>(p.chunks)) * p.tokens_per_block;
    const int tokens = min(p.tokens_per_block, view.tokens - token0);
    const int first = static_cast<int>(blockIdx.x % static_cast<unsigned>(p.chunks)) * kSegments * kHeadsPerLane + segment;
    const bool holds = lane * 8 < view.head_dim;
    const int k_begin = p.q_heads;
    const int v_begin = p.q_heads + (p.k != nullptr ? view.kv_heads : 0);

    // This thread's pieces of a token's heads.
    auto load = [&](int token, uint4 (&x)[kHeadsPerLane]) {
#pragma unroll
        for (int u = 0; u < kHeadsPerLane; ++u) {
            const int h = first + u * kSegments;
            x[u] = make_uint4(0u, 0u, 0u, 0u);
            if (h >= p.heads || !holds) continue;
            const uint8_t* base;
            long long at;
            if (h < k_begin) {
                base = p.q;
                at = token * p.q_token + h * p.q_head;
            } else if (h < v_begin) {
                base = p.k;
                at = token * p.k_token + (h - k_begin) * p.k_head;
            } else {
                base = p.v;
                at = token * p.v_token + (h - v_begin) * p.v_head;
            }
            x[u] = *reinterpret_cast<const uint4*>(base + 2 * (at + lane * 8));
        }
    };
    // This lane's cosines and sines: of its 8 elements, or of its 4 pairs in the interleaved form.
    const int half = p.rotary_dim / 2;
    const bool turns = p.rotary != nullptr && lane * 8 < p.rotary_dim;
    const int in_row = p.interleaved ? lane * 4 : (lane * 8) % half;
    auto load_turn = [&](int row, float4 (&cs)[2], float4 (&sn)[2]) {
        if (!turns || row < 0) return;
        const float* c = p.rotary + static_cast<long long>(row) * p.rotary_dim + in_row;
        cs[0] = __ldg(reinterpret_cast<const float4*>(c));
        sn[0] = __ldg(reinterpret_cast<const float4*>(c + half));
        if (!p.interleaved) {
            cs[1] = __ldg(reinterpret_cast<const float4*>(c + 4));
            sn[1] = __ldg(reinterpret_cast<const float4*>(c + half + 4));
        }
    };

    uint4 x[kHeadsPerLane];
    load(token0, x);
    if (tid / 32 < tokens) {
        const int token = token0 + tid / 32;
        const int s = sequence_of(view, token, tid & 31);
        if ((tid & 31) == 0) {
            Place place{-1, -2};
            if (s < view.sequences) {
                const long long end = view.starts[s + 1];
                const long long at = view.lengths[s] - end + token;  // negative: not among the cached ones
                const int position = static_cast<int>(max(at, -1LL));
                const long long turn = p.positions != nullptr ? p.positions[token] : at;
                place.row = 0;
                if (p.rotary != nullptr) place.row = turn >= 0 && turn < p.rotary_rows ? static_cast<int>(turn) : -1;
                if (p.k != nullptr && place.row >= 0) place.slot = slot_offset(view, s, position);
            }
            s_place[tid / 32] = place;
        }
    }
    __syncthreads();
    float4 cs[2] = {}, sn[2] = {};
    load_turn(s_place[0].row, cs, sn);
    // The lane that holds the other element of this lane's pairs (split form), and the sign of its
    // part: a cos - b sin, b cos + a sin.
    const int apart = half / 8;
    const int partner = (lane < apart ? lane + apart : lane - apart) & (LANES - 1);
    const float sign = lane < apart ? -1.0f : 1.0f;

#pragma unroll 1
    for (int i = 0; i < tokens; ++i) {
        const int token = token0 + i;
        const Place place = s_place[i];
        uint4 ahead[kHeadsPerLane];
        float4 cs_ahead[2] = {}, sn_ahead[2] = {};
        if (i + 1 < tokens) {
            load(token + 1, ahead);
            load_turn(s_place[i + 1].row, cs_ahead, sn_ahead);
        }
        if (place.row != -2) {
            const bool turned = turns && place.row >= 0;
            const float c8[8] = {cs[0].x, cs[0].y, cs[0].z, cs[0].w, cs[1].x, cs[1].y, cs[1].z, cs[1].w};
            const float s8[8] = {sn[0].x, sn[0].y, sn[0].z, sn[0].w, sn[1].x, sn[1].y, sn[1].z, sn[1].w};
#pragma unroll
            for (int u = 0; u < kHeadsPerLane; ++u) {
                const int h = first + u * kSegments;
                if (first - segment + u * kSegments >= p.heads) break;  // for the whole block, so that the shuffles see every lane
                const uint8_t* weight = h < k_begin ? p.q_norm : p.k_norm;
                const bool is_value = h >= v_begin;
                float f[8];
                const uint32_t packed[4] = {x[u].x, x[u].y, x[u].z, x[u].w};
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const float2 t = unpack2<T>(packed[j]);
                    f[2 * j] = t.x;
                    f[2 * j + 1] = t.y;
                }
                float sum = 0.0f;
#pragma unroll
                for (int j = 0; j < 8; ++j) sum += f[j] * f[j];
#pragma unroll
                for (int o = LANES / 2; o >= 1; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o, LANES);
                if (!is_value && weight != nullptr && holds) {
                    const float inv = rsqrtf(sum / static_cast<float>(view.head_dim) + p.eps);
                    const uint4 w = __ldg(reinterpret_cast<const uint4*>(weight) + lane);
                    const uint32_t ws[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const float2 t = unpack2<T>(ws[j]);
                        f[2 * j] *= inv * t.x;
                        f[2 * j + 1] *= inv * t.y;
                    }
                }
                if (p.rotary != nullptr) {
                    if (p.interleaved) {
                        if (turned && !is_value) {
#pragma unroll
                            for (int j = 0; j < 4; ++j) {
                                const float a = f[2 * j], b = f[2 * j + 1];
                                f[2 * j] = a * c8[j] - b * s8[j];
                                f[2 * j + 1] = b * c8[j] + a * s8[j];
                            }
                        }
                    } else {
#pragma unroll
                        for (int j = 0; j < 8; ++j) {
                            const float other = __shfl_sync(0xffffffffu, f[j], partner, LANES);
                            if (turned && !is_value) f[j] = f[j] * c8[j] + sign * other * s8[j];
                        }
                    }
                }
                uint4 y = make_uint4(pack2<T>(f[0], f[1]), pack2<T>(f[2], f[3]), pack2<T>(f[4], f[5]), pack2<T>(f[6], f[7]));
                if (is_value) y = x[u];  // bit for bit, NaN payloads included
                if (h >= p.heads || !holds) continue;
                if (h < k_begin) {
                    if (place.row < 0) y = make_uint4(0u, 0u, 0u, 0u);
                    *reinterpret_cast<uint4*>(p.q_out + 2 * (token * p.q_out_token + h * p.q_out_head + lane * 8)) = y;
                } else if (place.slot >= 0) {
                    const int head = is_value ? h - v_begin : h - k_begin;
                    uint8_t* base = is_value ? view.values : view.keys;
                    *reinterpret_cast<uint4*>(base + 2 * (place.slot + head * view.head_stride + lane * 8)) = y;
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kHeadsPerLane; ++u) x[u] = ahead[u];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            cs[j] = cs_ahead[j];
            sn[j] = sn_ahead[j];
        }
    }
}

template <typename T>
cudaError_t launch_append(const AppendParams& p, unsigned blocks, bool narrow, cudaStream_t stream) {
    KernelTimer timer("kv_append", stream);
    if (narrow) {
        append_kernel<T, 8><<<blocks, kThreads, 0, stream>>>(p);
    } else {
        append_kernel<T, 16><<<blocks, kThreads, 0, stream>>>(p);
    }
    return cudaGetLastError();
}

}  // namespace
}  // namespace paged
}  // namespace zc

extern "C" int zcgvs_kv_append(const zcgvs_paged_cache* cache, const zcgvs_step_batch* batch, const void* q,
                               int64_t q_token_stride, int64_t q_head_stride, int q_heads, const void* k,
                               int64_t k_token_stride, int64_t k_head_stride, const void* v, int64_t v_token_stride,
                               int64_t v_head_stride, const void* q_norm, const void* k_norm, float eps,
                               const float* rotary, int64_t rotary_rows, int rotary_dim, int interleaved,
                               const int* positions, void* q_out, int64_t q_out_token_stride,
                               int64_t q_out_head_stride, void* stream) {
    using namespace zc;
    using namespace zc::paged;
    const char* what = "zcgvs_kv_append";
    if (cache == nullptr || batch == nullptr) return invalid(what, "null cache or batch");
    if (batch->tokens <= 0 || batch->sequences <= 0) return ok();
    AppendParams p{};
    int status = make_view(what, cache, batch, p.view);
    if (status != ZCGVS_OK) return status;
    if ((k == nullptr) != (v == nullptr)) return invalid(what, "keys and values come together");
    if (q == nullptr) q_heads = 0;
    if (q_heads < 0 || (q != nullptr && q_heads == 0)) return invalid(what, "q_heads must be positive where q is given");
    if (q == nullptr && k == nullptr) return ok();
    if (q != nullptr) {
        if (q_out == nullptr) return invalid(what, "null q_out");
        status = check_rows(what, "q", q, q_token_stride, q_head_stride);
        if (status == ZCGVS_OK) status = check_rows(what, "q_out", q_out, q_out_token_stride, q_out_head_stride);
        if (status != ZCGVS_OK) return status;
    }
    if (k != nullptr) {
        status = check_rows(what, "k", k, k_token_stride, k_head_stride);
        if (status == ZCGVS_OK) status = check_rows(what, "v", v, v_token_stride, v_head_stride);
        if (status != ZCGVS_OK) return status;
    }
    if (!aligned_to(q_norm, 16) || !aligned_to(k_norm, 16) || !aligned_to(rotary, 16)) {
        return invalid(what, "q_norm, k_norm and rotary must be 16-byte aligned");
    }
    if (rotary != nullptr) {
        if (rotary_dim <= 0 || rotary_dim % 16 != 0 || rotary_dim > cache->head_dim) {
            return invalid(what, "rotary_dim must be a multiple of 16 in 16..head_dim");
        }
        if (rotary_rows <= 0 || rotary_rows > INT_MAX) return invalid(what, "rotary_rows must be in 1..2^31 - 1");
    } else {
        rotary_dim = 16;  // not used
    }
    const bool narrow = cache->head_dim <= 64;
    const int per_block = kThreads / (narrow ? 8 : 16) * kHeadsPerLane;
    const long long heads = static_cast<long long>(q_heads) + (k != nullptr ? 2LL * cache->kv_heads : 0);
    const long long chunks = (heads + per_block - 1) / per_block;
    if (heads > INT_MAX / 2 || chunks * batch->tokens > INT_MAX) return invalid(what, "too many tokens and heads for one call");
    p.q = static_cast<const uint8_t*>(q);
    p.k = static_cast<const uint8_t*>(k);
    p.v = static_cast<const uint8_t*>(v);
    p.q_token = q_token_stride;
    p.q_head = q_head_stride;
    p.k_token = k_token_stride;
    p.k_head = k_head_stride;
    p.v_token = v_token_stride;
    p.v_head = v_head_stride;
    p.q_norm = static_cast<const uint8_t*>(q_norm);
    p.k_norm = static_cast<const uint8_t*>(k_norm);
    p.eps = eps;
    p.rotary = rotary;
    p.rotary_rows = rotary_rows;
    p.rotary_dim = rotary_dim;
    p.interleaved = interleaved != 0;
    p.positions = positions;
    p.q_out = static_cast<uint8_t*>(q_out);
    p.q_out_token = q_out_token_stride;
    p.q_out_head = q_out_head_stride;
    p.q_heads = q_heads;
    p.heads = static_cast<int>(heads);
    p.chunks = static_cast<int>(chunks);
    // Enough blocks to fill the SMs twice over come first, then more tokens per block.
    const long long fill = 4LL * device_sm_count();
    p.tokens_per_block = static_cast<int>(std::min<long long>(std::max<long long>(chunks * batch->tokens / fill, 1), kMaxTokens));
    const unsigned blocks = static_cast<unsigned>(chunks * ((batch->tokens + p.tokens_per_block - 1) / p.tokens_per_block));
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    const cudaError_t e = cache->dtype == ZCGVS_DTYPE_F16 ? launch_append<__half>(p, blocks, narrow, s)
                                                          : launch_append<__nv_bfloat16>(p, blocks, narrow, s);
    if (e != cudaSuccess) return fail_cuda(e, what);
    return ok();
}
