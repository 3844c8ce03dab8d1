// zcgvs_sample: one token per row of logits by temperature, top-k, top-p and min-p with a given
// uniform number.
//
// Weights are whole numbers, w_i = rint(2^40 exp((x_i - m) / t)) (at most 327,680 of at most 2^40:
// sums stay below 2^59), so every sum below is exact, whatever its order: the token does not
// depend on the split over CTAs, and integer atomics may build histograms.
//
// Bound by reading the logits once. A cluster of 1 to 8 CTAs takes a row; each keeps its slice in
// shared memory in the logits' own type, so that everything after the first pass stays on chip:
//   1. load, maximum and minimum of the row (cluster-wide);
//   2. where top-k or top-p cuts: a histogram of the slice over 2048 bins of the distance m - x,
//      linear up to the distance where weights become 0 (tokens beyond weigh nothing and rank
//      last, so they change no result); each CTA then sums its share of the bins over the cluster;
//   3. a cut by count or by weight: the bin where the running sum reaches it, then the bin's few
//      tokens are ranked against one another by (logit descending, id ascending). A bin of more
//      than 1024 (equal or clustered logits) is cut into 2048 again by the tokens' 64-bit rank
//      order, as often as needed (each time 11 bits of at most 64);
//   4. the kept weights are summed per warp in ascending id order, and the warp that the drawn
//      number falls into walks its tokens.
#include <cooperative_groups.h>

#include <algorithm>

#include "common.cuh"
#include "paged.h"

namespace cg = cooperative_groups;

namespace zc {
namespace sampling {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 2048;
constexpr int kList = 1024;       // tokens of a bin that are ranked directly
constexpr float kUnits = 1099511627776.0f;  // 2^40
constexpr float kWeightless = 28.5f;        // exp(-28.5) * 2^40 rounds to 0
constexpr int kMaxCluster = 8;

struct SampleParams {
    const void* logits;
    long long row_stride;
    int vocab;
    int slice;      // tokens per CTA, a multiple of 32 * 8 * kWarps
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    const float* uniforms;
    int* tokens;
    float* logprobs;
};

// What the CTAs of a cluster show one another.
struct Shared {
    float top, low;            // of the slice
    u64 best;                  // smallest rank order value etc. (see the passes)
    u64 weight;                // kept weight of the slice
    unsigned chunk_count[2];   // of this CTA's share of the bins, per level
    u64 chunk_mass[2];
    unsigned listed;           // entries of this CTA's list
    u64 range_hi, range_lo;    // rank order values of a bin's members
    // Within the CTA.
    u64 warp_u64[kWarps];
    unsigned warp_u32[kWarps];
    float warp_f32[2][kWarps];
    int bin;
    unsigned bin_count, before_count;
    u64 before_mass;
    u64 cut, cut_mass;
};

template <typename T>
struct Vec;  // 16 bytes of T
template <>
struct Vec<float> {
    static constexpr int kN = 4;
    static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[4]) {
        x[0] = __uint_as_float(v.x);
        x[1] = __uint_as_float(v.y);
        x[2] = __uint_as_float(v.z);
        x[3] = __uint_as_float(v.w);
    }
    static __device__ __forceinline__ float load(const float* p) { return *p; }
    static __device__ __forceinline__ float lowest() { return -INFINITY; }
};
template <typename T>
struct Vec16 {
    static constexpr int kN = 8;
    static __device__ __forceinline__ void unpack(const uint4& v, float (&x)[8]) {
        const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float2 t = paged::unpack2<T>(w[i]);
            x[2 * i] = t.x;
            x[2 * i + 1] = t.y;
        }
    }
};
template <>
struct Vec<__half> : Vec16<__half> {
    static __device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
    static __device__ __forceinline__ __half lowest() { return __ushort_as_half(0xfc00); }
};
template <>
struct Vec<__nv_bfloat16> : Vec16<__nv_bfloat16> {
    static __device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
    static __device__ __forceinline__ __nv_bfloat16 lowest() { return __ushort_as_bfloat16(0xff80); }
};

// Rank order value: larger is ranked earlier. 0 is below every token's.
__device__ __forceinline__ u64 rank_value(float x, int id) { return make_key(x, static_cast<uint32_t>(id)); }

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

template <typename T>
struct Row {
    using V = Vec<T>;
    const SampleParams& p;
    Shared& sh;
    cg::cluster_group cluster;
    T* data;                 // [slice]
    unsigned* raw_count;     // [kBins]
    u64* raw_mass;           // [kBins]
    u64* own_list;           // [2][kList]: rank values, weights; shares memory with the histogram
    u64* list;               // [2][kList]
    unsigned* merged_count;  // [2][kBins / C]
    u64* merged_mass;        // [2][kBins / C]
    int ranks, rank, first;  // CTAs of the cluster, this one, its slice's first token
    int tid, lane, warp;
    float top, t, spread, to_bin;
    bool need_mass;

    __device__ Row(const SampleParams& params, Shared& shared) : p(params), sh(shared), cluster(cg::this_cluster()) {}

    // Calls f(x, id) for every token of the slice that can be drawn; ids ascend within a warp's
    // share, which is contiguous.
    template <typename F>
    __device__ __forceinline__ void each(F f) const {
        const int share = p.slice / kWarps;
        for (int at = warp * share + lane * V::kN; at < (warp + 1) * share; at += 32 * V::kN) {
            float x[V::kN];
            V::unpack(*reinterpret_cast<const uint4*>(data + at), x);
#pragma unroll
            for (int i = 0; i < V::kN; ++i) {
                if (x[i] != -INFINITY) f(x[i], first + at + i);
            }
        }
    }

    __device__ __forceinline__ float distance(float x) const { return x == top ? 0.0f : top - x; }
    __device__ __forceinline__ float share_of(float x) const { return x == top ? 1.0f : expf(__fdiv_rn(x - top, t)); }
    __device__ __forceinline__ u64 weight(float x) const { return static_cast<u64>(__float2ll_rn(share_of(x) * kUnits)); }
    __device__ __forceinline__ int bin_of(float d) const { return min(kBins - 1, static_cast<int>(d * to_bin)); }

    __device__ void clear_histogram() {
        for (int b = tid; b < kBins; b += kThreads) {
            raw_count[b] = 0u;
            raw_mass[b] = 0ull;
        }
        __syncthreads();
    }

    __device__ __forceinline__ void count(int b, float x) {
        atomicAdd(raw_count + b, 1u);
        if (need_mass) atomicAdd(raw_mass + b, weight(x));
    }

    // Sums this CTA's share of the bins over the cluster.
    __device__ void merge(int level) {
        cluster.sync();
        const int n = kBins / ranks;
        unsigned c_all = 0;
        u64 m_all = 0;
        for (int b = tid; b < n; b += kThreads) {
            unsigned c = 0;
            u64 m = 0;
            for (int r = 0; r < ranks; ++r) {
                c += cluster.map_shared_rank(raw_count, r)[rank * n + b];
                if (need_mass) m += cluster.map_shared_rank(raw_mass, r)[rank * n + b];
            }
            merged_count[level * n + b] = c;
            merged_mass[level * n + b] = m;
            c_all += c;
            m_all += m;
        }
        c_all = __reduce_add_sync(0xffffffffu, c_all);
        m_all = warp_sum_u64(m_all);
        if (lane == 0) {
            sh.warp_u32[warp] = c_all;
            sh.warp_u64[warp] = m_all;
        }
        __syncthreads();
        if (tid == 0) {
            unsigned c = 0;
            u64 m = 0;
            for (int w = 0; w < kWarps; ++w) {
                c += sh.warp_u32[w];
                m += sh.warp_u64[w];
            }
            sh.chunk_count[level] = c;
            sh.chunk_mass[level] = m;
        }
        cluster.sync();
    }

    // Where the running count reaches k (by_mass false) or the running weight `target`.
    __device__ __forceinline__ bool reached(bool by_mass, unsigned count, u64 mass, unsigned k, double target) const {
        return by_mass ? !(static_cast<double>(mass) < target) : count >= k;
    }

    // Finds the bin of `level` where the cut lies; false when no bin reaches it.
    __device__ bool find_bin(int level, bool by_mass, unsigned k, double target, unsigned count, u64 mass) {
        const int n = kBins / ranks;
        int owner = -1;
        for (int r = 0; r < ranks; ++r) {
            const Shared* other = cluster.map_shared_rank(&sh, r);
            const unsigned c = other->chunk_count[level];
            const u64 m = other->chunk_mass[level];
            if (reached(by_mass, count + c, mass + m, k, target)) {
                owner = r;
                break;
            }
            count += c;
            mass += m;
        }
        if (owner < 0) return false;
        const unsigned* counts = cluster.map_shared_rank(merged_count, owner) + level * n;
        const u64* masses = cluster.map_shared_rank(merged_mass, owner) + level * n;
        // Each thread takes `per` consecutive bins.
        const int per = (n + kThreads - 1) / kThreads;
        unsigned c_mine = 0;
        u64 m_mine = 0;
        for (int i = 0; i < per; ++i) {
            const int b = tid * per + i;
            if (b < n) {
                c_mine += counts[b];
                m_mine += masses[b];
            }
        }
        unsigned c_in = c_mine;
        u64 m_in = m_mine;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned tc = __shfl_up_sync(0xffffffffu, c_in, o);
            const u64 tm = __shfl_up_sync(0xffffffffu, m_in, o);
            if (lane >= o) {
                c_in += tc;
                m_in += tm;
            }
        }
        if (lane == 31) {
            sh.warp_u32[warp] = c_in;
            sh.warp_u64[warp] = m_in;
        }
        __syncthreads();
        for (int w = 0; w < warp; ++w) {
            c_in += sh.warp_u32[w];
            m_in += sh.warp_u64[w];
        }
        unsigned c = count + c_in - c_mine;
        u64 m = mass + m_in - m_mine;
        if (!reached(by_mass, c, m, k, target) || (c == 0 && m == 0)) {
            for (int i = 0; i < per; ++i) {
                const int b = tid * per + i;
                if (b >= n) break;
                const unsigned tc = counts[b];
                const u64 tm = masses[b];
                if (tc != 0u && reached(by_mass, c + tc, m + tm, k, target)) {
                    sh.bin = owner * n + b;
                    sh.bin_count = tc;
                    sh.before_count = c;
                    sh.before_mass = m;
                    break;
                }
                c += tc;
                m += tm;
            }
        }
        __syncthreads();
        return true;
    }

    // The cut: the rank value of the last kept token (0 when all are kept), and in `kept` the
    // weight up to it. Level 0 of the histogram has been merged.
    __device__ u64 cut(bool by_mass, unsigned k, double target, u64& kept) {
        if (!find_bin(0, by_mass, k, target, 0u, 0ull)) return 0ull;
        int level = 0;
        int bin = sh.bin;
        unsigned members = sh.bin_count, before_count = sh.before_count;
        u64 before_mass = sh.before_mass;
        u64 hi = 0ull, lo = 0ull;  // rank values of the bin's members, from level 1 on
        while (members > static_cast<unsigned>(kList)) {
            if (level == 0) {
                u64 a = 0ull, b = ~0ull;
                each([&](float x, int id) {
                    const float d = distance(x);
                    if (d <= spread && bin_of(d) == bin) {
                        const u64 v = rank_value(x, id);
                        a = v > a ? v : a;
                        b = v < b ? v : b;
                    }
                });
                a = warp_max_u64(a);
                b = ~warp_max_u64(~b);
                __syncthreads();
                if (tid == 0) {
                    sh.range_hi = 0ull;
                    sh.range_lo = ~0ull;
                }
                __syncthreads();
                if (lane == 0) {
                    atomicMax(&sh.range_hi, a);
                    atomicMin(&sh.range_lo, b);
                }
                cluster.sync();
                hi = 0ull;
                lo = ~0ull;
                for (int r = 0; r < ranks; ++r) {
                    const Shared* other = cluster.map_shared_rank(&sh, r);
                    hi = max(hi, other->range_hi);
                    lo = min(lo, other->range_lo);
                }
            }
            const int bits = 64 - __clzll(static_cast<long long>(hi - lo) | 1ll);
            const int shift = bits > 11 ? bits - 11 : 0;
            clear_histogram();
            each([&](float x, int id) {
                const u64 v = rank_value(x, id);
                if (v <= hi && v >= lo) count(static_cast<int>((hi - v) >> shift), x);
            });
            merge(1);
            find_bin(1, by_mass, k, target, before_count, before_mass);
            level = 1;
            bin = sh.bin;
            members = sh.bin_count;
            before_count = sh.before_count;
            before_mass = sh.before_mass;
            hi -= static_cast<u64>(bin) << shift;
            const u64 width = (1ull << shift) - 1ull;
            lo = hi - lo > width ? hi - width : lo;
            __syncthreads();
        }
        // The bin's members, from all CTAs.
        if (tid == 0) sh.listed = 0u;
        __syncthreads();
        each([&](float x, int id) {
            u64 v;
            if (level == 0) {
                const float d = distance(x);
                if (!(d <= spread) || bin_of(d) != bin) return;
                v = rank_value(x, id);
            } else {
                v = rank_value(x, id);
                if (v > hi || v < lo) return;
            }
            const unsigned at = atomicAdd(&sh.listed, 1u);
            own_list[at] = v;
            own_list[kList + at] = need_mass ? weight(x) : 0ull;
        });
        cluster.sync();
        int n = 0;
        for (int r = 0; r < ranks; ++r) {
            const int m = static_cast<int>(cluster.map_shared_rank(&sh, r)->listed);
            const u64* theirs = cluster.map_shared_rank(own_list, r);
            for (int i = tid; i < m; i += kThreads) {
                list[n + i] = theirs[i];
                list[kList + n + i] = theirs[kList + i];
            }
            n += m;
        }
        __syncthreads();
        for (int i = tid; i < n; i += kThreads) {
            const u64 v = list[i];
            unsigned c = before_count;
            u64 m = before_mass;
            for (int j = 0; j < n; ++j) {
                if (list[j] > v) {
                    ++c;
                    m += list[kList + j];
                }
            }
            const u64 with = m + list[kList + i];
            // Every token of the bin ranked at or before the one that reaches the cut is kept.
            const bool open = by_mass ? (static_cast<double>(m) < target || c == 0) : c < k;
            if (open && reached(by_mass, c + 1, with, k, target)) {
                sh.cut = v;
                sh.cut_mass = with;
            }
        }
        cluster.sync();  // the lists are free again in every CTA
        kept = sh.cut_mass;
        return sh.cut;
    }

    __device__ void run();
};

template <typename T>
__device__ void Row<T>::run() {
    const int row = static_cast<int>(blockIdx.x) / ranks;
    const T* src = static_cast<const T*>(p.logits) + row * p.row_stride + first;
    const int have = max(0, min(p.slice, p.vocab - first));
    const int share = p.slice / kWarps;

    // ---- load, maximum and minimum ----
    float hi = -INFINITY, lo = INFINITY;
    const bool wide = (reinterpret_cast<uintptr_t>(src) & 15u) == 0;
#pragma unroll 4
    for (int at = warp * share + lane * V::kN; at < (warp + 1) * share; at += 32 * V::kN) {
        uint4 v;
        T* e = reinterpret_cast<T*>(&v);
        if (wide && at + V::kN <= have) {
            v = __ldg(reinterpret_cast<const uint4*>(src + at));
        } else {
#pragma unroll
            for (int i = 0; i < V::kN; ++i) e[i] = at + i < have ? src[at + i] : V::lowest();
        }
        float x[V::kN];
        V::unpack(v, x);
#pragma unroll
        for (int i = 0; i < V::kN; ++i) {
            if (x[i] != x[i]) {  // NaN: never drawn
                e[i] = V::lowest();
                x[i] = -INFINITY;
            }
            hi = fmaxf(hi, x[i]);
            if (x[i] != -INFINITY) lo = fminf(lo, x[i]);
        }
        *reinterpret_cast<uint4*>(data + at) = v;
    }
    hi = warp_max_f32(hi);
    lo = -warp_max_f32(-lo);
    if (lane == 0) {
        sh.warp_f32[0][warp] = hi;
        sh.warp_f32[1][warp] = lo;
    }
    __syncthreads();
    if (tid == 0) {
        for (int w = 0; w < kWarps; ++w) {
            hi = fmaxf(hi, sh.warp_f32[0][w]);
            lo = fminf(lo, sh.warp_f32[1][w]);
        }
        sh.top = hi;
        sh.low = lo;
        sh.best = 0ull;
    }
    cluster.sync();
    top = -INFINITY;
    lo = INFINITY;
    for (int r = 0; r < ranks; ++r) {
        const Shared* other = cluster.map_shared_rank(&sh, r);
        top = fmaxf(top, other->top);
        lo = fminf(lo, other->low);
    }
    if (top == -INFINITY) {
        if (rank == 0 && tid == 0) {
            p.tokens[row] = -1;
            if (p.logprobs != nullptr) p.logprobs[row] = -FLT_MAX;
        }
        return;
    }

    t = p.temperature != nullptr ? p.temperature[row] : 1.0f;
    unsigned k = p.top_k != nullptr && p.top_k[row] > 0 ? static_cast<unsigned>(p.top_k[row]) : 0u;
    float top_p = p.top_p != nullptr ? p.top_p[row] : 1.0f;
    float min_p = p.min_p != nullptr ? p.min_p[row] : 0.0f;
    if (!(min_p > 0.0f)) min_p = 0.0f;
    if (!(t > 0.0f) || k == 1u || top_p <= 0.0f || min_p > 1.0f) {
        // Only the first ranked token is kept.
        u64 best = 0ull;
        each([&](float x, int id) {
            if (x == top) best = max(best, rank_value(x, id));
        });
        best = warp_max_u64(best);
        if (lane == 0) atomicMax(&sh.best, best);
        cluster.sync();
        if (rank == 0 && tid == 0) {
            for (int r = 0; r < ranks; ++r) best = max(best, cluster.map_shared_rank(&sh, r)->best);
            p.tokens[row] = key_id(best);
            if (p.logprobs != nullptr) p.logprobs[row] = 0.0f;
        }
        return;
    }

    u64 limit = 0ull;  // kept: rank value >= limit
    need_mass = top_p < 1.0f;
    if (need_mass || k != 0u) {
        spread = fminf(top - lo, kWeightless * t);
        if (!(spread > 0.0f)) spread = 0.0f;
        to_bin = spread > 0.0f ? fminf((kBins - 0.01f) / spread, 1e30f) : 0.0f;
        clear_histogram();
        each([&](float x, int) {
            const float d = distance(x);
            if (d <= spread) count(bin_of(d), x);
        });
        merge(0);
        u64 total = 0ull;
        for (int r = 0; r < ranks; ++r) total += cluster.map_shared_rank(&sh, r)->chunk_mass[0];
        if (k != 0u) limit = cut(false, k, 0.0, total);
        if (need_mass) {
            const u64 l = cut(true, 0u, static_cast<double>(top_p) * static_cast<double>(total), total);
            limit = max(limit, l);
        }
    }

    // ---- the kept weight, in ascending id order ----
    u64 mine = 0ull;
    each([&](float x, int id) {
        if (rank_value(x, id) < limit) return;
        const float e = share_of(x);
        if (e >= min_p) mine += static_cast<u64>(__float2ll_rn(e * kUnits));
    });
    mine = warp_sum_u64(mine);
    __syncthreads();
    if (lane == 0) sh.warp_u64[warp] = mine;
    __syncthreads();
    if (tid == 0) {
        u64 all = 0ull;
        for (int w = 0; w < kWarps; ++w) all += sh.warp_u64[w];
        sh.weight = all;
    }
    cluster.sync();
    u64 total = 0ull, before = 0ull;
    for (int r = 0; r < ranks; ++r) {
        const u64 w = cluster.map_shared_rank(&sh, r)->weight;
        if (r < rank) before += w;
        total += w;
    }
    float u = p.uniforms[row];
    u = u >= 0.0f ? fminf(u, 0.99999994f) : 0.0f;
    u64 target = static_cast<u64>(floor(static_cast<double>(u) * static_cast<double>(total)));
    if (target >= total) target = total - 1ull;
    for (int w = 0; w < warp; ++w) before += sh.warp_u64[w];
    if (target < before || target >= before + mine) return;
    for (int base = warp * share; base < (warp + 1) * share; base += 32 * V::kN) {
        const int at = base + lane * V::kN;
        float x[V::kN];
        V::unpack(*reinterpret_cast<const uint4*>(data + at), x);
        u64 w[V::kN], sum = 0ull;
#pragma unroll
        for (int i = 0; i < V::kN; ++i) {
            w[i] = 0ull;
            if (x[i] != -INFINITY && rank_value(x[i], first + at + i) >= limit) {
                const float e = share_of(x[i]);
                if (e >= min_p) w[i] = static_cast<u64>(__float2ll_rn(e * kUnits));
            }
            sum += w[i];
        }
        u64 upto = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const u64 v = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += v;
        }
        const u64 all = __shfl_sync(0xffffffffu, upto, 31);
        if (target < before + all) {
            u64 at_mine = before + upto - sum;
            if (target >= at_mine && target < at_mine + sum) {
#pragma unroll
                for (int i = 0; i < V::kN; ++i) {
                    if (target >= at_mine && target < at_mine + w[i]) {
                        p.tokens[row] = first + at + i;
                        if (p.logprobs != nullptr) {
                            p.logprobs[row] = static_cast<float>(log(static_cast<double>(w[i]) / static_cast<double>(total)));
                        }
                    }
                    at_mine += w[i];
                }
            }
            break;
        }
        before += all;
    }
}

// Shared memory after the slice: [histogram | own list and list share it] [merged, two levels].
constexpr size_t kWorkBytes = 4ull * kList * 8 > 12ull * kBins ? 4ull * kList * 8 : 12ull * kBins;

size_t smem_bytes(int slice, int cluster, size_t element) { return slice * element + kWorkBytes + 2ull * (kBins / cluster) * 12; }

template <typename T>
__global__ void __launch_bounds__(kThreads) sample_kernel(const SampleParams p) {
    extern __shared__ __align__(16) uint8_t smem[];
    __shared__ Shared sh;
    Row<T> row(p, sh);
    row.ranks = static_cast<int>(row.cluster.num_blocks());
    row.rank = static_cast<int>(row.cluster.block_rank());
    row.first = row.rank * p.slice;
    row.tid = threadIdx.x;
    row.lane = threadIdx.x & 31;
    row.warp = threadIdx.x >> 5;
    row.data = reinterpret_cast<T*>(smem);
    uint8_t* work = smem + static_cast<size_t>(p.slice) * sizeof(T);
    row.raw_mass = reinterpret_cast<u64*>(work);
    row.raw_count = reinterpret_cast<unsigned*>(work + 8 * kBins);
    row.own_list = reinterpret_cast<u64*>(work);
    row.list = row.own_list + 2 * kList;
    row.merged_mass = reinterpret_cast<u64*>(work + kWorkBytes);
    row.merged_count = reinterpret_cast<unsigned*>(row.merged_mass + 2 * (kBins / row.ranks));
    row.run();
    row.cluster.sync();  // no CTA leaves while another may still read its shared memory
}

int slice_of(int vocab, int cluster) {
    const int step = 32 * 8 * kWarps;
    const int each = (vocab + cluster - 1) / cluster;
    return (each + step - 1) / step * step;
}

template <typename T>
int launch(const SampleParams& base, int rows, cudaStream_t stream) {
    const auto kernel = sample_kernel<T>;
    cudaError_t e = ensure_smem_optin(reinterpret_cast<const void*>(kernel));
    if (e != cudaSuccess) return fail_cuda(e, "zcgvs_sample");
    const size_t limit = static_cast<size_t>(device_max_smem()) - sizeof(Shared) - 1024;
    // CTAs per row: enough to hold the row, then more while the rows leave SMs idle and a CTA
    // still has 4096 tokens.
    int cluster = 1;
    while (cluster < kMaxCluster && smem_bytes(slice_of(base.vocab, cluster), cluster, sizeof(T)) > limit) cluster *= 2;
    while (cluster < kMaxCluster && static_cast<long long>(rows) * cluster * 2 <= device_sm_count() && base.vocab / (cluster * 2) >= 4096) {
        cluster *= 2;
    }
    SampleParams p = base;
    p.slice = slice_of(p.vocab, cluster);
    const size_t smem = smem_bytes(p.slice, cluster, sizeof(T));
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(static_cast<unsigned>(rows * cluster));
    config.blockDim = dim3(kThreads);
    config.dynamicSmemBytes = smem;
    config.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = static_cast<unsigned>(cluster);
    attr[0].val.clusterDim.y = 1;
    attr[0].val.clusterDim.z = 1;
    config.attrs = attr;
    config.numAttrs = 1;
    KernelTimer timer("sample", stream);
    e = cudaLaunchKernelEx(&config, kernel, p);
    if (e != cudaSuccess) return fail_cuda(e, "zcgvs_sample");
    return ok();
}

}  // namespace
}  // namespace sampling
}  // namespace zc

extern "C" int zcgvs_sample(const void* logits, int dtype, int64_t row_stride, int rows, int vocab, const float* temperature,
                            const int* top_k, const float* top_p, const float* min_p, const float* uniforms, int* out_tokens,
                            float* out_logprobs, void* stream) {
    using namespace zc;
    using namespace zc::sampling;
    if (rows <= 0 || vocab <= 0) return ok();
    if (dtype != ZCGVS_DTYPE_F32 && dtype != ZCGVS_DTYPE_F16 && dtype != ZCGVS_DTYPE_BF16) {
        return fail(ZCGVS_ERR_INVALID_ARG, "zcgvs_sample: logits must be F32, F16 or BF16");
    }
    if (vocab > ZCGVS_MAX_VOCAB) return fail(ZCGVS_ERR_UNSUPPORTED, "zcgvs_sample: vocab exceeds ZCGVS_MAX_VOCAB");
    if (logits == nullptr || uniforms == nullptr || out_tokens == nullptr) {
        return fail(ZCGVS_ERR_INVALID_ARG, "zcgvs_sample: null logits, uniforms or out_tokens");
    }
    if (rows > 1 && row_stride < vocab) return fail(ZCGVS_ERR_INVALID_ARG, "zcgvs_sample: row_stride is smaller than vocab");
    if (!paged::aligned_to(logits, dtype == ZCGVS_DTYPE_F32 ? 4 : 2)) {
        return fail(ZCGVS_ERR_INVALID_ARG, "zcgvs_sample: logits are not aligned to their type");
    }
    if (rows > (1 << 26)) return fail(ZCGVS_ERR_INVALID_ARG, "zcgvs_sample: too many rows for one call");
    SampleParams p{};
    p.logits = logits;
    p.row_stride = row_stride;
    p.vocab = vocab;
    p.temperature = temperature;
    p.top_k = top_k;
    p.top_p = top_p;
    p.min_p = min_p;
    p.uniforms = uniforms;
    p.tokens = out_tokens;
    p.logprobs = out_logprobs;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    if (dtype == ZCGVS_DTYPE_F32) return launch<float>(p, rows, s);
    if (dtype == ZCGVS_DTYPE_F16) return launch<__half>(p, rows, s);
    return launch<__nv_bfloat16>(p, rows, s);
}
