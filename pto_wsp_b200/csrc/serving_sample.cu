// Token sampling: temperature, top-k, min-p and top-p, then one inverse of the cumulated weights per row.
//
// A weight is w = expf((x - max) / T), held as the whole number of 2^-40 below it: sums of whole numbers are exact, so the
// result depends on no order of summation and no atomics' order.  Candidates are ordered by composite = (key of x,
// ~index), a 64-bit number that falls with the logit and rises with the index, so every cut is one composite and ties
// need no counting.
//
// A cluster of CTAs holds a row in shared memory: it is read from HBM once, and every pass after that -- maximum,
// counts, masses, the pick -- runs over the copy.  A cut is found by a histogram over the logits' distance from the
// maximum (evenly spaced, where a radix over the bits would put most of a row into a few bins), and the elements of the
// bin that holds it are ranked against one another; a bin with too many is divided again over its range of composites.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <algorithm>

#include "serving.hpp"

namespace cg = cooperative_groups;

namespace ptowsp::dev {

namespace {

constexpr int kThreads = 512;
constexpr int kWarps = kThreads / 32;
constexpr int kBins = 1024;
constexpr int kList = 256;      // elements that are ranked by comparing all pairs
constexpr int kMaxCluster = 8;  // the portable size
constexpr float kReach = 28.f;  // e^-28 < 2^-40: what is further below the maximum weighs nothing
constexpr float kBinsPerUnit = kBins / kReach;

__device__ __forceinline__ float as_float(float x) { return x; }
__device__ __forceinline__ float as_float(__half x) { return __half2float(x); }
__device__ __forceinline__ float as_float(__nv_bfloat16 x) { return __bfloat162float(x); }

// Order-preserving keys: NaN as -inf, -0 as +0.
__device__ __forceinline__ uint32_t key_of(float x) {
    x = x == x ? x + 0.f : -INFINITY;
    const uint32_t u = __float_as_uint(x);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t k) {
    return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k);
}
__device__ __forceinline__ uint64_t composite(float x, int i) {
    return static_cast<uint64_t>(key_of(x)) << 32 | static_cast<uint32_t>(~i);
}

struct Element {
    uint64_t c;
    int64_t w;
};

// What a CTA shows to the others of its cluster.  Each step has a place of its own, written once between two barriers.
struct Board {
    uint64_t best;
    int64_t mass[3];
    int count[3];
    uint64_t low, high;
    int listed;
};

struct Shared {
    Board board;
    int64_t part[kWarps];
    uint64_t part64[kWarps];
    int64_t region[kWarps];
    uint64_t cut;
    int64_t cut_mass;
    int bin;
    int64_t before;
};
// only where a cut may be looked for
struct SharedCut {
    uint32_t hist[4][kBins];  // counts, and the masses' low 14, middle 14 and high bits: no sum passes 32 bits
    Element list[kList];      // this CTA's share
    Element all[kList];       // the cluster's
};

template <typename V, typename F>
__device__ V block_reduce(V v, F op, V* part) {
#pragma unroll
    for (int d = 16; d; d >>= 1) v = op(v, __shfl_xor_sync(~0u, v, d));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) part[threadIdx.x >> 5] = v;
    __syncthreads();
    v = part[threadIdx.x & (kWarps - 1)];
#pragma unroll
    for (int d = kWarps / 2; d; d >>= 1) v = op(v, __shfl_xor_sync(~0u, v, d));
    return v;
}

// Inclusive scan over the block.
__device__ int64_t block_inclusive(int64_t v, int64_t* part) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int64_t o = __shfl_up_sync(~0u, v, d);
        if (lane >= d) v += o;
    }
    __syncthreads();
    if (lane == 31) part[warp] = v;
    __syncthreads();
    for (int w = 0; w < warp; ++w) v += part[w];
    return v;
}

template <typename T, int CL, bool CUTS>
struct Row {
    const T* x;            // this CTA's slice, in shared memory
    Shared& sh;
    SharedCut* cuts;
    int first, n;          // its first index and its length
    float top, t, min_p;
    float low;             // what is below is no candidate
    uint64_t cut = 0;      // candidates are at or above

    __device__ void sync() const {
        if constexpr (CL > 1) cg::this_cluster().sync();
        else __syncthreads();
    }
    template <typename V>
    __device__ const V* of(const V* p, int rank) const {
        if constexpr (CL > 1) return cg::this_cluster().map_shared_rank(const_cast<V*>(p), rank);
        else return p;
    }
    __device__ float distance(float v) const { return __fdiv_rn(v - top, t); }
    // the candidate's weight, 0: none.  `v` is at or above `low`.
    __device__ int64_t weigh(float v, int i) const {
        float w = 1.f;
        if (v != top) {
            w = expf(distance(v));
            if (!(w >= min_p) || !(v > -INFINITY)) return 0;
        }
        if (CUTS && composite(v, first + i) < cut) return 0;
        return static_cast<int64_t>(w * 1099511627776.f);
    }
    __device__ int bin_of(float v) const {
        const float b = -distance(v) * kBinsPerUnit;
        return b < kBins ? static_cast<int>(b) : kBins - 1;  // NaN (an infinite row's rest) is in the last bin
    }

    // Calls f(value, index) for the slice's elements at or above `low`.
    template <typename F>
    __device__ void each(F f) const {
        for (int i = threadIdx.x; i < n; i += kThreads) {
            const float v = as_float(x[i]);
            if (!(v < low) && v == v) f(v, i);
        }
    }

    // Masses of the warps' regions, and the cluster's mass and count of candidates.
    __device__ void weigh_regions(int step, int64_t* mass, int* count) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const int size = region_size();
        int64_t m = 0;
        int k = 0;
        for (int i = warp * size + lane; i < min(n, (warp + 1) * size); i += 32) {
            const float v = as_float(x[i]);
            if (!(v < low) && v == v) {
                const int64_t w = weigh(v, i);
                m += w;
                k += w > 0;
            }
        }
#pragma unroll
        for (int d = 16; d; d >>= 1) m += __shfl_xor_sync(~0u, m, d);
        k = __reduce_add_sync(~0u, k);
        __syncthreads();
        if (lane == 0) {
            sh.region[warp] = m;
            sh.part[warp] = k;
        }
        __syncthreads();
        if (threadIdx.x == 0) {
            int64_t all = 0;
            int c = 0;
            for (int w = 0; w < kWarps; ++w) {
                all += sh.region[w];
                c += static_cast<int>(sh.part[w]);
            }
            sh.board.mass[step] = all;
            sh.board.count[step] = c;
        }
        sync();
        *mass = 0;
        *count = 0;
        for (int r = 0; r < CL; ++r) {
            const Board* b = of(&sh.board, r);
            *mass += b->mass[step];
            *count += b->count[step];
        }
    }
    __device__ int region_size() const { return ((n + kWarps - 1) / kWarps + 31) & ~31; }

    // Gathers the cluster's lists (at most kList elements in all) and finds the element at which the running measure,
    // from `before` on, reaches `target`: sets `cut` to it and returns the measure with it.
    template <bool MASS>
    __device__ int64_t rank_list(int64_t before, int64_t target, int total) {
        int at = 0;
        for (int r = 0; r < CL; ++r) {
            const int k = of(&sh.board, r)->listed;
            const Element* from = of(cuts->list, r);
            for (int i = threadIdx.x; i < k; i += kThreads) cuts->all[at + i] = from[i];
            at += k;
        }
        __syncthreads();
        // two threads per element, each against half of the list
        const int e = threadIdx.x >> 1, half = threadIdx.x & 1;
        const Element me = e < total ? cuts->all[e] : Element{0, 0};
        int64_t m = 0;
        for (int j = half; j < total; j += 2) {
            const Element o = cuts->all[j];
            if (o.c > me.c) m += MASS ? o.w : 1;
        }
        m += __shfl_xor_sync(~0u, m, 1);
        m += before;
        const int64_t with = m + (MASS ? me.w : 1);
        if (e < total && half == 0 && m < target && with >= target) {
            sh.cut = me.c;
            sh.cut_mass = with;
        }
        __syncthreads();
        cut = sh.cut;
        return sh.cut_mass;
    }

    // Lists the candidates that `in` takes; the cluster's number of them (the lists hold them all if it is <= kList).
    template <typename F>
    __device__ int list(F in) {
        sync();  // the last list has been read
        if (threadIdx.x == 0) sh.board.listed = 0;
        __syncthreads();
        each([&](float v, int i) {
            int64_t w;
            if (in(v, i, &w)) {
                const int at = atomicAdd(&sh.board.listed, 1);
                if (at < kList) cuts->list[at] = Element{composite(v, first + i), w};
            }
        });
        sync();
        int total = 0;
        for (int r = 0; r < CL; ++r) total += of(&sh.board, r)->listed;
        return total;
    }

    // Finds the element at which the measure of the candidates, in falling order, reaches `target` (>= 1, at most the
    // whole): the count (MASS false: every element within reach is a candidate) or the mass (those of at least `least`).
    template <bool MASS>
    __device__ int64_t find_cut(int64_t target, int64_t least) {
        uint64_t lo = 0, hi = ~0ull;  // range of composites that holds the element
        int shift = -1;               // bins: of the distance (-1), else of the composite's distance from hi
        int64_t before = 0;
        for (;;) {
            sync();  // the histograms and the board have been read
            for (int i = threadIdx.x; i < 4 * kBins; i += kThreads) (&cuts->hist[0][0])[i] = 0;
            __syncthreads();
            const auto place = [&](float v, int i, int64_t* w, int* bin) {
                const uint64_t c = composite(v, first + i);
                if (c < lo || c > hi) return false;
                if (MASS) {
                    *w = weigh(v, i);
                    if (*w < least || *w == 0) return false;
                } else {
                    *w = 0;
                }
                *bin = shift < 0 ? bin_of(v) : static_cast<int>((hi - c) >> shift);
                return true;
            };
            each([&](float v, int i) {
                int64_t w;
                int b;
                if (!place(v, i, &w, &b)) return;
                atomicAdd(&cuts->hist[0][b], 1u);
                if (MASS) {
                    if (w & 0x3fff) atomicAdd(&cuts->hist[1][b], static_cast<uint32_t>(w & 0x3fff));
                    if (w >> 14 & 0x3fff) atomicAdd(&cuts->hist[2][b], static_cast<uint32_t>(w >> 14 & 0x3fff));
                    if (w >> 28) atomicAdd(&cuts->hist[3][b], static_cast<uint32_t>(w >> 28));
                }
            });
            sync();
            // each thread sums consecutive bins over the cluster; the thread in whose bins the target lies says which
            constexpr int PER = kBins / kThreads;
            int64_t mine[PER], sum = 0;
            int counts[PER];
#pragma unroll
            for (int b = 0; b < PER; ++b) {
                mine[b] = 0;
                counts[b] = 0;
            }
            for (int r = 0; r < CL; ++r) {
                const uint32_t* h = of(&cuts->hist[0][0], r);
#pragma unroll
                for (int b = 0; b < PER; ++b) {
                    const int at = threadIdx.x * PER + b;
                    const uint32_t k = h[at];
                    counts[b] += k;
                    if (MASS) {
                        if (k)
                            mine[b] += static_cast<int64_t>(h[kBins + at]) + (static_cast<int64_t>(h[2 * kBins + at]) << 14) +
                                       (static_cast<int64_t>(h[3 * kBins + at]) << 28);
                    } else {
                        mine[b] += k;
                    }
                }
            }
#pragma unroll
            for (int b = 0; b < PER; ++b) sum += mine[b];
            int64_t run = before + block_inclusive(sum, sh.part) - sum;
#pragma unroll
            for (int b = 0; b < PER; ++b) {
                if (run < target && run + mine[b] >= target) {
                    sh.bin = threadIdx.x * PER + b;
                    sh.before = run;
                    sh.cut_mass = counts[b];
                }
                run += mine[b];
            }
            __syncthreads();
            const int bin = sh.bin;
            before = sh.before;
            const int64_t in_bin = sh.cut_mass;
            const auto inside = [&](float v, int i, int64_t* w) {
                int b;
                return place(v, i, w, &b) && b == bin;
            };
            if (in_bin <= kList) {
                const int total = list(inside);
                return rank_list<MASS>(before, target, total);
            }
            // too many for the list: divide the range of their composites
            uint64_t a = ~0ull, z = 0;
            each([&](float v, int i) {
                int64_t w;
                if (!inside(v, i, &w)) return;
                const uint64_t c = composite(v, first + i);
                a = min(a, c);
                z = max(z, c);
            });
            a = block_reduce(a, [](uint64_t p, uint64_t q) { return min(p, q); }, sh.part64);
            z = block_reduce(z, [](uint64_t p, uint64_t q) { return max(p, q); }, sh.part64);
            if (threadIdx.x == 0) {
                sh.board.low = a;
                sh.board.high = z;
            }
            sync();
            lo = ~0ull;
            hi = 0;
            for (int r = 0; r < CL; ++r) {
                const Board* b = of(&sh.board, r);
                lo = min(lo, b->low);
                hi = max(hi, b->high);
            }
            shift = 0;
            while ((hi - lo) >> shift >= kBins) ++shift;
        }
    }
};

template <typename T, int CL, bool CUTS>
__global__ void __launch_bounds__(kThreads, CUTS ? 2 : 3) sample_kernel(SampleArgs a, int slice) {
    extern __shared__ __align__(16) char smem[];
    __shared__ Shared sh;
    SharedCut* cuts = reinterpret_cast<SharedCut*>(smem);
    T* x = reinterpret_cast<T*>(smem + (CUTS ? sizeof(SharedCut) : 0));
    const int r = blockIdx.x / CL, rank = CL > 1 ? static_cast<int>(cg::this_cluster().block_rank()) : 0;
    const int first = rank * slice, n = max(0, min(a.vocab - first, slice));
    const T* from = static_cast<const T*>(a.logits) + r * a.row_stride + first;

    // -- read the slice once: 16 bytes at a time where the row allows it --
    constexpr int V = 16 / sizeof(T);
    uint64_t best = 0;
    const int head = static_cast<int>(min(static_cast<int64_t>(n), static_cast<int64_t>(
                                                                       (16 - (reinterpret_cast<uintptr_t>(from) & 15)) & 15) /
                                                                       static_cast<int64_t>(sizeof(T))));
    const int packs = (n - head) / V;
    const auto take = [&](T v, int i) {
        x[i] = v;
        best = max(best, composite(as_float(v), first + i));
    };
    for (int i = threadIdx.x; i < head; i += kThreads) take(from[i], i);
    constexpr int U = 4;
    for (int p0 = threadIdx.x; p0 < packs; p0 += kThreads * U) {
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (p0 + u * kThreads < packs) w[u] = __ldcs(reinterpret_cast<const uint4*>(from + head) + p0 + u * kThreads);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (p0 + u * kThreads >= packs) continue;
            const T* v = reinterpret_cast<const T*>(&w[u]);
#pragma unroll
            for (int k = 0; k < V; ++k) take(v[k], head + (p0 + u * kThreads) * V + k);
        }
    }
    for (int i = head + packs * V + threadIdx.x; i < n; i += kThreads) take(from[i], i);
    best = block_reduce(best, [](uint64_t p, uint64_t q) { return max(p, q); }, sh.part64);

    Row<T, CL, CUTS> row{x, sh, cuts, first, n};
    if (threadIdx.x == 0) sh.board.best = best;
    row.sync();
    for (int c = 0; c < CL; ++c) best = max(best, row.of(&sh.board, c)->best);
    row.top = value_of(static_cast<uint32_t>(best >> 32));
    const float temperature = a.temperature ? a.temperature[r] : 1.f;
    const bool none = row.top == -INFINITY, greedy = !(temperature > 0.f);
    if (none || greedy) {
        if (rank == 0 && threadIdx.x == 0) {
            a.token[r] = none ? -1 : static_cast<int>(~static_cast<uint32_t>(best));
            if (a.logprob) a.logprob[r] = none ? -INFINITY : 0.f;
        }
        row.sync();  // no CTA leaves while another may read its board
        return;
    }
    row.t = temperature;
    row.min_p = a.min_p ? fminf(a.min_p[r], 1.f) : 0.f;
    // NaN, where both are infinite, takes everything
    row.low = row.top - (kReach + 0.5f) * temperature;
    int64_t mass;
    int count;
    if constexpr (CUTS) {
        const int k = a.top_k ? a.top_k[r] : 0;
        const float top_p = a.top_p ? a.top_p[r] : 1.f;
        if (k > 0) {
            // fewer within reach than k: no cut
            int near = 0;
            row.each([&](float, int) { ++near; });
            near = static_cast<int>(block_reduce<int64_t>(near, [](int64_t p, int64_t q) { return p + q; }, sh.part));
            if (threadIdx.x == 0) sh.board.count[2] = near;
            row.sync();
            near = 0;
            for (int c = 0; c < CL; ++c) near += row.of(&sh.board, c)->count[2];
            if (k < near) {
                row.template find_cut<false>(k, 0);
                row.low = fmaxf(row.low, value_of(static_cast<uint32_t>(row.cut >> 32)));
            }
        }
        row.weigh_regions(0, &mass, &count);
        if (top_p < 1.f) {
            int64_t limit = static_cast<int64_t>(ceil(static_cast<double>(top_p) * static_cast<double>(mass)));
            if (limit < 1) limit = 1;
            if (limit < mass) {
                // weights below (1 - p) mass / (2 count) are together less than what stays out
                const double least = 0.5 * (1.0 - static_cast<double>(top_p)) * static_cast<double>(mass) / count;
                row.template find_cut<true>(limit, static_cast<int64_t>(fmax(least, 0.0)));
                row.low = fmaxf(row.low, value_of(static_cast<uint32_t>(row.cut >> 32)));
                row.weigh_regions(1, &mass, &count);
            }
        }
    } else {
        row.weigh_regions(0, &mass, &count);
    }

    // -- the pick: the CTA, then the warp's region, then the element --
    int64_t pick = static_cast<int64_t>(static_cast<double>(a.u[r]) * static_cast<double>(mass));
    if (pick > mass - 1) pick = mass - 1;
    if (pick < 0) pick = 0;
    // this CTA's masses, as every CTA of the cluster knows its own
    int64_t mine = 0;
    for (int w = 0; w < kWarps; ++w) mine += sh.region[w];
    if (threadIdx.x == 0) sh.board.mass[2] = mine;
    row.sync();
    int64_t before = 0;
    for (int c = 0; c < rank; ++c) before += row.of(&sh.board, c)->mass[2];
    if (pick >= before && pick < before + mine) {
        int region = 0;
        while (pick >= before + sh.region[region]) before += sh.region[region++];
        const int size = row.region_size(), begin = region * size, end = min(n, begin + size);
        const int per = (size + kThreads - 1) / kThreads;
        const int i0 = begin + threadIdx.x * per, i1 = min(end, i0 + per);
        int64_t sum = 0;
        const auto weight = [&](int i) -> int64_t {
            const float v = as_float(x[i]);
            return !(v < row.low) && v == v ? row.weigh(v, i) : 0;
        };
        for (int i = i0; i < i1; ++i) sum += weight(i);
        int64_t run = before + block_inclusive(sum, sh.part) - sum;
        if (pick >= run && pick < run + sum) {
            for (int i = i0; i < i1; ++i) {
                const int64_t w = weight(i);
                if (pick < run + w) {
                    a.token[r] = first + i;
                    if (a.logprob) a.logprob[r] = logf(static_cast<float>(w) / static_cast<float>(mass));
                    break;
                }
                run += w;
            }
        }
    }
    row.sync();
}

template <typename T, int CL, bool CUTS>
cudaError_t launch(const SampleArgs& a, int slice, cudaStream_t s) {
    const int smem = slice * static_cast<int>(sizeof(T)) + (CUTS ? static_cast<int>(sizeof(SharedCut)) : 0);
    static SmemOptIn opt_in;
    cudaError_t e = opt_in.once(reinterpret_cast<const void*>(sample_kernel<T, CL, CUTS>), kSampleMaxSmem);
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3(static_cast<unsigned>(a.rows) * CL);
    cfg.blockDim = dim3(kThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = CL;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = CL > 1 ? 1 : 0;
    return cudaLaunchKernelEx(&cfg, sample_kernel<T, CL, CUTS>, a, slice);
}

template <typename T, bool CUTS>
cudaError_t launch_cluster(const SampleArgs& a, int sms, cudaStream_t s) {
    const int extra = CUTS ? static_cast<int>(sizeof(SharedCut)) : 0;
    const auto slice_of = [&](int cl) { return ((a.vocab + cl - 1) / cl + 7) & ~7; };
    const auto bytes_of = [&](int cl) { return slice_of(cl) * static_cast<int64_t>(sizeof(T)) + extra; };
    const auto per_sm = [&](int cl) { return std::min<int64_t>(CUTS ? 2 : 3, (227 << 10) / (bytes_of(cl) + 2048)); };
    // Few rows: the most CTAs per row that the GPU holds at once.  More rows than that: the fewest that still let one
    // row be read while others on the SM are worked on.
    int cl = 0;
    for (int c = kMaxCluster; c >= 1 && !cl; c /= 2)
        if ((c == 1 || slice_of(c) >= 512) && static_cast<int64_t>(a.rows) * c <= per_sm(c) * sms) cl = c;
    for (int c = 1; c <= kMaxCluster && !cl; c *= 2)
        if (per_sm(c) >= (CUTS ? 2 : 3) || c == kMaxCluster) cl = c;
    if (bytes_of(cl) > kSampleMaxSmem) return cudaErrorInvalidValue;
    switch (cl) {
        case 1: return launch<T, 1, CUTS>(a, slice_of(1), s);
        case 2: return launch<T, 2, CUTS>(a, slice_of(2), s);
        case 4: return launch<T, 4, CUTS>(a, slice_of(4), s);
        default: return launch<T, 8, CUTS>(a, slice_of(8), s);
    }
}

template <typename T>
cudaError_t launch_type(const SampleArgs& a, int sms, cudaStream_t s) {
    return a.top_k || a.top_p ? launch_cluster<T, true>(a, sms, s) : launch_cluster<T, false>(a, sms, s);
}

}  // namespace

cudaError_t launch_sample(const SampleArgs& a, int sms, cudaStream_t s) {
    if (a.rows == 0) return cudaSuccess;
    switch (a.dtype) {
        case PTOWSP_F32: return launch_type<float>(a, sms, s);
        case PTOWSP_F16: return launch_type<__half>(a, sms, s);
        default: return launch_type<__nv_bfloat16>(a, sms, s);
    }
}

}  // namespace ptowsp::dev
