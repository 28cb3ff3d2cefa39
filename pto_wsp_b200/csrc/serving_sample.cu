// Token sampling: temperature, top-k, min-p and top-p, then one inverse of the cumulated weights per row.
//
// A weight is w = expf((x - max) / T), held as the whole number of 2^-40 below it: sums of whole numbers are exact, so the
// result depends on no order of summation and no atomics' order.  Candidates are ordered by composite = (key of x,
// ~index), a 64-bit number that falls with the logit and rises with the index, so every cut is one composite and ties
// need no counting.
//
// A cluster of CTAs holds a row in shared memory: it is read from HBM once, and every pass after that -- maximum,
// counts, masses, the pick -- runs over the copy.  The logits' distance from the maximum is cut into even bins, where a
// radix over the bits would put most of a row into a few.  Top-k lists the likely elements and ranks them against one
// another.  Top-p counts the elements of each bin; a bin's edges bound its mass, so counts alone leave a window of few
// bins that can hold the cut, and only the window is summed by mass.  A bin with too many elements is divided again
// over its range of composites.
//
// Bound by a row's chain of barriers: a pass over a slice in shared memory takes about a microsecond, and each pass waits
// for the one before.  One row of 50,021 (top-p) takes 15 to 43 us on the device: 15 to 22 where the counts leave no
// more candidates than can be ranked at once, 32 to 43 where the window has to be summed by mass, as in 14 of 24 drawn
// rows.  64 rows of 131,072 with all filters take 29 us as a whole call (17 MB, 0.6 TB/s), 509 rows of 32,000 without filters 37.6 (65 MB,
// 1.7 TB/s).  Two rows in flight per cluster took 60 for the last, slices read from L1 and L2 instead of shared memory
// 37-52.
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
constexpr float kSmallest = 9.094947e-13f;  // 2^-40

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

// w * 2^40 without its fraction, for 0 <= w <= 1: the 24 significant bits, moved (the conversion instruction for 64-bit
// integers has a sixteenth of this rate).
__device__ __forceinline__ int64_t whole_of(float w) {
    const uint32_t u = __float_as_uint(w);
    const int e = static_cast<int>(u >> 23) - 110;  // w = m * 2^(e - 40)
    const uint64_t m = (u & 0x7fffffu) | 0x800000u;
    return e >= 0 ? static_cast<int64_t>(m << e) : e > -24 ? static_cast<int64_t>(static_cast<uint32_t>(m) >> -e) : 0;
}

// What a CTA shows to the others of its cluster.  Each step has a place of its own, written once between two barriers.
struct Board {
    float top;
    int index;
    int64_t mass[3];
    int count[3];
    uint64_t low, high;
    int64_t above;
    int listed;
};

struct Shared {
    Board board;
    int64_t part[kWarps];
    uint64_t part64[kWarps];
    int64_t region[kWarps];
    uint64_t cut;
    int bin;
    int64_t before;
    int first_bin, last_bin, near;
};
// only where a cut may be looked for
struct SharedCut {
    uint32_t hist[3][kBins];  // counts, or the masses' low 14, middle 14 and high bits: no sum passes 32 bits
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
    float inv;             // RN(1 / t) where the quotient may be made from it, else 0
    float low;             // what is below is no candidate
    uint64_t cut = 0;      // candidates are at or above
    bool raised = false;   // `low` leaves out elements that have a weight

    __device__ void sync() const {
        if constexpr (CL > 1) cg::this_cluster().sync();
        else __syncthreads();
    }
    template <typename V>
    __device__ const V* of(const V* p, int rank) const {
        if constexpr (CL > 1) return cg::this_cluster().map_shared_rank(const_cast<V*>(p), rank);
        else return p;
    }
    // (v - top) / t, correctly rounded: Markstein's theorem gives that from RN(1 / t) by one fused correction of a
    // quotient that is within an ulp, which the first correction makes it.  For t within 2^-40 .. 2^40 no step
    // underflows, but where the quotient is so small that its exponential is 1.
    __device__ float distance(float v) const {
        const float a = v - top;
        float q = a * inv;
        q = fmaf(fmaf(-q, t, a), inv, q);
        return fmaf(fmaf(-q, t, a), inv, q);
    }
    __device__ float any_distance(float v) const { return inv != 0.f ? distance(v) : __fdiv_rn(v - top, t); }
    // the candidate's weight, 0: none.  `v` is at or above `low`, `d` its distance.
    __device__ int64_t weigh(float v, int i) const { return weigh(v, i, any_distance(v)); }
    __device__ int64_t weigh(float v, int i, float d) const {
        float w = 1.f;
        if (v != top) {
            w = expf(d);
            if (!(w >= min_p) || !(v > -INFINITY)) return 0;
        }
        if (CUTS && composite(v, first + i) < cut) return 0;
        return whole_of(w);
    }
    __device__ int bin_of(float v) const { return bin_at(any_distance(v)); }
    __device__ static int bin_at(float d) {
        const float b = -d * kBinsPerUnit;
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
    // COUNT: also the candidates' histogram of counts, over cleared bins; false where the row does not take that pass.
    template <bool COUNT>
    __device__ bool weigh_regions(int step, int64_t* mass, int* count) {
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        const int size = region_size(), end = min(n, (warp + 1) * size);
        int64_t m = 0;
        int k = 0;
        const bool open = inv != 0.f && top < INFINITY && !(CUTS && (cut || raised));
        if (open) {
            // The whole row, with no branch: the weight of -inf or NaN comes out as NaN and is none, what is out of reach
            // has no whole part.  w * 2^40 is taken in two parts of 20 bits: adding 2^23 with rounding towards zero
            // leaves floor(w * 2^20) in the low bits, and the rest of the product is exact.  A thread's parts sum to
            // less than 2^32: it has some 200 elements at most, and a part is at most 2^20.
            uint32_t hi = 0, lo = 0;
#pragma unroll 4
            for (int i = warp * size + lane; i < end; i += 32) {
                const float d = distance(as_float(x[i]));
                float w = expf(d);
                w = w >= min_p ? w : 0.f;
                const float h = __fmaf_rz(w, 1048576.f, 8388608.f);
                const float rest = fmaf(w, 1048576.f, 8388608.f - h);
                const float l = __fmaf_rz(rest, 1048576.f, 8388608.f);
                hi += __float_as_uint(h) - 0x4b000000u;
                lo += __float_as_uint(l) - 0x4b000000u;
                if (CUTS) k += w >= kSmallest;
                if (COUNT && w >= kSmallest) atomicAdd(&cuts->hist[0][bin_at(d)], 1u);
            }
            m = (static_cast<int64_t>(hi) << 20) + lo;
        } else {
            for (int i = warp * size + lane; i < end; i += 32) {
                const float v = as_float(x[i]);
                if (!(v < low) && v == v) {
                    const int64_t w = weigh(v, i);
                    m += w;
                    k += w > 0;
                }
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
#pragma unroll
        for (int r = 0; r < CL; ++r) {
            const Board* b = of(&sh.board, r);
            *mass += b->mass[step];
            *count += b->count[step];
        }
        return open;
    }
    __device__ int region_size() const { return ((n + kWarps - 1) / kWarps + 31) & ~31; }

    // Gathers the cluster's lists, at most kList elements in all.
    __device__ void gather() {
        int at = 0;
#pragma unroll
        for (int r = 0; r < CL; ++r) {
            const int k = of(&sh.board, r)->listed;
            const Element* from = of(cuts->list, r);
            for (int i = threadIdx.x; i < k; i += kThreads) cuts->all[at + i] = from[i];
            at += k;
        }
        __syncthreads();
    }

    // The element of the gathered list at which the running measure, from `before` on, reaches `target`: sets `cut`.
    template <bool MASS>
    __device__ void rank_list(int64_t before, int64_t target, int total) {
        gather();
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
        if (e < total && half == 0 && m < target && with >= target) sh.cut = me.c;
        __syncthreads();
        cut = sh.cut;
    }

    // All that is left to do where the lists hold every candidate: the first k of them (0: all), of these the shortest
    // prefix of mass `limit` (0: of top_p of their mass; top_p >= 1: all), and the pick by index.
    __device__ void finish_list(const SampleArgs& a, int r, int rank, int total, int k, float top_p, int64_t limit) {
        gather();
        const int e = threadIdx.x >> 1, half = threadIdx.x & 1;
        const bool real = e < total;
        const Element me = real ? cuts->all[e] : Element{0, 0};
        int64_t before = 0;
        int place = 0;
        for (int j = half; j < total; j += 2) {
            const Element o = cuts->all[j];
            if (o.c > me.c) {
                before += o.w;
                ++place;
            }
        }
        before += __shfl_xor_sync(~0u, before, 1);
        place += __shfl_xor_sync(~0u, place, 1);
        const auto add = [](int64_t p, int64_t q) { return p + q; };
        bool in = real && me.w > 0 && (k <= 0 || place < k);
        if (top_p < 1.f) {
            if (limit == 0) {
                const int64_t mass = block_reduce<int64_t>(in && half == 0 ? me.w : 0, add, sh.part);
                limit = limit_of(top_p, mass);
            }
            in = in && before < limit;
        }
        const int64_t mass = block_reduce<int64_t>(in && half == 0 ? me.w : 0, add, sh.part);
        const int64_t pick = pick_of(a.u[r], mass);
        if (half == 0 && real && !in) cuts->all[e].w = 0;
        __syncthreads();
        const uint32_t index = ~static_cast<uint32_t>(me.c);
        int64_t run = 0;
        for (int j = half; j < total; j += 2) {
            const Element o = cuts->all[j];
            if (~static_cast<uint32_t>(o.c) < index) run += o.w;
        }
        run += __shfl_xor_sync(~0u, run, 1);
        if (rank == 0 && half == 0 && in && pick >= run && pick < run + me.w) {
            a.token[r] = static_cast<int>(index);
            if (a.logprob) a.logprob[r] = logf(static_cast<float>(me.w) / static_cast<float>(mass));
        }
        sync();  // no CTA leaves while another may read its lists
    }
    __device__ static int64_t limit_of(float top_p, int64_t mass) {
        const int64_t limit = static_cast<int64_t>(ceil(static_cast<double>(top_p) * static_cast<double>(mass)));
        return limit < 1 ? 1 : limit;
    }
    __device__ static int64_t pick_of(float u, int64_t mass) {
        const int64_t pick = static_cast<int64_t>(static_cast<double>(u) * static_cast<double>(mass));
        return pick < 0 ? 0 : pick > mass - 1 ? mass - 1 : pick;
    }

    __device__ bool near_few() const {
        int k = 0;
        each([&](float, int) { ++k; });
        return block_reduce(k, [](int p, int q) { return p + q; }, reinterpret_cast<int*>(sh.part)) <= kList;
    }

    // Lists the candidates that `in` takes; the cluster's number of them (the lists hold them all if it is <= kList).
    // `sure`: `in` takes whatever is at or above `low`, so that counting these tells a list that is too short.
    template <typename F>
    __device__ int list(bool sure, F in) {
        sync();  // the last list has been read
        if (threadIdx.x == 0) sh.board.listed = 0;
        __syncthreads();
        if (sure && !near_few()) {
            if (threadIdx.x == 0) sh.board.listed = kList + 1;
        } else
        each([&](float v, int i) {
            int64_t w;
            // past the list's end only the fact counts, not how many
            if (in(v, i, &w) && *const_cast<volatile int*>(&sh.board.listed) <= kList) {
                const int at = atomicAdd(&sh.board.listed, 1);
                if (at < kList) cuts->list[at] = Element{composite(v, first + i), w};
            }
        });
        sync();
        int total = 0;
#pragma unroll
        for (int r = 0; r < CL; ++r) total += of(&sh.board, r)->listed;
        return total;
    }

    // Adds an element to the histogram: to its count, or to the three parts of its mass.
    template <bool MASS>
    __device__ void count_in(int bin, int64_t w) {
        if (!MASS) {
            atomicAdd(&cuts->hist[0][bin], 1u);
            return;
        }
        if (w & 0x3fff) atomicAdd(&cuts->hist[0][bin], static_cast<uint32_t>(w & 0x3fff));
        if (w >> 14 & 0x3fff) atomicAdd(&cuts->hist[1][bin], static_cast<uint32_t>(w >> 14 & 0x3fff));
        if (w >> 28) atomicAdd(&cuts->hist[2][bin], static_cast<uint32_t>(w >> 28));
    }
    // Sums the cluster's histograms and finds the bin in which the running measure, from `before` on, reaches `target`:
    // sh.bin (-1: none) and sh.before, the measure before it.
    template <bool MASS>
    __device__ void find_bin(int64_t before, int64_t target) {
        static_assert(kBins == 2 * kThreads, "two bins per thread");
        if (threadIdx.x == 0) sh.bin = -1;
        sync();
        int64_t m0 = 0, m1 = 0;
#pragma unroll
        for (int r = 0; r < CL; ++r) {
            const uint2* h = reinterpret_cast<const uint2*>(of(&cuts->hist[0][0], r)) + threadIdx.x;
            const uint2 a = h[0];
            m0 += a.x;
            m1 += a.y;
            if (MASS) {
                const uint2 b = h[kBins / 2], c = h[kBins];
                m0 += (static_cast<int64_t>(b.x) << 14) + (static_cast<int64_t>(c.x) << 28);
                m1 += (static_cast<int64_t>(b.y) << 14) + (static_cast<int64_t>(c.y) << 28);
            }
        }
        const int64_t end = before + block_inclusive(m0 + m1, sh.part), mid = end - m1, begin = mid - m0;
        if (begin < target && end >= target) {
            sh.bin = 2 * threadIdx.x + (mid >= target ? 0 : 1);
            sh.before = mid >= target ? begin : mid;
        }
        __syncthreads();
    }
    __device__ void clear_bins() {
        sync();  // the histograms have been read
        for (int i = threadIdx.x; i < 3 * kBins; i += kThreads) (&cuts->hist[0][0])[i] = 0;
        __syncthreads();
    }

    // Raises `low` to a logit that at least k candidates reach, because so many of the threads' own largest ones do.  The
    // likely tokens are few and mostly in shares of different threads, so few others are left above it, whatever the
    // vocabulary's size.
    __device__ void raise_low(int k, float own_top) {
        if (k > CL * kThreads / 2) return;
        clear_bins();
        if (!(own_top < low)) count_in<false>(bin_of(own_top), 1);
        find_bin<false>(0, k);
        if (sh.bin >= 0 && sh.bin < kBins - 1) drop_behind(sh.bin);
    }
    // Candidates are in the bins up to this one: `low` at its far edge, and a little more for the roundings.
    __device__ void drop_behind(int bin) {
        low = fmaxf(low, top - t * ((bin + 1) * (kReach / kBins) * 1.0001f));
        raised = true;
    }

    // The bins in which the running mass can reach `limit`, from the counts: a bin's weights lie between those of its
    // edges.  sh.first_bin, sh.last_bin, and sh.near candidates in the bins up to that.
    __device__ void window(int64_t limit) {
        if (threadIdx.x == 0) {
            sh.last_bin = kBins - 1;
            sh.near = INT32_MAX;
        }
        uint32_t c0 = 0, c1 = 0;
#pragma unroll
        for (int r = 0; r < CL; ++r) {
            const uint2 k = reinterpret_cast<const uint2*>(of(cuts->hist[0], r))[threadIdx.x];
            c0 += k.x;
            c1 += k.y;
        }
        const int b = 2 * threadIdx.x;
        const float e0 = expf(-b / kBinsPerUnit), e1 = expf(-(b + 1) / kBinsPerUnit), e2 = expf(-(b + 2) / kBinsPerUnit);
        // with room for the roundings of the bins and of the weights
        const auto above = [](float e) { return whole_of(fminf(e * 1.0001f, 1.f)) + 1; };
        const auto below = [](float e) { return whole_of(e * 0.9999f); };
        const int64_t u0 = c0 * above(e0), u1 = c1 * above(e1);
        const int64_t l0 = c0 * below(e1), l1 = b + 2 < kBins ? c1 * below(e2) : 0;  // the last bin has no far edge
        const int64_t ue = block_inclusive(u0 + u1, sh.part), le = block_inclusive(l0 + l1, sh.part);
        const int64_t ce = block_inclusive(c0 + c1, sh.part);
        if (ue >= limit && ue - u0 - u1 < limit) sh.first_bin = ue - u1 >= limit ? b : b + 1;
        if (le >= limit && le - l0 - l1 < limit) {
            const bool one = le - l1 >= limit;
            sh.last_bin = one ? b : b + 1;
            sh.near = static_cast<int>(one ? ce - c1 : ce);
        }
        __syncthreads();
    }

    // The cut at mass `limit` (less than all) from the counts of weigh_regions<true>: only the weights in front of the
    // window are summed, and only those inside it go into a histogram, of as many bins over the window.  False where
    // that leaves too many alike.
    __device__ bool window_cut(int64_t limit) {
        const int b0 = sh.first_bin, b1 = sh.last_bin;
        const float fine = static_cast<float>(kBins) / (b1 - b0 + 1);
        clear_bins();
        // -1: in front of the window or not in it; the candidate's weight where it is in or before it
        const auto place = [&](float v, int i, int64_t* w) -> int {
            const float d = any_distance(v);
            const int b = bin_at(d);
            if (b > b1) {
                *w = 0;
                return -1;
            }
            *w = weigh(v, i, d);
            return b < b0 ? -1 : min(kBins - 1, static_cast<int>((-d * kBinsPerUnit - b0) * fine));
        };
        int64_t front = 0;
        each([&](float v, int i) {
            int64_t w;
            const int b = place(v, i, &w);
            if (b < 0) front += w;
            else if (w > 0) count_in<true>(b, w);
        });
        front = block_reduce<int64_t>(front, [](int64_t p, int64_t q) { return p + q; }, sh.part);
        if (threadIdx.x == 0) sh.board.above = front;
        sync();
        front = 0;
#pragma unroll
        for (int r = 0; r < CL; ++r) front += of(&sh.board, r)->above;
        find_bin<true>(front, limit);
        const int bin = sh.bin;
        const int64_t before = sh.before;
        if (bin < 0) return false;
        const int total = list(false, [&](float v, int i, int64_t* w) { return place(v, i, w) == bin && *w > 0; });
        if (total > kList) return false;
        rank_list<true>(before, limit, total);
        return true;
    }

    // Finds the element at which the measure of the candidates, in falling order, reaches `target` (>= 1, at most the
    // whole): the count (MASS false: every element within reach is a candidate) or the mass (those of at least `least`).
    template <bool MASS>
    __device__ void find_cut(int64_t target, int64_t least) {
        uint64_t lo = 0, hi = ~0ull;  // range of composites that holds the element
        int shift = -1;               // bins: of the distance (-1), else of the composite's distance from hi
        int64_t before = 0;
        for (;;) {
            clear_bins();
            // the bin of an element in range, -1 if it is not; its distance in *d
            const auto place = [&](float v, int i, float* d) -> int {
                const uint64_t c = composite(v, first + i);
                if (c < lo || c > hi) return -1;
                *d = any_distance(v);
                return shift < 0 ? bin_at(*d) : static_cast<int>((hi - c) >> shift);
            };
            each([&](float v, int i) {
                float d;
                const int b = place(v, i, &d);
                if (b < 0) return;
                const int64_t w = MASS ? weigh(v, i, d) : 1;
                if (!MASS || (w >= least && w > 0)) count_in<MASS>(b, w);
            });
            find_bin<MASS>(before, target);
            const int bin = sh.bin;
            if (bin < 0) return;  // not reached: the callers ask for less than there is
            before = sh.before;
            const auto inside = [&](float v, int i, int64_t* w) {
                float d;
                if (place(v, i, &d) != bin) return false;
                *w = MASS ? weigh(v, i, d) : 0;
                return !MASS || (*w >= least && *w > 0);
            };
            const int total = list(false, inside);
            if (total <= kList) {
                rank_list<MASS>(before, target, total);
                return;
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

    // -- read the slice once: 16 bytes at a time between its ragged ends, to the same offset from a 16-byte boundary --
    constexpr int V = 16 / sizeof(T), U = 4;
    const int skew = static_cast<int>(reinterpret_cast<uintptr_t>(from) & 15);
    x = reinterpret_cast<T*>(reinterpret_cast<char*>(x) + skew);
    const int head = min(n, ((16 - skew) & 15) / static_cast<int>(sizeof(T))), packs = (n - head) / V;
    float top = -INFINITY;  // fmaxf passes over NaN
    for (int p0 = threadIdx.x; p0 < packs; p0 += kThreads * U) {
        uint4 w[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (p0 + u * kThreads < packs) w[u] = __ldcs(reinterpret_cast<const uint4*>(from + head) + p0 + u * kThreads);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (p0 + u * kThreads >= packs) continue;
            reinterpret_cast<uint4*>(x + head)[p0 + u * kThreads] = w[u];
            const T* v = reinterpret_cast<const T*>(&w[u]);
#pragma unroll
            for (int k = 0; k < V; ++k) top = fmaxf(top, as_float(v[k]));
        }
    }
    const int ends = n - packs * V;  // the head, then what the packs leave
    for (int j = threadIdx.x; j < ends; j += kThreads) {
        const int i = j < head ? j : j + packs * V;
        x[i] = from[i];
        top = fmaxf(top, as_float(x[i]));
    }
    const float own_top = top;  // of this thread's elements
    const auto larger = [](float p, float q) { return fmaxf(p, q); };
    top = block_reduce(top, larger, reinterpret_cast<float*>(sh.part));
    Row<T, CL, CUTS> row{x, sh, cuts, first, n};
    if (threadIdx.x == 0) sh.board.top = top;
    row.sync();
#pragma unroll
    for (int c = 0; c < CL; ++c) top = fmaxf(top, row.of(&sh.board, c)->top);
    row.top = top;
    const float temperature = a.temperature ? a.temperature[r] : 1.f;
    const bool none = top == -INFINITY, greedy = !(temperature > 0.f);
    if (none || greedy) {
        int at = INT32_MAX;  // the first of the largest
        for (int i = threadIdx.x; i < n && !none; i += kThreads)
            if (as_float(x[i]) == top) {
                at = first + i;
                break;
            }
        at = block_reduce(at, [](int p, int q) { return min(p, q); }, reinterpret_cast<int*>(sh.part));
        if (threadIdx.x == 0) sh.board.index = at;
        row.sync();
        if (rank == 0 && threadIdx.x == 0) {
            for (int c = 0; c < CL; ++c) at = min(at, row.of(&sh.board, c)->index);
            a.token[r] = none ? -1 : at;
            if (a.logprob) a.logprob[r] = none ? -INFINITY : 0.f;
        }
        row.sync();  // no CTA leaves while another may read its board
        return;
    }
    row.t = temperature;
    row.inv = temperature > 9.094947e-13f && temperature < 1.0995e12f ? __frcp_rn(temperature) : 0.f;
    row.min_p = a.min_p ? fminf(a.min_p[r], 1.f) : 0.f;
    // NaN, where both are infinite, takes everything
    row.low = row.top - (kReach + 0.5f) * temperature;
    int64_t mass;
    int count;
    if constexpr (CUTS) {
        const int k = a.top_k ? a.top_k[r] : 0;
        const float top_p = a.top_p ? a.top_p[r] : 1.f;
        const auto weighed = [&](float v, int i, int64_t* w) {
            *w = row.weigh(v, i);
            return true;
        };
        if (k > 0) {
            row.raise_low(k, own_top);
            const int total = row.list(true, weighed);
            if (total <= kList) {
                row.finish_list(a, r, rank, total, k, top_p, 0);
                return;
            }
            // fewer within reach than k: no cut
            int near = 0;
            row.each([&](float, int) { ++near; });
            near = block_reduce(near, [](int p, int q) { return p + q; }, reinterpret_cast<int*>(sh.part));
            if (threadIdx.x == 0) sh.board.count[2] = near;
            row.sync();
            near = 0;
#pragma unroll
            for (int c = 0; c < CL; ++c) near += row.of(&sh.board, c)->count[2];
            if (k < near) {
                row.template find_cut<false>(k, 0);
                row.low = fmaxf(row.low, value_of(static_cast<uint32_t>(row.cut >> 32)));
            }
        }
        bool counted = false;
        if (top_p < 1.f && !row.raised) {
            row.clear_bins();
            counted = row.template weigh_regions<true>(0, &mass, &count);
        } else {
            row.template weigh_regions<false>(0, &mass, &count);
        }
        const int64_t limit = row.limit_of(top_p, mass);
        if (top_p < 1.f && limit < mass) {
            bool found = false;
            if (counted) {
                row.window(limit);
                if (sh.near <= kList && sh.last_bin < kBins - 1) {
                    row.drop_behind(sh.last_bin);
                    const int total = row.list(true, weighed);
                    if (total <= kList) {
                        row.finish_list(a, r, rank, total, 0, top_p, limit);
                        return;
                    }
                }
                found = row.window_cut(limit);
            }
            if (!found) {
                // weights below (1 - p) mass / (2 count) are together less than what stays out
                const double least = 0.5 * (1.0 - static_cast<double>(top_p)) * static_cast<double>(mass) / count;
                row.template find_cut<true>(limit, static_cast<int64_t>(fmax(least, 0.0)));
            }
            row.low = fmaxf(row.low, value_of(static_cast<uint32_t>(row.cut >> 32)));
            row.template weigh_regions<false>(1, &mass, &count);
        }
    } else {
        row.template weigh_regions<false>(0, &mass, &count);
    }

    // -- the pick: the CTA, then the warp's region, then the element --
    const int64_t pick = row.pick_of(a.u[r], mass);
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
    const int smem = slice * static_cast<int>(sizeof(T)) + 16 + (CUTS ? static_cast<int>(sizeof(SharedCut)) : 0);
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
    const auto bytes_of = [&](int cl) { return slice_of(cl) * static_cast<int64_t>(sizeof(T)) + 16 + extra; };
    const auto per_sm = [&](int cl) { return std::min<int64_t>(CUTS ? 2 : 3, (227 << 10) / (bytes_of(cl) + 2048)); };
    // Slices of 8000 elements or more: below that the cluster's barriers and remote reads cost what the passes save, or more.
    // One row with top-p in 1, 2, 4 and 8 CTAs, device us: of 8000 10.5, 10.8, 10.8, 12.8; of 16000 13.4, 12.3, 11.4, 13.3
    // (taken: two); of 32000 20.4, 16.4, 13.7, 14.8; of 50000 28.4, 21.3, 16.6, 16.9, and 70, 46, 32, 30 where its window has
    // to be summed; of 131072 24.8 in four and 21.4 in eight, 81 and 55 with the window.  Few rows are spread over the SMs, one CTA
    // each; many rows share them, so that one is read while another is worked on.
    int cl = 1;
    while (cl < kMaxCluster && (slice_of(cl) > 32768 || bytes_of(cl) > kSampleMaxSmem ||
                                (static_cast<int64_t>(a.rows) * cl * 2 <= sms && slice_of(cl * 2) >= 8000) ||
                                (static_cast<int64_t>(a.rows) * cl > sms && per_sm(cl) < 2 && slice_of(cl * 2) >= 8000)))
        cl *= 2;
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
