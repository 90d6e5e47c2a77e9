// tb_sample_rows.cu -- one token per logits row, by temperature, top-k, top-p
// and min-p from a given uniform number.
//
// With m the row's maximum and w_i = exp((x_i - m) / T):
//   order   descending x, equal values by ascending index;
//   top-k   the first k of that order;
//   top-p   the shortest prefix of those whose mass reaches p times theirs;
//   min-p   of those, the ones with w_i >= min_p (the largest weight is 1);
//   token   the first kept index, in index order, whose running mass passes
//           u times the kept mass.
// T = 0 takes the maximum (its first index).  NaN counts as -inf, and a row of
// -inf alone yields token -1.
//
// A whole-number result has to come out the same whatever the launch shape, so
// nothing here depends on the order in which threads arrive: the weights are
// fp64 exponentials; the masses that place the top-p boundary are 64-bit
// fixed-point numbers (one is about 2^62 / V), whose integer sums are associative;
// the drawing sums are fp64 in a fixed order.
//
// A row is read once, by a cluster of P CTAs (P = 1, 2, 4, 8) that keep it in
// shared memory, each of their warps a run of consecutive elements.  A truncated
// row then takes one histogram of 1024 bins over (m - x) / T -- counts for top-k,
// masses for top-p -- and the elements of the one bin that holds the boundary,
// which every CTA ranks for itself (no sort: a select needs the boundary, not the
// order).  A bin of more elements than the list holds is narrowed by histograms
// over its keys.  Last come the kept masses and the search in the run that holds
// the draw.  Bound by the steps' latency for few rows, by the fp64 exponentials
// and the histogram's atomics for many.
#include "tb_common.cuh"
#include "tb_stream_entry.h"
#include "tb_unit.cuh"

namespace tb {
namespace {

constexpr int kRowThreads = 512;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kRowBins = 1024;
constexpr int kMaxCluster = 8;
constexpr int kList = 512;           // boundary elements that a CTA notes, and that are ranked
constexpr int kStagedMax = 44 * 1024;  // elements of a CTA that fit its shared memory
constexpr double kBinSpan = 40.0;    // nats below the maximum that the histogram resolves

struct RowsParams {
    const float* logits;
    long long ld;
    int V;
    double one;  // fixed-point masses: 1.0 as an integer, a power of two with V * one <= 2^62
    const float* temperature;
    const int* top_k;
    const float* top_p;
    const float* min_p;
    const float* uniform;
    int* token;
    float* prob;
    float* entropy;
};

typedef unsigned long long u64;

struct __align__(16) RowShared {
    u64 mass[kRowBins];             // as low, high words
    unsigned int count[kRowBins];
    u64 red[2][kMaxCluster * kRowWarps];  // a reduction's values from all CTAs, alternating
    u64 list[kList];                // the CTA's boundary elements: key, then the index's complement
    int listed[2];                  // how many, for top-k and for top-p
    u64 all[kList], weight[kList];  // all CTAs'
    int all_n;
    u64 scan[kRowWarps];
    u64 found[3];
    double mass_of[kMaxCluster * kRowWarps], moment_of[kMaxCluster * kRowWarps];  // by run
    int ties[kMaxCluster * kRowWarps];
    u64 tie_index[kMaxCluster];
};

__device__ __forceinline__ u64 dsmem_ld_u64(uint32_t addr) {
    u64 v;
    asm volatile("ld.shared::cluster.u64 %0, [%1];" : "=l"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ unsigned int dsmem_ld_u32(uint32_t addr) {
    unsigned int v;
    asm volatile("ld.shared::cluster.u32 %0, [%1];" : "=r"(v) : "r"(addr) : "memory");
    return v;
}
__device__ __forceinline__ void dsmem_st_u64(uint32_t addr, u64 v) {
    asm volatile("st.shared::cluster.u64 [%0], %1;" ::"r"(addr), "l"(v) : "memory");
}
__device__ __forceinline__ void dsmem_st_u32(uint32_t addr, unsigned int v) {
    asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(addr), "r"(v) : "memory");
}

// -0 becomes +0 (equal values are ties) and NaN -inf.
__device__ __forceinline__ float clean(float x) {
    x += 0.0f;
    return x == x ? x : -INFINITY;
}

constexpr __host__ __device__ int run_length(int V, int P) {
    const int runs = P * kRowWarps;
    return ((V + runs - 1) / runs + 31) & ~31;
}

template <int P, bool STAGED>
struct Row {
    static constexpr int kRuns = P * kRowWarps;
    const RowsParams& p;
    RowShared& sh;
    const float* x;   // the row
    float* kept;      // STAGED: the CTA's part of it
    int cta_begin, begin, end;  // the CTA's first element, the warp's run
    int lane, warp, rank;
    int turn = 0;     // which of the alternating buffers is next
    float top = 0.0f;
    double inv_t = 0.0;
    float bin_scale = 0.0f;
    // the last element of the kept prefix
    float cut = -INFINITY;
    int cut_index = -1;

    __device__ Row(const RowsParams& p_, RowShared& s, float* stage, int row) : p(p_), sh(s), kept(stage) {
        lane = threadIdx.x & 31;
        warp = threadIdx.x >> 5;
        rank = P == 1 ? 0 : (int)cluster_ctarank();
        x = p.logits + row * p.ld;
        const int len = run_length(p.V, P);
        cta_begin = min(rank * kRowWarps * len, p.V);
        begin = min((rank * kRowWarps + warp) * len, p.V);
        end = min(begin + len, p.V);
    }
    static __device__ __forceinline__ void sync() {
        if (P == 1)
            __syncthreads();
        else
            cluster_sync();
    }

    __device__ __forceinline__ float at(int i) const { return STAGED ? kept[i - cta_begin] : clean(x[i]); }
    __device__ __forceinline__ bool in_prefix(float v, int i) const { return v > cut || (v == cut && i <= cut_index); }
    // f(value, index) over the warp's run, in steps of 32 consecutive elements
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        int i = begin + lane;
        for (; i + 96 < end; i += 128) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = at(i + 32 * k);
#pragma unroll
            for (int k = 0; k < 4; ++k) f(v[k], i + 32 * k);
        }
        for (; i < end; i += 32) f(at(i), i);
    }
    // the first reading, which stages the row
    template <class F>
    __device__ __forceinline__ void read(F f) {
        int i = begin + lane;
        for (; i + 224 < end; i += 256) {
            float v[8];
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = clean(x[i + 32 * k]);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                if (STAGED) kept[i + 32 * k - cta_begin] = v[k];
                f(v[k], i + 32 * k);
            }
        }
        for (; i < end; i += 32) {
            const float v = clean(x[i]);
            if (STAGED) kept[i - cta_begin] = v;
            f(v, i);
        }
    }

    __device__ __forceinline__ double exponent(float v) const {
        return v == top ? 0.0 : ((double)v - (double)top) * inv_t;
    }
    __device__ __forceinline__ double weight(float v) const { return v == top ? 1.0 : exp(exponent(v)); }
    __device__ __forceinline__ u64 fixed(float v) const {
        const double w = weight(v);  // NaN where an infinite maximum meets an infinite T: no mass
        return w > 0.0 ? (u64)__double2ll_rn(w * p.one) : 0ull;
    }
    // Monotone in the value: 0 for the maximum, the last bin for all that lies
    // kBinSpan nats or more below it.
    __device__ __forceinline__ int bin_of(float v) const {
        if (v == top) return 0;
        return (int)fminf((top - v) * bin_scale, (float)(kRowBins - 1));
    }

    // Reduction over the cluster by an associative, commutative f with f(v, v) = v:
    // every thread gets the result.
    template <class F>
    __device__ u64 reduce(u64 v, F f) {
        for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
        u64* r = sh.red[turn];
        if (lane < P) dsmem_st_u64(dsmem_map(r + rank * kRowWarps + warp, lane), v);
        sync();
#pragma unroll
        for (int i = 0; i < kRuns; i += 32) v = f(v, r[i + lane % (kRuns < 32 ? kRuns : 32)]);
        for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
        turn ^= 1;
        return v;
    }

    __device__ __forceinline__ void add_mass(int bin, u64 w) {
        unsigned int* m = reinterpret_cast<unsigned int*>(sh.mass + bin);
        const unsigned int lo = (unsigned int)w;
        unsigned int hi = (unsigned int)(w >> 32);
        if (lo && atomicAdd(m, lo) + lo < lo) ++hi;  // carry
        if (hi) atomicAdd(m + 1, hi);
    }
    // After sync(): bins 2 t and 2 t + 1 of all CTAs (BY_MASS: masses, else counts)
    // and what stands before them in the order of the bins; the result is the sum.
    template <bool BY_MASS>
    __device__ u64 bins(u64 (&b)[2], u64& before) {
        u64 part[P][2];
#pragma unroll
        for (int r = 0; r < P; ++r) {
            if (BY_MASS) {
                asm volatile("ld.shared::cluster.v2.u64 {%0, %1}, [%2];"
                             : "=l"(part[r][0]), "=l"(part[r][1])
                             : "r"(dsmem_map(sh.mass + 2 * threadIdx.x, r)));
            } else {
                unsigned int c0, c1;
                asm volatile("ld.shared::cluster.v2.u32 {%0, %1}, [%2];"
                             : "=r"(c0), "=r"(c1)
                             : "r"(dsmem_map(sh.count + 2 * threadIdx.x, r)));
                part[r][0] = c0;
                part[r][1] = c1;
            }
        }
        b[0] = b[1] = 0;
#pragma unroll
        for (int r = 0; r < P; ++r) {
            b[0] += part[r][0];
            b[1] += part[r][1];
        }
        u64 incl = b[0] + b[1];
        for (int o = 1; o < 32; o <<= 1) {
            const u64 t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        if (lane == 31) sh.scan[warp] = incl;
        if (threadIdx.x == 0) sh.found[0] = ~0ull;
        __syncthreads();
        before = incl - b[0] - b[1];
        const u64 warps = lane < kRowWarps ? sh.scan[lane] : 0;
        u64 sum = warps, lower = lane < warp ? warps : 0;
        for (int o = kRowWarps / 2; o; o >>= 1) {
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
            lower += __shfl_xor_sync(0xffffffffu, lower, o);
        }
        before += __shfl_sync(0xffffffffu, lower, 0);
        return __shfl_sync(0xffffffffu, sum, 0);
    }
    // After bins(): the bin where the running weight, from `base` on, reaches target
    // (-1: it does not), and the weight before it.
    __device__ __forceinline__ int bin_at(const u64 (&b)[2], u64 before, u64 base, u64 target, u64* above) {
        before += base;
#pragma unroll
        for (int k = 0; k < 2; ++k) {
            if (before < target && before + b[k] >= target) {
                sh.found[0] = 2 * threadIdx.x + k;
                sh.found[1] = before;
            }
            before += b[k];
        }
        __syncthreads();
        *above = sh.found[1];
        return (int)sh.found[0];
    }

    // The prefix's elements in a bin, from all CTAs, as sh.all; false: more than the
    // list holds.
    __device__ bool gather(int bin, int which) {
        each([&](float v, int i) {
            if (bin_of(v) == bin && in_prefix(v, i)) {
                const int n = atomicAdd(&sh.listed[which], 1);
                if (n < kList) sh.list[n] = ((u64)float_order_key(v) << 32) | (uint32_t)~i;
            }
        });
        sync();
        int here = lane < P ? (int)dsmem_ld_u32(dsmem_map(&sh.listed[which], lane)) : 0, incl = here;
        for (int o = 1; o < P; o <<= 1) {
            const int t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        const int n = __shfl_sync(0xffffffffu, incl, P - 1);
        if (n <= kList) {
            const int r = warp % P, count = __shfl_sync(0xffffffffu, here, r);
            const int first = __shfl_sync(0xffffffffu, incl, r) - count;
            for (int i = warp / P * 32 + lane; i < count; i += kRowThreads / P)
                sh.all[first + i] = dsmem_ld_u64(dsmem_map(sh.list + i, r));
        }
        if (threadIdx.x == 0) sh.all_n = n;
        __syncthreads();
        return n <= kList;
    }
    // The list's element where its running weight, in descending order, reaches
    // `target`, becomes the prefix's last; BY_MASS: of their masses, else counts.
    // The weights of what stands above an element are added by 1 to 32 lanes.
    template <bool BY_MASS>
    __device__ void cut_in_list(u64 target) {
        const int n = sh.all_n;
        if (BY_MASS) {
            for (int i = threadIdx.x; i < n; i += kRowThreads)
                sh.weight[i] = fixed(float_from_order_key((uint32_t)(sh.all[i] >> 32)));
            __syncthreads();
        }
        int lanes = 32;
        while (lanes > 1 && n * lanes > kRowThreads) lanes >>= 1;
        const int i = threadIdx.x / lanes;  // n <= kList = kRowThreads
        const u64 e = i < n ? sh.all[i] : ~0ull;
        u64 upto = 0;
        for (int j = threadIdx.x % lanes; j < n; j += lanes)
            upto += sh.all[j] >= e ? (BY_MASS ? sh.weight[j] : 1ull) : 0ull;
        for (int o = 1; o < lanes; o <<= 1) upto += __shfl_xor_sync(0xffffffffu, upto, o);
        if (i < n && threadIdx.x % lanes == 0) {
            const u64 own = BY_MASS ? sh.weight[i] : 1ull;
            if (upto - own < target && upto >= target) sh.found[2] = e;
        }
        __syncthreads();
        cut = float_from_order_key((uint32_t)(sh.found[2] >> 32));
        cut_index = (int)~(uint32_t)sh.found[2];
    }

    // The same for a bin with more elements than the list: its keys, 1024 bins at a
    // time, until one key is left, and among its elements by index.  `above`: the
    // weight before the bin.
    template <bool BY_MASS>
    __device__ void cut_in_bin(int bin, u64 target, u64 above) {
        uint32_t lo_key = 0xffffffffu, hi_key = 0;
        each([&](float v, int i) {
            const uint32_t k = float_order_key(v);
            if (bin_of(v) == bin && in_prefix(v, i)) {
                lo_key = min(lo_key, k);
                hi_key = max(hi_key, k);
            }
        });
        // both ends in one reduction: the high key, and the low key's complement
        const u64 ends = reduce(((u64)hi_key << 32) | (uint32_t)~lo_key, [](u64 a, u64 b) {
            const uint32_t low = max((uint32_t)a, (uint32_t)b);
            return ((a > b ? a : b) & 0xffffffff00000000ull) | low;
        });
        hi_key = (uint32_t)(ends >> 32);
        lo_key = ~(uint32_t)ends;
        u64 b[2], before;
        while (lo_key < hi_key) {
            int shift = 0;
            while (((hi_key - lo_key) >> shift) >= (uint32_t)kRowBins) ++shift;
            sync();  // the bins have been read
            for (int i = threadIdx.x; i < kRowBins; i += kRowThreads) {
                if (BY_MASS)
                    sh.mass[i] = 0;
                else
                    sh.count[i] = 0;
            }
            __syncthreads();
            each([&](float v, int i) {
                const uint32_t k = float_order_key(v);
                if (k < lo_key || k > hi_key || !in_prefix(v, i)) return;
                const int to = (int)((hi_key - k) >> shift);
                if (BY_MASS)
                    add_mass(to, fixed(v));
                else
                    atomicAdd(&sh.count[to], 1u);
            });
            sync();
            bins<BY_MASS>(b, before);
            const int found = bin_at(b, before, above, target, &above);
            if (found < 0) break;  // cannot be: the bin's weight reaches the target, and sums are exact
            hi_key -= (uint32_t)found << shift;
            const uint32_t width = (1u << shift) - 1u;
            if (hi_key - lo_key > width) lo_key = hi_key - width;
        }
        // how many of the equal elements, and the last one's index
        const float value = float_from_order_key(hi_key);
        const u64 w = BY_MASS ? fixed(value) : 1ull;
        const u64 need = w ? (target - above + w - 1) / w : 1ull;
        int mine = 0;
        each([&](float v, int i) { mine += v == value && in_prefix(v, i); });
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (lane < P) dsmem_st_u32(dsmem_map(sh.ties + rank * kRowWarps + warp, lane), (unsigned int)mine);
        if (threadIdx.x < P) sh.tie_index[threadIdx.x] = 0;
        sync();
        const int me = rank * kRowWarps + warp;
        u64 rank_of = 0;
        for (int i = lane; i < me; i += 32) rank_of += sh.ties[i];
        for (int o = 16; o; o >>= 1) rank_of += __shfl_xor_sync(0xffffffffu, rank_of, o);
        if (rank_of < need && rank_of + mine >= need) {
            for (int i0 = begin; i0 < end; i0 += 32) {
                const int i = i0 + lane;
                const float v = i < end ? at(i) : -INFINITY;
                const bool same = i < end && v == value && in_prefix(v, i);
                const unsigned who = __ballot_sync(0xffffffffu, same);
                if (same && rank_of + __popc(who & ((2u << lane) - 1u)) == need)
                    for (int r = 0; r < P; ++r) dsmem_st_u64(dsmem_map(sh.tie_index + rank, r), (u64)i + 1);
                rank_of += __popc(who);
            }
        }
        sync();
        u64 index = 0;
#pragma unroll
        for (int r = 0; r < P; ++r) index += sh.tie_index[r];
        cut = value;
        cut_index = (int)index - 1;
    }
};

template <int P, bool STAGED>
__global__ void __launch_bounds__(kRowThreads) sample_rows_kernel(RowsParams p) {
    extern __shared__ float stage[];
    __shared__ RowShared sh;
    const int row = blockIdx.x / P;
    Row<P, STAGED> r(p, sh, stage, row);
    const bool writer = r.rank == 0 && threadIdx.x == 0;

    // 1. the row, its maximum and that one's first index
    for (int i = threadIdx.x; i < kRowBins; i += kRowThreads) {
        sh.mass[i] = 0;
        sh.count[i] = 0;
    }
    if (threadIdx.x < 2) sh.listed[threadIdx.x] = 0;
    if (P > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const float T = p.temperature ? p.temperature[row] : 1.0f;
    const int k = p.top_k ? p.top_k[row] : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.0f;
    const double floor_w = p.min_p ? (double)fminf(fmaxf(p.min_p[row], 0.0f), 1.0f) : 0.0;
    const double u = fminf(fmaxf(p.uniform[row], 0.0f), 0.99999994f);
    float best = -INFINITY;
    int best_i = 0;
    r.read([&](float v, int i) {
        if (v > best) {
            best = v;
            best_i = i;
        }
    });
    // the others have started: their shared memory may be written
    if (P > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const u64 key =
        r.reduce(best > -INFINITY ? argmax_key(best, best_i) : 0ull, [](u64 a, u64 b) { return a > b ? a : b; });
    if (key == 0 || !(T > 0.0f) || k == 1) {
        if (writer) {
            p.token[row] = key ? (int)(0xffffffffu - (uint32_t)key) : -1;
            if (p.prob) p.prob[row] = key ? 1.0f : 0.0f;
            if (p.entropy) p.entropy[row] = 0.0f;
        }
        return;  // (the others' writes came before the barrier)
    }
    r.top = float_from_order_key((uint32_t)(key >> 32));
    r.inv_t = 1.0 / (double)T;
    r.bin_scale = (float)((double)kRowBins / kBinSpan * r.inv_t);

    // 2. the kept prefix's last element: top-k's, and top-p's within it
    u64 b[2], before, above;
    if (k > 0 && k < p.V) {
        r.each([&](float v, int) {
            if (v > -INFINITY) atomicAdd(&sh.count[r.bin_of(v)], 1u);
        });
        r.sync();
        if (r.template bins<false>(b, before) > (u64)k) {  // else all there is
            const int bin = r.bin_at(b, before, 0, (u64)k, &above);
            if (r.gather(bin, 0))
                r.template cut_in_list<false>((u64)k - above);
            else
                r.template cut_in_bin<false>(bin, (u64)k, above);
        }
    }
    if (!(top_p >= 1.0f)) {
        r.each([&](float v, int i) {
            if (r.in_prefix(v, i)) r.add_mass(r.bin_of(v), r.fixed(v));
        });
        r.sync();
        const u64 mass = r.template bins<true>(b, before);
        const double want = ceil((double)top_p * (double)mass);
        const u64 target = want > 1.0 ? min((u64)want, mass) : 1ull;
        const int bin = r.bin_at(b, before, 0, target, &above);
        if (r.gather(bin, 1))
            r.template cut_in_list<true>(target - above);
        else
            r.template cut_in_bin<true>(bin, target, above);
    }

    // 3. the kept mass, run by run
    const auto weight_of = [&](float v, int i) -> double {
        if (!r.in_prefix(v, i)) return 0.0;
        const double w = r.weight(v);
        return w >= floor_w ? w : 0.0;
    };
    double mass = 0.0, moment = 0.0;
    r.each([&](float v, int i) {
        const double w = weight_of(v, i);
        if (w > 0.0) {
            mass += w;
            moment += w * r.exponent(v);
        }
    });
    for (int o = 16; o; o >>= 1) {
        mass += __shfl_xor_sync(0xffffffffu, mass, o);
        moment += __shfl_xor_sync(0xffffffffu, moment, o);
    }
    const int me = r.rank * kRowWarps + r.warp;
    if (r.lane < P) {
        dsmem_st_u64(dsmem_map(sh.mass_of + me, r.lane), (u64)__double_as_longlong(mass));
        dsmem_st_u64(dsmem_map(sh.moment_of + me, r.lane), (u64)__double_as_longlong(moment));
    }
    r.sync();  // the last: nothing of another CTA is touched from here on

    // 4. the run that holds the draw, found by every warp alike (4 runs a lane)
    double part[4], sum4 = 0.0, mom = 0.0;
    for (int j = 0; j < 4; ++j) {
        const int i = r.lane * 4 + j;
        part[j] = i < r.kRuns ? sh.mass_of[i] : 0.0;
        sum4 += part[j];
        mom += i < r.kRuns ? sh.moment_of[i] : 0.0;
    }
    double incl = sum4;
    for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, incl, o);
        if (r.lane >= o) incl += t;
    }
    for (int o = 16; o; o >>= 1) mom += __shfl_xor_sync(0xffffffffu, mom, o);
    const double all = __shfl_sync(0xffffffffu, incl, 31);
    const double goal = u * all;
    double upto_lane = __shfl_up_sync(0xffffffffu, incl, 1);
    if (r.lane == 0) upto_lane = 0.0;
    int run = -1;
    double run_before = 0.0;
    for (int j = 0; j < 4; ++j) {
        const double next = j == 3 ? incl : upto_lane + part[j];
        if (run < 0 && part[j] > 0.0 && next > goal) {
            run = r.lane * 4 + j;
            run_before = upto_lane;
        }
        upto_lane = next;
    }
    const unsigned who = __ballot_sync(0xffffffffu, run >= 0);
    const int src = who ? __ffs(who) - 1 : 0;
    run = __shfl_sync(0xffffffffu, run, src);
    run_before = __shfl_sync(0xffffffffu, run_before, src);
    if (run != me) return;
    // 5. the element: 256 at a time by their sum, then 32 at a time by a scan
    const auto weight_at = [&](int i) { return i < r.end ? weight_of(r.at(i), i) : 0.0; };
    int last = -1;
    double last_w = 0.0, running = run_before;
    bool done = false;
    for (int i0 = r.begin; i0 < r.end && !done; i0 += 256) {
        double s = 0.0;
#pragma unroll
        for (int j = 0; j < 256; j += 32) s += weight_at(i0 + j + r.lane);
        for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
        if (s == 0.0) continue;
        // what ends just short of the goal is searched too: a sum in another order
        // may end a rounding lower, and the run's last element is then the one
        if (running + s >= goal * (1.0 - 1e-12)) {
            double upto = running;
            for (int j = 0; j < 256 && i0 + j < r.end && !done; j += 32) {
                const double w = weight_at(i0 + j + r.lane);
                double c = w;
                for (int o = 1; o < 32; o <<= 1) {
                    const double t = __shfl_up_sync(0xffffffffu, c, o);
                    if (r.lane >= o) c += t;
                }
                const unsigned hit = __ballot_sync(0xffffffffu, w > 0.0 && upto + c > goal);
                const unsigned any = __ballot_sync(0xffffffffu, w > 0.0);
                const int pick = hit ? __ffs(hit) - 1 : any ? 31 - __clz(any) : -1;
                if (pick >= 0) {
                    last = i0 + j + pick;
                    last_w = __shfl_sync(0xffffffffu, w, pick);
                }
                done = hit != 0;
                upto += __shfl_sync(0xffffffffu, c, 31);
            }
        }
        running += s;
    }
    if (r.lane == 0) {
        p.token[row] = last;
        if (p.prob) p.prob[row] = (float)(last_w / all);
        if (p.entropy) p.entropy[row] = (float)fmax(log(all) - mom / all, 0.0);
    }
}

template <int P, bool STAGED>
cudaError_t launch_rows(const RowsParams& p, int rows, cudaStream_t stream) {
    const size_t smem = STAGED ? (size_t)run_length(p.V, P) * kRowWarps * sizeof(float) : 0;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * P));
    cfg.blockDim = dim3(kRowThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)P;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaSuccess;
    if (smem + sizeof(RowShared) > 48 * 1024)  // what needs no asking
        e = cudaFuncSetAttribute(sample_rows_kernel<P, STAGED>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kStagedMax * (int)sizeof(float));
    if (e == cudaSuccess) e = cudaLaunchKernelEx(&cfg, sample_rows_kernel<P, STAGED>, p);
    return e;
}

}  // namespace
}  // namespace tb

using namespace tb;

extern "C" tb_status tb_sample_rows_dev(void* stream, const float* logits, int64_t ld, int32_t rows, int32_t V,
                                        const float* temperature, const int32_t* top_k, const float* top_p,
                                        const float* min_p, const float* uniform, int32_t* token, float* prob,
                                        float* entropy) {
    TB_ENTRY_CHECK(logits && uniform && token, "NULL argument");
    TB_ENTRY_CHECK(rows >= 0 && V >= 1 && V <= (1 << 24) && ld >= V && rows <= INT32_MAX / kMaxCluster,
                   "bad rows / vocabulary / row stride");
    if (rows == 0) return TB_OK;
    StreamEntry entry(logits, "logits");
    if (entry.status != TB_OK) return entry.status;
    int log_v = 0;
    while ((1ll << log_v) < V) ++log_v;
    const RowsParams p{logits, ld, V, std::ldexp(1.0, 62 - log_v), temperature, top_k, top_p, min_p, uniform, token,
                       prob, entropy};
    // CTAs of a row: while the rows leave SMs idle and a CTA would still have 2048
    // elements to read, or while a CTA's part leaves no room for others on its SM
    int P = 1;
    while (P < kMaxCluster &&
           (((long long)rows * P < 2ll * entry.num_sms && V / (2 * P) >= 2048) || V / P > 16 * 1024))
        P *= 2;
    const cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e;
    if (P == 1)
        e = launch_rows<1, true>(p, rows, s);
    else if (P == 2)
        e = launch_rows<2, true>(p, rows, s);
    else if (P == 4)
        e = launch_rows<4, true>(p, rows, s);
    else if (run_length(V, P) * kRowWarps <= kStagedMax)
        e = launch_rows<8, true>(p, rows, s);
    else  // the passes read the row from L2
        e = launch_rows<8, false>(p, rows, s);
    return launch_status(e, "sampling launch");
}
