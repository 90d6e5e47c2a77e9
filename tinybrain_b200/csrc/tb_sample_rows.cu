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
// -inf alone yields token -1.  Weights below e^-700 count as 0.
//
// A whole-number result has to come out the same whatever the launch shape, so
// nothing here depends on the order in which threads arrive: the weights are
// fp64 exponentials; the masses that place the top-p boundary are 64-bit
// fixed-point numbers (one is about 2^62 / V), whose integer sums are associative;
// the drawing sums are fp64 in a fixed order.
//
// A row is read once, by a cluster of P CTAs (P = 1, 2, 4, 8) that keep it in
// shared memory, each of their warps a run of consecutive elements.  A truncated
// row then takes one histogram of 2048 bins over (m - x) / T -- counts for top-k,
// then masses of what that leaves for top-p -- and the elements of the one bin
// that holds the boundary, which are ranked (no sort: a select needs the boundary,
// not the order).  A bin of more elements than the list holds is narrowed by
// histograms over its keys.  Last come the kept masses, run by run, and the search
// in the run that holds the draw.  What the CTAs tell one another they push into
// each other's shared memory ahead of a barrier, after which it is read locally.
//
// Bound by the barriers' and reads' latency for few rows, by instruction issue for
// many.  Measured: one row of 32000 12 us, 64 rows 24 us; 256 rows of 131072, each
// with its own settings, 161 us (0.8 TB/s); greedy alone 43 us, without truncation
// 114, top-k 40 153, top-p 0.9 219 (at temperature 0.8).
#include <cfloat>
#include <climits>

#include "tb_common.cuh"
#include "tb_sample_cut.h"
#include "tb_stream_entry.h"
#include "tb_unit.cuh"

namespace tb {
namespace {

constexpr int kRowThreads = 512;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kRowBins = 2048;
constexpr int kBinsEach = kRowBins / kRowThreads;
constexpr int kBinGroups = kRowBins / 32;
constexpr int kMaxCluster = 8;
constexpr int kList = 512;           // boundary elements that a CTA notes, and that are ranked
constexpr int kStagedMax = 44 * 1024;  // elements of a CTA that fit its shared memory
constexpr float kBinSpan = 24.0f;      // nats below the maximum that the histogram resolves
constexpr int kRoots = 64;
constexpr int kBatch = 16;             // loads of a lane in flight while the row is read

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
    union {
        unsigned int count[kRowBins];
        struct {
            u64 all[kList], weight[kList];  // the listed elements of all CTAs, once the counts have been read
        };
    };
    u64 red[2][kMaxCluster * kRowWarps];  // a reduction's values from all CTAs, alternating
    u64 list[kList];                // the CTA's boundary elements: key, then the index's complement
    int listed[2];                  // how many, for top-k and for top-p
    int all_n;
    u64 groups[2][kMaxCluster][kBinGroups];  // sums of 32 bins from all CTAs, alternating
    u64 found[3];
    double root[kRoots];            // 2^(j / kRoots)
    double mass_of[kMaxCluster * kRowWarps], moment_of[kMaxCluster * kRowWarps];  // by run
    int ties[kMaxCluster * kRowWarps];
    double chunk[kRowWarps], pick_weight;
    int pick;
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
__device__ __forceinline__ float clean(float x) { return fmaxf(x + 0.0f, -INFINITY); }

constexpr __host__ __device__ int run_length(int V, int P) {
    const int runs = P * kRowWarps;
    return ((V + runs - 1) / runs + 127) & ~127;
}

template <int P, bool STAGED>
struct Row {
    static constexpr int kRuns = P * kRowWarps;
    const RowsParams& p;
    RowShared& sh;
    const float* x;   // the row
    float* kept;      // STAGED: the warp's run of it, -inf behind the row's end
    int base, n;      // the run's first element, and its elements
    int lane, warp, rank;
    int turn = 0, group_turn = 0;  // which of the alternating buffers is next
    u64 group[2], before_group;    // the lane's groups of bins, and what stands before them
    float top = 0.0f;
    double inv_t = 0.0;
    float bin_scale = 0.0f;
    double floor_w = 0.0;  // min-p's
    // the last element of the kept prefix
    float cut = -INFINITY;
    int cut_index = -1;

    __device__ Row(const RowsParams& p_, RowShared& s, float* stage, int row) : p(p_), sh(s) {
        lane = threadIdx.x & 31;
        warp = threadIdx.x >> 5;
        rank = P == 1 ? 0 : (int)cluster_ctarank();
        x = p.logits + row * p.ld;
        const int len = run_length(p.V, P);
        base = (rank * kRowWarps + warp) * len;
        n = min(max(p.V - base, 0), len);
        kept = stage + warp * len;
    }
    // the run of the CTA's warp w, instead of its own
    __device__ void turn_to(int w) {
        const int len = run_length(p.V, P);
        base += (w - warp) * len;
        kept += (w - warp) * len;
        n = min(max(p.V - base, 0), len);
    }
    static __device__ __forceinline__ void sync() {
        if (P == 1)
            __syncthreads();
        else
            cluster_sync();
    }

    __device__ __forceinline__ bool in_prefix(float v, int i) const { return v > cut || (v == cut && i <= cut_index); }
    // the four elements that start at base + o; -inf behind the run's end
    __device__ __forceinline__ void load4(int o, float (&v)[4]) const {
        if (STAGED) {
            const float4 f = *reinterpret_cast<const float4*>(kept + o);
            v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = o + k < n ? clean(x[base + o + k]) : -INFINITY;
        }
    }
    // f(values, index of the first) over the warp's run, a lane four consecutive
    // elements at a time
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        for (int o = 4 * lane; o - 4 * lane < n; o += 128) {
            float v[4];
            load4(o, v);
            f(v, base + o);
        }
    }
    // The first reading, which stages the row: the lane's largest element, and where
    // asked for, the first index of that value.
    __device__ __forceinline__ float read(bool want_index, int& index) {
        float best = -INFINITY;
        index = 0;
        const float* run = x + base;
        int o = lane;
        float v[kBatch];
        for (; o - lane + 32 * kBatch <= n; o += 32 * kBatch) {
#pragma unroll
            for (int k = 0; k < kBatch; ++k) v[k] = clean(run[o + 32 * k]);
            float m = v[0];
#pragma unroll
            for (int k = 1; k < kBatch; ++k) m = fmaxf(m, v[k]);
            if (m > best) {
                best = m;
                if (want_index) {
#pragma unroll
                    for (int k = kBatch - 1; k >= 0; --k) index = v[k] == m ? base + o + 32 * k : index;
                }
            }
            if (STAGED) {
#pragma unroll
                for (int k = 0; k < kBatch; ++k) kept[o + 32 * k] = v[k];
            }
        }
        for (; o < ((n + 127) & ~127); o += 128) {
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = o + 32 * k < n ? clean(run[o + 32 * k]) : -INFINITY;
            const float m = fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3]));
            if (m > best) {
                best = m;
#pragma unroll
                for (int k = 3; k >= 0; --k) index = v[k] == m ? base + o + 32 * k : index;
            }
            if (STAGED) {
#pragma unroll
                for (int k = 0; k < 4; ++k) kept[o + 32 * k] = v[k];
            }
        }
        return best;
    }
    // exp(y) of y = (v - top) / T in [-700, 0] (lowest_weighted) as 2^q 2^(j / 64) e^r, |r| <= ln 2 / 128,
    // the root of two from a table and e^r by its series to r^5 / 5! (the next term is
    // below 2^-54): the table-driven method of P. T. P. Tang, ACM TOMS 15 (1989).  exp()
    // itself has a branch for its ends, across which four elements do not overlap.
    __device__ __forceinline__ double weight(float v, double& y) const {
        const double ln2 = 0.6931471805599453094, ln2_rest = 2.319046813846299558e-17;
        y = ((double)fminf(v, FLT_MAX) - (double)fminf(top, FLT_MAX)) * inv_t;
        const double shift = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to a whole number
        const double sum = fma(y, kRoots / ln2, shift), t = sum - shift;
        const int n = __double2loint(sum);
        const double r = fma(t, -ln2_rest / kRoots, fma(t, -ln2 / kRoots, y));
        double e = fma(r, 1.0 / 120.0, 1.0 / 24.0);
        e = fma(e, r, 1.0 / 6.0);
        e = fma(e, r, 0.5);
        e = fma(e, r, 1.0);
        const double root = sh.root[n & (kRoots - 1)];
        e = fma(root * r, e, root);
        return __hiloint2double(__double2hiint(e) + ((n >> 6) << 20), __double2loint(e));
    }
    __device__ __forceinline__ u64 fixed(float v) const {
        double y;
        return (u64)__double2ll_rn(weight(v, y) * p.one);
    }
    // The weights of four elements of the kept prefix, 0 for others and those that
    // min-p leaves out, and their exponents.
    __device__ __forceinline__ void weights(const float (&v)[4], int i, double (&w)[4], double (&y)[4]) const {
        bool in[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            in[k] = in_prefix(v[k], i + k);
            w[k] = y[k] = 0.0;
        }
        if (in[0] || in[1] || in[2] || in[3]) {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const double e = weight(in[k] ? v[k] : top, y[k]);
                w[k] = in[k] ? e : 0.0;
            }
            if (floor_w > 0.0) {
#pragma unroll
                for (int k = 0; k < 4; ++k) w[k] = w[k] >= floor_w ? w[k] : 0.0;
            }
        }
    }
    // Monotone in the value: 0 for the maximum, the last bin for all that lies
    // kBinSpan nats or more below it (and for 0 * infinity).  As a float, the bin's
    // number above 2^23, to which adding that rounds.
    __device__ __forceinline__ float float_bin(float v) const {
        float b = fminf((top - v) * bin_scale, (float)(kRowBins - 1));
        if (!STAGED) b = fmaxf(b, 0.0f);  // a row that changes while it is read must not leave the bins
        return b + 8388608.0f;
    }
    __device__ __forceinline__ int bin_of(float v) const { return __float_as_int(float_bin(v)) - 0x4b000000; }

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

    // Adds four elements' masses; a bin of -1: none.
    __device__ __forceinline__ void add_masses(const float (&v)[4], const int (&bin)[4]) {
        if (bin[0] < 0 && bin[1] < 0 && bin[2] < 0 && bin[3] < 0) return;
        unsigned int lo[4], hi[4], sum[4];
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const u64 w = fixed(v[k]);
            lo[k] = bin[k] >= 0 ? (unsigned int)w : 0u;
            hi[k] = bin[k] >= 0 ? (unsigned int)(w >> 32) : 0u;
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            sum[k] = 0;
            if (lo[k]) sum[k] = atomicAdd(reinterpret_cast<unsigned int*>(sh.mass + bin[k]), lo[k]) + lo[k];
        }
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            if (sum[k] < lo[k]) ++hi[k];  // carry
            if (hi[k]) atomicAdd(reinterpret_cast<unsigned int*>(sh.mass + bin[k]) + 1, hi[k]);
        }
    }
    // Adds up the cluster's bins (BY_MASS: masses, else counts), 32 to a group; the
    // result is the sum.  Each CTA hands its groups' sums to the others: their bins
    // (128 KB for P = 8) would take 7 us.
    template <bool BY_MASS>
    __device__ u64 add_bins() {
        static_assert(kBinsEach == 4 && kBinGroups == 64 && P <= 8, "eight threads to a group");
        __syncthreads();
        u64 sum = 0;
#pragma unroll
        for (int k = 0; k < kBinsEach; ++k) {
            const int bin = kBinsEach * threadIdx.x + k;
            sum += BY_MASS ? sh.mass[bin] : sh.count[bin];
        }
        for (int o = 1; o < 8; o <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        u64(&groups)[kMaxCluster][kBinGroups] = sh.groups[group_turn ^= 1];
        if (lane % 8 < P) dsmem_st_u64(dsmem_map(&groups[rank][threadIdx.x / 8], lane % 8), sum);
        sync();
        group[0] = group[1] = 0;
#pragma unroll
        for (int r = 0; r < P; ++r) {
            group[0] += groups[r][2 * lane];
            group[1] += groups[r][2 * lane + 1];
        }
        u64 incl = group[0] + group[1];
        for (int o = 1; o < 32; o <<= 1) {
            const u64 t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        before_group = incl - group[0] - group[1];
        return __shfl_sync(0xffffffffu, incl, 31);
    }
    // After that: the bin where the running weight, from *above on, reaches target,
    // and the weight before it.
    template <bool BY_MASS>
    __device__ int bin_at(u64 target, u64* above) {
        if (warp == 0) {
            u64 before = *above + before_group;
            const bool second = before + group[0] < target;
            if (second) before += group[0];
            const bool here = before < target && before + (second ? group[1] : group[0]) >= target;
            const unsigned who = __ballot_sync(0xffffffffu, here);
            const int src = who ? __ffs(who) - 1 : 0;
            const int bin = 32 * __shfl_sync(0xffffffffu, 2 * lane + second, src) + lane;
            before = __shfl_sync(0xffffffffu, before, src);
            u64 part[P], own = 0;
#pragma unroll
            for (int r = 0; r < P; ++r)
                part[r] = BY_MASS ? dsmem_ld_u64(dsmem_map(sh.mass + bin, r)) : dsmem_ld_u32(dsmem_map(sh.count + bin, r));
#pragma unroll
            for (int r = 0; r < P; ++r) own += part[r];
            u64 incl = own;
            for (int o = 1; o < 32; o <<= 1) {
                const u64 t = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += t;
            }
            incl += before;
            if (incl >= target && incl - own < target) {
                sh.found[0] = bin;
                sh.found[1] = incl - own;
            }
        }
        __syncthreads();
        *above = sh.found[1];
        return (int)sh.found[0];
    }

    // The prefix's elements in a bin, from all CTAs, as sh.all; false: more than the
    // list holds.
    __device__ bool gather(int bin, int which) {
        const float wanted = (float)bin + 8388608.0f;
        each([&](const float (&v)[4], int i) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (float_bin(v[k]) == wanted && in_prefix(v[k], i + k)) {
                    const int n = atomicAdd(&sh.listed[which], 1);
                    if (n < kList) sh.list[n] = ((u64)float_order_key(v[k]) << 32) | (uint32_t) ~(i + k);
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
    // The weights of what stands above an element are added by 1 to 32 lanes; a long
    // list is split over the cluster (300 elements: 5 us of a CTA's time otherwise).
    template <bool BY_MASS>
    __device__ void cut_in_list(u64 target) {
        const int n = sh.all_n;
        if (BY_MASS) {
            for (int i = threadIdx.x; i < n; i += kRowThreads)
                sh.weight[i] = fixed(float_from_order_key((uint32_t)(sh.all[i] >> 32)));
            __syncthreads();
        }
        const bool split = P > 1 && n > 64;
        const int threads = split ? P * kRowThreads : kRowThreads;
        int lanes = 32;
        while (lanes > 1 && n * lanes > threads) lanes >>= 1;
        const int i = ((split ? rank * kRowThreads : 0) + threadIdx.x) / lanes;  // n <= kList = kRowThreads
        if (__any_sync(0xffffffffu, i < n)) {
            const u64 e = i < n ? sh.all[i] : ~0ull;
            u64 upto = 0;
#pragma unroll 4
            for (int j = threadIdx.x % lanes; j < n; j += lanes)
                upto += sh.all[j] >= e ? (BY_MASS ? sh.weight[j] : 1ull) : 0ull;
            for (int o = 1; o < lanes; o <<= 1) upto += __shfl_xor_sync(0xffffffffu, upto, o);
            if (i < n && threadIdx.x % lanes == 0) {
                const u64 own = BY_MASS ? sh.weight[i] : 1ull;
                if (upto - own < target && upto >= target) {
                    sh.found[2] = e;
                    if (split)
                        for (int r = 0; r < P; ++r) dsmem_st_u64(dsmem_map(sh.found + 2, r), e);
                }
            }
        }
        if (split)
            sync();
        else
            __syncthreads();
        cut = float_from_order_key((uint32_t)(sh.found[2] >> 32));
        cut_index = (int)~(uint32_t)sh.found[2];
    }

    // The same for a bin with more elements than the list: its keys, 2048 bins at a
    // time, until one key is left, and among its elements by index.  `above`: the
    // weight before the bin.
    template <bool BY_MASS>
    __device__ void cut_in_bin(int bin, u64 target, u64 above) {
        uint32_t lo_key = 0xffffffffu, hi_key = 0;
        const float wanted = (float)bin + 8388608.0f;
        each([&](const float (&v)[4], int i) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                if (float_bin(v[k]) == wanted && in_prefix(v[k], i + k)) {
                    lo_key = min(lo_key, float_order_key(v[k]));
                    hi_key = max(hi_key, float_order_key(v[k]));
                }
        });
        // both ends in one reduction: the high key, and the low key's complement
        const u64 ends = reduce(((u64)hi_key << 32) | (uint32_t)~lo_key, [](u64 a, u64 b) {
            const uint32_t low = max((uint32_t)a, (uint32_t)b);
            return ((a > b ? a : b) & 0xffffffff00000000ull) | low;
        });
        hi_key = (uint32_t)(ends >> 32);
        lo_key = ~(uint32_t)ends;
        for (int round = 0; lo_key < hi_key && round < 3; ++round) {  // 2^32 keys, 2^21, 2^10
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
            each([&](const float (&v)[4], int i) {
                int to[4];
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const uint32_t key = float_order_key(v[k]);
                    const bool in = key >= lo_key && key <= hi_key && in_prefix(v[k], i + k);
                    to[k] = in ? (int)((hi_key - key) >> shift) : -1;
                    if (!BY_MASS && in) atomicAdd(&sh.count[to[k]], 1u);
                }
                if (BY_MASS) add_masses(v, to);
            });
            add_bins<BY_MASS>();  // the bin's weight reaches the target, and sums are exact: one is found
            const int found = bin_at<BY_MASS>(target, &above);
            hi_key -= (uint32_t)found << shift;
            const uint32_t width = (1u << shift) - 1u;
            if (hi_key - lo_key > width) lo_key = hi_key - width;
        }
        // how many of the equal elements, and the last one's index
        const float value = float_from_order_key(hi_key);
        const u64 w = BY_MASS ? fixed(value) : 1ull;
        const u64 need = w ? (target - above + w - 1) / w : 1ull;
        int mine = 0;
        each([&](const float (&v)[4], int i) {
#pragma unroll
            for (int k = 0; k < 4; ++k) mine += v[k] == value && in_prefix(v[k], i + k);
        });
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (lane < P) dsmem_st_u32(dsmem_map(sh.ties + rank * kRowWarps + warp, lane), (unsigned int)mine);
        if (threadIdx.x < P) sh.tie_index[threadIdx.x] = 0;
        sync();
        const int me = rank * kRowWarps + warp;
        u64 rank_of = 0;
        for (int i = lane; i < me; i += 32) rank_of += sh.ties[i];
        for (int o = 16; o; o >>= 1) rank_of += __shfl_xor_sync(0xffffffffu, rank_of, o);
        if (rank_of < need && rank_of + mine >= need) {
            for (int o = 4 * lane; o - 4 * lane < n; o += 128) {
                float v[4];
                load4(o, v);
                int same = 0;
#pragma unroll
                for (int k = 0; k < 4; ++k) same += v[k] == value && in_prefix(v[k], base + o + k);
                int incl = same;
                for (int s = 1; s < 32; s <<= 1) {
                    const int t = __shfl_up_sync(0xffffffffu, incl, s);
                    if (lane >= s) incl += t;
                }
                u64 at = rank_of + incl - same;
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    if (v[k] == value && in_prefix(v[k], base + o + k) && ++at == need)
                        for (int r = 0; r < P; ++r) dsmem_st_u64(dsmem_map(sh.tie_index + rank, r), (u64)(base + o + k) + 1);
                rank_of += __shfl_sync(0xffffffffu, incl, 31);
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
    extern __shared__ __align__(16) float stage[];
    __shared__ RowShared sh;
    const int row = blockIdx.x / P;
    Row<P, STAGED> r(p, sh, stage, row);
    const bool writer = r.rank == 0 && threadIdx.x == 0;

    // 1. the row, its maximum and that one's first index
    for (int i = threadIdx.x; i < kRowBins; i += kRowThreads) {
        sh.mass[i] = 0;
        sh.count[i] = 0;
    }
    if (threadIdx.x < kRoots) sh.root[threadIdx.x] = exp2((double)threadIdx.x / kRoots);
    if (threadIdx.x < 2) sh.listed[threadIdx.x] = 0;
    if (P > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    const float T = p.temperature ? p.temperature[row] : 1.0f;
    const int k = p.top_k ? p.top_k[row] : 0;
    const float top_p = p.top_p ? p.top_p[row] : 1.0f;
    r.floor_w = p.min_p ? (double)fminf(fmaxf(p.min_p[row], 0.0f), 1.0f) : 0.0;
    const double u = fminf(fmaxf(p.uniform[row], 0.0f), 0.99999994f);
    const bool greedy = !(T > 0.0f) || k == 1;
    int index;
    const float best = r.read(greedy, index);
    // the others have started: their shared memory may be written
    if (P > 1) asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    const u64 key = r.reduce(argmax_key(best, index), [](u64 a, u64 b) { return a > b ? a : b; });
    r.top = float_from_order_key((uint32_t)(key >> 32));
    if (greedy || r.top == -INFINITY) {
        if (writer) {
            const bool any = r.top > -INFINITY;
            p.token[row] = any ? (int)(0xffffffffu - (uint32_t)key) : -1;
            if (p.prob) p.prob[row] = any ? 1.0f : 0.0f;
            if (p.entropy) p.entropy[row] = 0.0f;
        }
        return;  // (the others' writes came before the barrier)
    }
    r.inv_t = 1.0 / (double)T;
    r.bin_scale = (float)((double)kRowBins / kBinSpan * r.inv_t);
    // below this there is no weight; an infinite maximum shares it with its like alone
    r.cut = r.top == INFINITY ? INFINITY : lowest_weighted(r.top, T);
    r.cut_index = r.cut > -INFINITY ? INT_MAX : -1;

    // 2. the kept prefix's last element: top-k's, and top-p's within it
    u64 above = 0;
    if (k > 0 && k < p.V) {
        r.each([&](const float (&v)[4], int i) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
                if (r.in_prefix(v[j], i + j)) atomicAdd(&sh.count[r.bin_of(v[j])], 1u);
        });
        if (r.template add_bins<false>() > (u64)k) {  // else all there is
            const int bin = r.template bin_at<false>((u64)k, &above);
            if (r.gather(bin, 0))
                r.template cut_in_list<false>((u64)k - above);
            else
                r.template cut_in_bin<false>(bin, (u64)k, above);
        }
    }
    if (!(top_p >= 1.0f)) {
        r.each([&](const float (&v)[4], int i) {
            int bin[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) bin[j] = r.in_prefix(v[j], i + j) ? r.bin_of(v[j]) : -1;
            r.add_masses(v, bin);
        });
        const u64 mass = r.template add_bins<true>();
        const double want = ceil((double)top_p * (double)mass);
        const u64 target = want > 1.0 ? min((u64)want, mass) : 1ull;
        above = 0;
        const int bin = r.template bin_at<true>(target, &above);
        if (r.gather(bin, 1))
            r.template cut_in_list<true>(target - above);
        else
            r.template cut_in_bin<true>(bin, target, above);
    }

    // 3. the kept mass, run by run
    double mass = 0.0, moment = 0.0;
    r.each([&](const float (&v)[4], int i) {
        double w[4], y[4];
        r.weights(v, i, w, y);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            mass += w[j];
            moment += w[j] * y[j];
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
    // (one always has it, unless the row changes while it is read: no run before the first then)
    run = max(__shfl_sync(0xffffffffu, run, src), 0);
    run_before = __shfl_sync(0xffffffffu, run_before, src);
    // 5. the element, by the warps of the CTA that has the run: each scans the lanes'
    // fours of 128 elements, and the first whose sum passes the goal has it
    if (run / kRowWarps != r.rank) return;
    r.turn_to(run % kRowWarps);
    if (threadIdx.x == 0) {  // a draw that finds none (here: at the start the stores took 0.2 us)
        sh.pick = -1;
        sh.pick_weight = 0.0;
    }
    double running = run_before;
    for (int first = 0; first < r.n; first += 128 * kRowWarps) {
        const int o = first + 128 * r.warp + 4 * r.lane;
        float v[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
        double w[4], y[4];
        if (o - 4 * r.lane < r.n) r.load4(o, v);
        r.weights(v, r.base + o, w, y);
        const double own = (w[0] + w[1]) + (w[2] + w[3]);
        double incl4 = own;
        for (int s = 1; s < 32; s <<= 1) {
            const double t = __shfl_up_sync(0xffffffffu, incl4, s);
            if (r.lane >= s) incl4 += t;
        }
        if (r.lane == 31) sh.chunk[r.warp] = incl4;
        __syncthreads();
        int chunk = -1, last = -1;
        double before = running;
        for (int c = 0; c < kRowWarps; ++c) {
            const double sum = sh.chunk[c];
            if (sum > 0.0 && chunk < 0) {
                last = c;
                if (running + sum > goal) {
                    chunk = c;
                    before = running;
                }
            }
            running += sum;
        }
        // A sum in another order may end a rounding lower, so that the goal is not
        // passed: the last element with a weight is then the one.
        if (r.warp == (chunk >= 0 ? chunk : last)) {
            double upto = before + (incl4 - own), pick_w = 0.0;
            int pick = -1;  // the lane's first element that passes the goal, else its last one
            bool hit = false;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                upto += w[j];
                if (w[j] > 0.0 && !hit) {
                    pick = j;
                    pick_w = w[j];
                    hit = chunk >= 0 && upto > goal;
                }
            }
            const unsigned hits = __ballot_sync(0xffffffffu, hit), any = __ballot_sync(0xffffffffu, pick >= 0);
            if (r.lane == (hits ? __ffs(hits) - 1 : 31 - __clz(any))) {
                sh.pick = r.base + o + pick;
                sh.pick_weight = pick_w;
            }
        }
        __syncthreads();
        if (chunk >= 0) break;
    }
    if (threadIdx.x == 0) {
        p.token[row] = sh.pick;
        if (p.prob) p.prob[row] = (float)(sh.pick_weight / all);
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
    if (STAGED) e = kernel_attributes<sample_rows_kernel<P, STAGED>>(kStagedMax * sizeof(float));
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
    // elements to read, or while a CTA's part leaves no room for others on its SM.
    // Measured, us by P = 1, 2, 4, 8: rows of 32000: one 22, 16, 13, 12; 16 36, 25, 19, 19;
    // 64 41, 28, 24, 29; 128 41, 34, 33, 52; 256 53, 46, 58, 101.  Of 4096: one 8, 9, 10,
    // 10; 64 13, 13, 17, 24.  256 rows of 131072: P = 4 177, 8 161
    int P = 1;
    while (P < kMaxCluster &&
           (((long long)rows * P < entry.num_sms && V / (2 * P) >= 2048) || V / P > 16 * 1024))
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
