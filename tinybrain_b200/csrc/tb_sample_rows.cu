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
    int P;
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

struct RowShared {
    uint2 mass[kRowBins];           // low, high words
    unsigned int count[kRowBins];
    u64 red[2][kRowWarps];          // a reduction's values, alternating
    u64 list[2][kList];             // the CTA's boundary elements: key, then the index's complement
    int listed[2];
    u64 all[kList], weight[kList];  // all CTAs'
    int all_n;
    u64 scan[2][kRowWarps];
    u64 found[4];
    double run_mass[kRowWarps], run_moment[kRowWarps];
    double all_mass[kMaxCluster * kRowWarps], all_moment[kMaxCluster * kRowWarps];
    int ties[kRowWarps];
    u64 tie_index;
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

// -0 becomes +0 (equal values are ties) and NaN -inf.
__device__ __forceinline__ float clean(float x) {
    x += 0.0f;
    return x == x ? x : -INFINITY;
}

template <bool STAGED>
struct Row {
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

    __device__ Row(const RowsParams& p_, RowShared& s, float* stage, int row) : p(p_), sh(s), kept(stage) {
        lane = threadIdx.x & 31;
        warp = threadIdx.x >> 5;
        rank = (int)cluster_ctarank();
        x = p.logits + row * p.ld;
        const int len = run_length(p.V, p.P);
        cta_begin = min(rank * kRowWarps * len, p.V);
        begin = min((rank * kRowWarps + warp) * len, p.V);
        end = min(begin + len, p.V);
    }
    __host__ __device__ static int run_length(int V, int P) {
        const int runs = P * kRowWarps;
        return ((V + runs - 1) / runs + 31) & ~31;
    }

    __device__ __forceinline__ float at(int i) const { return STAGED ? kept[i - cta_begin] : clean(x[i]); }
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
        if (lane == 0) r[warp] = v;
        cluster_sync();
        for (int i = lane; i < p.P * kRowWarps; i += 32)
            v = f(v, dsmem_ld_u64(dsmem_map(r + i % kRowWarps, i / kRowWarps)));
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
    // After cluster_sync: bins 2 t and 2 t + 1 of all CTAs, and what stands before
    // them in the order of the bins; `which` 0: counts, 1: masses.
    __device__ __forceinline__ u64 bins(int which, u64 (&b)[2], u64& before) {
        b[0] = b[1] = 0;
        for (int r = 0; r < p.P; ++r) {
            if (which == 0) {
                const u64 c = dsmem_ld_u64(dsmem_map(sh.count + 2 * threadIdx.x, r));
                b[0] += (unsigned int)c;
                b[1] += c >> 32;
            } else {
                b[0] += dsmem_ld_u64(dsmem_map(sh.mass + 2 * threadIdx.x, r));
                b[1] += dsmem_ld_u64(dsmem_map(sh.mass + 2 * threadIdx.x + 1, r));
            }
        }
        u64 incl = b[0] + b[1];
        for (int o = 1; o < 32; o <<= 1) {
            const u64 t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        __syncthreads();
        if (lane == 31) sh.scan[which][warp] = incl;
        __syncthreads();
        before = incl - b[0] - b[1];
        u64 sum = 0;
        for (int w = 0; w < kRowWarps; ++w) {
            if (w < warp) before += sh.scan[which][w];
            sum += sh.scan[which][w];
        }
        return sum;
    }
    // The bin where the running weight reaches target (-1: it does not), and the
    // weight before it.
    __device__ __forceinline__ int bin_at(const u64 (&b)[2], u64 before, u64 target, u64* above) {
        __syncthreads();
        if (threadIdx.x == 0) sh.found[0] = ~0ull;
        __syncthreads();
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
    __device__ __forceinline__ void clear_bins() {
        for (int i = threadIdx.x; i < kRowBins; i += kRowThreads) {
            sh.mass[i] = make_uint2(0, 0);
            sh.count[i] = 0;
        }
    }

    // The elements of a bin from all CTAs, as sh.all; false: more than the list holds.
    __device__ bool gather(int bin, int buffer) {
        each([&](float v, int i) {
            if (v > -INFINITY && bin_of(v) == bin) {
                const int n = atomicAdd(&sh.listed[buffer], 1);
                if (n < kList) sh.list[buffer][n] = ((u64)float_order_key(v) << 32) | (uint32_t)~i;
            }
        });
        cluster_sync();
        int n = 0;
        for (int r = 0; r < p.P; ++r) {
            const int here = (int)dsmem_ld_u32(dsmem_map(&sh.listed[buffer], r));
            if (n + here <= kList)
                for (int i = threadIdx.x; i < here; i += kRowThreads)
                    sh.all[n + i] = dsmem_ld_u64(dsmem_map(&sh.list[buffer][i], r));
            n += here;
        }
        if (threadIdx.x == 0) sh.all_n = n;
        __syncthreads();
        return n <= kList;
    }
    // sh.weight[i] = the list's elements' masses
    __device__ void weigh() {
        for (int i = threadIdx.x; i < sh.all_n; i += kRowThreads)
            sh.weight[i] = fixed(float_from_order_key((uint32_t)(sh.all[i] >> 32)));
        __syncthreads();
    }
    // The list's element where its running weight, in descending order, reaches
    // `target`; by_mass: of sh.weight, else counts.
    template <bool BY_MASS>
    __device__ u64 list_at(u64 target) {
        const int n = sh.all_n;
        for (int i = threadIdx.x; i < n; i += kRowThreads) {
            const u64 e = sh.all[i];
            u64 upto = 0;
            for (int j = 0; j < n; ++j) upto += sh.all[j] >= e ? (BY_MASS ? sh.weight[j] : 1ull) : 0ull;
            const u64 own = BY_MASS ? sh.weight[i] : 1ull;
            if (upto - own < target && upto >= target) sh.found[2] = e;
        }
        __syncthreads();
        return sh.found[2];
    }
    // Mass of the list's elements from `e` up.
    __device__ u64 list_mass(u64 e) {
        u64 sum = 0;
        for (int i = lane; i < sh.all_n; i += 32) sum += sh.all[i] >= e ? sh.weight[i] : 0ull;
        for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        return sum;
    }

    // A bin with more elements than the list: its keys, 1024 bins at a time, until
    // one key is left, and among its elements by index.  The element where the
    // weight (counts or masses) from `above` reaches target; *taken: the weight up
    // to and with it, in masses too where `mass_too`.
    template <bool BY_MASS>
    __device__ u64 narrow(int bin, u64 target, u64 above, u64 mass_above, bool mass_too, u64* mass_taken) {
        uint32_t lo_key = 0xffffffffu, hi_key = 0;
        each([&](float v, int) {
            const uint32_t k = float_order_key(v);
            if (v > -INFINITY && bin_of(v) == bin) {
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
            cluster_sync();  // the bins have been read
            clear_bins();
            __syncthreads();
            each([&](float v, int) {
                const uint32_t k = float_order_key(v);
                if (k < lo_key || k > hi_key) return;
                const int at = (int)((hi_key - k) >> shift);
                if (!BY_MASS) atomicAdd(&sh.count[at], 1u);
                if (BY_MASS || mass_too) add_mass(at, fixed(v));
            });
            cluster_sync();
            bins(BY_MASS ? 1 : 0, b, before);
            const u64 base = above;
            const int found = bin_at(b, before + base, target, &above);
            if (found < 0) break;  // cannot be: the bin's weight passes the target, and sums are exact
            if (!BY_MASS && mass_too) {  // the mass before the same bin
                u64 m[2], m_before;
                bins(1, m, m_before);
                __syncthreads();
                if ((int)threadIdx.x == found / 2) sh.found[1] = m_before + (found % 2 ? m[0] : 0ull);
                __syncthreads();
                mass_above += sh.found[1];
            }
            hi_key -= (uint32_t)found << shift;
            const uint32_t width = (1u << shift) - 1u;
            if (hi_key - lo_key > width) lo_key = hi_key - width;
        }
        const u64 w = BY_MASS || mass_too ? fixed(float_from_order_key(hi_key)) : 0ull;
        // how many of the equal elements, and the last one's index
        const u64 need = BY_MASS ? (w ? (target - above + w - 1) / w : 1ull) : target - above;
        int mine = 0;
        each([&](float v, int) { mine += float_order_key(v) == hi_key; });
        for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
        if (lane == 0) sh.ties[warp] = mine;
        if (threadIdx.x == 0) sh.tie_index = 0;
        cluster_sync();
        const int me = rank * kRowWarps + warp;
        u64 rank_of = 0;
        for (int i = lane; i < me; i += 32) rank_of += dsmem_ld_u32(dsmem_map(sh.ties + i % kRowWarps, i / kRowWarps));
        for (int o = 16; o; o >>= 1) rank_of += __shfl_xor_sync(0xffffffffu, rank_of, o);
        if (rank_of < need && rank_of + mine >= need) {
            for (int i0 = begin; i0 < end; i0 += 32) {
                const int i = i0 + lane;
                const bool same = i < end && float_order_key(at(i)) == hi_key;
                const unsigned who = __ballot_sync(0xffffffffu, same);
                if (same && rank_of + __popc(who & ((2u << lane) - 1u)) == need) sh.tie_index = (u64)i + 1;
                rank_of += __popc(who);
            }
        }
        cluster_sync();
        u64 index = 0;
        for (int r = 0; r < p.P; ++r) index += dsmem_ld_u64(dsmem_map(&sh.tie_index, r));
        // (equal weights that round to no mass may not reach the target: all of them, then)
        *mass_taken = mass_above + need * w;
        return ((u64)hi_key << 32) | (uint32_t) ~(uint32_t)(index ? index - 1 : 0xffffffffull);
    }
};

template <bool STAGED>
__global__ void __launch_bounds__(kRowThreads) sample_rows_kernel(RowsParams p) {
    extern __shared__ float stage[];
    __shared__ RowShared sh;
    const int row = blockIdx.x / p.P;
    Row<STAGED> r(p, sh, stage, row);
    const bool writer = r.rank == 0 && threadIdx.x == 0;

    // 1. the row, its maximum and that one's first index
    r.clear_bins();
    if (threadIdx.x < 2) sh.listed[threadIdx.x] = 0;
    float best = -INFINITY;
    int best_i = 0;
    r.read([&](float v, int i) {
        if (v > best) {
            best = v;
            best_i = i;
        }
    });
    const u64 key =
        r.reduce(best > -INFINITY ? argmax_key(best, best_i) : 0ull, [](u64 a, u64 b) { return a > b ? a : b; });
    const float T = p.temperature ? p.temperature[row] : 1.0f;
    const int k = p.top_k ? p.top_k[row] : 0;
    if (key == 0 || !(T > 0.0f) || k == 1) {
        if (writer) {
            p.token[row] = key ? (int)(0xffffffffu - (uint32_t)key) : -1;
            if (p.prob) p.prob[row] = key ? 1.0f : 0.0f;
            if (p.entropy) p.entropy[row] = 0.0f;
        }
        cluster_sync();  // no CTA leaves while another reads its shared memory
        return;
    }
    r.top = float_from_order_key((uint32_t)(key >> 32));
    r.inv_t = 1.0 / (double)T;
    r.bin_scale = (float)((double)kRowBins / kBinSpan * r.inv_t);

    // 2. the last element of the kept prefix, as (key, complement of the index):
    // what compares greater or equal is kept
    u64 cut = ((u64)float_order_key(-INFINITY) << 32) | 0xffffffffull;  // everything above -inf
    const float tp = p.top_p ? p.top_p[row] : 1.0f;
    bool by_count = k > 0 && k < p.V;
    const bool by_mass = !(tp >= 1.0f);
    if (by_count || by_mass) {
        r.each([&](float v, int) {
            if (v == -INFINITY) return;
            const int bin = r.bin_of(v);
            if (by_count) atomicAdd(&sh.count[bin], 1u);
            if (by_mass) r.add_mass(bin, r.fixed(v));
        });
        cluster_sync();
        u64 c[2], c_before = 0, m[2], m_before = 0, mass = 0, above = 0;
        if (by_mass) mass = r.bins(1, m, m_before);
        if (by_count) by_count = r.bins(0, c, c_before) > (u64)k;  // else all there is
        u64 mass_above = mass;  // before the bin of the k-th element
        int k_bin = kRowBins;
        bool listed = false;
        if (by_count) {
            k_bin = r.bin_at(c, c_before, (u64)k, &above);
            if (by_mass) {
                __syncthreads();
                if ((int)threadIdx.x == k_bin / 2) sh.found[3] = m_before + (k_bin % 2 ? m[0] : 0ull);
                __syncthreads();
                mass_above = sh.found[3];
            }
            listed = r.gather(k_bin, 0);
            if (listed) {
                cut = r.template list_at<false>((u64)k - above);
                if (by_mass) {
                    r.weigh();
                    mass = mass_above + r.list_mass(cut);
                }
            } else {
                cut = r.template narrow<false>(k_bin, (u64)k, above, mass_above, by_mass, &mass);
            }
        }
        if (by_mass) {
            const double want = ceil((double)tp * (double)mass);
            const u64 target = want > 1.0 ? min((u64)want, mass) : 1ull;
            if (target > mass_above) {  // among the last bin that top-k keeps
                if (listed) {
                    cut = r.template list_at<true>(target - mass_above);
                } else {
                    const u64 p_cut = r.template narrow<true>(k_bin, target, mass_above, 0, false, &mass);
                    cut = max(cut, p_cut);
                }
            } else {
                const int p_bin = r.bin_at(m, m_before, target, &above);
                if (r.gather(p_bin, 1)) {
                    r.weigh();
                    cut = r.template list_at<true>(target - above);
                } else {
                    cut = r.template narrow<true>(p_bin, target, above, 0, false, &mass);
                }
            }
        }
    }

    // 3. the kept mass, run by run
    const double floor_w = p.min_p ? (double)fminf(fmaxf(p.min_p[row], 0.0f), 1.0f) : 0.0;
    const auto weight_of = [&](float v, int i) -> double {
        if (v == -INFINITY || (((u64)float_order_key(v) << 32) | (uint32_t)~i) < cut) return 0.0;
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
    if (r.lane == 0) {
        sh.run_mass[r.warp] = mass;
        sh.run_moment[r.warp] = moment;
    }
    cluster_sync();
    const int runs = p.P * kRowWarps;
    for (int i = threadIdx.x; i < runs; i += kRowThreads) {
        sh.all_mass[i] = __longlong_as_double((long long)dsmem_ld_u64(dsmem_map(sh.run_mass + i % kRowWarps, i / kRowWarps)));
        sh.all_moment[i] =
            __longlong_as_double((long long)dsmem_ld_u64(dsmem_map(sh.run_moment + i % kRowWarps, i / kRowWarps)));
    }
    __syncthreads();

    // 4. the run that holds the draw, found by every warp alike (4 runs a lane)
    double part[4], sum4 = 0.0, mom = 0.0;
    for (int j = 0; j < 4; ++j) {
        const int i = r.lane * 4 + j;
        part[j] = i < runs ? sh.all_mass[i] : 0.0;
        sum4 += part[j];
        mom += i < runs ? sh.all_moment[i] : 0.0;
    }
    double incl = sum4;
    for (int o = 1; o < 32; o <<= 1) {
        const double t = __shfl_up_sync(0xffffffffu, incl, o);
        if (r.lane >= o) incl += t;
    }
    for (int o = 16; o; o >>= 1) mom += __shfl_xor_sync(0xffffffffu, mom, o);
    const double all = __shfl_sync(0xffffffffu, incl, 31);
    const double u = fminf(fmaxf(p.uniform[row], 0.0f), 0.99999994f);
    const double goal = u * all;
    double before = __shfl_up_sync(0xffffffffu, incl, 1);
    if (r.lane == 0) before = 0.0;
    int run = -1;
    double run_before = 0.0;
    for (int j = 0; j < 4; ++j) {
        const double next = j == 3 ? incl : before + part[j];
        if (run < 0 && part[j] > 0.0 && next > goal) {
            run = r.lane * 4 + j;
            run_before = before;
        }
        before = next;
    }
    const unsigned who = __ballot_sync(0xffffffffu, run >= 0);
    const int src = who ? __ffs(who) - 1 : 0;
    run = __shfl_sync(0xffffffffu, run, src);
    run_before = __shfl_sync(0xffffffffu, run_before, src);
    if (run == r.rank * kRowWarps + r.warp) {
        // 5. the element: 256 at a time by their sum, then 32 at a time by a scan
        const auto weight_at = [&](int i) { return i < r.end ? weight_of(r.at(i), i) : 0.0; };
        int last = -1;
        double last_w = 0.0, running = run_before;
        bool done = false;
        for (int b = r.begin; b < r.end && !done; b += 256) {
            double s = 0.0;
#pragma unroll
            for (int j = 0; j < 256; j += 32) s += weight_at(b + j + r.lane);
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (s == 0.0) continue;
            // what ends just short of the goal is searched too: a sum in another order
            // may end a rounding lower, and the run's last element is then the one
            if (running + s >= goal * (1.0 - 1e-12)) {
                double upto = running;
                for (int j = 0; j < 256 && b + j < r.end && !done; j += 32) {
                    const double w = weight_at(b + j + r.lane);
                    double c = w;
                    for (int o = 1; o < 32; o <<= 1) {
                        const double t = __shfl_up_sync(0xffffffffu, c, o);
                        if (r.lane >= o) c += t;
                    }
                    const unsigned hit = __ballot_sync(0xffffffffu, w > 0.0 && upto + c > goal);
                    const unsigned any = __ballot_sync(0xffffffffu, w > 0.0);
                    const int pick = hit ? __ffs(hit) - 1 : any ? 31 - __clz(any) : -1;
                    if (pick >= 0) {
                        last = b + j + pick;
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
    cluster_sync();
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
    RowsParams p{logits, ld, V, 1, 0.0, temperature, top_k, top_p, min_p, uniform, token, prob, entropy};
    // CTAs of a row: while the rows leave SMs idle and a CTA would still have 2048
    // elements to read, or while a CTA's part leaves no room for others on its SM
    while (p.P < kMaxCluster && (((long long)rows * p.P < 2ll * entry.num_sms && V / (2 * p.P) >= 2048) ||
                                 V / p.P > 16 * 1024))
        p.P *= 2;
    int log_v = 0;
    while ((1ll << log_v) < V) ++log_v;
    p.one = std::ldexp(1.0, 62 - log_v);
    const int part = Row<true>::run_length(V, p.P) * kRowWarps;
    const bool staged = part <= kStagedMax;  // else the passes read the row from L2
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * p.P));
    cfg.blockDim = dim3(kRowThreads);
    cfg.dynamicSmemBytes = staged ? (size_t)part * sizeof(float) : 0;
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.P;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaError_t e = cudaSuccess;
    if (cfg.dynamicSmemBytes > 16 * 1024)  // with the static part beyond the 48 KB that need no asking
        e = cudaFuncSetAttribute(sample_rows_kernel<true>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                 kStagedMax * (int)sizeof(float));
    if (e == cudaSuccess)
        e = staged ? cudaLaunchKernelEx(&cfg, sample_rows_kernel<true>, p)
                   : cudaLaunchKernelEx(&cfg, sample_rows_kernel<false>, p);
    return launch_status(e, "sampling launch");
}
