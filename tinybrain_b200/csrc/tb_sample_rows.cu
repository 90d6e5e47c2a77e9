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
// A row is read by a cluster of P CTAs (P = 1, 2, 4, 8: enough that a few rows
// still fill the GPU), each of whose warps owns a run of consecutive elements.
// The row is not staged: a CTA's share stays in its L1 between the passes, and
// all rows in flight fit L2.  Passes: the maximum; for a truncated row a
// histogram of 1024 bins over (m - x) / T, then two or three of 1024 bins over
// the keys of the bin that holds the boundary (no sort: a select needs the
// boundary, not the order); the kept masses; and a search in the one run that
// holds the draw.  Bound by the fp64 exponentials of rows that keep most of
// their vocabulary, else by the passes' latency.
#include "tb_common.cuh"
#include "tb_stream_entry.h"
#include "tb_unit.cuh"

namespace tb {
namespace {

constexpr int kRowThreads = 512;
constexpr int kRowWarps = kRowThreads / 32;
constexpr int kRowBins = 1024;
constexpr int kMaxCluster = 8;
constexpr double kBinSpan = 40.0;  // nats below the maximum that the first histogram resolves

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

struct RowShared {
    unsigned int lo[2][kRowBins], hi[2][kRowBins];  // a level's histogram, alternating
    unsigned long long red[2][kRowWarps];           // a reduction's values, alternating
    double mass[kRowWarps], moment[kRowWarps];
    double all_mass[kMaxCluster * kRowWarps], all_moment[kMaxCluster * kRowWarps];
    int ties[kRowWarps];
    unsigned long long scan[kRowWarps];
    unsigned long long found_above[2];
    int found_bin[2];
};

__device__ __forceinline__ unsigned long long dsmem_ld_u64(uint32_t addr) {
    unsigned long long v;
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

struct Row {
    const RowsParams& p;
    RowShared& sh;
    const float* x;
    int begin, end;  // the warp's run
    int lane, warp, rank;
    int turn = 0;    // which of the alternating buffers is next
    float top = 0.0f;
    double inv_t = 0.0;
    float bin_scale = 0.0f;

    __device__ Row(const RowsParams& p_, RowShared& s, int row) : p(p_), sh(s) {
        lane = threadIdx.x & 31;
        warp = threadIdx.x >> 5;
        rank = (int)cluster_ctarank();
        x = p.logits + row * p.ld;
        const int runs = p.P * kRowWarps;
        const int len = ((p.V + runs - 1) / runs + 31) & ~31;
        begin = min((rank * kRowWarps + warp) * len, p.V);
        end = min(begin + len, p.V);
    }

    // f(value, index) over the warp's run, four loads in flight
    template <class F>
    __device__ __forceinline__ void each(F f) const {
        int i = begin + lane;
        for (; i + 96 < end; i += 128) {
            float v[4];
#pragma unroll
            for (int k = 0; k < 4; ++k) v[k] = x[i + 32 * k];
#pragma unroll
            for (int k = 0; k < 4; ++k) f(clean(v[k]), i + 32 * k);
        }
        for (; i < end; i += 32) f(clean(x[i]), i);
    }

    __device__ __forceinline__ double exponent(float v) const {
        return v == top ? 0.0 : ((double)v - (double)top) * inv_t;
    }
    __device__ __forceinline__ double weight(float v) const { return v == top ? 1.0 : exp(exponent(v)); }
    __device__ __forceinline__ unsigned long long fixed(float v) const {
        const double w = weight(v);  // NaN where an infinite maximum meets an infinite T: no mass
        return w > 0.0 ? (unsigned long long)__double2ll_rn(w * p.one) : 0ull;
    }
    // Monotone in the value: 0 for the maximum, the last bin for all that lies
    // kBinSpan nats or more below it.
    __device__ __forceinline__ int first_bin(float v) const {
        if (v == top) return 0;
        return (int)fminf((top - v) * bin_scale, (float)(kRowBins - 1));
    }

    // Reduction over the cluster by an associative, commutative f with f(v, v) = v:
    // every thread gets the result.
    template <class F>
    __device__ unsigned long long reduce(unsigned long long v, F f) {
        for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
        unsigned long long* r = sh.red[turn];
        if (lane == 0) r[warp] = v;
        cluster_sync();
        for (int i = lane; i < p.P * kRowWarps; i += 32)
            v = f(v, dsmem_ld_u64(dsmem_map(r + i % kRowWarps, i / kRowWarps)));
        for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
        turn ^= 1;
        return v;
    }

    // One histogram: fill(add) adds every member's weight to its bin (0 =
    // largest values).  The result is the bin where the running weight, from
    // `above`, reaches target = target_of(weight of all), or -1; *above
    // becomes the weight before that bin and *total the weight of all.
    template <class Fill, class Target>
    __device__ int level(Fill fill, Target target_of, unsigned long long* above, unsigned long long* total) {
        unsigned int *lo = sh.lo[turn], *hi = sh.hi[turn];
        for (int i = threadIdx.x; i < kRowBins; i += kRowThreads) lo[i] = hi[i] = 0;
        if (threadIdx.x == 0) sh.found_bin[turn] = -1;
        __syncthreads();
        fill([&](int bin, unsigned long long w) {
            const unsigned int wl = (unsigned int)w;
            unsigned int wh = (unsigned int)(w >> 32);
            if (wl && atomicAdd(lo + bin, wl) + wl < wl) ++wh;  // carry
            if (wh) atomicAdd(hi + bin, wh);
        });
        cluster_sync();
        static_assert(kRowBins == 2 * kRowThreads, "two bins a thread");
        unsigned long long b[2] = {0, 0};
        for (int r = 0; r < p.P; ++r)
            for (int k = 0; k < 2; ++k)
                b[k] += dsmem_ld_u32(dsmem_map(lo + 2 * threadIdx.x + k, r)) +
                        ((unsigned long long)dsmem_ld_u32(dsmem_map(hi + 2 * threadIdx.x + k, r)) << 32);
        unsigned long long incl = b[0] + b[1];
        for (int o = 1; o < 32; o <<= 1) {
            const unsigned long long t = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += t;
        }
        if (lane == 31) sh.scan[warp] = incl;
        __syncthreads();
        unsigned long long before = *above + incl - b[0] - b[1], sum = 0;
        for (int w = 0; w < kRowWarps; ++w) {
            if (w < warp) before += sh.scan[w];
            sum += sh.scan[w];
        }
        const unsigned long long target = target_of(sum);
        for (int k = 0; k < 2; ++k) {
            if (before < target && before + b[k] >= target) {
                sh.found_bin[turn] = 2 * threadIdx.x + k;
                sh.found_above[turn] = before;
            }
            before += b[k];
        }
        __syncthreads();
        const int bin = sh.found_bin[turn];
        if (bin >= 0) *above = sh.found_above[turn];
        *total = sum;
        turn ^= 1;
        return bin;
    }

    // The key T at which the running weight, over the values above key
    // `floor` in descending order, reaches target = target_of(their weight):
    // *above of it lies above T.  false: the target exceeds their weight.
    template <class Weight, class Target>
    __device__ bool select(uint32_t floor, Weight w, Target target_of, uint32_t* T, unsigned long long* above,
                           unsigned long long* total, unsigned long long* target) {
        unsigned long long ignored;
        *above = 0;
        int bin = level(
            [&](auto add) {
                each([&](float v, int) {
                    if (float_order_key(v) > floor) add(first_bin(v), w(v));
                });
            },
            target_of, above, total);
        if (bin < 0) return false;
        *target = target_of(*total);
        uint32_t lo_key = 0xffffffffu, hi_key = 0;
        each([&](float v, int) {
            const uint32_t k = float_order_key(v);
            if (k > floor && first_bin(v) == bin) {
                lo_key = min(lo_key, k);
                hi_key = max(hi_key, k);
            }
        });
        // both ends in one reduction: the high key, and the low key's complement
        const unsigned long long ends =
            reduce(((unsigned long long)hi_key << 32) | (uint32_t)~lo_key,
                   [](unsigned long long a, unsigned long long b) {
                       const uint32_t low = max((uint32_t)a, (uint32_t)b);
                       return ((a > b ? a : b) & 0xffffffff00000000ull) | low;
                   });
        hi_key = (uint32_t)(ends >> 32);
        lo_key = ~(uint32_t)ends;
        while (lo_key < hi_key) {
            int shift = 0;
            while (((hi_key - lo_key) >> shift) >= (uint32_t)kRowBins) ++shift;
            bin = level(
                [&](auto add) {
                    each([&](float v, int) {
                        const uint32_t k = float_order_key(v);
                        if (k >= lo_key && k <= hi_key) add((int)((hi_key - k) >> shift), w(v));
                    });
                },
                [&](unsigned long long) { return *target; }, above, &ignored);
            hi_key -= (uint32_t)bin << shift;
            const uint32_t width = (1u << shift) - 1u;
            if (hi_key - lo_key > width) lo_key = hi_key - width;
        }
        *T = hi_key;
        return true;
    }
};

__global__ void __launch_bounds__(kRowThreads) sample_rows_kernel(RowsParams p) {
    __shared__ RowShared sh;
    const int row = blockIdx.x / p.P;
    Row r(p, sh, row);
    const bool writer = r.rank == 0 && threadIdx.x == 0;

    // 1. the maximum and its first index
    float best = -INFINITY;
    int best_i = 0;
    r.each([&](float v, int i) {
        if (v > best) {
            best = v;
            best_i = i;
        }
    });
    const auto larger = [](unsigned long long a, unsigned long long b) { return a > b ? a : b; };
    const unsigned long long key = r.reduce(best > -INFINITY ? argmax_key(best, best_i) : 0ull, larger);
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

    // 2. the boundary of the kept prefix: all above key `cut`, and the first
    // `need` elements at it
    uint32_t cut = float_order_key(-INFINITY);
    long long need = 0;
    unsigned long long above = 0, total = 0, target = 0;
    if (k > 0 && k < p.V) {
        uint32_t t;
        if (r.select(cut, [](float) { return 1ull; }, [&](unsigned long long) { return (unsigned long long)k; }, &t,
                     &above, &total, &target)) {
            cut = t;
            need = k - (long long)above;
        }
    }
    const float tp = p.top_p ? p.top_p[row] : 1.0f;
    if (!(tp >= 1.0f)) {
        const unsigned long long tie = need ? r.fixed(float_from_order_key(cut)) : 0ull;
        const auto share = [&](unsigned long long mass) -> unsigned long long {
            const double want = (double)tp * (double)(mass + (unsigned long long)need * tie);
            return want > 1.0 ? (unsigned long long)ceil(want) : 1ull;
        };
        uint32_t t;
        unsigned long long mass = 0;
        if (r.select(cut, [&](float v) { return r.fixed(v); }, share, &t, &above, &mass, &target)) {
            const unsigned long long each = r.fixed(float_from_order_key(t));
            cut = t;
            need = each ? (long long)((target - above + each - 1) / each) : 1;
        } else if (need) {  // the boundary lies among top-k's last, equal elements
            const double want = fmax((double)tp, 0.0) * (double)(mass + (unsigned long long)need * tie);
            const double rest = want - (double)mass;
            const long long n = tie ? (long long)ceil(rest / (double)tie) : need;
            need = min(need, max(n, mass ? 0ll : 1ll));
        }
    }

    // 3. the ties' places, where some of them may be left out
    int tie_rank = 0;
    if (need) {
        int n = 0;
        r.each([&](float v, int) { n += float_order_key(v) == cut; });
        for (int o = 16; o; o >>= 1) n += __shfl_xor_sync(0xffffffffu, n, o);
        if (r.lane == 0) sh.ties[r.warp] = n;
        cluster_sync();
        const int me = r.rank * kRowWarps + r.warp;
        for (int i = r.lane; i < me; i += 32)
            tie_rank += (int)dsmem_ld_u32(dsmem_map(sh.ties + i % kRowWarps, i / kRowWarps));
        for (int o = 16; o; o >>= 1) tie_rank += __shfl_xor_sync(0xffffffffu, tie_rank, o);
    }

    // 4. the kept mass, run by run.  The elements of 32 lanes are consecutive,
    // so a tie's place is the ties of earlier steps and of lower lanes.
    const double floor_w = p.min_p ? (double)fminf(fmaxf(p.min_p[row], 0.0f), 1.0f) : 0.0;
    const auto weight_at = [&](int i, int& ties_before) -> double {
        const float v = i < r.end ? clean(r.x[i]) : -INFINITY;
        const uint32_t kx = float_order_key(v);
        bool in = kx > cut;
        if (need) {
            const unsigned same = __ballot_sync(0xffffffffu, kx == cut);
            if (kx == cut) in = ties_before + __popc(same & ((1u << r.lane) - 1u)) < need;
            ties_before += __popc(same);
        }
        if (!in) return 0.0;
        const double w = r.weight(v);
        return w >= floor_w ? w : 0.0;
    };
    double mass = 0.0, moment = 0.0;
    {
        int ties = tie_rank;
        for (int b = r.begin; b < r.end; b += 32) {
            const double w = weight_at(b + r.lane, ties);
            if (w > 0.0) {
                mass += w;
                moment += w * r.exponent(clean(r.x[b + r.lane]));
            }
        }
    }
    for (int o = 16; o; o >>= 1) {
        mass += __shfl_xor_sync(0xffffffffu, mass, o);
        moment += __shfl_xor_sync(0xffffffffu, moment, o);
    }
    if (r.lane == 0) {
        sh.mass[r.warp] = mass;
        sh.moment[r.warp] = moment;
    }
    cluster_sync();
    const int runs = p.P * kRowWarps;
    for (int i = threadIdx.x; i < runs; i += kRowThreads) {
        sh.all_mass[i] = __longlong_as_double((long long)dsmem_ld_u64(dsmem_map(sh.mass + i % kRowWarps, i / kRowWarps)));
        sh.all_moment[i] =
            __longlong_as_double((long long)dsmem_ld_u64(dsmem_map(sh.moment + i % kRowWarps, i / kRowWarps)));
    }
    __syncthreads();

    // 5. the run that holds the draw, found by every warp alike (4 runs a lane)
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
        // 6. the element: 256 at a time by their sum, then 32 at a time by a scan
        int ties = tie_rank, last = -1;
        double last_w = 0.0, running = run_before;
        bool done = false;
        for (int b = r.begin; b < r.end && !done; b += 256) {
            const int ties_here = ties;
            double s = 0.0;
            for (int j = 0; j < 256 && b + j < r.end; j += 32) s += weight_at(b + j + r.lane, ties);
            for (int o = 16; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
            if (s == 0.0) continue;
            // the last 256 with any mass are searched in any case: a sum in another
            // order may end a rounding short of the goal
            const bool cross = running + s > goal;
            int t2 = ties_here;
            double run2 = running;
            if (cross || running + s >= goal * (1.0 - 1e-12)) {
                for (int j = 0; j < 256 && b + j < r.end && !done; j += 32) {
                    const int i = b + j + r.lane;
                    const double w = weight_at(i, t2);
                    double c = w;
                    for (int o = 1; o < 32; o <<= 1) {
                        const double t = __shfl_up_sync(0xffffffffu, c, o);
                        if (r.lane >= o) c += t;
                    }
                    const unsigned hit = __ballot_sync(0xffffffffu, w > 0.0 && run2 + c > goal);
                    const unsigned any = __ballot_sync(0xffffffffu, w > 0.0);
                    const int pick = hit ? __ffs(hit) - 1 : any ? 31 - __clz(any) : -1;
                    if (pick >= 0) {
                        last = b + j + pick;
                        last_w = __shfl_sync(0xffffffffu, w, pick);
                    }
                    done = hit != 0;
                    run2 += __shfl_sync(0xffffffffu, c, 31);
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
    // CTAs of a row: while the rows leave SMs idle and a CTA would still have
    // 2048 elements to read
    while (p.P < kMaxCluster && (long long)rows * p.P < 2ll * entry.num_sms && V / (2 * p.P) >= 2048) p.P *= 2;
    int log_v = 0;
    while ((1ll << log_v) < V) ++log_v;
    p.one = std::ldexp(1.0, 62 - log_v);
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)(rows * p.P));
    cfg.blockDim = dim3(kRowThreads);
    cfg.stream = static_cast<cudaStream_t>(stream);
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = (unsigned)p.P;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return launch_status(cudaLaunchKernelEx(&cfg, sample_rows_kernel, p), "sampling launch");
}
