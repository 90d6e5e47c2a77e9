// tb_chunk_units.cuh -- what the kernels of the chunk attention (tb_chunk.cu,
// tb_chunk_few.cuh) share beside the walk over units (tb_chunk_walk.h): their waits,
// the search for a CTA's share, the partial sums of units that several CTAs hold,
// and one row in plain fp32.
#pragma once

#include <climits>

#include "tb_chunk_walk.h"
#include "tb_common.cuh"
#include "tb_stream_entry.h"

namespace tb {

// Pool page of a table entry, -1 where there is none (evicted, or reported as bad).
__device__ __forceinline__ int checked_page(const ChunkParams& p, int page) {
    if (page >= p.num_pages) {
        record_error(p.err, kDevBadPage);
        return -1;
    }
    return page;
}
__device__ __forceinline__ int page_at(const ChunkParams& p, int s, int pos) {
    return checked_page(p, p.table[(size_t)s * p.stride + pos / kPageTokens]);
}

template <int D>
__device__ __forceinline__ const float* head_rows(const ChunkParams& p, int page, int kv, int head) {
    return p.pool + ((((size_t)page * p.num_layers + p.layer) * 2 + kv) * p.Hkv + head) * (size_t)(kPageTokens * D);
}

// One query row of one head over positions [t0, t1) by one warp: lane = token
// for the scores, lane = dim for the sums; fp32 throughout.
template <int D>
struct RowSum {
    float m = -INFINITY, l = 0.0f;
    float acc[(D + 31) / 32] = {};

    __device__ void add_range(const ChunkParams& p, const float* q, float scale, int s, int head, int t0, int t1) {
        const int lane = threadIdx.x & 31;
        for (int base = t0; base < t1; base += 32) {
            const int t = base + lane;
            float score = -INFINITY;
            int page = -1;
            if (t < t1) {
                page = page_at(p, s, t);
                score = 0.0f;
                if (page >= 0) {
                    const float4* k = reinterpret_cast<const float4*>(head_rows<D>(p, page, 0, head) +
                                                                      (t % kPageTokens) * D);
#pragma unroll 4
                    for (int i = 0; i < D / 4; ++i) {  // q may be aligned to 4 bytes only
                        const float4 a = k[i];
                        score = fmaf(a.x, q[4 * i], fmaf(a.y, q[4 * i + 1],
                                                         fmaf(a.z, q[4 * i + 2], fmaf(a.w, q[4 * i + 3], score))));
                    }
                    score *= scale;
                }
            }
            float mx = score;
            for (int o = 16; o; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
            mx = fmaxf(mx, m);
            const float off = mx == -INFINITY ? 0.0f : mx;  // nothing but -inf so far
            const float w = t < t1 ? expf(score - off) : 0.0f, r = expf(m - off);
            m = mx;
            float sum = w;
            for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
            l = l * r + sum;
#pragma unroll
            for (int i = 0; i < (D + 31) / 32; ++i) acc[i] *= r;
            const int n = min(32, t1 - base);
            for (int j = 0; j < n; ++j) {
                const int pg = __shfl_sync(0xffffffffu, page, j);
                const float wj = __shfl_sync(0xffffffffu, w, j);
                if (pg < 0) continue;
                const float* v = head_rows<D>(p, pg, 1, head) + ((base + j) % kPageTokens) * D;
#pragma unroll
                for (int i = 0; i < (D + 31) / 32; ++i)
                    if (lane + 32 * i < D) acc[i] = fmaf(wj, v[lane + 32 * i], acc[i]);
            }
        }
    }
};

constexpr int kChunkCtas = 148; // most CTAs of a launch (the workspace's size)

// Sleeps until the phase completes or a millisecond has passed.  Without the
// hint the waiting warps poll, and took a third of the issue slots.
__device__ __forceinline__ bool sleep_on(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2, %3;\n\t"
        "selp.u32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(smem_u32(bar)), "r"(parity), "r"(1000000u)
        : "memory");
    return ok != 0;
}
// What the waits of a CTA go by.  One that takes longer than `limit` (ns) sets `dead`,
// after which nobody waits any more.  Rows summed in fp32 add their own time to the
// limit: 128 of them over 65536 positions take 0.7 s, for which the other warps wait.
struct ChunkWatch {
    volatile int dead;
    unsigned long long limit;
};
__device__ __forceinline__ void watch_init(ChunkWatch& watch) {
    watch.dead = 0;
    watch.limit = kWaitLimitNs;
}
__device__ __forceinline__ bool chunk_wait(ChunkWatch* watch, uint64_t* bar, uint32_t parity, int* err) {
    if (sleep_on(bar, parity)) return true;
    const unsigned long long t0 = global_timer_ns();
    while (!watch->dead) {
        if (sleep_on(bar, parity)) return true;
        if (global_timer_ns() - t0 > *static_cast<volatile unsigned long long*>(&watch->limit)) {
            record_error(err, kDevWaitTimeout);
            watch->dead = 1;
        }
    }
    return false;
}
// After a wait that ran out: time for the CTA's copies in flight to land (they
// take microseconds) before it ends.
__device__ __forceinline__ void land_copies() {
    const uint64_t t0 = global_timer_ns();
    while (global_timer_ns() - t0 < 50000000ull) {
    }
}
// The same for several barriers at once: every lane with one of its own (bar not
// null) waits for it, all return together.  With the roles' code spread over the
// instruction cache a wait costs some 300 cycles even where nothing is missing.
__device__ __forceinline__ void lanes_wait(ChunkWatch* watch, uint64_t* bar, uint32_t parity, int* err) {
    bool ok = !bar || sleep_on(bar, parity);
    if (__all_sync(0xffffffffu, ok)) return;
    if (!ok) chunk_wait(watch, bar, parity, err);
    __syncwarp();
}
// What a share leaves for chunk_combine_kernel: its last unit, if that begins
// here and goes on in the next `more` shares.
struct alignas(16) ChunkSplit {
    int more;   // -1: no unit
    int head, row, rows;  // KV head, the output's row of the unit's first token, rows in use
    int blank;  // rows in front that see no position
    int unused[3];
};
template <int ROWS>
__device__ __forceinline__ ChunkSplit split_of(const ChunkParams& p, const Unit& u, int more) {
    const int G = p.H / p.Hkv, per = ROWS / G, t0 = u.tile * per;
    return ChunkSplit{more, u.head, u.first + t0, min(per, u.n - t0) * G, max(u.n - u.len - t0, 0) * G, {0, 0, 0}};
}
// Partial sums of one unit in the workspace: O [rows][D], then M and l [rows].
__host__ __device__ constexpr size_t partial_floats(int rows, int d) { return (size_t)rows * (d + 2); }

struct ShareShared {
    long long scan[32], at;
    Unit start;  // the share's first unit
    int tile;    // and its first tile of that
};
// Every CTA counts for itself: a thread takes a run of sequences, then a run of
// the row tiles of the sequence that the share begins in.  sh.start and sh.tile
// may be read after the caller's next barrier.
template <int NT, int ROWS, int THREADS>
__device__ __forceinline__ Share find_share(const ChunkParams& p, ShareShared& sh) {
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const int run = (p.batch + THREADS - 1) / THREADS;
    const int s0 = min(tid * run, p.batch), s1 = min(s0 + run, p.batch);
    long long mine = 0;
    for (int s = s0; s < s1; ++s) {
        mine += tiles_of_sequence<NT, ROWS>(p, s);
        int first, n;
        rows_of(p, s, first, n);
        if (n && p.total_lens[s] > p.stride * kPageTokens) record_error(p.err, kDevBadPage);
    }
    long long incl = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl += t;
    }
    if (lane == 31) sh.scan[warp] = incl;
    __syncthreads();
    Share share;
    long long before = incl - mine;
    share.total = 0;
    for (int w = 0; w < THREADS / 32; ++w) {
        if (w < warp) before += sh.scan[w];
        share.total += sh.scan[w];
    }
    share.index = blockIdx.x;
    share.shares = min((long long)gridDim.x, share.total);  // every share has a tile
    const bool has = share.index < share.shares;
    const long long begin = has ? share.total * share.index / share.shares : 0;
    share.end = has ? share.total * (share.index + 1) / share.shares : 0;
    share.count = (int)(share.end - begin);
    if (share.count > 0 && mine > 0 && before <= begin && begin < before + mine) {
        Unit u;
        long long at = begin - before;
        for (u.s = s0; u.s + 1 < s1; ++u.s) {
            const long long here = tiles_of_sequence<NT, ROWS>(p, u.s);
            if (at < here) break;
            at -= here;
        }
        set_sequence(p, u);
        u.head = u.tile = 0;
        sh.start = u;
        sh.at = at;
    }
    __syncthreads();
    if (share.count > 0) {
        Unit u = sh.start;
        const int per = ROWS / (p.H / p.Hkv), all = (u.n + per - 1) / per, each = (all + THREADS - 1) / THREADS;
        const int t0 = min(tid * each, all), t1 = min(t0 + each, all);
        long long here = 0;
        for (u.tile = t0; u.tile < t1; ++u.tile) {
            set_tile<NT, ROWS>(p, u);
            here += (long long)u.tiles * p.Hkv;
        }
        long long upto = here;
        if (all > each) {
            for (int o = 1; o < 32; o <<= 1) {
                const long long t = __shfl_up_sync(0xffffffffu, upto, o);
                if (lane >= o) upto += t;
            }
            if (lane == 31) sh.scan[warp] = upto;
            __syncthreads();
            for (int w = 0; w < warp; ++w) upto += sh.scan[w];
        }
        long long at = sh.at - (upto - here);
        __syncthreads();
        if (here > 0 && at >= 0 && at < here) {
            for (u.tile = t0;; ++u.tile) {
                set_tile<NT, ROWS>(p, u);
                if (at < (long long)u.tiles * p.Hkv) break;
                at -= (long long)u.tiles * p.Hkv;
            }
            u.head = (int)(at / u.tiles);
            sh.start = u;
            sh.tile = (int)(at % u.tiles);
        }
    }
    return share;
}

// Row r of a unit over positions [t0, t1) in fp32 by one warp, to the output or
// to the unit's partial sums (whose weights carry 2^shift, and whose row sums are
// multiplied by sum_scale).  false: the unit has no such row.
template <int D, int ROWS>
__device__ bool row_in_fp32(const ChunkParams& p, const Unit& u, int r, int t0, int t1, float* partial, float shift,
                            float sum_scale) {
    const int G = p.H / p.Hkv, per = ROWS / G, lane = threadIdx.x & 31, token = u.tile * per + r / G;
    if (r >= per * G || token >= u.n) return false;
    const int h = u.head * G + r % G, sees = min(u.len - u.n + token + 1, u.limit);
    RowSum<D> sum;
    sum.add_range(p, p.q + (u.first + token) * p.ld_q + (size_t)h * D, rsqrtf((float)D), u.s, u.head, t0,
                  min(t1, sees));
    for (int i = 0; i < (D + 31) / 32; ++i) {
        const int dim = lane + 32 * i;
        if (dim >= D) continue;
        if (partial)
            partial[(size_t)r * D + dim] = sum.acc[i];
        else
            p.out[(u.first + token) * p.ld_out + (size_t)h * D + dim] = sees > 0 ? sum.acc[i] / sum.l : 0.0f;
    }
    if (partial && lane == 0) {
        partial[ROWS * D + r] = sum.m * 1.4426950408889634f + shift;
        partial[ROWS * (D + 1) + r] = sum.l * sum_scale;
    }
    return true;
}

// Joins the parts of the units that several shares hold.  A block takes eight rows
// of the units that begin in eight consecutive shares.  Of few parts a warp joins
// a unit's alone; of many all warps do, one unit after the other (there are then
// no more than two or three such units in eight shares).  A lane has four dims
// of kEach rows, and reads the parts with their maxima and sums side by side: what
// the call waits for here is a chain of loads (the share's record, the parts).
constexpr int kCombineThreads = 256, kCombineWarps = 8, kCombineRows = 8;
constexpr int kCombineAlone = 4;  // parts that a warp joins alone

template <int D>
struct CombineSum {
    static constexpr int kEach = D / 16;
    float top[kEach], l[kEach];
    float4 sum[kEach];
    __device__ __forceinline__ void clear() {
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            top[i] = -INFINITY;
            l[i] = 0.0f;
            sum[i] = make_float4(0, 0, 0, 0);
        }
    }
    __device__ __forceinline__ void add(int i, float m, float ll, const float4& x) {
        const float both = fmaxf(top[i], m), off = both == -INFINITY ? 0.0f : both;
        const float a = exp2f(top[i] - off), b = exp2f(m - off);
        top[i] = both;
        l[i] = l[i] * a + ll * b;
        sum[i].x = sum[i].x * a + x.x * b, sum[i].y = sum[i].y * a + x.y * b;
        sum[i].z = sum[i].z * a + x.z * b, sum[i].w = sum[i].w * a + x.w * b;
    }
};

template <int D, int ROWS>
__global__ void __launch_bounds__(kCombineThreads, 2)
    chunk_combine_kernel(ChunkParams p, const float* partials, const ChunkSplit* splits, int shares, bool wide_out,
                         float sum_scale) {
    constexpr int kGroups = ROWS / kCombineRows, kEach = CombineSum<D>::kEach, kAcross = D / 4;
    constexpr int kAtOnce = D == 128 ? 1 : D == 64 ? 2 : 4;  // parts in flight
    __shared__ float4 sums[kCombineWarps][kEach][32];
    __shared__ float tops[kCombineWarps][kCombineRows], ls[kCombineWarps][kCombineRows];
    __shared__ ChunkSplit items[kCombineWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, G = p.H / p.Hkv;
    const int share0 = (int)blockIdx.x / kGroups * kCombineWarps, r0 = (int)blockIdx.x % kGroups * kCombineRows;
    pdl_wait();
    ChunkSplit s{-1, 0, 0, 0, 0, {0, 0, 0}};
    if (share0 + warp < shares) s = splits[share0 + warp];
    if (r0 >= s.rows) s.more = -1;
    if (lane == 0) items[warp] = s;

    CombineSum<D> sum;
    const auto row_of = [&](int i) { return (lane + 32 * i) / kAcross; };
    // adds parts k0, k0 + step, ... of the unit that begins in `share`
    const auto join = [&](const ChunkSplit& t, int share, int k0, int step) {
        sum.clear();
        for (int k = k0; k <= t.more; k += kAtOnce * step) {
            float m[kAtOnce][kEach], l[kAtOnce][kEach];
            float4 x[kAtOnce][kEach];
#pragma unroll
            for (int a = 0; a < kAtOnce; ++a) {
                if (k + a * step > t.more) break;
                const float* part = partials + ((size_t)(share + k + a * step) * 2 + (k + a * step == 0)) *
                                                   partial_floats(ROWS, D);
#pragma unroll
                for (int i = 0; i < kEach; ++i) {
                    const int r = r0 + row_of(i);
                    if (r >= t.rows) continue;  // not written
                    m[a][i] = part[ROWS * D + r];
                    l[a][i] = part[ROWS * (D + 1) + r];
                    x[a][i] = *reinterpret_cast<const float4*>(part + (size_t)r * D + (lane + 32 * i) % kAcross * 4);
                }
            }
#pragma unroll
            for (int a = 0; a < kAtOnce; ++a) {
                if (k + a * step > t.more) break;
#pragma unroll
                for (int i = 0; i < kEach; ++i)
                    if (r0 + row_of(i) < t.rows) sum.add(i, m[a][i], l[a][i], x[a][i]);
            }
        }
    };
    const auto write = [&](const ChunkSplit& t, int i, float l, const float4& v) {
        const int r = r0 + row_of(i);
        if (r >= t.rows) return;
        float* dst = p.out + (t.row + r / G) * p.ld_out + (size_t)(t.head * G + r % G) * D + (lane + 32 * i) % kAcross * 4;
        const float n = sum_scale / l;  // the parts' sums are multiplied by it
        float4 y = make_float4(v.x * n, v.y * n, v.z * n, v.w * n);
        if (r < t.blank) y = make_float4(0, 0, 0, 0);  // whatever the parts hold
        if (wide_out)
            *reinterpret_cast<float4*>(dst) = y;
        else
            dst[0] = y.x, dst[1] = y.y, dst[2] = y.z, dst[3] = y.w;
    };
    if (s.more >= 0 && s.more < kCombineAlone) {
        join(s, share0 + warp, 0, 1);
#pragma unroll
        for (int i = 0; i < kEach; ++i) write(s, i, sum.l[i], sum.sum[i]);
    }
    __syncthreads();
    for (int w = 0; w < kCombineWarps; ++w) {
        const ChunkSplit t = items[w];
        if (t.more < kCombineAlone) continue;
        join(t, share0 + w, warp, kCombineWarps);
#pragma unroll
        for (int i = 0; i < kEach; ++i) {
            sums[warp][i][lane] = sum.sum[i];
            if ((lane + 32 * i) % kAcross == 0) {
                tops[warp][row_of(i)] = sum.top[i];
                ls[warp][row_of(i)] = sum.l[i];
            }
        }
        __syncthreads();
        if (warp < kEach) {
            const int r = row_of(warp);
            sum.clear();
#pragma unroll
            for (int k = 0; k < kCombineWarps; ++k) sum.add(0, tops[k][r], ls[k][r], sums[k][warp][lane]);
            write(t, warp, sum.l[0], sum.sum[0]);
        }
        __syncthreads();
    }
}

template <int D, int ROWS>
cudaError_t launch_combine(const ChunkParams& p, int shares, const float* partials, const ChunkSplit* splits,
                           bool wide_out, float sum_scale, cudaStream_t stream) {
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)((shares + kCombineWarps - 1) / kCombineWarps * (ROWS / kCombineRows)));
    cfg.blockDim = dim3(kCombineThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, chunk_combine_kernel<D, ROWS>, p, partials, splits, shares, wide_out, sum_scale);
}

}  // namespace tb
