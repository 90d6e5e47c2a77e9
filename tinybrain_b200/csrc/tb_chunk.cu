// tb_chunk.cu -- attention of each sequence's new tokens over its paged cache.
//
// Row i of a sequence with n new tokens and length L (the new ones included)
// has position p = L - n + i and attends over positions 0..p:
//     out = sum_j softmax_j(q . k_j / sqrt(d)) v_j,
// keys and values out of the page pool, the new tokens' own among them (they
// are in the cache before the call).  Query head h reads KV head h / (H/Hkv).
// Rows of an evicted page (table entry -1) are zeros, as in the decode
// attention (ModelRunner.swift:519-579 over KVCache.swift's pages).
#include <climits>

#include "tb_chunk_mma.cuh"
#include "tb_common.cuh"
#include "tb_stream_entry.h"

namespace tb {
namespace {

struct ChunkParams {
    const float* q;
    long long ld_q;
    const int* row_offsets;
    const int* total_lens;
    int batch, rows;
    const float* pool;
    int num_pages;
    const int* table;
    int stride;
    int layer, num_layers, H, Hkv;
    float* out;
    long long ld_out;
    int* err;
};

// The rows of sequence s that the call holds.
__device__ __forceinline__ void rows_of(const ChunkParams& p, int s, int& first, int& count) {
    first = min(max(p.row_offsets[s], 0), p.rows);
    count = max(min(p.row_offsets[s + 1], p.rows) - first, 0);
}

// Pool page of a position, -1 where there is none (evicted, or reported as bad).
__device__ __forceinline__ int page_at(const ChunkParams& p, int s, int pos) {
    const int page = p.table[(size_t)s * p.stride + pos / kPageTokens];
    if (page >= p.num_pages) {
        record_error(p.err, kDevBadPage);
        return -1;
    }
    return page;
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

// ---------------------------------------------------------------------------
// Tiles on the tensor cores.
//
// A unit is 128 query rows of one KV head (the G = H / Hkv query heads of
// 128 / G consecutive tokens) over the positions they see, cut into tiles of NT
// positions.  Per tile S = Q K^T and O += P V are three fp16 products each
// (tb_chunk_mma.cuh), Q and P from tensor memory, K and V from shared memory.
//
// One CTA per SM walks an equal share of all units' tiles (a share may begin
// and end inside a unit), so a ragged batch, one long sequence and a large
// prompt all load the SMs evenly without a plan made on the host.  A unit that
// several CTAs hold leaves partial sums in the workspace; chunk_combine_kernel
// adds them in the order of the CTAs.
//
// Roles (14 warps of 16):
//   producer   one lane per page of a tile: page table, then a bulk copy of the
//              page's K or V rows of this head into a ring of fp32 pages;
//   converters (8 warps) one page at a time: the page's largest magnitude gives
//              a power-of-two scale, the halves go to the K and V operand rings;
//   issuer     one thread: S(i + 1) before P V(i), so the softmax of a tile runs
//              while the tensor cores do the next S and the last P V;
//   softmax    (4 warps, a row a thread) base-2 softmax over the tile, P as
//              halves over S in tensor memory, and the last tile's P V added to
//              the row's sums in registers, which are rescaled only where the
//              running maximum grew by more than 2^8.
//
// With c the row's scale times the page's, a score is c S and a weighted value
// 2^(c S - M) v = 2^(c S + e - M) (v 2^-e): the page's value exponent e enters
// the exponent of P, and its inverse the row sum.  P of the largest term is
// thus always near the top of fp16's range, and a page's precision does not
// depend on the sizes of other pages.  Pages with values of 2^20 and more or
// that are not finite have no such operands (one of them may be masked for some
// rows of the tile), nor have scores beyond 2^20: the unit's rows are then summed
// in fp32 on the CUDA cores.
// ---------------------------------------------------------------------------
constexpr int kSoftmaxWarps = 4, kConvertWarps = 8;
constexpr int kIssueWarp = kSoftmaxWarps + kConvertWarps, kLoadWarp = kIssueWarp + 1;
constexpr int kChunkThreads = 512;  // four warpgroups, the last one with two idle warps
// registers of a thread: 128 at launch, then the softmax warpgroup (a tile's
// row of S and the row's sums) takes what the other three leave
constexpr int kLaunchRegs = 128, kSoftmaxRegs = 224, kOtherRegs = 96;
static_assert(kSoftmaxRegs + 3 * kOtherRegs == 4 * kLaunchRegs, "registers");
constexpr int kChunkCtas = 148;   // most CTAs of a launch (the workspace's size)
constexpr int kTileRows = 128;
constexpr int kStages = 2;        // K and V operand tiles each
constexpr int kScaleRing = 4;     // tiles whose page scales are kept
constexpr uint32_t kWildBits = (127u + 20u) << 23;    // a K or V value of 2^20
constexpr uint32_t kWildQueryBits = (127u + 40u) << 23;
constexpr float kPShift = 6.0f;   // P = 2^(6 + score - M), M within 2^8 of the maximum: at most 2^14
constexpr float kLazy = 8.0f;
constexpr float kWildMark = 3e38f;
constexpr float kHuge = 1048576.0f;  // a score whose rounding could carry P out of fp16's range

template <int D>
struct Shape {
    static constexpr int NT = D == 128 ? 64 : 128;     // positions of a tile
    static constexpr int PG = NT / kPageTokens;        // its pages
    static constexpr int kPageBytes = kPageTokens * D * 4;
    static constexpr int kHalf = NT * D * 2;           // bytes of one operand half
    static constexpr int kSlots = D == 128 ? 12 : D == 64 ? 24 : 32;
    static constexpr size_t kSmem = (size_t)kStages * 4 * kHalf + (size_t)kSlots * kPageBytes;
    // tensor memory columns
    static constexpr int kS = 0, kO = 2 * NT, kQ = kO + 2 * D;  // S / P and O twice
    static_assert(kQ + D <= 512, "tensor memory");
};

struct Unit {
    int s, tile, head;
    int first, n, len;  // the sequence's first row, rows and length
    int limit;          // positions that the unit's last row sees
    int tiles;          // of NT positions, at least one
};

struct ChunkBars {
    uint64_t slot_full[32], slot_empty[32];
    uint64_t k_full[kStages], k_empty[kStages], v_full[kStages], v_empty[kStages];
    uint64_t scales[kScaleRing];
    uint64_t s_full[2], p_full[2];
    uint64_t pv_done[2], q_full, drained;
};

__device__ __forceinline__ int tokens_of_tile(int G) { return kTileRows / G; }

template <int D>
__device__ __forceinline__ void set_tile(const ChunkParams& p, Unit& u) {
    const int per = tokens_of_tile(p.H / p.Hkv);
    const int last = min((u.tile + 1) * per, u.n) - 1;
    u.limit = min(max(u.len - u.n + last + 1, 0), p.stride * kPageTokens);
    u.tiles = max(1, (u.limit + Shape<D>::NT - 1) / Shape<D>::NT);
}
__device__ __forceinline__ void set_sequence(const ChunkParams& p, Unit& u) {
    rows_of(p, u.s, u.first, u.n);
    u.len = p.total_lens[u.s];
}
template <int D>
__device__ __forceinline__ void next_unit(const ChunkParams& p, Unit& u) {
    if (++u.head < p.Hkv) return;
    u.head = 0;
    ++u.tile;
    if (u.tile * tokens_of_tile(p.H / p.Hkv) >= u.n) {
        u.tile = 0;
        do {
            ++u.s;
            set_sequence(p, u);
        } while (u.n == 0 && u.s + 1 < p.batch);
    }
    set_tile<D>(p, u);
}
// Tiles of all units of a sequence.
template <int D>
__device__ __forceinline__ long long tiles_of_sequence(const ChunkParams& p, int s) {
    Unit u;
    u.s = s;
    set_sequence(p, u);
    long long sum = 0;
    for (u.tile = 0; u.tile * tokens_of_tile(p.H / p.Hkv) < u.n; ++u.tile) {
        set_tile<D>(p, u);
        sum += u.tiles;
    }
    return sum * p.Hkv;
}

// What a CTA leaves for chunk_combine_kernel: its last unit, if that begins
// here and goes on in the next `more` CTAs.
struct ChunkSplit {
    int s, tile, head, more;
};
// Partial sums of one unit in the workspace: O [128][D], then M and l [128].
template <int D>
struct Partial {
    static constexpr size_t kFloats = (size_t)kTileRows * (D + 2);
};

struct ChunkShared {
    ChunkBars bars;
    float k_scale[kScaleRing][8], v_exp[kScaleRing][8];
    int slot_page[32];
    Unit start;
    int start_tile;
    long long total, ctas, begin, end;
    long long scan[kChunkThreads / 32];
    uint32_t tmem;
    volatile int dead;  // a wait ran out: nobody waits any more
};

__device__ __forceinline__ bool chunk_wait(ChunkShared& sh, uint64_t* bar, uint32_t parity, int* err) {
    if (mbar_try_wait(bar, parity)) return true;
    const uint64_t t0 = global_timer_ns();
    while (!sh.dead) {
        if (mbar_try_wait(bar, parity)) return true;
        if (global_timer_ns() - t0 > kWaitLimitNs) {
            record_error(err, kDevWaitTimeout);
            sh.dead = 1;
        }
    }
    return false;
}
__device__ __forceinline__ void warp_wait(ChunkShared& sh, uint64_t* bar, uint32_t parity, int* err) {
    if ((threadIdx.x & 31) == 0) chunk_wait(sh, bar, parity, err);
    __syncwarp();
}

// Largest magnitude of the warp's values, as bits.
__device__ __forceinline__ uint32_t warp_max_bits(uint32_t m) { return __reduce_max_sync(0xffffffffu, m); }

// K page -> rows `page * 16 ..` of the K operand.  A lane takes 8 consecutive
// dims of a token; the dims are staggered over the tokens so that eight lanes'
// reads (rows of D floats) and writes (16-byte rows of a core matrix) both fall
// into different banks.
template <int D>
__device__ __forceinline__ void convert_k(const float* src, int valid, uint8_t* hi, uint8_t* lo, int page,
                                          float* scale_out) {
    constexpr int C = D / 8, kTasks = C / 2;
    const int lane = threadIdx.x & 31, l7 = lane & 7, swap = (lane >> 2) & 1;
    const int r = l7 + 8 * ((lane >> 3) & 1), c0 = l7 + (lane >> 4) * kTasks;
    float4 x[kTasks][2];
    uint32_t m = 0;
#pragma unroll
    for (int t = 0; t < kTasks; ++t) {
        const float* at = src + r * D + ((c0 + t) % C) * 8;
        float4 a = make_float4(0, 0, 0, 0), b = a;
        if (r < valid) {
            a = lds128f(at + 4 * swap);
            b = lds128f(at + 4 * (swap ^ 1));
        }
        x[t][0] = swap ? b : a;
        x[t][1] = swap ? a : b;
#pragma unroll
        for (int h = 0; h < 2; ++h)
            m = max(max(m, max(abs_bits(x[t][h].x), abs_bits(x[t][h].y))),
                    max(abs_bits(x[t][h].z), abs_bits(x[t][h].w)));
    }
    m = warp_max_bits(m);
    const int e = block_exponent(m);
    const float s = exp2_int(-e);
    if (lane == 0) *scale_out = m >= kWildBits ? kWildMark : exp2_int(e);
#pragma unroll
    for (int t = 0; t < kTasks; ++t) {
        uint4 h, l;
        split_pair(x[t][0].x * s, x[t][0].y * s, h.x, l.x);
        split_pair(x[t][0].z * s, x[t][0].w * s, h.y, l.y);
        split_pair(x[t][1].x * s, x[t][1].y * s, h.z, l.z);
        split_pair(x[t][1].z * s, x[t][1].w * s, h.w, l.w);
        const int row = page * kPageTokens + r, at = (row >> 3) * (C * 128) + ((c0 + t) % C) * 128 + (row & 7) * 16;
        *reinterpret_cast<uint4*>(hi + at) = h;
        *reinterpret_cast<uint4*>(lo + at) = l;
    }
}

// V page -> columns (k) `page * 16 ..` of the V^T operand: a lane takes 8
// consecutive tokens of a dim.
template <int D>
__device__ __forceinline__ void convert_v(const float* src, int valid, uint8_t* hi, uint8_t* lo, int page,
                                          float* exp_out) {
    constexpr int NT = Shape<D>::NT, kTasks = D / 16;
    const int lane = threadIdx.x & 31;
    float x[kTasks][8];
    uint32_t m = 0;
#pragma unroll
    for (int t = 0; t < kTasks; ++t) {
        const int task = lane + 32 * t, n = task % D, kc = task / D;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            x[t][j] = kc * 8 + j < valid ? src[(kc * 8 + j) * D + n] : 0.0f;
            m = max(m, abs_bits(x[t][j]));
        }
    }
    m = warp_max_bits(m);
    const int e = block_exponent(m);
    const float s = exp2_int(-e);
    if (lane == 0) *exp_out = m >= kWildBits ? kWildMark : (float)e;
#pragma unroll
    for (int t = 0; t < kTasks; ++t) {
        const int task = lane + 32 * t, n = task % D, kc = task / D;
        uint4 h, l;
        split_pair(x[t][0] * s, x[t][1] * s, h.x, l.x);
        split_pair(x[t][2] * s, x[t][3] * s, h.y, l.y);
        split_pair(x[t][4] * s, x[t][5] * s, h.z, l.z);
        split_pair(x[t][6] * s, x[t][7] * s, h.w, l.w);
        const int at = (n >> 3) * (NT * 16) + (page * 2 + kc) * 128 + (n & 7) * 16;
        *reinterpret_cast<uint4*>(hi + at) = h;
        *reinterpret_cast<uint4*>(lo + at) = l;
    }
}

template <int D>
__device__ __forceinline__ void load_row4(const float* q, bool wide, int i, float (&x)[4]) {
    if (wide) {
        const float4 f = *reinterpret_cast<const float4*>(q + i);
        x[0] = f.x, x[1] = f.y, x[2] = f.z, x[3] = f.w;
    } else {
        x[0] = q[i], x[1] = q[i + 1], x[2] = q[i + 2], x[3] = q[i + 3];
    }
}

// The unit's query rows as halves in tensor memory; the thread's row factor
// (2^e log2(e) / sqrt(D)) is the result, negative for a row without operands.
template <int D>
__device__ __forceinline__ float load_queries(const ChunkParams& p, const float* q, bool valid, bool wide,
                                              uint32_t tq) {
    uint32_t m = 0;
    if (valid)
        for (int i = 0; i < D; i += 4) {
            float x[4];
            load_row4<D>(q, wide, i, x);
            m = max(max(m, max(abs_bits(x[0]), abs_bits(x[1]))), max(abs_bits(x[2]), abs_bits(x[3])));
        }
    const int e = m < kWildQueryBits ? block_exponent(m) : 0;
    const float s = exp2_int(-e);
    constexpr int W = D < 32 ? D : 32;
#pragma unroll 1
    for (int i = 0; i < D; i += W) {
        uint32_t hi[W / 2], lo[W / 2];
#pragma unroll
        for (int j = 0; j < W; j += 4) {
            float x[4] = {0, 0, 0, 0};
            if (valid && m < kWildQueryBits) load_row4<D>(q, wide, i + j, x);
            split_pair(x[0] * s, x[1] * s, hi[j / 2], lo[j / 2]);
            split_pair(x[2] * s, x[3] * s, hi[j / 2 + 1], lo[j / 2 + 1]);
        }
        if constexpr (W == 32) {
            tmem_st16(tq + i / 2, hi);
            tmem_st16(tq + D / 2 + i / 2, lo);
        } else {
            tmem_st8(tq + i / 2, hi);
            tmem_st8(tq + D / 2 + i / 2, lo);
        }
    }
    return m < kWildQueryBits ? exp2_int(e) * (1.4426950408889634f * rsqrtf((float)D)) : -1.0f;
}

// A unit's rows of one warp in fp32 (pages or queries without fp16 operands).
template <int D>
__device__ __noinline__ void rows_without_operands(const ChunkParams& p, const Unit& u, int t0, int t1, float* partial) {
    const int G = p.H / p.Hkv, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int r = warp * 32; r < warp * 32 + 32; ++r) {
        const int token = u.tile * tokens_of_tile(G) + r / G;
        if (r >= tokens_of_tile(G) * G || token >= u.n) break;
        const int h = u.head * G + r % G;
        const int sees = min(u.len - u.n + token + 1, u.limit);
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
            partial[kTileRows * D + r] = sum.m * 1.4426950408889634f + kPShift;
            partial[kTileRows * (D + 1) + r] = sum.l;
        }
    }
}

template <int D>
__global__ void __launch_bounds__(kChunkThreads, 1) chunk_tiles_kernel(ChunkParams p, float* partials,
                                                                        ChunkSplit* splits, bool wide_q, bool wide_out) {
    using S = Shape<D>;
    constexpr int NT = S::NT, PG = S::PG;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ ChunkShared sh;
    static_assert(S::kSmem + sizeof(ChunkShared) <= 227 * 1024, "shared memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t* k_ops = smem;                                // [stage][hi, lo]
    uint8_t* v_ops = smem + kStages * 2 * S::kHalf;
    uint8_t* pages = smem + kStages * 4 * S::kHalf;
    ChunkBars& b = sh.bars;

    // the CTA's share: tiles [total c / C, total (c + 1) / C) of all units' tiles
    long long sum = 0;
    for (int s = tid; s < p.batch; s += kChunkThreads) {
        sum += tiles_of_sequence<D>(p, s);
        int first, n;
        rows_of(p, s, first, n);
        if (n && p.total_lens[s] > p.stride * kPageTokens) record_error(p.err, kDevBadPage);
    }
    for (int o = 16; o; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
    if (lane == 0) sh.scan[warp] = sum;
    if (tid == 0) {
        sh.dead = 0;
        for (int i = 0; i < S::kSlots; ++i) {
            mbar_init(b.slot_full + i, 1);
            mbar_init(b.slot_empty + i, 1);
        }
        for (int i = 0; i < kStages; ++i) {
            mbar_init(b.k_full + i, PG);
            mbar_init(b.v_full + i, PG);
            mbar_init(b.k_empty + i, 1);
            mbar_init(b.v_empty + i, 1);
        }
        for (int i = 0; i < kScaleRing; ++i) mbar_init(b.scales + i, 2 * PG);
        for (int i = 0; i < 2; ++i) {
            mbar_init(b.s_full + i, 1);
            mbar_init(b.p_full + i, kSoftmaxWarps);
            mbar_init(b.pv_done + i, 1);
        }
        mbar_init(&b.drained, 1);
        mbar_init(&b.q_full, kSoftmaxWarps);
        fence_barrier_init();
        fence_proxy_async_shared();
    }
    __syncthreads();
    if (tid == 0) {
        long long total = 0;
        for (int w = 0; w < kChunkThreads / 32; ++w) total += sh.scan[w];
        const long long c = blockIdx.x, ctas = min((long long)gridDim.x, total);  // every share has a tile
        sh.total = total;
        sh.ctas = ctas;
        sh.begin = c < ctas ? total * c / ctas : 0;
        sh.end = c < ctas ? total * (c + 1) / ctas : 0;
        sh.start.s = -1;
    }
    __syncthreads();
    const long long begin = sh.begin, count = sh.end - begin;
    if (count > 0) {
        long long carry = 0;
        for (int base = 0; base < p.batch; base += kChunkThreads) {
            const int s = base + tid;
            const long long mine = s < p.batch ? tiles_of_sequence<D>(p, s) : 0;
            long long incl = mine;
            for (int o = 1; o < 32; o <<= 1) {
                const long long t = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += t;
            }
            __syncthreads();
            if (lane == 31) sh.scan[warp] = incl;
            __syncthreads();
            long long before = carry + incl - mine;
            for (int w = 0; w < kChunkThreads / 32; ++w) {
                if (w < warp) before += sh.scan[w];
                carry += sh.scan[w];
            }
            if (mine > 0 && before <= begin && begin < before + mine) {
                Unit u;
                u.s = s;
                u.head = 0;
                set_sequence(p, u);
                long long at = begin - before;
                for (u.tile = 0;; ++u.tile) {
                    set_tile<D>(p, u);
                    if (at < (long long)u.tiles * p.Hkv) break;
                    at -= (long long)u.tiles * p.Hkv;
                }
                u.head = (int)(at / u.tiles);
                sh.start = u;
                sh.start_tile = (int)(at % u.tiles);
            }
            if (carry > begin) break;
        }
    }
    if (warp == kIssueWarp) tmem_alloc(&sh.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = sh.tmem;
    Unit u = sh.start;
    int at = sh.start_tile;

    // (a warpgroup's warps all move the same way, each in its own role)
    if (count > 0 && warp == kLoadWarp) {
        // ---- producer ----
        set_registers_down<kOtherRegs>();
        long long job0 = 0;
        for (long long left = count; left > 0 && !sh.dead; at = 0) {
            const int take = (int)min((long long)(u.tiles - at), left);
            for (int j = at; j < at + take; ++j, job0 += 2 * PG) {
                if (lane < 2 * PG) {
                    const int kv = lane / PG, pos = j * NT + (lane % PG) * kPageTokens;
                    const int page = pos < u.limit ? page_at(p, u.s, pos) : -1;
                    const long long job = job0 + lane;
                    const int slot = (int)(job % S::kSlots);
                    if (chunk_wait(sh, b.slot_empty + slot, (uint32_t)(job / S::kSlots & 1) ^ 1, p.err)) {
                        sh.slot_page[slot] = page;
                        if (page >= 0) {
                            mbar_arrive_expect_tx(b.slot_full + slot, S::kPageBytes);
                            bulk_g2s(pages + slot * S::kPageBytes, head_rows<D>(p, page, kv, u.head), S::kPageBytes,
                                     b.slot_full + slot);
                        } else {
                            mbar_arrive(b.slot_full + slot);
                        }
                    }
                }
                __syncwarp();
            }
            left -= take;
            if (left > 0) next_unit<D>(p, u);
        }
        if (sh.dead) {  // copies still in flight must land before the CTA ends
            const uint64_t t0 = global_timer_ns();
            for (int s = lane; s < S::kSlots; s += 32) {
                // the slot's last fill, counted in jobs
                const long long fills = (job0 - 1 - s >= 0) ? (job0 - 1 - s) / S::kSlots + 1 : 0;
                while (fills && !mbar_try_wait(b.slot_full + s, (uint32_t)(fills - 1) & 1) &&
                       global_timer_ns() - t0 < kWaitLimitNs) {
                }
            }
        }
    } else if (count > 0 && warp == kIssueWarp) {
        // ---- issuer ----
        set_registers_down<kOtherRegs>();
        if (lane == 0) {
            const uint32_t k0 = smem_u32(k_ops), v0 = smem_u32(v_ops);
            long long i = 0, unit = 0;
            const auto issue_s = [&](long long item, bool first, long long un) {
                const int st = (int)(item % kStages);
                if (first) chunk_wait(sh, &b.q_full, (uint32_t)(un & 1), p.err);
                chunk_wait(sh, b.k_full + st, (uint32_t)(item / kStages & 1), p.err);
                tc_fence_after();
                const uint32_t kb = k0 + st * 2 * S::kHalf;
                tc_mma_split<NT, D>(tmem + S::kS + (uint32_t)(item & 1) * NT, tmem + S::kQ,
                                    [](int s) { return 8 * s; }, D / 2, kb, kb + S::kHalf);
                tc_commit(b.s_full + (item & 1));
                tc_commit(b.k_empty + st);
            };
            for (long long left = count; left > 0; at = 0) {
                const int take = (int)min((long long)(u.tiles - at), left);
                issue_s(i, true, unit);
                for (int j = 0; j < take; ++j, ++i) {
                    if (j + 1 < take) issue_s(i + 1, false, unit);
                    const int st = (int)(i % kStages);
                    chunk_wait(sh, b.v_full + st, (uint32_t)(i / kStages & 1), p.err);
                    chunk_wait(sh, b.p_full + (i & 1), (uint32_t)(i / 2 & 1), p.err);
                    tc_fence_after();
                    const uint32_t vb = v0 + st * 2 * S::kHalf;
                    // P: 16 columns of high, 16 of low halves per 32 positions.  O of two
                    // tiles before was read before P of this one arrived.
                    tc_mma_split<D, NT>(tmem + S::kO + (uint32_t)(i & 1) * D, tmem + S::kS + (uint32_t)(i & 1) * NT,
                                        [](int s) { return 32 * (s / 2) + 8 * (s % 2); }, 16, vb, vb + S::kHalf);
                    tc_commit(b.v_empty + st);
                    tc_commit(b.pv_done + (i & 1));
                }
                left -= take;
                ++unit;
                if (left > 0) next_unit<D>(p, u);
            }
            // every product has been read and written before tensor memory goes
            tc_commit(&b.drained);
            const uint64_t t0 = global_timer_ns();
            while (!mbar_try_wait(&b.drained, 0) && global_timer_ns() - t0 < kWaitLimitNs) {
            }
        }
        __syncwarp();
    } else if (count > 0 && warp >= kSoftmaxWarps && warp < kIssueWarp) {
        // ---- converters ----
        set_registers_down<kOtherRegs>();
        const int cw = warp - kSoftmaxWarps;
        long long i = 0;
        for (long long left = count; left > 0; at = 0) {
            const int take = (int)min((long long)(u.tiles - at), left);
            for (int j = at; j < at + take; ++j, ++i) {
                const int st = (int)(i % kStages), ring = (int)(i % kScaleRing);
                for (int jj = cw; jj < 2 * PG; jj += kConvertWarps) {
                    const bool is_v = jj >= PG;
                    const int page = jj % PG;
                    const long long job = i * (2 * PG) + jj;
                    const int slot = (int)(job % S::kSlots);
                    warp_wait(sh, b.slot_full + slot, (uint32_t)(job / S::kSlots & 1), p.err);
                    const int left_here = u.limit - (j * NT + page * kPageTokens);
                    const int valid = sh.slot_page[slot] < 0 ? 0 : max(0, min(left_here, kPageTokens));
                    warp_wait(sh, (is_v ? b.v_empty : b.k_empty) + st, (uint32_t)(i / kStages & 1) ^ 1, p.err);
                    const float* src = reinterpret_cast<const float*>(pages + slot * S::kPageBytes);
                    uint8_t* op = (is_v ? v_ops : k_ops) + st * 2 * S::kHalf;
                    if (is_v)
                        convert_v<D>(src, valid, op, op + S::kHalf, page, &sh.v_exp[ring][page]);
                    else
                        convert_k<D>(src, valid, op, op + S::kHalf, page, &sh.k_scale[ring][page]);
                    fence_proxy_async_shared();
                    __syncwarp();
                    if (lane == 0) {
                        mbar_arrive((is_v ? b.v_full : b.k_full) + st);
                        mbar_arrive(b.slot_empty + slot);
                        mbar_arrive(b.scales + ring);
                    }
                }
            }
            left -= take;
            if (left > 0) next_unit<D>(p, u);
        }
    } else if (count > 0 && warp < kSoftmaxWarps) {
        // ---- softmax ----
        set_registers_up<kSoftmaxRegs>();
        const uint32_t lanes = (uint32_t)(warp * 32) << 16;
        const int G = p.H / p.Hkv, per = tokens_of_tile(G);
        const int row = tid, tok = row / G, sub = row % G;
        long long i = 0;
        ChunkSplit split{0, 0, 0, -1};
        const auto queries = [&](const Unit& w) {
            const int token = w.tile * per + tok;
            const bool valid = row < per * G && token < w.n;
            float f = 1.0f;
            if (__any_sync(0xffffffffu, valid)) {
                f = load_queries<D>(p, p.q + (w.first + (valid ? token : 0)) * p.ld_q + (size_t)(w.head * G + sub) * D, valid,
                                    wide_q, tmem + S::kQ + lanes);
                tmem_st_wait();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(&b.q_full);
            return f;
        };
        float c = queries(u);
        for (long long left = count; left > 0;) {
            const int take = (int)min((long long)(u.tiles - at), left);
            const int token = u.tile * per + tok;
            const bool valid = row < per * G && token < u.n;
            const bool busy = __any_sync(0xffffffffu, valid);
            const int sees = min(u.len - u.n + token + 1, u.limit);  // the row's own limit, may be <= 0
            const int first_sees = __shfl_sync(0xffffffffu, sees, 0);  // tokens ascend with the lanes
            bool wild = __any_sync(0xffffffffu, valid && c < 0.0f);
            bool huge = false;
            float M = -INFINITY, l = 0.0f;
            float2 acc[D / 2];
#pragma unroll
            for (int x = 0; x < D / 2; ++x) acc[x] = make_float2(0.0f, 0.0f);
            // adds P V of tile `item`, whose scale the sums still have
            const auto collect = [&](long long item) {
                warp_wait(sh, b.pv_done + (item & 1), (uint32_t)(item / 2 & 1), p.err);
                tc_fence_after();
                const uint32_t to = tmem + S::kO + (uint32_t)(item & 1) * D + lanes;
                if constexpr (D == 16) {
                    int v[16];
                    tmem_ld16(to, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        acc[x] = __fadd2_rn(acc[x], make_float2(__int_as_float(v[2 * x]), __int_as_float(v[2 * x + 1])));
                } else {
#pragma unroll
                    for (int o = 0; o < D; o += 32) {
                        int v[32];
                        tmem_ld32(to + o, v);
                        tmem_ld_wait();
#pragma unroll
                        for (int x = 0; x < 16; ++x)
                            acc[o / 2 + x] = __fadd2_rn(acc[o / 2 + x], make_float2(__int_as_float(v[2 * x]),
                                                                                     __int_as_float(v[2 * x + 1])));
                    }
                }
            };
            for (int j = at; j < at + take; ++j, ++i) {
                const uint32_t ts = tmem + S::kS + (uint32_t)(i & 1) * NT + lanes;
                const int ring = (int)(i % kScaleRing);
                warp_wait(sh, b.scales + ring, (uint32_t)(i / kScaleRing & 1), p.err);
                warp_wait(sh, b.s_full + (i & 1), (uint32_t)(i / 2 & 1), p.err);
                tc_fence_after();
                float r = 1.0f;
                if (busy) {
                    const float *ks = sh.k_scale[ring], *ve = sh.v_exp[ring];
                    int v[NT / 32][32];
#pragma unroll
                    for (int g = 0; g < NT / 32; ++g) tmem_ld32(ts + 32 * g, v[g]);
                    tmem_ld_wait();
                    if (first_sees < (j + 1) * NT) {  // some row does not see all of the tile
                        const int room = sees - j * NT;
#pragma unroll
                        for (int x = 0; x < NT; ++x)
                            if (x >= room) v[x / 32][x % 32] = __float_as_int(-INFINITY);
                    }
                    // the row's maximum of score + value exponent: per page the largest S decides
                    float top = -INFINITY;
#pragma unroll
                    for (int g = 0; g < PG; ++g) {
                        float m0 = __int_as_float(v[g / 2][g % 2 * 16]), m1 = __int_as_float(v[g / 2][g % 2 * 16 + 1]);
#pragma unroll
                        for (int x = 2; x < 16; x += 2) {
                            m0 = fmaxf(m0, __int_as_float(v[g / 2][g % 2 * 16 + x]));
                            m1 = fmaxf(m1, __int_as_float(v[g / 2][g % 2 * 16 + x + 1]));
                        }
                        wild |= ks[g] == kWildMark || ve[g] == kWildMark;
                        top = fmaxf(top, fmaf(fmaxf(m0, m1), c * ks[g], ve[g]));
                    }
                    huge |= valid && top > -INFINITY && fabsf(top) > kHuge;
                    if (top > M + kLazy || (M == -INFINITY && top > -INFINITY)) {
                        r = M == -INFINITY ? 0.0f : ex2(M - top);
                        M = top;
                        l *= r;
                    }
                    const float shift = kPShift - (M == -INFINITY ? 0.0f : M);
#pragma unroll
                    for (int g = 0; g < NT / 32; ++g) {
                        uint32_t hi[16], lo[16];
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            const float e = ve[2 * g + h];
                            const float2 kk = make_float2(c * ks[2 * g + h], c * ks[2 * g + h]);
                            const float2 bb = make_float2(e + shift, e + shift);
                            float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                            for (int x = 16 * h; x < 16 * h + 16; x += 2) {
                                const float2 t = __ffma2_rn(
                                    make_float2(__int_as_float(v[g][x]), __int_as_float(v[g][x + 1])), kk, bb);
                                const float2 w = make_float2(ex2(t.x), ex2(t.y));
                                sum = __fadd2_rn(sum, w);
                                split_pair(w.x, w.y, hi[x / 2], lo[x / 2]);
                            }
                            l = fmaf(sum.x + sum.y, ex2(-e), l);
                        }
                        tmem_st16(ts + 32 * g, hi);
                        tmem_st16(ts + 32 * g + 16, lo);
                    }
                    tmem_st_wait();
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(b.p_full + (i & 1));
                if (busy) {
                    if (j > at) collect(i - 1);
                    if (__any_sync(0xffffffffu, r != 1.0f)) {
#pragma unroll
                        for (int x = 0; x < D / 2; ++x) acc[x] = __fmul2_rn(acc[x], make_float2(r, r));
                    }
                }
            }
            const Unit done = u;
            const int from = at;
            left -= take;
            if (left > 0) {  // the next unit's queries, while the last products run
                next_unit<D>(p, u);
                c = queries(u);
            }
            const bool whole = from == 0 && take == done.tiles;
            float* part = nullptr;
            if (!whole) {
                part = partials + ((size_t)blockIdx.x * 2 + (from == 0)) * Partial<D>::kFloats;
                if (from == 0) {  // goes on in the next CTAs: up to the one that holds its last tile
                    const long long last = sh.end + (done.tiles - take) - 1;
                    int more = 0;
                    while (sh.total * (blockIdx.x + more + 2) / sh.ctas <= last) ++more;
                    split = ChunkSplit{done.s, done.tile, done.head, more + 1};
                }
            }
            if (busy) collect(i - 1);
            wild |= __any_sync(0xffffffffu, huge);
            if (valid && !wild) {
                float* dst = part ? part + (size_t)row * D
                                  : p.out + (done.first + token) * p.ld_out + (size_t)(done.head * G + sub) * D;
                const float inv = part ? 1.0f : sees > 0 ? 1.0f / l : 0.0f;
                if (part || wide_out) {
#pragma unroll
                    for (int x = 0; x < D / 2; x += 2)
                        *reinterpret_cast<float4*>(dst + 2 * x) = make_float4(acc[x].x * inv, acc[x].y * inv,
                                                                              acc[x + 1].x * inv, acc[x + 1].y * inv);
                } else {
#pragma unroll
                    for (int x = 0; x < D / 2; ++x) {
                        dst[2 * x] = acc[x].x * inv;
                        dst[2 * x + 1] = acc[x].y * inv;
                    }
                }
                if (part) {
                    part[kTileRows * D + row] = M;
                    part[kTileRows * (D + 1) + row] = l;
                }
            }
            if (busy && wild) rows_without_operands<D>(p, done, from * NT, (from + take) * NT, part);
            at = 0;
        }
        if (tid == 0) splits[blockIdx.x] = split;
    } else if (count > 0) {
        set_registers_down<kOtherRegs>();
    } else if (tid == 0) {
        splits[blockIdx.x] = ChunkSplit{0, 0, 0, -1};
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kIssueWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Block c: the unit that begins in CTA c and goes on in the next ones.
constexpr int kCombineThreads = 256;
template <int D>
__global__ void __launch_bounds__(kCombineThreads) chunk_combine_kernel(ChunkParams p, const float* partials,
                                                                         const ChunkSplit* splits) {
    pdl_wait();
    const ChunkSplit s = splits[blockIdx.x];
    if (s.more < 0) return;
    Unit u;
    u.s = s.s, u.tile = s.tile, u.head = s.head;
    set_sequence(p, u);
    set_tile<D>(p, u);
    const int G = p.H / p.Hkv, per = tokens_of_tile(G);
    const int rows = min(per, u.n - u.tile * per) * G;
    const auto part = [&](int k) {
        return partials + ((size_t)(blockIdx.x + k) * 2 + (k == 0)) * Partial<D>::kFloats;
    };
    for (int e = threadIdx.x; e < rows * D; e += kCombineThreads) {
        const int row = e / D, token = u.tile * per + row / G;
        float top = -INFINITY;
        for (int k = 0; k <= s.more; ++k) top = fmaxf(top, part(k)[kTileRows * D + row]);
        const float off = top == -INFINITY ? 0.0f : top;
        float o = 0.0f, l = 0.0f;
        for (int k = 0; k <= s.more; ++k) {
            const float* x = part(k);
            const float w = exp2f(x[kTileRows * D + row] - off);
            o = fmaf(w, x[e], o);
            l = fmaf(w, x[kTileRows * (D + 1) + row], l);
        }
        p.out[(u.first + token) * p.ld_out + (size_t)(u.head * G + row % G) * D + e % D] =
            u.len - u.n + token >= 0 ? o / l : 0.0f;
    }
}

// CTAs of a launch: one per tile of work that the caller's bounds allow, at
// most one per SM.
int chunk_ctas(long long rows, long long batch, long long max_new, long long max_len, int H, int Hkv, int d) {
    const long long G = H / Hkv, per = kTileRows / G, nt = d == 128 ? 64 : 128;
    const long long units = std::min(batch * ((std::min(max_new, rows) + per - 1) / per), batch + rows / per) * Hkv;
    const long long tiles = units * ((max_len + nt - 1) / nt);
    return (int)std::max<long long>(1, std::min<long long>(tiles, kChunkCtas));
}
size_t chunk_workspace(int ctas, int d) {
    return (size_t)ctas * (2 * (size_t)kTileRows * (d + 2) * sizeof(float) + sizeof(ChunkSplit));
}

template <int D>
cudaError_t launch_chunk(const ChunkParams& p, int ctas, void* workspace, cudaStream_t stream) {
    float* partials = static_cast<float*>(workspace);
    ChunkSplit* splits = reinterpret_cast<ChunkSplit*>(partials + (size_t)ctas * 2 * Partial<D>::kFloats);
    const bool wide_q = p.ld_q % 4 == 0 && aligned_to(p.q, 16), wide_out = p.ld_out % 4 == 0 && aligned_to(p.out, 16);
    cudaError_t e = cudaFuncSetAttribute(chunk_tiles_kernel<D>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                         (int)Shape<D>::kSmem);
    if (e != cudaSuccess) return e;
    // setmaxnreg moves registers within what the CTA was launched with: with
    // fewer than planned the softmax warps would wait for them
    cudaFuncAttributes attr_regs{};
    e = cudaFuncGetAttributes(&attr_regs, chunk_tiles_kernel<D>);
    if (e != cudaSuccess) return e;
    if (attr_regs.numRegs != kLaunchRegs) return cudaErrorNotSupported;
    chunk_tiles_kernel<D><<<ctas, kChunkThreads, Shape<D>::kSmem, stream>>>(p, partials, splits, wide_q, wide_out);
    e = cudaGetLastError();
    if (e != cudaSuccess) return e;
    cudaLaunchConfig_t cfg{};
    cfg.gridDim = dim3((unsigned)ctas);
    cfg.blockDim = dim3(kCombineThreads);
    cfg.stream = stream;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, chunk_combine_kernel<D>, p, (const float*)partials, (const ChunkSplit*)splits);
}

}  // namespace
}  // namespace tb

using namespace tb;

static tb_status check_chunk(int rows, int batch, int max_new, int max_len, int H, int Hkv, int d) {
    TB_ENTRY_CHECK(rows >= 0 && batch >= 1 && max_new >= 1 && max_len >= 1, "bad rows / batch / lengths");
    TB_ENTRY_CHECK(H >= 1 && Hkv >= 1 && H % Hkv == 0, "heads must divide: H %d, Hkv %d", H, Hkv);
    if ((d != 16 && d != 32 && d != 64 && d != 128) || H / Hkv > kTileRows)
        return (tb_status)report_error(TB_ERR_UNSUPPORTED,
                                       "head dimension %d is not 16, 32, 64 or 128, or %d query heads share a KV head "
                                       "(at most %d)",
                                       d, H / Hkv, kTileRows);
    return TB_OK;
}

extern "C" tb_status tb_paged_attention_chunk_workspace(int32_t rows, int32_t batch, int32_t max_new, int32_t max_len,
                                                        int32_t H, int32_t Hkv, int32_t d, int64_t* bytes) {
    TB_ENTRY_CHECK(bytes, "NULL argument");
    *bytes = 0;
    tb_status st = check_chunk(rows, batch, max_new, max_len, H, Hkv, d);
    if (st == TB_OK && rows > 0)
        *bytes = (int64_t)chunk_workspace(chunk_ctas(rows, batch, max_new, max_len, H, Hkv, d), d);
    return st;
}

extern "C" tb_status tb_paged_attention_chunk_dev(void* stream, const float* q, int64_t ld_q, int32_t rows,
                                                  const int32_t* row_offsets, const int32_t* total_lens, int32_t batch,
                                                  const float* pool, int32_t num_pages, const int32_t* table,
                                                  int32_t stride, int32_t max_new, int32_t max_len, int32_t layer,
                                                  int32_t num_layers, int32_t H, int32_t Hkv, int32_t d, float* out,
                                                  int64_t ld_out, void* workspace, int64_t workspace_bytes) {
    TB_ENTRY_CHECK(q && row_offsets && total_lens && pool && table && out, "NULL argument");
    tb_status st = check_chunk(rows, batch, max_new, max_len, H, Hkv, d);
    if (st != TB_OK) return st;
    TB_ENTRY_CHECK(num_pages >= 1 && stride >= 1 && stride <= INT_MAX / kPageTokens && layer >= 0 &&
                       layer < num_layers,
                   "bad pages / page table stride / layer");
    TB_ENTRY_CHECK(ld_q >= (int64_t)H * d && ld_out >= (int64_t)H * d, "a row stride is shorter than its row");
    TB_ENTRY_CHECK(aligned_to(pool, 16), "kv_pool must be 16-byte aligned");
    if (rows == 0) return TB_OK;
    const int ctas = chunk_ctas(rows, batch, max_new, max_len, H, Hkv, d);
    TB_ENTRY_CHECK(workspace && aligned_to(workspace, 16) && workspace_bytes >= (int64_t)chunk_workspace(ctas, d),
                   "the workspace must be 16-byte aligned and hold %lld bytes", (long long)chunk_workspace(ctas, d));
    StreamEntry entry(pool, "kv_pool");
    if (entry.status != TB_OK) return entry.status;
    ChunkParams p{q, ld_q, row_offsets, total_lens, batch, rows, pool, num_pages, table, stride, layer, num_layers, H,
                  Hkv, out, ld_out, entry.err};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = d == 16   ? launch_chunk<16>(p, ctas, workspace, s)
                    : d == 32 ? launch_chunk<32>(p, ctas, workspace, s)
                    : d == 64 ? launch_chunk<64>(p, ctas, workspace, s)
                              : launch_chunk<128>(p, ctas, workspace, s);
    return launch_status(e, "chunk attention launch");
}
