// tb_chunk.cu -- attention of each sequence's new tokens over its paged cache.
//
// Row i of a sequence with n new tokens and length L (the new ones included)
// has position p = L - n + i and attends over positions 0..p:
//     out = sum_j softmax_j(q . k_j / sqrt(d)) v_j,
// keys and values out of the page pool, the new tokens' own among them (they
// are in the cache before the call).  Query head h reads KV head h / (H/Hkv).
// Rows of an evicted page (table entry -1) are zeros, as in the decode
// attention (ModelRunner.swift:519-579 over KVCache.swift's pages).
#include "tb_chunk_mma.cuh"
#include "tb_chunk_few.cuh"
#include "tb_chunk_units.cuh"

namespace tb {
namespace {

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
// Roles:
//   producers  (2 warps: K, V) a lane per page of a tile: page table, then a bulk
//              copy of the page's rows of this head into a ring of fp32 pages;
//   converters (8 warps) the K and the V page of 16 tokens at a time (of D = 128 two
//              warps a page, half the dims each): a page's largest magnitude gives
//              a power-of-two scale, the halves go to the operand tiles;
//   issuer     one thread: S(i + 1) (or i + 2) before P V(i), so the softmax of a tile
//              runs while the tensor cores do the next S and the last P V;
//   softmax    a warpgroup, a row a thread: base-2 softmax over the tile, P as
//              halves over S in tensor memory, and the P V of the last tile added
//              to the row's sums in registers, which are rescaled only where the
//              running maximum grew by more than 2^8.
// Where the operands are made beforehand (long prompts) there are no converters;
// the producer copies operand tiles, and a second softmax warpgroup takes the
// odd tiles: one warp per scheduler waits for its own instructions, two fill
// each other's gaps.  Each keeps its own maximum and sums, and at a unit's end
// the odd one hands its to the even one, which writes the unit.  Tensor memory
// then holds three S and one O: S runs two tiles ahead, so that a warpgroup finds
// its next tile ready (two of each: 391 us for the prompt below), and O is read
// before the weights of the next tile are formed.
//
// Bound by the softmax warps' instructions (a weight takes an exponential, two
// conversions and some ten others).  Measured: 2048 tokens over 8192 positions, 32
// query and 4 KV heads of 64, 305 to 314 us (by card), 0.70 of the three products'
// time at the measured 1679 TFLOP/s; 8 us for the operands.  Converted by the CTAs
// that read them, 713 tokens of seven sequences of 664 to 1694, 32 heads of 128:
// 167 us; 64 tokens over 1920, 32 and 4 heads of 64: 23 us, of which 4 pass before
// the share is known and 2 in reading the queries.
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
// The roles' warps, and the registers of a thread: the launch's, then what the
// softmax warpgroups (with the rows' sums) take and the others keep.
template <bool PRE>
struct Roles {
    static constexpr int kGroups = PRE ? 2 : 1;  // softmax warpgroups
    static constexpr int kSoftmaxWarps = 4 * kGroups, kConvertWarps = PRE ? 0 : 8;
    static constexpr int kIssueWarp = kSoftmaxWarps + kConvertWarps, kLoadWarp = kIssueWarp + 1;
    static constexpr int kLoadWarps = PRE ? 1 : 2;  // K pages, V pages
    static constexpr int kThreads = PRE ? 384 : 512;
    static constexpr int kLaunchRegs = PRE ? 168 : 128, kSoftmaxRegs = PRE ? 208 : 224, kOtherRegs = PRE ? 88 : 96;
    static_assert(kGroups * 128 * kSoftmaxRegs + (kThreads - kGroups * 128) * kOtherRegs == kThreads * kLaunchRegs,
                  "registers");
    static_assert(kLoadWarp + kLoadWarps <= kThreads / 32, "warps");
};
constexpr int kTileRows = 128;
constexpr int kScaleRing = 8;     // tiles whose page scales are kept, at least two more than operand tiles
// Barriers that free the operand tiles, more than there are tiles: a phase two back
// on the same barrier looks like the one that a warp waits for.
constexpr int kEmptyRing = 4;
constexpr int kUnitRing = 4;      // units whose queries' scales are kept: with units of one tile, one
                                  // softmax warpgroup can be two units ahead of the other
constexpr uint32_t kWildBits = (127u + 20u) << 23;    // a K or V value of 2^20
constexpr uint32_t kWildQueryBits = (127u + 40u) << 23;
constexpr float kPShift = 6.0f;   // P = 2^(6 + score - M), M within 2^8 of the maximum: at most 2^14
constexpr float kLazy = 8.0f;
// The pages' value exponents are kept with 32 added (the reference maximum has it too,
// so P does not), and the row sums thus count in 2^32: over pages of zeros a term is up
// to 2^(14 + 100), and 2^31 of them have to fit; the smallest sum is 2^(6 - 6 - 32).
constexpr int kSumShift = 32;
constexpr float kSumScale = 1.0f / 4294967296.0f;
constexpr float kWildMark = 3e38f;
constexpr float kHuge = 1048576.0f;  // a score whose rounding could carry P out of fp16's range

template <int D>
struct Shape {
    static constexpr int NT = D == 128 ? 64 : 128;     // positions of a tile
    static constexpr int PG = NT / kPageTokens;        // its pages
    static constexpr int kPageBytes = kPageTokens * D * 4;
    static constexpr int kHalf = NT * D * 2;           // bytes of one operand half
    // fp32 pages on their way: a page takes about 3 us under load, so what streams
    // from HBM is bound by the bytes in flight (80 KB: 3.7 TB/s)
    static constexpr int kSlots = D == 128 ? 14 : D == 64 ? 28 : 64;
    // K and V operand tiles, and the bytes of shared memory.  K is free once S is
    // done, V only after P V, one softmax later.
    template <bool PRE>
    static constexpr int kKStages = PRE ? 3 : 1;
    template <bool PRE>
    static constexpr int kVStages = PRE ? 3 : 2;
    template <bool PRE>
    static constexpr size_t kSmem = (size_t)(kKStages<PRE> + kVStages<PRE>) * 2 * kHalf +
                                    (PRE ? 0 : (size_t)kSlots * kPageBytes);
    // tensor memory columns: S / P and O, each a few times, and Q
    template <bool PRE>
    static constexpr int kSBufs = PRE ? 3 : 2;
    template <bool PRE>
    static constexpr int kOBufs = PRE ? 1 : 2;
    template <bool PRE>
    static constexpr int kO = kSBufs<PRE> * NT;
    template <bool PRE>
    static constexpr int kQ = kO<PRE> + kOBufs<PRE> * D;
    static_assert(kQ<false> + D <= 512 && kQ<true> + D <= 512, "tensor memory");
};

struct ChunkBars {
    // By fill: a slot's fills come from two producers and go to converters that may be a
    // tile apart, so one barrier's parity would not tell a fill from the one two before
    // it.  With two, that one is four fills and at least two V tiles back.
    uint64_t slot_full[2][64], slot_empty[2][64];
    uint64_t k_full[3], v_full[3];
    uint64_t k_empty[kEmptyRing], v_empty[kEmptyRing];  // by tile, see kEmptyRing
    uint64_t scales[kScaleRing];
    uint64_t s_full[3], p_full[3];
    uint64_t pv_done[2], o_read[2], q_full[kUnitRing], merge_full[4], merge_read[4], drained;
};

// Operands made beforehand (chunk_operands_kernel): per sequence, KV head and
// tile [K high, K low, V high, V low] as the kernel holds them, and the tile's
// 16 page scales.  tiles = 0: none, the kernel converts pages itself.
struct Operands {
    uint8_t* ops;
    float* scales;
    int tiles;  // of a sequence
};
template <int D>
__device__ __forceinline__ size_t operand_tile(const ChunkParams& p, const Operands& o, int s, int head, int tile) {
    return ((size_t)s * p.Hkv + head) * o.tiles + tile;
}

struct ChunkShared {
    ChunkBars bars;
    alignas(16) float scale[kScaleRing][16];  // of a tile's pages: K factors, then V exponents
    int slot_page[64];
    uint32_t page_top[2][8];  // of K and V pages that two warps convert
    ShareShared share;
    uint32_t tmem;
    float q_scale[kUnitRing][kTileRows];              // of the units' rows
    float merge_m[kTileRows], merge_l[kTileRows];     // the odd warpgroup's
    float quad_m[kTileRows], quad_l[kTileRows];       // the even warpgroup's warps', in small units
    float quad_sum[3][32][17];
    int merge_wild[4], quad_wild[4];
    ChunkWatch watch;
};

// What frees the operand tile that position tile i goes to: the product with its
// last user, `stages` tiles before.
__device__ __forceinline__ uint64_t* free_bar(uint64_t* ring, int i, int stages) {
    return i < stages ? nullptr : ring + (i - stages) % kEmptyRing;
}
__device__ __forceinline__ uint32_t free_parity(int i, int stages) { return (uint32_t)((i - stages) / kEmptyRing & 1); }
__device__ __forceinline__ void warp_wait(ChunkShared& sh, uint64_t* bar, uint32_t parity, int* err) {
    if ((threadIdx.x & 31) == 0) chunk_wait(&sh.watch, bar, parity, err);
    __syncwarp();
}

// Exponent of a page's block from the lanes' largest magnitudes (all lanes get it).
__device__ __forceinline__ uint32_t warp_max_bits(float m) {
    return __reduce_max_sync(0xffffffffu, __float_as_uint(m) & 0x7fffffffu);
}
__device__ __forceinline__ void split4(const float4& a, float s, uint2& hi, uint2& lo) {
    const float2 ss = make_float2(s, s);
    const float2 x = __fmul2_rn(make_float2(a.x, a.y), ss), y = __fmul2_rn(make_float2(a.z, a.w), ss);
    split_pair(x.x, x.y, hi.x, lo.x);
    split_pair(y.x, y.y, hi.y, lo.y);
}

// The largest magnitude of a page that PARTS warps convert, each its dims: they
// tell one another (tops[page][part]) and meet at the page's named barrier.
template <int PARTS>
struct PageTop {
    volatile uint32_t* tops;
    __device__ __forceinline__ uint32_t operator()(uint32_t bits, int page, int part) const {
        if (PARTS == 1) return bits;
        if ((threadIdx.x & 31) == 0) tops[page * PARTS + part] = bits;
        named_bar_sync(2 + page, 32 * PARTS);
        for (int k = 0; k < PARTS; ++k) bits = max(bits, tops[page * PARTS + k]);
        return bits;
    }
};

// K page -> rows `page * 16 ..` of the K operand, four dims of a token at a
// time.  Lane (r, q) of a step takes dims 4 g .. of token r + 8 (q & 1) with g
// staggered over the lanes, so that the reads (rows of D floats, 16 bytes a
// lane) and the writes (8 bytes of a core matrix's 16-byte rows) fall into
// different banks.
template <int D, int PARTS>
__device__ __forceinline__ void convert_k(const float* src, int valid, uint8_t* hi, uint8_t* lo, int page, int part,
                                          PageTop<PARTS> both, float* scale_out) {
    constexpr int C = D / 4 / PARTS, kTasks = C / 2;  // 16-byte columns of a token, steps of a lane
    const int lane = threadIdx.x & 31, r = lane & 15;
    const int g0 = (lane & 7) + ((lane >> 3) & 1) + (lane >> 4) * kTasks;
    const float* row = src + r * D;
    float4 x[kTasks];
#pragma unroll
    for (int t = 0; t < kTasks; ++t)
        x[t] = r < valid ? lds128f(row + (part * C + (g0 + t) % C) * 4) : make_float4(0, 0, 0, 0);
    float m = 0.0f;
#pragma unroll
    for (int t = 0; t < kTasks; ++t) m = max_abs(max_abs(m, x[t].x, x[t].y), x[t].z, x[t].w);
    const uint32_t bits = both(warp_max_bits(m), page, part);
    const int e = block_exponent(bits, kLowestFactor);
    const float s = exp2_int(-e);
    if (lane == 0 && part == 0) *scale_out = bits >= kWildBits ? kWildMark : exp2_int(e);
    const int at0 = (page * 2 + (r >> 3)) * (D * 16) + (r & 7) * 16;
#pragma unroll
    for (int t = 0; t < kTasks; ++t) {
        const int g = part * C + (g0 + t) % C, at = at0 + (g >> 1) * 128 + (g & 1) * 8;
        uint2 h, l;
        split4(x[t], s, h, l);
        *reinterpret_cast<uint2*>(hi + at) = h;
        *reinterpret_cast<uint2*>(lo + at) = l;
    }
}

// V page -> columns (k) `page * 16 ..` of the V^T operand of NT columns: a lane
// takes 8 consecutive tokens of a dim.
template <int D, int NT, int PARTS>
__device__ __forceinline__ void convert_v(const float* src, int valid, uint8_t* hi, uint8_t* lo, int page, int part,
                                          PageTop<PARTS> both, float* exp_out) {
    constexpr int kDims = D / PARTS, kTasks = kDims / 16;
    const int lane = threadIdx.x & 31;
    float x[kTasks][8];
    float m = 0.0f;
#pragma unroll
    for (int t = 0; t < kTasks; ++t) {
        const int task = lane + 32 * t, n = part * kDims + task % kDims, kc = task / kDims;
#pragma unroll
        for (int j = 0; j < 8; ++j) x[t][j] = kc * 8 + j < valid ? src[(kc * 8 + j) * D + n] : 0.0f;
    }
#pragma unroll
    for (int t = 0; t < kTasks; ++t)
#pragma unroll
        for (int j = 0; j < 8; j += 2) m = max_abs(m, x[t][j], x[t][j + 1]);
    const uint32_t bits = both(warp_max_bits(m), page, part);
    const int e = block_exponent(bits, kLowestValue);
    const float s = exp2_int(-e);
    if (lane == 0 && part == 0) *exp_out = bits >= kWildBits ? kWildMark : (float)(e + kSumShift);
#pragma unroll
    for (int t = 0; t < kTasks; ++t) {
        const int task = lane + 32 * t, n = part * kDims + task % kDims, kc = task / kDims;
        uint2 h0, l0, h1, l1;
        split4(make_float4(x[t][0], x[t][1], x[t][2], x[t][3]), s, h0, l0);
        split4(make_float4(x[t][4], x[t][5], x[t][6], x[t][7]), s, h1, l1);
        const int at = (n >> 3) * (NT * 16) + (page * 2 + kc) * 128 + (n & 7) * 16;
        *reinterpret_cast<uint4*>(hi + at) = make_uint4(h0.x, h0.y, h1.x, h1.y);
        *reinterpret_cast<uint4*>(lo + at) = make_uint4(l0.x, l0.y, l1.x, l1.y);
    }
}

// A thread's 4 of every 16 values of a query row (N of them in all), all loads in
// flight: a branch at each would make them wait for one another.
template <int N>
__device__ __forceinline__ void load_row(const float* q, bool wide, float (&x)[N]) {
    if (wide) {
#pragma unroll
        for (int j = 0; j < N; j += 4) {
            const float4 f = *reinterpret_cast<const float4*>(q + 4 * j);
            x[j] = f.x, x[j + 1] = f.y, x[j + 2] = f.z, x[j + 3] = f.w;
        }
    } else {
#pragma unroll
        for (int j = 0; j < N; ++j) x[j] = q[j / 4 * 16 + j % 4];
    }
}

// A warp's 32 query rows (row(r): where row r is) as halves in tensor memory, 16 at a
// time, four threads to a row, so that a load touches 8 rows and not 32 (a thread a
// row: 311 us for the prompt above instead of 305).  scale[r] becomes the row's factor
// (2^e log2(e) / sqrt(D)), negative for a row without operands.  What rows that are
// not the unit's (row() is then a neighbour's) or have no operands hold reaches no
// other row.
template <int D, class Row>
__device__ __forceinline__ void load_queries(Row row, bool wide, uint32_t tq, float* scale) {
    constexpr int N = D < 64 ? D : 64, M = N / 4;  // dims at a time; all of them are read once
    const int lane = threadIdx.x & 31, own = lane / 4, dims = 4 * (lane % 4);
#pragma unroll 1
    for (int half = 0; half < 2; ++half) {
        const float* q[2] = {row(16 * half + own) + dims, row(16 * half + own + 8) + dims};
        float x[2][M], s[2];
        float top[2] = {0.0f, 0.0f};
#pragma unroll 1
        for (int i = 0; i < D; i += N) {
            load_row(q[0] + i, wide, x[0]);
            load_row(q[1] + i, wide, x[1]);
#pragma unroll
            for (int a = 0; a < 2; ++a)
#pragma unroll
                for (int j = 0; j < M; j += 2) top[a] = max_abs(top[a], x[a][j], x[a][j + 1]);
        }
#pragma unroll
        for (int a = 0; a < 2; ++a) {
            for (int o = 1; o < 4; o <<= 1)
                top[a] = max_abs(top[a], __shfl_xor_sync(0xffffffffu, top[a], o), 0.0f);
            const uint32_t m = __float_as_uint(top[a]) & 0x7fffffffu;
            const int e = m < kWildQueryBits ? block_exponent(m, kLowestFactor) : 0;
            s[a] = exp2_int(-e);
            if (dims == 0)
                scale[16 * half + own + 8 * a] =
                    m < kWildQueryBits ? exp2_int(e) * (1.4426950408889634f * rsqrtf((float)D)) : -1.0f;
        }
        const uint32_t to = tq + ((uint32_t)(16 * half) << 16);
#pragma unroll 1
        for (int i = 0; i < D; i += N) {
            if (N < D) {
                load_row(q[0] + i, wide, x[0]);
                load_row(q[1] + i, wide, x[1]);
            }
            uint32_t hi[M], lo[M];
#pragma unroll
            for (int j = 0; j < M; j += 4)
#pragma unroll
                for (int a = 0; a < 2; ++a) {
                    split_pair(x[a][j] * s[a], x[a][j + 1] * s[a], hi[j + 2 * a], lo[j + 2 * a]);
                    split_pair(x[a][j + 2] * s[a], x[a][j + 3] * s[a], hi[j + 2 * a + 1], lo[j + 2 * a + 1]);
                }
            tmem_st_rows<N / 16>(to + i / 2, hi);
            tmem_st_rows<N / 16>(to + D / 2 + i / 2, lo);
        }
    }
}

// A unit's rows of one warp in fp32 (pages or queries without fp16 operands).
template <int D>
__device__ __noinline__ void rows_without_operands(const ChunkParams& p, const Unit& u, int t0, int t1, float* partial,
                                                   ChunkWatch* watch) {
    const int first = (threadIdx.x >> 5) * 32;
    for (int r = first; r < first + 32; ++r) {  // the even warpgroup's warps 0 to 3
        const unsigned long long since = global_timer_ns();
        if (!row_in_fp32<D, kTileRows>(p, u, r, t0, t1, partial, kPShift + kSumShift, kSumScale)) break;
        if ((threadIdx.x & 31) == 0) atomicAdd(&watch->limit, global_timer_ns() - since);
    }
}

template <int D, bool PRE>
__global__ void __launch_bounds__(Roles<PRE>::kThreads, 1)
    chunk_tiles_kernel(ChunkParams p, float* partials, ChunkSplit* splits, Operands pre, bool wide_q, bool wide_out) {
    using S = Shape<D>;
    using R = Roles<PRE>;
    constexpr int NT = S::NT, PG = S::PG, kChunkThreads = R::kThreads;
    constexpr int kKStages = S::template kKStages<PRE>, kVStages = S::template kVStages<PRE>;
    constexpr int kIssueWarp = R::kIssueWarp, kLoadWarp = R::kLoadWarp;
    constexpr int kSoftmaxRegs = R::kSoftmaxRegs, kOtherRegs = R::kOtherRegs, kSoftmaxWarps = R::kSoftmaxWarps;
    constexpr int kGroups = R::kGroups;
    constexpr int kSBufs = S::template kSBufs<PRE>, kOBufs = S::template kOBufs<PRE>;
    constexpr int kO = S::template kO<PRE>, kQ = S::template kQ<PRE>;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ ChunkShared sh;
    static_assert(S::template kSmem<PRE> + sizeof(ChunkShared) <= 227 * 1024, "shared memory");
    static_assert(S::kSlots <= 64 && kScaleRing >= kVStages + 2 && S::kSlots >= 2 * PG && PG <= 8, "rings");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    uint8_t* k_ops = smem;                                // [stage][hi, lo]
    uint8_t* v_ops = smem + kKStages * 2 * S::kHalf;
    uint8_t* pages = v_ops + kVStages * 2 * S::kHalf;
    ChunkBars& b = sh.bars;

    if (tid == 0) {
        watch_init(sh.watch);
        for (int i = 0; i < S::kSlots; ++i) {
            for (int f = 0; f < 2; ++f) {
                mbar_init(b.slot_full[f] + i, 1);
                mbar_init(b.slot_empty[f] + i, 8 / PG);
            }
        }
        for (int i = 0; i < 3; ++i) {
            mbar_init(b.s_full + i, 1);
            mbar_init(b.p_full + i, 4);
            mbar_init(b.k_full + i, PRE ? 1 : 8);
            mbar_init(b.v_full + i, PRE ? 1 : 8);
        }
        for (int i = 0; i < kEmptyRing; ++i) {
            mbar_init(b.k_empty + i, 1);
            mbar_init(b.v_empty + i, 1);
        }
        for (int i = 0; i < kScaleRing; ++i) mbar_init(b.scales + i, PRE ? 1 : 2 * PG);
        for (int i = 0; i < 2; ++i) {
            mbar_init(b.pv_done + i, 1);
            mbar_init(b.o_read + i, 4);
        }
        for (int i = 0; i < kUnitRing; ++i) mbar_init(b.q_full + i, 4);
        for (int i = 0; i < 4; ++i) {
            mbar_init(b.merge_full + i, 1);
            mbar_init(b.merge_read + i, 1);
        }
        mbar_init(&b.drained, 1);
        fence_barrier_init();
        fence_proxy_async_shared();
    }
    const Share share = find_share<NT, kTileRows, kChunkThreads>(p, sh.share);
    const int count = share.count;
    if (warp == kIssueWarp) tmem_alloc(&sh.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    pdl_launch_dependents();
    const uint32_t tmem = sh.tmem;
    Unit u = sh.share.start;
    int at = sh.share.tile;

    // (a warpgroup's warps all move the same way, each in its own role)
    if (count > 0 && warp >= kLoadWarp && warp < kLoadWarp + R::kLoadWarps) {
        // ---- producer ----
        set_registers_down<kOtherRegs>();
        if constexpr (PRE) {
            int i = 0;
            if (lane == 0) {
                for (int left = count; left > 0 && !sh.watch.dead; at = 0) {
                    const int take = min(u.tiles - at, left);
                    for (int j = at; j < at + take; ++j, ++i) {
                        const int sk = i % kKStages, sv = i % kVStages, ring = i % kScaleRing;
                        const bool made = u.len <= pre.tiles * NT;  // a longer one goes without operands
                        const size_t t = made ? operand_tile<D>(p, pre, u.s, u.head, j) : 0;
                        const uint8_t* src = pre.ops + t * (4 * S::kHalf);
                        if (i >= kKStages && !chunk_wait(&sh.watch, free_bar(b.k_empty, i, kKStages), free_parity(i, kKStages), p.err)) break;
                        mbar_arrive_expect_tx(b.scales + ring, 64);
                        bulk_g2s(sh.scale[ring], pre.scales + t * 16, 64, b.scales + ring);
                        mbar_arrive_expect_tx(b.k_full + sk, 2 * S::kHalf);
                        bulk_g2s(k_ops + sk * 2 * S::kHalf, src, 2 * S::kHalf, b.k_full + sk);
                        if (i >= kVStages && !chunk_wait(&sh.watch, free_bar(b.v_empty, i, kVStages), free_parity(i, kVStages), p.err)) break;
                        mbar_arrive_expect_tx(b.v_full + sv, 2 * S::kHalf);
                        bulk_g2s(v_ops + sv * 2 * S::kHalf, src + 2 * S::kHalf, 2 * S::kHalf, b.v_full + sv);
                    }
                    left -= take;
                    if (left > 0) next_unit<NT, kTileRows>(p, u);
                }
                if (sh.watch.dead) land_copies();
            }
            __syncwarp();
        } else {
        // Table entries are read a tile ahead: their latency would otherwise stand
        // in front of every tile's copies.  Four pages go at a time: one by one the
        // lanes' branches take longer than the copies, and a whole tile would wait
        // for its last slot.
        const int kv = warp - kLoadWarp;
        int slot = kv * PG + lane, fill = 0;  // the lane's page slot, and its fills before
        const bool mine = lane < PG;
        const auto entry = [&](int j) {
            const int pos = j * NT + lane * kPageTokens;
            return mine && pos < u.limit ? p.table[(size_t)u.s * p.stride + pos / kPageTokens] : -1;
        };
        int left = count, j = at, end_j = at + min(u.tiles - at, left), page = entry(j);
        while (left > 0 && !sh.watch.dead) {
            const int id = checked_page(p, page);
            const float* src = head_rows<D>(p, max(id, 0), kv, u.head);
            if (--left > 0) {
                if (++j == end_j) {
                    next_unit<NT, kTileRows>(p, u);
                    j = 0;
                    end_j = min(u.tiles, left);
                }
                page = entry(j);
            }
#pragma unroll 1
            for (int g = 0; g < PG; g += 4) {
                const bool turn = lane >= g && lane < g + 4;
                const int last = fill - 1;
                lanes_wait(&sh.watch, turn && fill ? b.slot_empty[last & 1] + slot : nullptr, (uint32_t)(last >> 1) & 1,
                           p.err);
                if (turn && !sh.watch.dead) {
                    sh.slot_page[slot] = id;
                    uint64_t* full = b.slot_full[fill & 1] + slot;
                    mbar_arrive_expect_tx(full, id >= 0 ? S::kPageBytes : 0);
                    if (id >= 0) bulk_g2s(pages + slot * S::kPageBytes, src, S::kPageBytes, full);
                }
                __syncwarp();
            }
            slot += 2 * PG;
            if (slot >= S::kSlots) {
                slot -= S::kSlots;
                ++fill;
            }
        }
        if (sh.watch.dead) land_copies();
        }
    } else if (count > 0 && warp == kIssueWarp) {
        // ---- issuer ----
        set_registers_down<kOtherRegs>();
        if (elect_one()) {
            const uint32_t k0 = smem_u32(k_ops), v0 = smem_u32(v_ops);
            int i = 0, unit = 0;
            const auto issue_s = [&](int item, bool first, int un) {
                const int st = item % kKStages;
                if (first) chunk_wait(&sh.watch, b.q_full + un % kUnitRing, (uint32_t)(un / kUnitRing & 1), p.err);
                chunk_wait(&sh.watch, b.k_full + st, (uint32_t)(item / kKStages & 1), p.err);
                tc_fence_after();
                const uint32_t kb = k0 + st * 2 * S::kHalf;
                tc_mma_split<NT, D>(tmem + (uint32_t)(item % kSBufs) * NT, tmem + kQ, [](int s) { return 8 * s; }, D / 2,
                                    kb, kb + S::kHalf);
                tc_commit(b.s_full + item % kSBufs);
                tc_commit(b.k_empty + item % kEmptyRing);
            };
            for (int left = count; left > 0; at = 0) {
                const int take = min(u.tiles - at, left);
                // S goes kAhead tiles ahead, over a P whose product has been issued before
                constexpr int kAhead = kSBufs - 1;
                for (int j = 0; j < kAhead && j < take; ++j) issue_s(i + j, j == 0, unit);
                for (int j = 0; j < take; ++j, ++i) {
                    if (j + kAhead < take) issue_s(i + kAhead, false, unit);
                    const int st = i % kVStages;
                    chunk_wait(&sh.watch, b.v_full + st, (uint32_t)(i / kVStages & 1), p.err);
                    chunk_wait(&sh.watch, b.p_full + i % kSBufs, (uint32_t)(i / kSBufs & 1), p.err);
                    // (of two buffers, O of two tiles before was read before P of this one arrived)
                    if (kOBufs == 1 && i > 0)
                        chunk_wait(&sh.watch, b.o_read + (i - 1 & 1), (uint32_t)((i - 1) / 2 & 1), p.err);
                    tc_fence_after();
                    const uint32_t vb = v0 + st * 2 * S::kHalf;
                    // P: 16 columns of high, 16 of low halves per 32 positions
                    tc_mma_split<D, NT>(tmem + kO + (uint32_t)(i % kOBufs) * D, tmem + (uint32_t)(i % kSBufs) * NT,
                                        [](int s) { return 32 * (s / 2) + 8 * (s % 2); }, 16, vb, vb + S::kHalf);
                    tc_commit(b.v_empty + i % kEmptyRing);
                    tc_commit(b.pv_done + (i & 1));
                }
                left -= take;
                ++unit;
                if (left > 0) next_unit<NT, kTileRows>(p, u);
            }
            // every product has been read and written before tensor memory goes
            tc_commit(&b.drained);
            const uint64_t t0 = global_timer_ns();
            while (!mbar_try_wait(&b.drained, 0) && global_timer_ns() - t0 < kWaitLimitNs) {
            }
        }
        __syncwarp();
    } else if (!PRE && count > 0 && warp >= kSoftmaxWarps && warp < kIssueWarp) {
        // ---- converters: a warp takes the same page of every tile, or of a tile of four
        //      pages half the dims of one (one K operand tile: the next tile's conversion
        //      waits for this one's, and a page by one warp takes 5600 cycles of D = 128) ----
        set_registers_down<kOtherRegs>();
        constexpr int kParts = 8 / PG;
        const int cw = warp - kSoftmaxWarps, page = cw % PG, part = cw / PG;
        int i = 0;  // the CTA's tile
        int left = count;
        for (; left > 0; at = 0) {
            const int take = min(u.tiles - at, left);
            for (int j = at; j < at + take; ++j, ++i) {
                const int ring = i % kScaleRing, valid_here = u.limit - (j * NT + page * kPageTokens);
                const int job = i * (2 * PG) + page;
                for (int kv = 0; kv < 2; ++kv) {
                    const int slot = (job + kv * PG) % S::kSlots, fill = (job + kv * PG) / S::kSlots;
                    const int st = kv ? i % kVStages : i % kKStages, stages = kv ? kVStages : kKStages;
                    // lane 0: the page, lane 1: its place in the operand tile
                    lanes_wait(&sh.watch,
                               lane == 0   ? b.slot_full[fill & 1] + slot
                               : lane == 1 ? free_bar(kv ? b.v_empty : b.k_empty, i, stages)
                                           : nullptr,
                               lane == 0 ? (uint32_t)(fill >> 1) & 1 : free_parity(i, stages), p.err);
                    const int valid = sh.slot_page[slot] < 0 ? 0 : max(0, min(valid_here, kPageTokens));
                    const float* src = reinterpret_cast<const float*>(pages + slot * S::kPageBytes);
                    uint8_t* op = (kv ? v_ops : k_ops) + st * 2 * S::kHalf;
                    if (kv)
                        convert_v<D, NT, kParts>(src, valid, op, op + S::kHalf, page, part, {sh.page_top[1]},
                                                 &sh.scale[ring][8 + page]);
                    else
                        convert_k<D, kParts>(src, valid, op, op + S::kHalf, page, part, {sh.page_top[0]},
                                             &sh.scale[ring][page]);
                    fence_proxy_async_shared();
                    __syncwarp();
                    if (lane < (part == 0 ? 3 : 2))
                        mbar_arrive(lane == 0   ? (kv ? b.v_full : b.k_full) + st
                                    : lane == 1 ? b.slot_empty[fill & 1] + slot
                                                : b.scales + ring);
                }
            }
            left -= take;
            if (left > 0) next_unit<NT, kTileRows>(p, u);
        }
    } else if (count > 0 && warp < kSoftmaxWarps) {
        // ---- softmax: of two warpgroups each takes the tiles of its parity ----
        set_registers_up<kSoftmaxRegs>();
        const int group = warp >> 2, quad = warp & 3;
        const uint32_t lanes = (uint32_t)(quad * 32) << 16;
        const int G = p.H / p.Hkv, per = (kTileRows / G);
        const uint32_t s0_addr = tmem + lanes, o0_addr = tmem + kO + lanes;
        ChunkSplit split{-1};
        // A unit of at most 32 rows would leave three of a warpgroup's four warps
        // idle: its rows stand in all four lane groups, each of which takes a
        // quarter of a tile's positions (P is zero elsewhere).
        const auto small_unit = [&](const Unit& w) { return min(per, w.n - w.tile * per) * G <= 32; };
        const auto queries = [&](const Unit& w, int unit) {
            const int row0 = small_unit(w) ? 0 : quad * 32, used = min(per, w.n - w.tile * per) * G;
            if (row0 < used) {
                load_queries<D>(
                    [&](int r) {  // (rows that are not the unit's: its first)
                        const int row = row0 + r < used ? row0 + r : 0;
                        return p.q + (w.first + w.tile * per + row / G) * p.ld_q + (size_t)(w.head * G + row % G) * D;
                    },
                    wide_q, tmem + kQ + lanes, sh.q_scale[unit % kUnitRing] + quad * 32);
                tmem_st_wait();
            }
            tc_fence_before();
            __syncwarp();
            if (lane == 0) mbar_arrive(b.q_full + unit % kUnitRing);
        };
        int i = 0, unit = 0, merges = 0;
        if (group == 0) queries(u, 0);
        for (int left = count; left > 0; ++unit) {
            const int take = min(u.tiles - at, left);
            const bool small = small_unit(u);
            const int row = small ? lane : quad * 32 + lane, sub = row % G;
            const int token = u.tile * per + row / G;
            const bool valid = row < per * G && token < u.n;
            const bool busy = __any_sync(0xffffffffu, valid);
            const int sees = min(u.len - u.n + token + 1, u.limit);  // the row's own limit, may be <= 0
            const int first_sees = __shfl_sync(0xffffffffu, sees, 0);  // tokens ascend with the lanes
            warp_wait(sh, b.q_full + unit % kUnitRing, (uint32_t)(unit / kUnitRing & 1), p.err);
            const float c = busy ? sh.q_scale[unit % kUnitRing][quad * 32 + lane] : 1.0f;
            bool wild = __any_sync(0xffffffffu, valid && c < 0.0f) || (PRE && u.len > pre.tiles * NT), huge = false;
            float M = -INFINITY, l = 0.0f;
            float2 acc[D / 2];
#pragma unroll
            for (int x = 0; x < D / 2; ++x) acc[x] = make_float2(0.0f, 0.0f);
            // adds P V of the warpgroup's tile `item`, whose scale the sums still have
            const auto collect = [&](int item) {
                warp_wait(sh, b.pv_done + (item & 1), (uint32_t)(item / 2 & 1), p.err);
                tc_fence_after();
                const uint32_t to = o0_addr + (uint32_t)(item % kOBufs) * D;
                if constexpr (D == 16) {
                    int v[16];
                    tmem_ld16(to, v);
                    tmem_ld_wait();
#pragma unroll
                    for (int x = 0; x < 8; ++x)
                        acc[x] = __fadd2_rn(acc[x],
                                            make_float2(__int_as_float(v[2 * x]), __int_as_float(v[2 * x + 1])));
                } else {
#pragma unroll
                    for (int o = 0; o < D; o += 64) {
                        int v[2][32];
                        tmem_ld32(to + o, v[0]);
                        if (o + 32 < D) tmem_ld32(to + o + 32, v[1]);
                        tmem_ld_wait();
#pragma unroll
                        for (int h = 0; h < 2 && o + 32 * h < D; ++h)
#pragma unroll
                            for (int x = 0; x < 16; ++x)
                                acc[o / 2 + 16 * h + x] = __fadd2_rn(
                                    acc[o / 2 + 16 * h + x], make_float2(__int_as_float(v[h][2 * x]),
                                                                         __int_as_float(v[h][2 * x + 1])));
                    }
                }
            };
            // after that, where there is one O: the next tile's product may go over it
            const auto release = [&](int item) {
                if (kOBufs > 1) return;
                // a warp without rows may not run ahead: its next arrival would count for this tile
                if (!busy) warp_wait(sh, b.pv_done + (item & 1), (uint32_t)(item / 2 & 1), p.err);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(b.o_read + (item & 1));
            };
            const int i0 = i;  // then this warpgroup's first tile of the unit:
            const int first = kGroups == 1 || (i0 & 1) == group ? i0 : i0 + 1;
            for (i = first; i < i0 + take; i += kGroups) {
                const uint32_t ts = s0_addr + (uint32_t)(i % kSBufs) * NT;
                const int j = at + (i - i0), ring = i % kScaleRing;
                lanes_wait(&sh.watch, lane == 0 ? b.scales + ring : lane == 1 ? b.s_full + i % kSBufs : nullptr,
                           (uint32_t)(lane == 0 ? i / kScaleRing : i / kSBufs) & 1, p.err);
                tc_fence_after();
                if (busy) {
                    const float *ks = sh.scale[ring], *ve = ks + 8;
                    const int room = sees - j * NT;                 // columns below it are seen
                    const bool masked = first_sees < (j + 1) * NT;  // some row does not see all of the tile
                    // A block of W positions: -inf where the row does not see one, the largest
                    // score + value exponent (per page the largest S decides), and the weights.
                    const auto mask = [&](auto& v, int col) {
                        constexpr int W = sizeof(v) / 4;
#pragma unroll
                        for (int x = 0; x < W; ++x)
                            if (col + x >= room) v[x] = __float_as_int(-INFINITY);
                    };
                    const auto page_top = [&](const int* v, int page) {
                        float m0 = __int_as_float(v[0]), m1 = __int_as_float(v[1]);
#pragma unroll
                        for (int x = 2; x < 14; x += 4) {
                            m0 = max3(m0, __int_as_float(v[x]), __int_as_float(v[x + 1]));
                            m1 = max3(m1, __int_as_float(v[x + 2]), __int_as_float(v[x + 3]));
                        }
                        m0 = max3(m0, __int_as_float(v[14]), __int_as_float(v[15]));
                        wild |= ks[page] == kWildMark || ve[page] == kWildMark;
                        return fmaf(fmaxf(m0, m1), c * ks[page], ve[page]);
                    };
                    const auto page_weights = [&](const int* v, int page, float shift, uint32_t* hi, uint32_t* lo) {
                        const float e = ve[page], k = c * ks[page];
                        const float2 kk = make_float2(k, k), bb = make_float2(e + shift, e + shift);
                        float2 sum = make_float2(0.0f, 0.0f);
#pragma unroll
                        for (int x = 0; x < 16; x += 2) {
                            const float2 t =
                                __ffma2_rn(make_float2(__int_as_float(v[x]), __int_as_float(v[x + 1])), kk, bb);
                            const float2 w = make_float2(ex2(t.x), ex2(t.y));
                            sum = __fadd2_rn(sum, w);
                            split_pair(w.x, w.y, hi[x / 2], lo[x / 2]);
                        }
                        l = fmaf(sum.x + sum.y, ex2(-e), l);
                    };
                    float r = 1.0f;
                    // takes the block's maximum into the reference; the result is P's shift
                    const auto refer = [&](float top) {
                        huge |= valid && top > -INFINITY && fabsf(top) > kHuge;
                        if (top > M + kLazy || (M == -INFINITY && top > -INFINITY)) {
                            r = M == -INFINITY ? 0.0f : ex2(M - top);
                            M = top;
                            l *= r;
                        }
                        return kPShift - (M == -INFINITY ? 0.0f : M);
                    };
                    // the last tile's P V, and the sums to the new reference: one O is given back
                    // before the weights are formed, of two the product has time until after
                    const auto settle = [&] {
                        if (i > first) {
                            collect(i - kGroups);
                            release(i - kGroups);
                        }
                        if (__any_sync(0xffffffffu, r != 1.0f)) {
#pragma unroll
                            for (int x = 0; x < D / 2; ++x) acc[x] = __fmul2_rn(acc[x], make_float2(r, r));
                        }
                    };
                    if (small) {  // the warp's quarter, kept in registers; zeros elsewhere
                        constexpr int W = NT / 4;
                        const int col = quad * W, g = col / 32;
                        int v[W];
                        if constexpr (W == 32)
                            tmem_ld32(ts + col, v);
                        else
                            tmem_ld16(ts + col, v);
                        tmem_ld_wait();
                        uint32_t zero[32];
#pragma unroll
                        for (int x = 0; x < 32; ++x) zero[x] = 0;
#pragma unroll
                        for (int k = 0; k < NT / 32; ++k)
                            if (W == 16 || k != g) tmem_st32(ts + 32 * k, zero);
                        if (masked) mask(v, col);
                        float top = page_top(v, col / 16);
                        if constexpr (W == 32) top = fmaxf(top, page_top(v + 16, col / 16 + 1));
                        const float shift = refer(top);
                        if (kOBufs == 1) settle();
                        uint32_t hi[W / 2], lo[W / 2];
                        page_weights(v, col / 16, shift, hi, lo);
                        if constexpr (W == 32) {
                            page_weights(v + 16, col / 16 + 1, shift, hi + 8, lo + 8);
                            tmem_st16(ts + 32 * g, hi);
                            tmem_st16(ts + 32 * g + 16, lo);
                        } else {
                            tmem_st_wait();  // over the zeros
                            tmem_st8(ts + 32 * g + col % 32 / 2, hi);
                            tmem_st8(ts + 32 * g + 16 + col % 32 / 2, lo);
                        }
                    } else {
                        float top = -INFINITY;
#pragma unroll 1
                        for (int g = 0; g < NT / 32; ++g) {
                            int v[32];
                            tmem_ld32(ts + 32 * g, v);
                            tmem_ld_wait();
                            if (masked) mask(v, 32 * g);
                            top = max3(top, page_top(v, 2 * g), page_top(v + 16, 2 * g + 1));
                        }
                        const float shift = refer(top);
                        if (kOBufs == 1) settle();
#pragma unroll 1
                        for (int g = 0; g < NT / 32; ++g) {
                            int v[32];
                            uint32_t hi[16], lo[16];
                            tmem_ld32(ts + 32 * g, v);
                            tmem_ld_wait();
                            if (masked) mask(v, 32 * g);
                            page_weights(v, 2 * g, shift, hi, lo);
                            page_weights(v + 16, 2 * g + 1, shift, hi + 8, lo + 8);
                            tmem_st16(ts + 32 * g, hi);
                            tmem_st16(ts + 32 * g + 16, lo);
                        }
                    }
                    tmem_st_wait();
                    if (kOBufs > 1) settle();
                } else if (i > first) {
                    release(i - kGroups);
                }
                // the odd sums of the last unit still stand where P V of this tile goes
                if (group == 1 && i == first && merges > 0)
                    warp_wait(sh, b.merge_read + quad, (uint32_t)(merges - 1) & 1, p.err);
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(b.p_full + i % kSBufs);
            }
            i = i0 + take;
            const Unit done = u;
            const int from = at;
            left -= take;
            at = 0;
            if (left > 0) {
                next_unit<NT, kTileRows>(p, u);
                // the warpgroup of the unit's last tile knows that its queries are read
                if (kGroups == 1 || ((i - 1) & 1) == group) queries(u, unit + 1);
            }
            if (first < i) {
                const int mine = kGroups == 1 || ((i - 1) & 1) == group ? i - 1 : i - 2;
                if (busy) collect(mine);
                release(mine);
            }
            wild |= __any_sync(0xffffffffu, huge);
            const bool merge = kGroups == 2 && ((i0 & 1) || take > 1);  // the odd warpgroup had a tile
            if (group == 1) {
                if (merge) {
                    // its sums go over O, which the even warpgroup may still be reading
                    if (((i - 1) & 1) == 0) warp_wait(sh, b.o_read, (uint32_t)((i - 1) / 2) & 1, p.err);
                    tc_fence_after();
                    if (busy) {
#pragma unroll
                        for (int o = 0; o < D; o += 16) {
                            uint32_t w[16];
#pragma unroll
                            for (int x = 0; x < 8; ++x) {
                                w[2 * x] = __float_as_uint(acc[o / 2 + x].x);
                                w[2 * x + 1] = __float_as_uint(acc[o / 2 + x].y);
                            }
                            tmem_st16(o0_addr + o, w);
                        }
                        sh.merge_m[quad * 32 + lane] = M;
                        sh.merge_l[quad * 32 + lane] = l;
                        if (lane == 0) sh.merge_wild[quad] = wild;
                        tmem_st_wait();
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(b.merge_full + quad);
                    ++merges;
                }
                continue;
            }
            const bool whole = from == 0 && take == done.tiles;
            float* part = nullptr;
            if (!whole) {
                part = partials + ((size_t)blockIdx.x * 2 + (from == 0)) * partial_floats(kTileRows, D);
                if (from == 0) {  // goes on in the next CTAs: up to the one that holds its last tile
                    const int more = share.followers(done.tiles - take);
                    split = split_of<kTileRows>(p, done, more);
                }
            }
            float w0 = 1.0f, w1 = 0.0f;
            if (merge) {
                warp_wait(sh, b.merge_full + quad, (uint32_t)merges & 1, p.err);
                tc_fence_after();
                ++merges;
                if (busy) {
                    const float m1 = sh.merge_m[quad * 32 + lane], both = fmaxf(M, m1);
                    const float off = both == -INFINITY ? 0.0f : both;
                    w0 = ex2(M - off);
                    w1 = ex2(m1 - off);
                    M = both;
                    l = l * w0 + sh.merge_l[quad * 32 + lane] * w1;
                    wild |= sh.merge_wild[quad] != 0;
                }
            }
            if (small) {  // the four warps' sums share a maximum and a row sum
                sh.quad_m[quad * 32 + lane] = M;
                sh.quad_l[quad * 32 + lane] = l;
                if (lane == 0) sh.quad_wild[quad] = wild;
                named_bar_sync(1, 128);
                float top = -INFINITY;
                for (int k = 0; k < 4; ++k) {
                    top = fmaxf(top, sh.quad_m[k * 32 + lane]);
                    wild |= sh.quad_wild[k] != 0;
                }
                const float off = top == -INFINITY ? 0.0f : top, w = ex2(M - off);
                w0 *= w;
                w1 *= w;
                M = top;
                l = 0.0f;
                for (int k = 0; k < 4; ++k) l = fmaf(ex2(sh.quad_m[k * 32 + lane] - off), sh.quad_l[k * 32 + lane], l);
            }
            const bool blank = !part && sees <= 0;  // zeros, whatever the sums hold
            if (!part) {
                const float inv = kSumScale / l;
                w0 *= inv;
                w1 *= inv;
            }
            float* dst = part ? part + (size_t)row * D
                              : p.out + (done.first + (valid ? token : 0)) * p.ld_out +
                                    (size_t)(done.head * G + sub) * D;
            const bool writes = valid && !wild && (!small || quad == 0);
            if (busy) {
#pragma unroll
                for (int o = 0; o < D; o += 16) {
                    int v[16];
                    if (merge) {
                        tmem_ld16(o0_addr + o, v);
                        tmem_ld_wait();
                    }
#pragma unroll
                    for (int x = 0; x < 8; ++x) {
                        float2 y = __fmul2_rn(acc[o / 2 + x], make_float2(w0, w0));
                        if (merge)
                            y = __ffma2_rn(make_float2(__int_as_float(v[2 * x]), __int_as_float(v[2 * x + 1])),
                                           make_float2(w1, w1), y);
                        acc[o / 2 + x] = blank ? make_float2(0.0f, 0.0f) : y;
                    }
                    if (small) {  // the first warp adds the others', 16 dims at a time
                        if (o) named_bar_sync(1, 128);
                        if (quad) {
#pragma unroll
                            for (int x = 0; x < 8; ++x) {
                                sh.quad_sum[quad - 1][lane][2 * x] = acc[o / 2 + x].x;
                                sh.quad_sum[quad - 1][lane][2 * x + 1] = acc[o / 2 + x].y;
                            }
                        }
                        named_bar_sync(1, 128);
                        if (!quad) {
#pragma unroll
                            for (int x = 0; x < 8; ++x)
#pragma unroll
                                for (int k = 0; k < 3; ++k)
                                    acc[o / 2 + x] = __fadd2_rn(
                                        acc[o / 2 + x], make_float2(sh.quad_sum[k][lane][2 * x],
                                                                    sh.quad_sum[k][lane][2 * x + 1]));
                        }
                    }
                    if (!writes) continue;
                    if (part || wide_out) {
#pragma unroll
                        for (int x = o / 2; x < o / 2 + 8; x += 2)
                            *reinterpret_cast<float4*>(dst + 2 * x) =
                                make_float4(acc[x].x, acc[x].y, acc[x + 1].x, acc[x + 1].y);
                    } else {
#pragma unroll
                        for (int x = o / 2; x < o / 2 + 8; ++x) {
                            dst[2 * x] = acc[x].x;
                            dst[2 * x + 1] = acc[x].y;
                        }
                    }
                }
                if (part && writes) {
                    part[kTileRows * D + row] = M;
                    part[kTileRows * (D + 1) + row] = l;
                }
                if (small) named_bar_sync(1, 128);  // the sums' buffer is free again
            }
            if (merge) {
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(b.merge_read + quad);
            }
            if (busy && wild)
                rows_without_operands<D>(p, done, from * NT, (from + take) * NT, part, &sh.watch);
        }
        if (tid == 0) splits[blockIdx.x] = split;
    } else if (count > 0) {
        set_registers_down<kOtherRegs>();  // idle
    } else if (tid == 0) {
        splits[blockIdx.x] = ChunkSplit{-1};
    }
    tc_fence_before();
    __syncthreads();
    if (warp == kIssueWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

// Operands of all K and V pages of a head: a warp a page, which it reads into
// shared memory, converts in place (the halves take as many bytes as the page) and
// writes to its part of the tile.  No warp waits for another; bound by HBM.
constexpr int kOperandWarps = 8;
template <int D>
__global__ void __launch_bounds__(kOperandWarps * 32) chunk_operands_kernel(ChunkParams p, Operands pre) {
    using S = Shape<D>;
    constexpr int PG = S::PG, kBlocks = 2 * PG / kOperandWarps;  // CTAs of a tile
    static_assert(kBlocks * kOperandWarps == 2 * PG, "a tile's pages");
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ uint64_t bar[kOperandWarps];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, head = blockIdx.y, s = blockIdx.z;
    const int tile = blockIdx.x / kBlocks, j = blockIdx.x % kBlocks * kOperandWarps + warp, page = j % PG;
    int first, n;
    rows_of(p, s, first, n);
    const int len = p.total_lens[s], limit = min(len, p.stride * kPageTokens);
    // (the units of a sequence without a position read its first tile too)
    if (n == 0 || tile * S::NT >= max(limit, 1) || len > pre.tiles * S::NT) return;
    const size_t t = operand_tile<D>(p, pre, s, head, tile);
    uint8_t* buf = smem + warp * S::kPageBytes;
    const int pos = tile * S::NT + page * kPageTokens, id = pos < limit ? page_at(p, s, pos) : -1;
    if (id >= 0) {
        if (lane == 0) {
            mbar_init(bar + warp, 1);
            fence_barrier_init();
            fence_proxy_async_shared();
            mbar_arrive_expect_tx(bar + warp, S::kPageBytes);
            bulk_g2s(buf, head_rows<D>(p, id, j / PG, head), S::kPageBytes, bar + warp);
        }
        __syncwarp();
        if (!mbar_wait(bar + warp, 0, p.err)) land_copies();
    }
    const int valid = id >= 0 ? min(limit - pos, kPageTokens) : 0;
    const float* src = reinterpret_cast<const float*>(buf);
    uint8_t* to = pre.ops + t * (4 * S::kHalf);
    constexpr int kPart = S::kPageBytes / 2;  // of the high halves, then of the low ones
    if (j < PG) {
        convert_k<D, 1>(src, valid, buf, buf + kPart, 0, 0, {}, pre.scales + t * 16 + page);
        to += page * kPart;
    } else {
        convert_v<D, kPageTokens, 1>(src, valid, buf, buf + kPart, 0, 0, {}, pre.scales + t * 16 + 8 + page);
        to += 2 * S::kHalf + page * 256;
    }
    __syncwarp();
#pragma unroll 4
    for (int i = lane; i < kPart / 16; i += 32) {
        const int at = j < PG ? i * 16 : i / 16 * (16 * S::NT) + i % 16 * 16;  // V: 256 bytes of every 8 dims
        *reinterpret_cast<uint4*>(to + at) = *reinterpret_cast<const uint4*>(buf + i * 16);
        *reinterpret_cast<uint4*>(to + S::kHalf + at) = *reinterpret_cast<const uint4*>(buf + kPart + i * 16);
    }
}

// The launches for a call's bounds, and their workspace: partial sums, what is
// split, and the operands where they are made beforehand.
struct ChunkPlan {
    bool whole;          // chunk_few_kernel by whole units
    int ctas, few_ctas;  // one per tile of work that the bounds allow, at most one per SM; 0: not launched
    int operand_tiles;   // of a sequence, 0: converted by the CTAs that read them
    size_t splits, few, few_splits, operands, scales, bytes;  // offsets, and all of it
};
ChunkPlan chunk_plan(long long rows, long long batch, long long max_new, long long max_len, int H, int Hkv, int d) {
    const long long G = H / Hkv, per = kTileRows / G, nt = d == 128 ? 64 : 128, len_tiles = (max_len + nt - 1) / nt;
    const auto most = [](long long n) { return std::min<long long>(n, kChunkCtas); };
    const auto ctas = [&](long long tokens) {  // for units of so many tokens
        const long long units = std::min(batch * ((std::min(max_new, rows) + tokens - 1) / tokens), batch + rows / tokens);
        return (int)std::max<long long>(1, most(most(units) * most(Hkv) * most(len_tiles)));
    };
    constexpr int kWholePages = 2;
    ChunkPlan c{};
    // Sequences with at most eight rows of a KV head go to chunk_few_kernel.  Where
    // the bounds say that all have so few it takes them all, where they say that
    // the one sequence has more the tensor-core kernel does; else each takes its own.
    const bool few = G <= kFewRows && (max_new * G <= kFewRows || batch > 1);
    const bool many = !few || max_new * G > kFewRows;
    if (few) {
        // every warp has a share, of kFewPages pages or more
        const long long units = std::min(batch * ((std::min(max_new, rows) + kFewRows / G - 1) / (kFewRows / G)),
                                         batch + rows / (kFewRows / G));
        const auto many_pages = [](long long n) { return std::min<long long>(n, 1 << 16); };
        const long long pages = many_pages(units) * many_pages(Hkv) * many_pages((max_len + kPageTokens - 1) / kPageTokens);
        c.few_ctas = (int)std::max<long long>(1, most((pages + kFewPages - 1) / kFewPages));
        // A CTA takes whole units, and nothing is left to join, where a warp then has
        // kWholePages or fewer.  Measured, us by shares / by units, one sequence of 4 KV
        // heads of 64: 129 tokens (1 page) 16.9 / 10.2, 256 (1) 13.0 / 11.7, 512 (2) 13.4 /
        // 14.3, 1024 (4) 14.6 / 19.4; 9 sequences of 16 heads: 512 18.7 / 16.3, 1024 28 / 22.
        const int warps = d == 128 ? 8 : 16;
        c.whole = !many && units <= kChunkCtas && units * Hkv <= kChunkCtas &&
                  max_len <= (long long)kWholePages * warps * kPageTokens;
        if (c.whole) c.few_ctas = (int)(units * Hkv);
    }
    const int few_shares = c.whole ? 0 : c.few_ctas * (d == 128 ? 8 : 16);
    if (many) c.ctas = ctas(per);
    // Made beforehand where every K and V tile is read by so many row tiles or more
    // (as far as the bounds tell), a CTA has some tiles to pay for the launch, and the
    // operands fit kPreBytes.  Measured, us without / with:
    //   D = 128: 4 row tiles 226 / 253 and 125 / 132, 8 204 / 188 and 539 / 603, 16 342 / 286
    //   D = 64:  2 row tiles 78 / 87 and 56 / 62, 4 120 / 115 and 208 / 182, 8 190 / 165;
    //            of a CTA's two tiles, 4 row tiles 30 / 33
    //   D = 32:  4 row tiles 97 / 78
    const long long reuse = d == 128 ? 12 : 4;
    constexpr long long kPreTiles = 4, kPreBytes = 1ll << 30;
    const long long tile_bytes = 8 * nt * d + 64;
    const bool fits = batch <= 65535 && len_tiles <= (1 << 24) && batch * Hkv * len_tiles <= kPreBytes / tile_bytes;
    if (many && fits && rows / per >= reuse * batch && rows / per * most(Hkv) * len_tiles >= kPreTiles * kChunkCtas)
        c.operand_tiles = (int)len_tiles;
    const long long all_tiles = batch * Hkv * c.operand_tiles;
    const auto up = [](size_t n) { return (n + 127) & ~(size_t)127; };
    c.splits = c.ctas * 2 * partial_floats(kTileRows, d) * sizeof(float);
    c.few = up(c.splits + c.ctas * sizeof(ChunkSplit));
    c.few_splits = c.few + few_shares * 2 * partial_floats(kFewRows, d) * sizeof(float);
    c.operands = up(c.few_splits + few_shares * sizeof(ChunkSplit));
    c.scales = c.operands + (size_t)all_tiles * 8 * nt * d;
    c.bytes = c.scales + (size_t)all_tiles * 64;
    return c;
}

bool wide_output(const ChunkParams& p) { return p.ld_out % 4 == 0 && aligned_to(p.out, 16); }

template <int D, bool PRE>
cudaError_t launch_tiles(const ChunkParams& p, const ChunkPlan& plan, float* partials, ChunkSplit* splits,
                         const Operands& pre, cudaStream_t stream) {
    const bool wide_q = p.ld_q % 4 == 0 && aligned_to(p.q, 16), wide_out = wide_output(p);
    cudaError_t e = kernel_attributes<chunk_tiles_kernel<D, PRE>>(Shape<D>::template kSmem<PRE>, Roles<PRE>::kLaunchRegs);
    if (e != cudaSuccess) return e;
    chunk_tiles_kernel<D, PRE><<<plan.ctas, Roles<PRE>::kThreads, Shape<D>::template kSmem<PRE>, stream>>>(p, partials, splits, pre,
                                                                                               wide_q, wide_out);
    return cudaGetLastError();
}

template <int D>
cudaError_t launch_chunk(ChunkParams p, const ChunkPlan& plan, void* workspace, cudaStream_t stream) {
    uint8_t* w = static_cast<uint8_t*>(workspace);
    cudaError_t e = cudaSuccess;
    if (plan.few_ctas) {
        float* partials = reinterpret_cast<float*>(w + plan.few);
        ChunkSplit* splits = reinterpret_cast<ChunkSplit*>(w + plan.few_splits);
        p.rows_upto = plan.ctas ? kFewRows : INT_MAX;
        if (plan.whole) {
            e = kernel_attributes<chunk_few_kernel<D, true>>(Few<D>::kSmem);
            if (e != cudaSuccess) return e;
            chunk_few_kernel<D, true><<<plan.few_ctas, Few<D>::kThreads, Few<D>::kSmem, stream>>>(p, nullptr, nullptr);
            return cudaGetLastError();
        }
        e = kernel_attributes<chunk_few_kernel<D, false>>(Few<D>::kSmem);
        if (e != cudaSuccess) return e;
        chunk_few_kernel<D, false><<<plan.few_ctas, Few<D>::kThreads, Few<D>::kSmem, stream>>>(p, partials, splits);
        e = cudaGetLastError();
        if (e == cudaSuccess)
            e = launch_combine<D, kFewRows>(p, plan.few_ctas * Few<D>::kWarps, partials, splits, wide_output(p), 1.0f,
                                            stream);
        p.rows_above = kFewRows;
        p.rows_upto = INT_MAX;
    }
    if (e != cudaSuccess || !plan.ctas) return e;
    float* partials = reinterpret_cast<float*>(w);
    ChunkSplit* splits = reinterpret_cast<ChunkSplit*>(w + plan.splits);
    const Operands pre{w + plan.operands, reinterpret_cast<float*>(w + plan.scales), plan.operand_tiles};
    if (plan.operand_tiles) {
        const size_t smem = kOperandWarps * Shape<D>::kPageBytes;
        e = kernel_attributes<chunk_operands_kernel<D>>(smem);
        if (e != cudaSuccess) return e;
        const unsigned blocks = (unsigned)plan.operand_tiles * (2 * Shape<D>::PG / kOperandWarps);
        chunk_operands_kernel<D><<<dim3(blocks, (unsigned)p.Hkv, (unsigned)p.batch), kOperandWarps * 32, smem, stream>>>(
            p, pre);
        e = cudaGetLastError();
        if (e == cudaSuccess) e = launch_tiles<D, true>(p, plan, partials, splits, pre, stream);
    } else {
        e = launch_tiles<D, false>(p, plan, partials, splits, pre, stream);
    }
    if (e != cudaSuccess) return e;
    return launch_combine<D, kTileRows>(p, plan.ctas, partials, splits, wide_output(p), kSumScale, stream);
}

}  // namespace
}  // namespace tb

using namespace tb;

static tb_status check_chunk(int rows, int batch, int max_new, int max_len, int H, int Hkv, int d) {
    TB_ENTRY_CHECK(rows >= 0 && batch >= 1 && max_new >= 1 && max_len >= 1, "bad rows / batch / lengths");
    TB_ENTRY_CHECK(H >= 1 && Hkv >= 1 && H % Hkv == 0 && Hkv <= 65535, "heads must divide: H %d, Hkv %d", H, Hkv);
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
        *bytes = (int64_t)chunk_plan(rows, batch, max_new, max_len, H, Hkv, d).bytes;
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
    const ChunkPlan plan = chunk_plan(rows, batch, max_new, max_len, H, Hkv, d);
    TB_ENTRY_CHECK(plan.bytes == 0 ||
                       (workspace && aligned_to(workspace, 16) && workspace_bytes >= (int64_t)plan.bytes),
                   "the workspace must be 16-byte aligned and hold %lld bytes", (long long)plan.bytes);
    StreamEntry entry(pool, "kv_pool");
    if (entry.status != TB_OK) return entry.status;
    ChunkParams p{q, ld_q, row_offsets, total_lens, batch, rows, pool, num_pages, table, stride, layer, num_layers, H,
                  Hkv, 0, INT_MAX, out, ld_out, entry.err};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    cudaError_t e = d == 16   ? launch_chunk<16>(p, plan, workspace, s)
                    : d == 32 ? launch_chunk<32>(p, plan, workspace, s)
                    : d == 64 ? launch_chunk<64>(p, plan, workspace, s)
                              : launch_chunk<128>(p, plan, workspace, s);
    return launch_status(e, "chunk attention launch");
}
