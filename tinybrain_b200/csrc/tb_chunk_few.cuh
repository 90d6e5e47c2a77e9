// tb_chunk_few.cuh -- chunk attention for sequences with at most eight rows of a
// KV head (one token of eight query heads, eight tokens of one): decode.
//
// The work is reading K and V once; eight rows leave a 128-row tensor-core tile
// empty, and making its operands costs more than the products.  Here every warp
// streams its own pages (every 16th of a unit, 8th for D = 128) through its own
// ring of bulk copies and needs no other warp until the unit ends:
//   scores  mma.sync m16n8k8 on the fp32 page as it lies: A = 16 tokens, B = the
//           rows' queries from registers, both split into a TF32 high part and
//           the rest (3 products in separate chains, the small ones apart);
//   weights base-2, relative to a maximum that moves only when a score exceeds
//           it by 2^8 (one vote a page);
//   sums    V in plain fp32 FMAs: a lane holds D / 32 dims of all rows, a row of
//           V is one conflict-free load, the weights are broadcast loads.
// At a unit's end the warps' sums meet in shared memory.  The dims of a lane in
// the scores' products are four neighbours: k is a label, the same for A and B.
//
// Bound by HBM: a 16-token page of K and V takes a warp about 450 instructions,
// a quarter of what the SM could issue while they arrive.
#pragma once

#include "tb_chunk_units.cuh"

namespace tb {
namespace {

constexpr int kFewRows = 8;

template <int D>
struct Few {
    static constexpr int NT = D == 128 ? 64 : 128, PG = NT / kPageTokens;
    static constexpr int kWarps = D == 128 ? 8 : 16, kThreads = kWarps * 32;
    static constexpr int kPageBytes = kPageTokens * D * 4;
    static constexpr int kRing = D >= 64 ? 3 : D == 32 ? 6 : 8;  // pages of a warp on their way
    static constexpr int kLaneDims = D < 32 ? 1 : D / 32;
    static constexpr int kSumDims = D < 32 ? D : 32;  // dims of a round of the final sum
    static constexpr size_t kSmem = (size_t)kWarps * kRing * kPageBytes;
};

template <int D>
struct FewShared {
    using F = Few<D>;
    alignas(16) float weight[F::kWarps][kPageTokens][kFewRows];
    float sum[F::kWarps][kFewRows][F::kSumDims + 1];
    float m[F::kWarps][kFewRows], l[F::kWarps][kFewRows];
    float inverse[kFewRows];  // of the rows' sums
    int wild[F::kWarps];
    uint64_t full[F::kWarps][F::kRing];
    int id[F::kWarps][F::kRing];
    ShareShared share;
    volatile int dead;
};

__device__ __forceinline__ void mma_tf32(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// The high part keeps TF32's 11 bits (rounded up by half a step, then cut), the
// rest is exact; the product reads 11 bits of it: 2^-22 of the value is lost.
__device__ __forceinline__ void split_tf32(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xffffe000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
}
__device__ __forceinline__ float few_ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// The pages of the CTA's share that a warp takes, in order.
template <int D>
struct WarpPages {
    using F = Few<D>;
    Unit u;
    int at, take, left;  // the piece's first tile and tiles, the tiles after it
    int page, end;       // the warp's page and the end of the piece's pages
    int ids, base;       // lane l: the pool page of page base + l * warps

    __device__ void piece(const ChunkParams& p, int warp) {
        take = min(u.tiles - at, left);
        left -= take;
        page = at * F::PG + warp;
        end = min((at + take) * F::PG, (u.limit + kPageTokens - 1) / kPageTokens);
        load(p);
    }
    __device__ void load(const ChunkParams& p) {
        base = page;
        const int mine = base + (threadIdx.x & 31) * F::kWarps;
        ids = mine < end ? checked_page(p, p.table[(size_t)u.s * p.stride + mine]) : -1;
    }
    __device__ bool next_piece(const ChunkParams& p, int warp) {
        if (left == 0) return false;
        next_unit<F::NT, kFewRows>(p, u);
        at = 0;
        piece(p, warp);
        return true;
    }
    // to the next page, over pieces without one; false: none is left
    __device__ bool settle(const ChunkParams& p, int warp) {
        while (page >= end)
            if (!next_piece(p, warp)) return false;
        if (page - base >= 32 * F::kWarps) load(p);
        return true;
    }
    __device__ int id() const { return __shfl_sync(0xffffffffu, ids, (page - base) / F::kWarps); }
};

template <int D>
__global__ void __launch_bounds__(Few<D>::kThreads, 1)
    chunk_few_kernel(ChunkParams p, float* partials, ChunkSplit* splits) {
    using F = Few<D>;
    constexpr int kSteps = D / 8, kRing = F::kRing, kDims = F::kLaneDims;
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ FewShared<D> sh;
    static_assert(F::kSmem + sizeof(FewShared<D>) <= 227 * 1024, "shared memory");
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, tig = lane & 3;
    uint8_t* ring = smem + (size_t)warp * kRing * F::kPageBytes;
    if (lane == 0) {
        for (int i = 0; i < kRing; ++i) mbar_init(&sh.full[warp][i], 1);
        if (warp == 0) sh.dead = 0;
        fence_barrier_init();
        fence_proxy_async_shared();
    }
    const Share share = find_share<F::NT, kFewRows, F::kThreads>(p, sh.share);
    __syncthreads();
    pdl_launch_dependents();
    if (share.count == 0) {
        if (tid == 0) splits[blockIdx.x] = ChunkSplit{0, 0, 0, -1};
        return;
    }
    const int G = p.H / p.Hkv, per = kFewRows / G;
    ChunkSplit split{0, 0, 0, -1};

    // K and V pages alternate through the ring; `fetch` runs ahead of the pieces
    WarpPages<D> fetch, now;
    fetch.u = now.u = sh.share.start;
    fetch.at = now.at = sh.share.tile;
    fetch.left = now.left = share.count;
    fetch.piece(p, warp);
    now.piece(p, warp);
    bool more = fetch.settle(p, warp);
    int fetch_kv = 0, fetch_slot = 0, held = 0;  // held: pages fetched and not yet read
    int slot = 0, phase = 0;
    const auto fill = [&]() {
        while (more && held < kRing && !sh.dead) {
            const int id = fetch.id();
            if (lane == 0) {
                uint64_t* bar = &sh.full[warp][fetch_slot];
                sh.id[warp][fetch_slot] = id;
                mbar_arrive_expect_tx(bar, id >= 0 ? F::kPageBytes : 0);
                if (id >= 0)
                    bulk_g2s(ring + fetch_slot * F::kPageBytes, head_rows<D>(p, id, fetch_kv, fetch.u.head),
                             F::kPageBytes, bar);
            }
            ++held;
            if (++fetch_slot == kRing) fetch_slot = 0;
            if (fetch_kv) {
                fetch.page += F::kWarps;
                more = fetch.settle(p, warp);
            }
            fetch_kv ^= 1;
        }
    };
    // the next page in the ring; its pool page (-1: zeros)
    const auto take_page = [&](const float*& rows) {
        if (lane == 0) chunk_wait(&sh.dead, &sh.full[warp][slot], (uint32_t)phase, p.err);
        __syncwarp();
        rows = reinterpret_cast<const float*>(ring + slot * F::kPageBytes);
        return sh.id[warp][slot];
    };
    const auto done_page = [&]() {
        __syncwarp();
        --held;
        if (++slot == kRing) {
            slot = 0;
            phase ^= 1;
        }
        fill();
    };
    fill();

    while (true) {
        const Unit& u = now.u;
        // the rows' queries, times log2(e) / sqrt(D): B fragments (k = dims, n = rows)
        uint32_t qh[kSteps][2], ql[kSteps][2];
        {
            const int token = u.tile * per + g / G;
            const bool valid = g < per * G && token < u.n;
            const float* q = p.q + (u.first + (valid ? token : 0)) * p.ld_q + (size_t)(u.head * G + g % G) * D;
            const float scale = 1.4426950408889634f * rsqrtf((float)D);
#pragma unroll
            for (int b = 0; b < D / 16; ++b)
#pragma unroll
                for (int x = 0; x < 4; ++x)
                    split_tf32(valid ? q[16 * b + 4 * tig + x] * scale : 0.0f, qh[2 * b + x / 2][x % 2],
                               ql[2 * b + x / 2][x % 2]);
        }
        // what rows 2 tig and 2 tig + 1 see, and the least that a row of the unit does
        const int held_tokens = u.len - u.n + u.tile * per;
        int sees[2];
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            const int r = 2 * tig + x, token = u.tile * per + r / G;
            sees[x] = r < per * G && token < u.n ? min(held_tokens + r / G + 1, u.limit) : u.limit;
        }
        const int rows = min(per, u.n - u.tile * per) * G, all_see = min(held_tokens + 1, u.limit);
        float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.0f, 0.0f};
        float acc[kFewRows][kDims];
#pragma unroll
        for (int r = 0; r < kFewRows; ++r)
#pragma unroll
            for (int d = 0; d < kDims; ++d) acc[r][d] = 0.0f;
        bool wild = false;
        float(*weight)[kFewRows] = sh.weight[warp];
        for (; now.page < now.end; now.page += F::kWarps) {
            const int pos0 = now.page * kPageTokens;
            const float* rows_k;
            const int id = take_page(rows_k);
            float c[4] = {0, 0, 0, 0};
            if (id >= 0) {
                float c1[4] = {0, 0, 0, 0}, c2[4] = {0, 0, 0, 0};
#pragma unroll
                for (int b = 0; b < D / 16; ++b) {
                    const float4 x = lds128f(rows_k + g * D + 16 * b + 4 * tig);
                    const float4 y = lds128f(rows_k + (g + 8) * D + 16 * b + 4 * tig);
                    uint32_t ah[4], al[4];
                    split_tf32(x.x, ah[0], al[0]);
                    split_tf32(y.x, ah[1], al[1]);
                    split_tf32(x.y, ah[2], al[2]);
                    split_tf32(y.y, ah[3], al[3]);
                    mma_tf32(c1, al, qh[2 * b][0], qh[2 * b][1]);
                    mma_tf32(c2, ah, ql[2 * b][0], ql[2 * b][1]);
                    mma_tf32(c, ah, qh[2 * b][0], qh[2 * b][1]);
                    split_tf32(x.z, ah[0], al[0]);
                    split_tf32(y.z, ah[1], al[1]);
                    split_tf32(x.w, ah[2], al[2]);
                    split_tf32(y.w, ah[3], al[3]);
                    mma_tf32(c1, al, qh[2 * b + 1][0], qh[2 * b + 1][1]);
                    mma_tf32(c2, ah, ql[2 * b + 1][0], ql[2 * b + 1][1]);
                    mma_tf32(c, ah, qh[2 * b + 1][0], qh[2 * b + 1][1]);
                }
#pragma unroll
                for (int x = 0; x < 4; ++x) c[x] += c1[x] + c2[x];
            }
            done_page();
            // c[0], c[1]: token g, rows 2 tig, 2 tig + 1; c[2], c[3]: token g + 8
            const bool masked = all_see < pos0 + kPageTokens;
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const bool vis = !masked || pos0 + g + (x / 2) * 8 < sees[x % 2];
                wild |= vis && !(fabsf(c[x]) <= 3.4028234e38f);
                if (!vis) c[x] = -INFINITY;
            }
            float top[2] = {fmaxf(c[0], c[2]), fmaxf(c[1], c[3])};
            bool grow = false;
#pragma unroll
            for (int x = 0; x < 2; ++x) grow |= top[x] > m[x] + 8.0f || (m[x] == -INFINITY && top[x] > -INFINITY);
            if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                for (int x = 0; x < 2; ++x) {
                    for (int o = 4; o < 32; o <<= 1) top[x] = fmaxf(top[x], __shfl_xor_sync(0xffffffffu, top[x], o));
                    const float next = fmaxf(m[x], top[x]);
                    const float r = m[x] == -INFINITY ? 0.0f : few_ex2(m[x] - next);
                    m[x] = next;
                    l[x] *= r;
                    if (g == 0) weight[0][2 * tig + x] = r;
                }
                __syncwarp();
#pragma unroll
                for (int r = 0; r < kFewRows; ++r)
#pragma unroll
                    for (int d = 0; d < kDims; ++d) acc[r][d] *= weight[0][r];
                __syncwarp();
            }
            float w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) w[x] = few_ex2(c[x] - (m[x % 2] == -INFINITY ? 0.0f : m[x % 2]));
            l[0] += w[0] + w[2];
            l[1] += w[1] + w[3];
            *reinterpret_cast<float2*>(&weight[g][2 * tig]) = make_float2(w[0], w[1]);
            *reinterpret_cast<float2*>(&weight[g + 8][2 * tig]) = make_float2(w[2], w[3]);
            const float* rows_v;
            const int id_v = take_page(rows_v);  // (its barrier orders the weights too)
            if (id_v >= 0 && (D >= 32 || lane < D)) {
                const int tokens = min(kPageTokens, u.limit - pos0);
                const auto load_v = [&](int t, float (&v)[kDims]) {
                    const float* at = rows_v + t * D + lane * kDims;
                    if constexpr (kDims == 4) {
                        const float4 f = lds128f(at);
                        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
                    } else if constexpr (kDims == 2) {
                        const float2 f = *reinterpret_cast<const float2*>(at);
                        v[0] = f.x, v[1] = f.y;
                    } else {
                        v[0] = at[0];
                    }
                };
                if (!masked) {
#pragma unroll 4
                    for (int t = 0; t < kPageTokens; ++t) {
                        float v[kDims];
                        load_v(t, v);
                        const float4 w0 = lds128f(&weight[t][0]), w1 = lds128f(&weight[t][4]);
                        const float ws[8] = {w0.x, w0.y, w0.z, w0.w, w1.x, w1.y, w1.z, w1.w};
#pragma unroll
                        for (int r = 0; r < kFewRows; ++r)
#pragma unroll
                            for (int d = 0; d < kDims; ++d) acc[r][d] = fmaf(ws[r], v[d], acc[r][d]);
                    }
                } else {  // what a row does not see may be anything
#pragma unroll 1
                    for (int t = 0; t < tokens; ++t) {
                        float v[kDims];
                        load_v(t, v);
#pragma unroll
                        for (int r = 0; r < kFewRows; ++r) {
                            if (r >= rows || pos0 + t >= held_tokens + r / G + 1) continue;
#pragma unroll
                            for (int d = 0; d < kDims; ++d) acc[r][d] = fmaf(weight[t][r], v[d], acc[r][d]);
                        }
                    }
                }
            }
            done_page();
        }

        // ---- the unit's end: the warps' sums on a common maximum ----
#pragma unroll
        for (int x = 0; x < 2; ++x) {
            for (int o = 4; o < 32; o <<= 1) l[x] += __shfl_xor_sync(0xffffffffu, l[x], o);
            if (g == 0) {
                sh.m[warp][2 * tig + x] = m[x];
                sh.l[warp][2 * tig + x] = l[x];
            }
        }
        wild = __any_sync(0xffffffffu, wild);
        if (lane == 0) sh.wild[warp] = wild;
        __syncthreads();
        float top = -INFINITY;
        for (int k = lane >> 3; k < F::kWarps; k += 4) {
            top = fmaxf(top, sh.m[k][lane & 7]);
            wild |= sh.wild[k] != 0;
        }
        wild = __any_sync(0xffffffffu, wild);
        for (int o = 8; o < 32; o <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        const float off = top == -INFINITY ? 0.0f : top;
        float all = 0.0f;
        for (int k = lane >> 3; k < F::kWarps; k += 4)
            all = fmaf(few_ex2(sh.m[k][lane & 7] - off), sh.l[k][lane & 7], all);
        for (int o = 8; o < 32; o <<= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
        const float mine = few_ex2(sh.m[warp][lane & 7] - off);  // of row lane % 8
        if (warp == 0 && lane < kFewRows) sh.inverse[lane] = 1.0f / all;
        const bool whole = now.at == 0 && now.take == u.tiles;
        float* part = nullptr;
        if (!whole) {
            part = partials + ((size_t)blockIdx.x * 2 + (now.at == 0)) * partial_floats(kFewRows, D);
            if (now.at == 0) split = ChunkSplit{u.s, u.tile, u.head, share.followers(u.tiles - now.take)};
        }
#pragma unroll
        for (int r = 0; r < kFewRows; ++r) {
            const float f = __shfl_sync(0xffffffffu, mine, r);
#pragma unroll
            for (int d = 0; d < kDims; ++d) acc[r][d] *= f;
        }
#pragma unroll 1
        for (int o = 0; o < D; o += F::kSumDims) {
            const int d0 = lane * kDims - o;
            if (d0 >= 0 && d0 < F::kSumDims)
#pragma unroll
                for (int r = 0; r < kFewRows; ++r)
#pragma unroll
                    for (int d = 0; d < kDims; ++d) sh.sum[warp][r][d0 + d] = acc[r][d];
            __syncthreads();
            for (int e = tid; e < kFewRows * F::kSumDims; e += F::kThreads) {
                const int r = e / F::kSumDims, d = e % F::kSumDims;
                float x = 0.0f;
#pragma unroll
                for (int k = 0; k < F::kWarps; ++k) x += sh.sum[k][r][d];
                if (r < rows && !wild) {
                    if (part) {
                        part[r * D + o + d] = x;
                    } else {
                        const int token = u.tile * per + r / G;
                        p.out[(u.first + token) * p.ld_out + (size_t)(u.head * G + r % G) * D + o + d] =
                            held_tokens + r / G + 1 > 0 ? x * sh.inverse[r] : 0.0f;
                    }
                }
            }
            __syncthreads();
        }
        if (part && warp == 0 && lane < rows && !wild) {
            part[kFewRows * D + lane] = top;
            part[kFewRows * (D + 1) + lane] = all;
        }
        if (wild)
            for (int r = warp; r < rows; r += F::kWarps)
                row_in_fp32<D, kFewRows>(p, u, r, now.at * F::NT, (now.at + now.take) * F::NT, part, 0.0f);
        __syncthreads();  // the sums' buffers are free again
        if (!now.next_piece(p, warp)) break;
    }
    if (tid == 0) splits[blockIdx.x] = split;
    if (sh.dead) land_copies();
}

}  // namespace
}  // namespace tb
