// tb_chunk_few.cuh -- chunk attention for sequences with at most eight rows of a
// KV head (one token of eight query heads, eight tokens of one): decode.
//
// The work is reading K and V once; eight rows leave a 128-row tensor-core tile
// empty, and making its operands costs more than the products.  Here every warp
// takes an equal share of all pages of all units, streams them through its own
// ring of bulk copies and waits for no other warp; units that several warps hold
// are joined by chunk_combine_kernel.  (In the 64-sequence step below, sixteen warps
// on one unit after the other, joined at each one's end, spent a fifth of their time
// at that barrier.)  WHOLE, for so little work that a second launch would cost more:
// the warps of a CTA do share a unit's pages and join them at its end.
// Per page of 16 tokens:
//   scores  mma.sync m16n8k8 on the fp32 page as it lies: A = 16 tokens, B = the
//           rows' queries from registers, both split into a TF32 high part and
//           the rest (3 products in separate chains, the small ones apart);
//   weights base-2, relative to a maximum that moves only when a score exceeds
//           it by 2^8 (one vote a page);
//   sums    V in plain fp32 FMAs: a lane holds D / 32 dims of all rows, a row of
//           V is one conflict-free load, the weights are broadcast loads.
// Bound by issue slots (45 % of the cycles) beside HBM.  Measured: 64 sequences of 512
// to 4224 tokens, 32 query and 4 KV heads of 64, 69 us for 290 MB, 4.2 TB/s; WHOLE, one
// token over 129 positions, 10 us.
// The dims of a lane in the scores' products are four neighbours: k is a label,
// the same for A and B.
#pragma once

#include "tb_chunk_units.cuh"

namespace tb {
namespace {

constexpr int kFewRows = 8;

template <int D>
struct Few {
    static constexpr int kWarps = D == 128 ? 8 : 16, kThreads = kWarps * 32;
    static constexpr int kPageBytes = kPageTokens * D * 4;
    static constexpr int kRing = D >= 64 ? 3 : D == 32 ? 6 : 8;  // pages of a warp on their way
    static constexpr int kLaneDims = D < 32 ? 1 : D / 32;
    static constexpr size_t kSmem = (size_t)kWarps * kRing * kPageBytes;
};
constexpr int kFewPages = 2;  // least pages of a share

template <int D>
struct FewShared {
    using F = Few<D>;
    alignas(16) float weight[F::kWarps][kPageTokens][kFewRows];
    uint64_t full[F::kWarps][F::kRing];
    int id[F::kWarps][F::kRing];
    long long scan[F::kWarps], before[F::kThreads], mine[F::kThreads];
    ChunkWatch watch;
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

// A warp's share of the pages, in order: units' pages are tiles of 16 positions.
struct WarpPages {
    Unit u;
    int page, end, left;  // the next page, the end of the piece's, and the pages after the piece
    int ids, base;        // lane l: the pool page of page base + l

    __device__ __forceinline__ void piece(const ChunkParams& p, int from) {
        page = from;
        end = min(u.tiles, from + left);
        left -= end - from;
        load(p);
    }
    __device__ __forceinline__ void load(const ChunkParams& p) {
        base = page;
        const int mine = base + (threadIdx.x & 31);  // (a unit without positions has one page, all of it beyond)
        ids = mine < end && mine * kPageTokens < u.limit
                  ? checked_page(p, p.table[(size_t)u.s * p.stride + mine])
                  : -1;
    }
    __device__ __forceinline__ bool next_piece(const ChunkParams& p) {
        if (left == 0) return false;
        next_unit<kPageTokens, kFewRows>(p, u);
        piece(p, 0);
        return true;
    }
    __device__ __forceinline__ bool next_page(const ChunkParams& p) {
        if (++page == end) return next_piece(p);
        if (page - base == 32) load(p);
        return true;
    }
    __device__ __forceinline__ int id() const { return __shfl_sync(0xffffffffu, ids, page - base); }
};

template <int D, bool WHOLE>
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
        if (warp == 0) watch_init(sh.watch);
        fence_barrier_init();
        fence_proxy_async_shared();
    }

    // ---- the work: the warp's share of all units' pages (shares w, w + CTAs, ... fall to
    //      one CTA, so that few pages spread over the SMs), or WHOLE the CTA's units ----
    const int G = p.H / p.Hkv, per = kFewRows / G;
    const int run = (p.batch + F::kThreads - 1) / F::kThreads;
    const auto work_of = [&](int s) -> long long {
        if (!WHOLE) return tiles_of_sequence<kPageTokens, kFewRows>(p, s);
        int first, n;
        rows_of(p, s, first, n);
        return (long long)((n + per - 1) / per) * p.Hkv;
    };
    long long mine = 0;
    {
        const int s0 = min(tid * run, p.batch), s1 = min(s0 + run, p.batch);
        for (int s = s0; s < s1; ++s) {
            mine += work_of(s);
            int first, n;
            rows_of(p, s, first, n);
            if (n && p.total_lens[s] > p.stride * kPageTokens) record_error(p.err, kDevBadPage);
        }
    }
    long long upto = mine;
    for (int o = 1; o < 32; o <<= 1) {
        const long long t = __shfl_up_sync(0xffffffffu, upto, o);
        if (lane >= o) upto += t;
    }
    if (lane == 31) sh.scan[warp] = upto;
    __syncthreads();
    Share share;
    share.total = 0;
    for (int w = 0; w < F::kWarps; ++w) {
        if (w < warp) upto += sh.scan[w];
        share.total += sh.scan[w];
    }
    sh.before[tid] = upto - mine;
    sh.mine[tid] = mine;
    __syncthreads();
    if (!WHOLE) pdl_launch_dependents();
    share.index = WHOLE ? blockIdx.x : warp * gridDim.x + blockIdx.x;
    share.shares = min((long long)gridDim.x * F::kWarps, (share.total + kFewPages - 1) / kFewPages);
    if (share.index >= (WHOLE ? share.total : share.shares)) {
        if (!WHOLE && lane == 0) splits[share.index] = ChunkSplit{-1};
        return;
    }
    WarpPages fetch, now;
    const auto seek = [&](long long begin) {  // the unit that holds it, and the place in its sequence's work
        int holder = 0;
        for (int t = lane; t < F::kThreads; t += 32) {
            const bool has = sh.before[t] <= begin && begin < sh.before[t] + sh.mine[t];
            if (has) holder = t + 1;
        }
        holder = max(__reduce_max_sync(0xffffffffu, holder) - 1, 0);
        long long at = begin - sh.before[holder];
        Unit& u = now.u;
        for (u.s = min(holder * run, p.batch - 1);; ++u.s) {
            const long long here = run == 1 || u.s + 1 >= p.batch ? LLONG_MAX : work_of(u.s);
            if (at < here) break;
            at -= here;
        }
        set_sequence(p, u);
        return at;
    };
    if (!WHOLE) {
        const long long begin = share.total * share.index / share.shares;
        share.end = share.total * (share.index + 1) / share.shares;
        long long at = seek(begin);
        Unit& u = now.u;
        for (u.tile = 0;; ++u.tile) {
            set_tile<kPageTokens, kFewRows>(p, u);
            if (at < (long long)u.tiles * p.Hkv) break;
            at -= (long long)u.tiles * p.Hkv;
        }
        u.head = (int)(at / u.tiles);
        now.left = (int)(share.end - begin);
        now.piece(p, (int)(at % u.tiles));
        fetch = now;
    }
    ChunkSplit split{-1};

    // K and V pages alternate through the ring; `fetch` runs ahead of `now`
    bool more = !WHOLE;
    int fetch_kv = 0, fetch_slot = 0, held = 0;  // held: pages fetched and not yet read
    int slot = 0, phase = 0;
    const size_t page_floats = (size_t)p.num_layers * 2 * p.Hkv * (kPageTokens * D);
    const float* fetch_at = nullptr;  // page 0's rows of fetch's head, K
    int fetch_id = -1;
    const auto fetch_next = [&]() {
        if (fetch_kv == 0) {
            fetch_id = fetch.id();
            fetch_at = head_rows<D>(p, 0, 0, fetch.u.head);
        }
        if (lane == 0) {
            uint64_t* bar = &sh.full[warp][fetch_slot];
            sh.id[warp][fetch_slot] = fetch_id;
            mbar_arrive_expect_tx(bar, fetch_id >= 0 ? F::kPageBytes : 0);
            if (fetch_id >= 0)
                bulk_g2s(ring + fetch_slot * F::kPageBytes,
                         fetch_at + fetch_id * page_floats + (fetch_kv ? p.Hkv * (kPageTokens * D) : 0), F::kPageBytes,
                         bar);
        }
        if (++fetch_slot == kRing) fetch_slot = 0;
        if (fetch_kv) more = fetch.next_page(p);
        fetch_kv ^= 1;
    };
    const auto fill = [&]() {
        for (; more && held < kRing; ++held) fetch_next();
    };
    // the next page in the ring; its pool page (-1: zeros)
    const auto take_page = [&](const float*& rows) {
        if (lane == 0) chunk_wait(&sh.watch, &sh.full[warp][slot], (uint32_t)phase, p.err);
        __syncwarp();
        rows = reinterpret_cast<const float*>(ring + slot * F::kPageBytes);
        return sh.id[warp][slot];
    };
    const auto done_page = [&]() {
        __syncwarp();
        if (++slot == kRing) {
            slot = 0;
            phase ^= 1;
        }
        if (more && !sh.watch.dead)
            fetch_next();
        else
            --held;
    };
    // a WHOLE unit's partial sums, one warp's after the other's, over the ring
    float* const parts = reinterpret_cast<float*>(smem);
    constexpr int kPartStride = F::kSmem / F::kWarps / sizeof(float);
    static_assert(kPartStride >= (int)partial_floats(kFewRows, D), "a warp's sums in its ring");

    do {
        if (WHOLE) {  // pages T w / warps to T (w + 1) / warps of the CTA's unit
            const long long at = seek(share.index);
            Unit& u = now.u;
            u.tile = (int)(at / p.Hkv);
            u.head = (int)(at % p.Hkv);
            set_tile<kPageTokens, kFewRows>(p, u);
            const int begin = (int)((long long)u.tiles * warp / F::kWarps);
            now.left = (int)((long long)u.tiles * (warp + 1) / F::kWarps) - begin;
            more = now.left > 0;
            now.piece(p, begin);
            fetch = now;
        }
        fill();
        const Unit& u = now.u;
        const int from = now.page;
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
        float2 acc[kFewRows / 2][kDims];  // two rows side by side
#pragma unroll
        for (int r = 0; r < kFewRows / 2; ++r)
#pragma unroll
            for (int d = 0; d < kDims; ++d) acc[r][d] = make_float2(0.0f, 0.0f);
        bool wild = false;
        float(*weight)[kFewRows] = sh.weight[warp];
        for (; now.page < now.end; ++now.page) {
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
            if (masked) {
#pragma unroll
                for (int x = 0; x < 4; ++x) {
                    const bool vis = pos0 + g + (x / 2) * 8 < sees[x % 2];
                    wild |= vis && !(fabsf(c[x]) <= 3.4028234e38f);
                    if (!vis) c[x] = -INFINITY;
                }
            } else {  // (a sum is finite only if its terms are)
                wild |= !(fabsf(c[0] * 0.25f + c[1] * 0.25f) + fabsf(c[2] * 0.25f + c[3] * 0.25f) <= 3.4028234e38f);
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
                for (int r = 0; r < kFewRows / 2; ++r)
#pragma unroll
                    for (int d = 0; d < kDims; ++d)
                        acc[r][d] = __fmul2_rn(acc[r][d], make_float2(weight[0][2 * r], weight[0][2 * r + 1]));
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
                const auto add_token = [&](int t, const float4& w0, const float4& w1) {
                    const float* at = rows_v + t * D + lane * kDims;
                    float v[kDims];
                    if constexpr (kDims == 4) {
                        const float4 f = lds128f(at);
                        v[0] = f.x, v[1] = f.y, v[2] = f.z, v[3] = f.w;
                    } else if constexpr (kDims == 2) {
                        const float2 f = *reinterpret_cast<const float2*>(at);
                        v[0] = f.x, v[1] = f.y;
                    } else {
                        v[0] = at[0];
                    }
                    const float2 ws[4] = {make_float2(w0.x, w0.y), make_float2(w0.z, w0.w), make_float2(w1.x, w1.y),
                                          make_float2(w1.z, w1.w)};
#pragma unroll
                    for (int d = 0; d < kDims; ++d)
#pragma unroll
                        for (int r = 0; r < kFewRows / 2; ++r)
                            acc[r][d] = __ffma2_rn(ws[r], make_float2(v[d], v[d]), acc[r][d]);
                };
                if (!masked) {
#pragma unroll 4
                    for (int t = 0; t < kPageTokens; ++t)
                        add_token(t, lds128f(&weight[t][0]), lds128f(&weight[t][4]));
                } else {  // what a row does not see may be anything
#pragma unroll 1
                    for (int t = 0; t < tokens; ++t) {
                        const float* at = rows_v + t * D + lane * kDims;
#pragma unroll
                        for (int r = 0; r < kFewRows; ++r) {
                            if (r >= rows || pos0 + t >= held_tokens + r / G + 1) continue;
                            const float wr = weight[t][r];
#pragma unroll
                            for (int d = 0; d < kDims; ++d) {
                                float& a = r % 2 ? acc[r / 2][d].y : acc[r / 2][d].x;
                                a = fmaf(wr, at[d], a);
                            }
                        }
                    }
                }
            }
            done_page();
        }

        // ---- the piece's end: the unit's rows, or their partial sums ----
#pragma unroll
        for (int x = 0; x < 2; ++x)
            for (int o = 4; o < 32; o <<= 1) l[x] += __shfl_xor_sync(0xffffffffu, l[x], o);
        wild = __any_sync(0xffffffffu, wild);
        const bool whole = from == 0 && now.end == u.tiles;
        float* part = nullptr;
        if (WHOLE) {
            part = parts + warp * kPartStride;
        } else if (!whole) {
            part = partials + (share.index * 2 + (from == 0)) * partial_floats(kFewRows, D);
            if (from == 0) split = split_of<kFewRows>(p, u, share.followers(u.tiles - now.end));
        }
        if (WHOLE && from == now.end) {  // no page
        } else if (wild) {
            for (int r = 0; r < rows; ++r)
                row_in_fp32<D, kFewRows>(p, u, r, from * kPageTokens, now.end * kPageTokens, part, 0.0f, 1.0f);
        } else {
#pragma unroll
            for (int r = 0; r < kFewRows; ++r) {
                const float lr = __shfl_sync(0xffffffffu, r % 2 ? l[1] : l[0], r / 2);
                const float mr = __shfl_sync(0xffffffffu, r % 2 ? m[1] : m[0], r / 2);
                if (r >= rows) continue;
                const int token = u.tile * per + r / G;
                float* dst = part ? part + r * D
                                  : p.out + (u.first + token) * p.ld_out + (size_t)(u.head * G + r % G) * D;
                const bool some = held_tokens + r / G + 1 > 0;
                const float f = part ? 1.0f : 1.0f / lr;
                if (D >= 32 || lane < D) {
#pragma unroll
                    for (int d = 0; d < kDims; ++d) {
                        const float a = r % 2 ? acc[r / 2][d].y : acc[r / 2][d].x;
                        dst[lane * kDims + d] = part || some ? a * f : 0.0f;
                    }
                }
                if (part && lane == 0) {
                    part[kFewRows * D + r] = mr;
                    part[kFewRows * (D + 1) + r] = lr;
                }
            }
        }
        if (WHOLE) {
            __syncthreads();
            for (int e = tid; e < kFewRows * D / 4; e += F::kThreads) {
                const int r = e / (D / 4), d4 = e % (D / 4) * 4;
                if (r >= rows) continue;
                CombineSum<D> sum;
                sum.clear();
#pragma unroll 4
                for (int w = 0; w < F::kWarps; ++w) {
                    const float* at = parts + w * kPartStride;
                    if ((long long)u.tiles * w / F::kWarps < (long long)u.tiles * (w + 1) / F::kWarps)
                        sum.add(0, at[kFewRows * D + r], at[kFewRows * (D + 1) + r],
                                *reinterpret_cast<const float4*>(at + r * D + d4));
                }
                const float f = 1.0f / sum.l[0];
                const bool some = held_tokens + r / G + 1 > 0;
                float* dst = p.out + (u.first + u.tile * per + r / G) * p.ld_out + (size_t)(u.head * G + r % G) * D + d4;
                dst[0] = some ? sum.sum[0].x * f : 0.0f;
                dst[1] = some ? sum.sum[0].y * f : 0.0f;
                dst[2] = some ? sum.sum[0].z * f : 0.0f;
                dst[3] = some ? sum.sum[0].w * f : 0.0f;
            }
            share.index += gridDim.x;
            if (share.index >= share.total) break;
            fence_proxy_async_shared();  // the ring takes copies again
            __syncthreads();
        }
    } while (WHOLE || now.next_piece(p));
    if (!WHOLE && lane == 0) splits[share.index] = split;
    if (sh.watch.dead) land_copies();
}

}  // namespace
}  // namespace tb
