// tb_cache.cu -- filling the paged KV cache of a step without the host: page
// tables and slot maps from the sequences' lengths, and the write of rotated
// keys and values to their slots.
//
// The runner keeps its page tables on the host (KVCache.swift:108-356 restated
// in tb_runtime.cu) and fuses RoPE and the cache write into its QKV launch.
// These entries are the same steps for a caller that runs its own projections
// over the same pool layout and cannot stop for the host between steps.
#include "tb_common.cuh"
#include "tb_stream_entry.h"

namespace tb {
namespace {

// ---------------------------------------------------------------------------
// Page tables and slot maps.
//
// Sequence s holds ceil(c/16) pages and needs ceil((c+n)/16).  With the
// exclusive sums R_s of n and P_s of the pages taken, row R_s + i has position
// c + i, and logical page ceil(c/16) + j becomes free[P_s + j].  Nothing here
// needs more than those two sums, so every CTA forms them for the whole batch
// by itself (8 bytes a sequence out of L2) instead of waiting for another CTA
// or another launch, and then writes its own tile of 1024 rows or of 1024
// taken pages.  Inside a tile each sequence leaves a mark at its first row; a
// running maximum over the marks gives every row its sequence without a search.
// A row's page is looked up where it comes from (the table for pages held
// before, the free list for new ones), never in entries that another CTA
// writes.  Bound by latency: launch, two walks over the lengths, a block scan, a
// dependent load.  Measured: 64 sequences of one token 4.0 us, 4096 sequences with
// 200 thousand rows 8.1 us.
// ---------------------------------------------------------------------------
constexpr int kTabThreads = 512;
constexpr int kTabWarps = kTabThreads / 32;
constexpr int kTabTile = 1024;   // rows or taken pages of a CTA

struct TableParams {
    const int* cached;
    const int* fresh;
    int batch;
    const int* free_pages;
    int num_free;
    int* table;
    int stride;
    int max_rows;
    int row_tiles;
    bool wide;  // the lengths may be read four at a time
    int* row_offsets;
    int* total_lens;
    int* row_seq;
    int* row_pos;
    long long* row_slot;
    int* info;
};

__device__ __forceinline__ int pages_of(int n) { return (int)(((unsigned)n + kPageTokens - 1) / kPageTokens); }

__global__ void __launch_bounds__(kTabThreads) page_tables_kernel(TableParams p) {
    __shared__ long long scan_r[kTabWarps], scan_p[kTabWarps];
    __shared__ int red_bad[kTabWarps], scan_a[kTabWarps];
    __shared__ int mark_seq[kTabTile], mark_at[kTabTile], mark_base[kTabTile], mark_len[kTabTile];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;

    // 1. A thread adds up a run of sequences, four at a time (one by one the strided
    // reads took 11 us at 4096 sequences), and finds the first whose lengths cannot be
    // (negative, or longer than its table row).
    const int run = (p.batch + kTabThreads * 4 - 1) / (kTabThreads * 4) * 4;
    const int s0 = min(tid * run, p.batch), s1 = min(s0 + run, p.batch);
    const auto walk = [&](auto f) {
#pragma unroll 2
        for (int base = s0; base < s1; base += 4) {
            int4 c, n;
            if (p.wide && base + 4 <= s1) {
                c = *reinterpret_cast<const int4*>(p.cached + base);
                n = *reinterpret_cast<const int4*>(p.fresh + base);
            } else {
                const auto load = [&](const int* from, int k) { return base + k < s1 ? from[base + k] : 0; };
                c = make_int4(load(p.cached, 0), load(p.cached, 1), load(p.cached, 2), load(p.cached, 3));
                n = make_int4(load(p.fresh, 0), load(p.fresh, 1), load(p.fresh, 2), load(p.fresh, 3));
            }
            f(base, c.x, n.x);
            if (base + 1 < s1) f(base + 1, c.y, n.y);
            if (base + 2 < s1) f(base + 2, c.z, n.z);
            if (base + 3 < s1) f(base + 3, c.w, n.w);
        }
    };
    long long rows = 0, taken = 0;
    int bad = INT32_MAX;
    walk([&](int s, int c, int n) {
        if (c < 0 || n < 0 || (long long)c + n > (long long)p.stride * kPageTokens) {
            bad = min(bad, s);
            return;
        }
        rows += n;
        taken += pages_of(c + n) - pages_of(c);
    });
    // 2. the sums before the thread's run, and all of them
    long long ir = rows, ip = taken;
    for (int o = 1; o < 32; o <<= 1) {
        const long long a = __shfl_up_sync(0xffffffffu, ir, o), b = __shfl_up_sync(0xffffffffu, ip, o);
        if (lane >= o) {
            ir += a;
            ip += b;
        }
    }
    bad = __reduce_min_sync(0xffffffffu, bad);
    if (lane == 31) {
        scan_r[warp] = ir;
        scan_p[warp] = ip;
        red_bad[warp] = bad;
    }
    for (int i = tid; i < kTabTile; i += kTabThreads) mark_seq[i] = -1;
    __syncthreads();
    long long r = ir - rows, q = ip - taken;
    rows = taken = 0;
#pragma unroll
    for (int w = 0; w < kTabWarps; ++w) {
        if (w < warp) {
            r += scan_r[w];
            q += scan_p[w];
        }
        rows += scan_r[w];
        taken += scan_p[w];
        bad = min(bad, red_bad[w]);
    }
    const int status = bad != INT32_MAX ? TB_PAGES_BAD_LENGTH
                       : rows > p.max_rows ? TB_PAGES_ROWS_EXCEEDED
                       : taken > p.num_free ? TB_PAGES_EXHAUSTED
                                            : TB_PAGES_OK;
    if (blockIdx.x == 0 && tid == 0) {
        p.info[0] = status ? 0 : (int)rows;
        p.info[1] = status ? 0 : (int)taken;
        p.info[2] = status;
        p.info[3] = status == TB_PAGES_BAD_LENGTH ? bad : -1;
        p.row_offsets[p.batch] = status ? 0 : (int)rows;
    }
    const bool row_tile = (int)blockIdx.x < p.row_tiles;
    const int t0 = (row_tile ? (int)blockIdx.x : (int)blockIdx.x - p.row_tiles) * kTabTile;
    const int tend = status ? 0 : min((long long)t0 + kTabTile, row_tile ? rows : taken);

    // 3. The per-sequence outputs, which the warps of the CTAs share out, and the
    // marks of the CTA's tile.
    const bool mine = warp % (int)gridDim.x == (int)blockIdx.x;
    if (mine || (!status && t0 < tend)) {
        walk([&](int s, int c, int n) {
            if (status) n = 0;
            if (mine) {
                p.row_offsets[s] = status ? 0 : (int)r;
                p.total_lens[s] = c + n;
            }
            const int more = status ? 0 : pages_of(c + n) - pages_of(c);
            const int first = (int)(row_tile ? r : q), count = row_tile ? n : more;
            const int at = max(first, t0);
            if (at < min(first + count, tend)) {
                mark_seq[at - t0] = s;
                mark_at[at - t0] = first;
                mark_base[at - t0] = (int)q;
                mark_len[at - t0] = c;
            }
            r += n;
            q += more;
        });
    }
    if (t0 >= tend) return;

    // 4. the tile: two neighbouring entries a thread, the last mark at or before each
    __syncthreads();
    static_assert(kTabTile == 2 * kTabThreads, "two entries a thread");
    const int i0 = 2 * tid;
    const int m0 = mark_seq[i0] >= 0 ? i0 : -1;
    const int m1 = mark_seq[i0 + 1] >= 0 ? i0 + 1 : m0;
    int incl = m1;
    for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, incl, o);
        if (lane >= o) incl = max(incl, a);
    }
    if (lane == 31) scan_a[warp] = incl;
    __syncthreads();
    int before = __shfl_up_sync(0xffffffffu, incl, 1);
    if (lane == 0) before = -1;
    for (int w = 0; w < warp; ++w) before = max(before, scan_a[w]);
#pragma unroll
    for (int k = 0; k < 2; ++k) {
        const int e = t0 + i0 + k;
        const int m = max(before, k ? m1 : m0);
        if (e >= tend || m < 0) continue;
        const int s = mark_seq[m], held = pages_of(mark_len[m]);
        if (row_tile) {
            const int pos = mark_len[m] + (e - mark_at[m]);
            const int lp = pos / kPageTokens;
            const int page = lp < held ? p.table[(size_t)s * p.stride + lp] : p.free_pages[mark_base[m] + lp - held];
            p.row_seq[e] = s;
            p.row_pos[e] = pos;
            p.row_slot[e] = page < 0 ? -1ll : (long long)page * kPageTokens + pos % kPageTokens;
        } else {
            p.table[(size_t)s * p.stride + held + (e - mark_at[m])] = p.free_pages[e];
        }
    }
}

// ---------------------------------------------------------------------------
// RoPE on q and k, k and v written to their slots.
//
// (x0, x1) -> (x0 cos - x1 sin, x0 sin + x1 cos) on neighbouring dims, with the
// same unfused roundings as the runner's QKV epilogue (tb_gemv.cu), so both
// writers leave the same bits in the cache.  Pure data movement: every input
// byte is read once and every output byte written once; bound by HBM for long
// prompts and by launch latency for a decode step.  One CTA takes 512 groups of
// W floats of one row (q, k and v columns side by side), two groups a thread,
// so that a row's position, slot and table row are read once per CTA and both
// loads of a thread are in flight together.
// Measured: 8192 rows of 32 query and 32 KV heads of 128 142 us, 0.87 of the copy
// rate; 64 rows 2.1 us.
// ---------------------------------------------------------------------------
constexpr int kRopeThreads = 256;
constexpr int kRopeGroups = 2;

struct RopeParams {
    const float* q;
    const float* k;
    const float* v;
    long long ld_q, ld_k, ld_v, ld_out;
    const int* num_rows;
    int rows;
    const int* pos;
    const long long* slot;
    const float* rope;
    int rope_positions;
    int layer, num_layers, H, Hkv, d;
    float* pool;
    long long num_slots;
    float* out;
    int* err;
};

template <int W>
struct Group {
    float x[W];
};
template <int W>
__device__ __forceinline__ Group<W> load_group(const float* p) {
    Group<W> g;
    if constexpr (W == 4) {
        const float4 f = *reinterpret_cast<const float4*>(p);
        g.x[0] = f.x, g.x[1] = f.y, g.x[2] = f.z, g.x[3] = f.w;
    } else {
        for (int i = 0; i < W; ++i) g.x[i] = p[i];
    }
    return g;
}
template <int W>
__device__ __forceinline__ void store_group(float* p, const Group<W>& g) {
    if constexpr (W == 4)
        *reinterpret_cast<float4*>(p) = make_float4(g.x[0], g.x[1], g.x[2], g.x[3]);
    else
        for (int i = 0; i < W; ++i) p[i] = g.x[i];
}

template <int W>
__global__ void __launch_bounds__(kRopeThreads) rope_append_kernel(RopeParams p) {
    const int row = blockIdx.x;
    if (p.num_rows && row >= *p.num_rows) return;
    const int pos = p.pos[row];
    const long long slot = p.slot[row];
    if (pos < 0 || pos >= p.rope_positions) {  // no angle for it: the row is left out
        if (threadIdx.x == 0) record_error(p.err, kDevBadPosition);
        return;
    }
    if (slot >= p.num_slots && threadIdx.x == 0) record_error(p.err, kDevBadPage);
    const bool keep = slot >= 0 && slot < p.num_slots;
    const int d = p.d, nq = p.H * d, nk = p.Hkv * d;
    const long long page = slot / kPageTokens, token = slot % kPageTokens;
    Group<W> g[kRopeGroups], cs[kRopeGroups];
    int at[kRopeGroups];
#pragma unroll
    for (int u = 0; u < kRopeGroups; ++u) {
        const int e = (blockIdx.y * (kRopeGroups * kRopeThreads) + u * kRopeThreads + threadIdx.x) * W;
        at[u] = e < nq + 2 * nk ? e : -1;
        if (at[u] < 0) continue;
        const float* src = e < nq ? p.q + row * p.ld_q + e
                           : e < nq + nk ? p.k + row * p.ld_k + (e - nq)
                                         : p.v + row * p.ld_v + (e - nq - nk);
        if (e >= nq && !keep) {
            at[u] = -1;
            continue;
        }
        g[u] = load_group<W>(src);
        if (e < nq + nk) cs[u] = load_group<W>(p.rope + (size_t)pos * d + (e < nq ? e : e - nq) % d);
    }
#pragma unroll
    for (int u = 0; u < kRopeGroups; ++u) {
        const int e = at[u];
        if (e < 0) continue;
        Group<W> o = g[u];
        if (e < nq + nk) {
#pragma unroll
            for (int i = 0; i < W; i += 2) {
                o.x[i] = __fsub_rn(__fmul_rn(g[u].x[i], cs[u].x[i]), __fmul_rn(g[u].x[i + 1], cs[u].x[i + 1]));
                o.x[i + 1] = __fadd_rn(__fmul_rn(g[u].x[i], cs[u].x[i + 1]), __fmul_rn(g[u].x[i + 1], cs[u].x[i]));
            }
        }
        if (e < nq) {
            store_group<W>(p.out + row * p.ld_out + e, o);
            continue;
        }
        const int kv = e < nq + nk ? 0 : 1, c = e - nq - kv * nk;
        const size_t tile = (((size_t)page * p.num_layers + p.layer) * 2 + kv) * p.Hkv + c / d;
        store_group<W>(p.pool + (tile * kPageTokens + token) * d + c % d, o);
    }
}

}  // namespace
}  // namespace tb

using namespace tb;

extern "C" tb_status tb_page_tables_build_dev(void* stream, const int32_t* cached, const int32_t* fresh, int32_t batch,
                                              const int32_t* free_pages, int32_t num_free, int32_t* table,
                                              int32_t stride, int32_t max_rows, int32_t* row_offsets,
                                              int32_t* total_lens, int32_t* row_seq, int32_t* row_pos,
                                              int64_t* row_slot, int32_t* info) {
    TB_ENTRY_CHECK(cached && fresh && table && row_offsets && total_lens && info, "NULL argument");
    TB_ENTRY_CHECK(batch >= 1 && stride >= 1 && stride <= INT32_MAX / kPageTokens, "bad batch / page table stride");
    TB_ENTRY_CHECK(num_free >= 0 && (free_pages || num_free == 0), "bad free list");
    TB_ENTRY_CHECK(max_rows >= 0 && (max_rows == 0 || (row_seq && row_pos && row_slot)), "bad row buffers");
    // every CTA reads the lengths while one writes
    const auto apart = [&](const int32_t* out, int64_t n) {
        return (out + n <= cached || cached + batch <= out) && (out + n <= fresh || fresh + batch <= out);
    };
    TB_ENTRY_CHECK(apart(total_lens, batch) && apart(row_offsets, (int64_t)batch + 1),
                   "total_lens and row_offsets must not overlap the lengths");
    StreamEntry entry(table, "page_table");
    if (entry.status != TB_OK) return entry.status;
    TableParams p{cached, fresh, batch, free_pages, num_free, table, stride, max_rows, 0,
                  aligned_to(cached, 16) && aligned_to(fresh, 16), row_offsets, total_lens,
                  row_seq, row_pos, reinterpret_cast<long long*>(row_slot), info};
    // a sequence takes at most n / 16 + 1 pages
    const long long most_pages = std::min<long long>(num_free, (long long)batch + max_rows / kPageTokens);
    p.row_tiles = std::max(1, (int)(((long long)max_rows + kTabTile - 1) / kTabTile));
    const int page_tiles = (int)((most_pages + kTabTile - 1) / kTabTile);
    page_tables_kernel<<<p.row_tiles + page_tiles, kTabThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return launch_status(cudaGetLastError(), "page table launch");
}

extern "C" tb_status tb_rope_append_paged_dev(void* stream, const float* q, int64_t ld_q, const float* k, int64_t ld_k,
                                              const float* v, int64_t ld_v, int32_t rows, const int32_t* num_rows,
                                              const int32_t* row_pos, const int64_t* row_slot, const float* rope,
                                              int32_t rope_positions, int32_t layer, int32_t num_layers, int32_t H,
                                              int32_t Hkv, int32_t d, float* pool, int32_t num_pages, float* out,
                                              int64_t ld_out) {
    TB_ENTRY_CHECK(q && k && v && row_pos && row_slot && rope && pool && out, "NULL argument");
    TB_ENTRY_CHECK(rows >= 0 && rope_positions >= 1 && num_pages >= 1 && layer >= 0 && layer < num_layers,
                   "bad rows / positions / pages / layer");
    TB_ENTRY_CHECK(H >= 1 && Hkv >= 1 && H % Hkv == 0 && d >= 2 && d % 2 == 0 && d <= 1024 &&
                       ((int64_t)H + 2 * (int64_t)Hkv) * d <= (1 << 24),
                   "bad head geometry: H %d, Hkv %d, d %d", H, Hkv, d);
    TB_ENTRY_CHECK(ld_q >= (int64_t)H * d && ld_out >= (int64_t)H * d && ld_k >= (int64_t)Hkv * d &&
                       ld_v >= (int64_t)Hkv * d,
                   "a row stride is shorter than its row");
    if (rows == 0) return TB_OK;
    StreamEntry entry(pool, "kv_pool");
    if (entry.status != TB_OK) return entry.status;
    RopeParams p{};
    p.q = q, p.k = k, p.v = v;
    p.ld_q = ld_q, p.ld_k = ld_k, p.ld_v = ld_v, p.ld_out = ld_out;
    p.num_rows = num_rows;
    p.rows = rows;
    p.pos = row_pos;
    p.slot = reinterpret_cast<const long long*>(row_slot);
    p.rope = rope;
    p.rope_positions = rope_positions;
    p.layer = layer, p.num_layers = num_layers, p.H = H, p.Hkv = Hkv, p.d = d;
    p.pool = pool;
    p.num_slots = (long long)num_pages * kPageTokens;
    p.out = out;
    p.err = entry.err;
    // 16-byte groups where every row and head starts on 16 bytes, else pairs of
    // scalars (a base or stride that is only 4-byte aligned, or d = 4n + 2)
    const bool wide = d % 4 == 0 && ((ld_q | ld_k | ld_v | ld_out) & 3) == 0 && aligned_to(q, 16) &&
                      aligned_to(k, 16) && aligned_to(v, 16) && aligned_to(out, 16) && aligned_to(pool, 16) &&
                      aligned_to(rope, 16);
    const int groups = (int)(((int64_t)H + 2 * Hkv) * d / (wide ? 4 : 2));
    const dim3 grid((unsigned)rows, (unsigned)((groups + kRopeGroups * kRopeThreads - 1) / (kRopeGroups * kRopeThreads)));
    if (wide)
        rope_append_kernel<4><<<grid, kRopeThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    else
        rope_append_kernel<2><<<grid, kRopeThreads, 0, static_cast<cudaStream_t>(stream)>>>(p);
    return launch_status(cudaGetLastError(), "RoPE and cache write launch");
}

extern "C" tb_status tb_rope_table(int32_t positions, int32_t d, float* table) {
    TB_ENTRY_CHECK(table && positions >= 1 && d >= 2 && d % 2 == 0, "bad table arguments");
    for (int pos = 0; pos < positions; ++pos)
        for (int i = 0; i < d; i += 2) rope_angle(pos, i, d, table + (size_t)pos * d + i);
    return TB_OK;
}
