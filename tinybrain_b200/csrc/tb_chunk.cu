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
                    for (int i = 0; i < D / 4; ++i) {
                        const float4 a = k[i], b = reinterpret_cast<const float4*>(q)[i];
                        score = fmaf(a.x, b.x, fmaf(a.y, b.y, fmaf(a.z, b.z, fmaf(a.w, b.w, score))));
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

constexpr int kRowWarps = 4;

template <int D>
__global__ void __launch_bounds__(kRowWarps * 32) chunk_rows_kernel(ChunkParams p) {
    __shared__ __align__(16) float qs[kRowWarps][D];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const long long item = (long long)blockIdx.x * kRowWarps + warp;
    const int row = (int)(item / p.H), h = (int)(item % p.H);
    if (row >= min(p.row_offsets[p.batch], p.rows)) return;
    int lo = 0, hi = p.batch;  // the last sequence whose rows begin at or before `row`
    while (hi - lo > 1) {
        const int mid = (lo + hi) / 2;
        if (p.row_offsets[mid] <= row) lo = mid; else hi = mid;
    }
    int first, count;
    rows_of(p, lo, first, count);
    int t1 = p.total_lens[lo] - count + (row - first) + 1;
    if (t1 > p.stride * kPageTokens) {  // longer than its table row
        record_error(p.err, kDevBadPage);
        t1 = p.stride * kPageTokens;
    }
    for (int i = lane; i < D; i += 32) qs[warp][i] = p.q[row * p.ld_q + (size_t)h * D + i];
    __syncwarp();
    RowSum<D> r;
    r.add_range(p, qs[warp], rsqrtf((float)D), lo, h / (p.H / p.Hkv), 0, t1);
#pragma unroll
    for (int i = 0; i < (D + 31) / 32; ++i)
        if (lane + 32 * i < D) p.out[row * p.ld_out + (size_t)h * D + lane + 32 * i] = t1 > 0 ? r.acc[i] / r.l : 0.0f;
}

template <int D>
cudaError_t launch_chunk(const ChunkParams& p, cudaStream_t stream) {
    const long long items = (long long)p.rows * p.H;
    chunk_rows_kernel<D><<<(unsigned)((items + kRowWarps - 1) / kRowWarps), kRowWarps * 32, 0, stream>>>(p);
    return cudaGetLastError();
}

}  // namespace
}  // namespace tb

using namespace tb;

extern "C" tb_status tb_paged_attention_chunk_workspace(int32_t rows, int32_t batch, int32_t max_new, int32_t max_len,
                                                        int32_t H, int32_t Hkv, int32_t d, int64_t* bytes) {
    TB_ENTRY_CHECK(bytes, "NULL argument");
    *bytes = 0;
    return TB_OK;
}

extern "C" tb_status tb_paged_attention_chunk_dev(void* stream, const float* q, int64_t ld_q, int32_t rows,
                                                  const int32_t* row_offsets, const int32_t* total_lens, int32_t batch,
                                                  const float* pool, int32_t num_pages, const int32_t* table,
                                                  int32_t stride, int32_t max_new, int32_t max_len, int32_t layer,
                                                  int32_t num_layers, int32_t H, int32_t Hkv, int32_t d, float* out,
                                                  int64_t ld_out, void* workspace, int64_t workspace_bytes) {
    TB_ENTRY_CHECK(q && row_offsets && total_lens && pool && table && out, "NULL argument");
    TB_ENTRY_CHECK(rows >= 0 && batch >= 1 && num_pages >= 1 && stride >= 1 && stride <= INT_MAX / kPageTokens &&
                       layer >= 0 && layer < num_layers && max_new >= 1 && max_len >= 1,
                   "bad rows / batch / pages / lengths / layer");
    TB_ENTRY_CHECK(H >= 1 && Hkv >= 1 && H % Hkv == 0, "heads must divide: H %d, Hkv %d", H, Hkv);
    TB_ENTRY_CHECK(ld_q >= (int64_t)H * d && ld_out >= (int64_t)H * d, "a row stride is shorter than its row");
    if ((d != 16 && d != 32 && d != 64 && d != 128) || H / Hkv > 128)
        return (tb_status)report_error(TB_ERR_UNSUPPORTED, "head dimension %d is not 16, 32, 64 or 128, or %d query heads share a KV head (at most 128)",
                                       d, H / Hkv);
    if (rows == 0) return TB_OK;
    StreamEntry entry(pool, "kv_pool");
    if (entry.status != TB_OK) return entry.status;
    ChunkParams p{q, ld_q, row_offsets, total_lens, batch, rows, pool, num_pages, table, stride, layer, num_layers, H,
                  Hkv, out, ld_out, entry.err};
    cudaStream_t s = static_cast<cudaStream_t>(stream);
    switch (d) {
        case 16: return launch_status(launch_chunk<16>(p, s), "chunk attention launch");
        case 32: return launch_status(launch_chunk<32>(p, s), "chunk attention launch");
        case 64: return launch_status(launch_chunk<64>(p, s), "chunk attention launch");
    }
    return launch_status(launch_chunk<128>(p, s), "chunk attention launch");
}
