// tb_chunk_walk.h -- how a call of the chunk attention (tb_chunk.cu, tb_chunk_few.cuh)
// falls into units and equal shares, and the walk from one unit to the next.
// Plain arithmetic on the lengths, for the device and the host alike: the tests
// compile it with the host's compiler and check that the shares of a call hold
// every tile once and read nothing beyond the caller's arrays.
#pragma once

#ifdef __CUDACC__
#include "tb_kernels.h"
#define TB_WALK __host__ __device__ __forceinline__
#else
#include <algorithm>
#include <cstddef>
#define TB_WALK inline
namespace tb {
constexpr int kPageTokens = 16;
using std::max;
using std::min;
}  // namespace tb
#endif

namespace tb {

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
    int rows_above, rows_upto;  // the kernel's sequences: those with more and at most so many rows of a KV head
    float* out;
    long long ld_out;
    int* err;
};

// The rows of sequence s that the call holds (none where another kernel has them).
TB_WALK void rows_of(const ChunkParams& p, int s, int& first, int& count) {
    first = min(max(p.row_offsets[s], 0), p.rows);
    count = max(min(p.row_offsets[s + 1], p.rows) - first, 0);
    const long long of_head = (long long)count * (p.H / p.Hkv);
    if (of_head <= p.rows_above || of_head > p.rows_upto) count = 0;
}

// A unit: ROWS query rows of one KV head (the G = H / Hkv query heads of ROWS / G
// consecutive tokens) over the positions they see, in tiles of NT positions.
struct Unit {
    int s, tile, head;
    int first, n, len;  // the sequence's first row, rows and length
    int limit;          // positions that the unit's last row sees
    int tiles;          // of NT positions, at least one
};

template <int NT, int ROWS>
TB_WALK void set_tile(const ChunkParams& p, Unit& u) {
    const int per = ROWS / (p.H / p.Hkv);
    const int last = min((u.tile + 1) * per, u.n) - 1;
    u.limit = min(max(u.len - u.n + last + 1, 0), p.stride * kPageTokens);
    u.tiles = max(1, (u.limit + NT - 1) / NT);
}
TB_WALK void set_sequence(const ChunkParams& p, Unit& u) {
    rows_of(p, u.s, u.first, u.n);
    u.len = p.total_lens[u.s];
}
// The unit after u; behind the batch's last one it stays in the last sequence, so
// that no lengths, whatever becomes of them during the call, lead out of the arrays.
template <int NT, int ROWS>
TB_WALK void next_unit(const ChunkParams& p, Unit& u) {
    if (++u.head < p.Hkv) return;
    u.head = 0;
    ++u.tile;
    // (a tile has ROWS / G whole tokens, also where G does not divide ROWS)
    if ((long long)u.tile * (ROWS / (p.H / p.Hkv)) >= u.n) {
        u.tile = 0;
        while (u.s + 1 < p.batch) {
            ++u.s;
            set_sequence(p, u);
            if (u.n > 0) break;
        }
    }
    set_tile<NT, ROWS>(p, u);
}
// sum of floor((a i + b) / m) over i < n, for a, b >= 0 and m > 0 (Euclid's
// algorithm on the lattice points under the line).
TB_WALK long long floor_sum(long long n, long long m, long long a, long long b) {
    long long sum = 0;
    while (n > 0) {
        sum += (a / m) * (n * (n - 1) / 2) + (b / m) * n;
        a %= m;
        b %= m;
        const long long top = a * n + b;
        if (top < m) break;
        n = top / m;
        b = top % m;
        const long long t = m;
        m = a;
        a = t;
    }
    return sum;
}
// Position tiles of the first `count` row tiles of u's sequence, for one head.
template <int NT, int ROWS>
TB_WALK long long tiles_before(const ChunkParams& p, Unit u, int count) {
    const int per = ROWS / (p.H / p.Hkv), held = u.len - u.n, all = (u.n + per - 1) / per;
    if (count > 4 && held >= 0 && u.len <= p.stride * kPageTokens) {
        // ceil((held + (t + 1) per) / NT) each, but for the last row tile of the sequence
        const int full = min(count, all - 1);
        long long sum = floor_sum(full, NT, per, (long long)held + per + NT - 1);
        if (count == all && all > 0) sum += (u.len + NT - 1) / NT;
        return sum;
    }
    long long sum = 0;  // a few, or lengths that do not fit (reported): one by one
    for (u.tile = 0; u.tile < count; ++u.tile) {
        set_tile<NT, ROWS>(p, u);
        sum += u.tiles;
    }
    return sum;
}
// Tiles of all units of a sequence.
template <int NT, int ROWS>
TB_WALK long long tiles_of_sequence(const ChunkParams& p, int s) {
    Unit u;
    u.s = s;
    set_sequence(p, u);
    const int per = ROWS / (p.H / p.Hkv);
    return tiles_before<NT, ROWS>(p, u, (u.n + per - 1) / per) * p.Hkv;
}

// A CTA's share: tiles [total c / C, total (c + 1) / C) of all units' tiles, one
// unit after the other.  A ragged batch, one long sequence and a large prompt
// thus load the SMs evenly without a plan made on the host.
struct Share {
    long long total, shares, index, end;  // all tiles; the shares and this one of them; where it ends
    int count;
    // shares after this one that hold the `left` tiles after its last
    TB_WALK int followers(int left) const {
        const long long last = end + left - 1;
        int n = (int)max(last * shares / total - index, 1ll);  // about: shares differ by a tile
        while (n > 1 && total * (index + n) / shares > last) --n;
        while (total * (index + n + 1) / shares <= last) ++n;
        return n;
    }
};

}  // namespace tb
