// embedding.hip — rows of a table by token, scaled, and the table's gradient by sorted tokens,
// hand-written for gfx950 (include/esgd_ops.h has the formulas).
//
// Lookup: a copy with a gather; HBM bounds it.  A wave moves 64 x 16 bytes of a row at a time,
// or as many short rows at once as fill its lanes.
//
// Gradient: sum of the output's gradient rows by token.  The tokens are sorted first
// (row_sort.hip), so equal tokens lie together and every sum has one order; float atomics would
// need none of that but give other bits at every call, and no run could be repeated.  The sorted rows are cut into tiles of equal length, whatever
// the tokens: a wave walks its tile's rows for 64 x 16 bytes of columns, adding in registers,
// and stores a table row where a token's run ends.  A run that crosses tiles leaves fp32
// partial sums, which k_row_join adds up in the order of the tiles; a token that half the
// batch consists of is thus spread over the chip like any other.  The whole table is zeroed while
// the sort runs; rows with a token are written a second time.
#include <hip/hip_runtime.h>

#include <algorithm>

#include "row_ops.h"

namespace esgd {

// elements a lane moves in one access: 16 bytes of the narrower type, at most two accesses of the wider
template <class A, class B>
constexpr int lane_elems = sizeof(A) == 4 && sizeof(B) == 4 ? 4 : 8;

template <class W, class O>
__global__ __launch_bounds__(256) void k_lookup(const W *table, int64_t table_pitch, int64_t rows, int64_t width,
                                                const void *token, int wide, int64_t n, float scale, O *out,
                                                int64_t out_pitch, int lanes_log2, int64_t chunks, int64_t items) {
    // an item: 1 << (6 - lanes_log2) rows, one chunk of (1 << lanes_log2) * E columns each
    constexpr int E = lane_elems<W, O>;
    const int lane = threadIdx.x & 63;
    const int64_t waves = int64_t(gridDim.x) * 4;
    for (int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6); item < items; item += waves) {
        const int64_t t = ((item / chunks) << (6 - lanes_log2)) + (lane >> lanes_log2);
        const int64_t c = inside<E>(((item % chunks) << lanes_log2) * E + (lane & ((1 << lanes_log2) - 1)) * E, width);
        if (t >= n || c >= width) continue;
        const int64_t v = wide ? static_cast<const int64_t *>(token)[t]
                               : int64_t(static_cast<const int32_t *>(token)[t]);
        float x[E] = {};
        if (v >= 0 && v < rows) {
            load_row<W, E>(table + v * table_pitch, c, width, x);
#pragma unroll
            for (int i = 0; i < E; ++i) x[i] *= scale;
        }
        store_row<O, E>(out + t * out_pitch, c, width, x);
    }
}

// ---- gradient: runs of equal keys summed, `per` sorted rows a tile ----
constexpr int kAhead = 4;   // rows whose loads are issued at once
// Elements a lane sums: 16 bytes of the table's type, so that a wave's store is 1 KB without gaps.  Two
// stores of 16 bytes a lane, 32 bytes apart, stream past the caches as halves of their lines (32768
// bf16 rows of 1024 into fp32: the whole gradient 151 us, 128 without them).
template <class W>
constexpr int sum_elems = 16 / int(sizeof(W));

template <class G, class W>
__global__ __launch_bounds__(256) void k_row_sums(const G *grad, int64_t grad_pitch, int64_t n, int64_t width,
                                                  const uint32_t *key, const uint32_t *place, uint32_t limit, int per,
                                                  float scale, W *table, int accumulate, float *part, int64_t chunks,
                                                  int64_t items) {
    constexpr int E = sum_elems<W>;
    const int lane = threadIdx.x & 63;
    const int64_t item = int64_t(blockIdx.x) * 4 + (threadIdx.x >> 6);
    if (item >= items) return;
    const int64_t tile = item / chunks, first = tile * per;
    int64_t c = (item % chunks) * (64 * E) + lane * E;
    if (!accumulate) c = inside<E>(c, width);   // (what is added to must be added to once)
    const int have = int(min(int64_t(per), n - first));
    const uint32_t k = lane < have ? key[first + lane] : limit;
    const uint32_t row = lane < have ? place[first + lane] : 0;
    const int count = __popcll(__ballot(k < limit));   // dropped tokens are the last
    if (!count) return;
    const uint32_t key_before = first ? key[first - 1] : limit;
    const uint32_t key_behind = first + have < n ? key[first + have] : limit;
    float sum[E] = {};
    bool whole = __builtin_amdgcn_readlane(k, 0) != key_before;   // the run began in this tile
    // Two batches of kAhead rows in turn: the loads of one are issued before the other's sums are
    // stored, since a wait for a load behind a store is one for the store too.
    vec<G, E> x[2][kAhead];
    auto load = [&](vec<G, E> (&to)[kAhead], int j0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int j = min(j0 + u, count - 1);
            const G *p = grad + int64_t(__builtin_amdgcn_readlane(row, j)) * grad_pitch;
            if (j0 + u < count && c < width) to[u] = load_packed<G, E>(p, c, width);
        }
    };
    auto add = [&](const vec<G, E> (&from)[kAhead], int j0) {
#pragma unroll
        for (int u = 0; u < kAhead; ++u) {
            const int j = j0 + u;
            if (j >= count) break;
#pragma unroll
            for (int i = 0; i < E; ++i) sum[i] += float(from[u][i]);
            const uint32_t now = __builtin_amdgcn_readlane(k, j);
            const uint32_t next = j + 1 < count ? __builtin_amdgcn_readlane(k, (j + 1) & 63)
                                                : (j + 1 < have ? limit : key_behind);
            if (next == now && j + 1 < count) continue;
            const bool ends = next != now;   // else the run goes on in the next tile
            if (c < width) {
                if (whole && ends) {
                    W *to = table + int64_t(now) * width;
                    float y[E];
                    if (accumulate) load_row<W, E>(to, c, width, y);
#pragma unroll
                    for (int i = 0; i < E; ++i) y[i] = accumulate ? y[i] + scale * sum[i] : scale * sum[i];
                    store_row<W, E>(to, c, width, y);
                } else {
                    // a tile's first run goes to its slot 0 unless it began here, its last to slot 1
                    // (kept for the join: 32768 rows of 512, all one token's, 68 us, past the caches 76)
                    store_row<float, E, true>(part + (tile * 2 + (whole ? 1 : 0)) * width, c, width, sum);
                }
            }
#pragma unroll
            for (int i = 0; i < E; ++i) sum[i] = 0.0f;
            whole = true;
        }
    };
    load(x[0], 0);
    for (int j0 = 0; j0 < count; j0 += 2 * kAhead) {
        load(x[1], j0 + kAhead);
        add(x[0], j0);
        load(x[0], j0 + 2 * kAhead);
        add(x[1], j0 + kAhead);
    }
}

// A run that crosses tiles: slot 1 of the tile where it begins, slot 0 of those behind.  One
// workgroup per tile and 256 columns; where no such run begins there is nothing to do.  A token
// that fills the batch has one run through all tiles: its workgroups have 8 loads a lane in flight
// (131072 tokens, all the same, width 1024: the whole gradient takes 134 us, 155 with 4 loads).
// Narrower rows leave lanes over: 64 >> lanes_log2 groups of them have a part of the tiles each.
template <class W>
__global__ __launch_bounds__(256) void k_row_join(const uint32_t *key, int64_t n, int64_t width, uint32_t limit, int per,
                                                  float scale, W *table, int accumulate, const float *part,
                                                  int lanes_log2, int64_t chunks) {
    constexpr int E = 4, PROBES = 4;
    const int64_t tile = blockIdx.x / chunks, first = tile * per;
    if (first + per >= n) return;   // the last tile: nothing behind it
    const uint32_t k = key[first + per - 1], behind = key[first + per], begin = key[first];
    const uint32_t before = first ? key[first - 1] : limit;
    const uint32_t later = first + 2 * per < n ? key[first + 2 * per] : limit;
    if (k >= limit || behind != k || (begin == k && before == k)) return;   // none, or it began before
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t more = 1;   // tiles behind this one that begin with k
    for (bool on = later == k; on;) {
        bool same[PROBES];
#pragma unroll
        for (int i = 0; i < PROBES; ++i) {
            const int64_t at = (tile + 1 + more + i * 64 + lane) * per;
            same[i] = at < n && key[min(at, n - 1)] == k;
        }
#pragma unroll
        for (int i = 0; i < PROBES; ++i) {
            const uint64_t no = __ballot(!same[i]);
            if (on) more += no ? __ffsll(static_cast<unsigned long long>(no)) - 1 : 64;
            on &= !no;
        }
    }
    const int group = lane >> lanes_log2, groups = 64 >> lanes_log2;
    int64_t c = ((blockIdx.x % chunks) << lanes_log2) * E + (lane & ((1 << lanes_log2) - 1)) * E;
    if (!accumulate) c = inside<E>(c, width);
    float sum[E] = {};
    if (c < width) {
        const int u = wave * groups + group;   // its tiles lie next to each other
        if (u == 0) load_row<float, E>(part + (tile * 2 + 1) * width, c, width, sum);
        const int64_t each = (more + 4 * groups - 1) / (4 * groups), t1 = min(more, (u + 1) * each);
#pragma unroll 8
        for (int64_t t = u * each; t < t1; ++t) {
            float x[E];
            load_row<float, E>(part + (tile + 1 + t) * 2 * width, c, width, x);
#pragma unroll
            for (int i = 0; i < E; ++i) sum[i] += x[i];
        }
    }
    for (int m = 1 << lanes_log2; m < 64; m <<= 1) {
#pragma unroll
        for (int i = 0; i < E; ++i) sum[i] += __shfl_down(sum[i], m);
    }
    __shared__ float sums[3][64][E];
    if (wave) {
#pragma unroll
        for (int i = 0; i < E; ++i) sums[wave - 1][lane][i] = sum[i];
    }
    __syncthreads();
    if (wave || group || c >= width) return;
#pragma unroll
    for (int w = 0; w < 3; ++w) {
#pragma unroll
        for (int i = 0; i < E; ++i) sum[i] += sums[w][lane][i];
    }
    W *to = table + int64_t(k) * width;
    float y[E];
    if (accumulate) load_row<W, E>(to, c, width, y);
#pragma unroll
    for (int i = 0; i < E; ++i) y[i] = accumulate ? y[i] + scale * sum[i] : scale * sum[i];
    store_row<W, E>(to, c, width, y);
}

namespace {

// Rows a tile: 64 (a lane has a row's key) where that leaves 2048 waves that load 16 bytes a lane, or
// 4096 of 8 bytes, else down to 8, so that short batches still spread over the chip and enough loads are
// on their way (32768 bf16 rows of 1024 into fp32, skewed: sums 34.9 us with tiles of 32, 47.4 with
// 64).  Longer tiles leave fewer partial sums (whole gradient, bf16 rows of 1024 into fp32: 131072
// tokens 114 us, with tiles of 32 121; 32768 of one token 128 us, 133 with 32, 154 with 16), shorter
// ones more waves (4096 tokens into bf16 27.1 us with 8, 30.0 with 16, 36.7 with 32).
int rows_per_tile(int64_t n, int64_t chunks, int lane_bytes) {
    int per = 64;
    while (per > 8 && (n + per - 1) / per * chunks * lane_bytes < 2048 * 16) per /= 2;
    return per;
}
template <class G, class W>
int rows_per_tile_of(int64_t n, int64_t width) {
    constexpr int E = sum_elems<W>;
    return rows_per_tile(n, (width + 64 * E - 1) / (64 * E), E * int(sizeof(G)));
}
// two rows a tile, with the shortest tiles that any of the types have
size_t part_bytes(int64_t n, int64_t width) {
    const int64_t per = std::min({rows_per_tile_of<f32_t, f32_t>(n, width), rows_per_tile_of<bf16_t, f32_t>(n, width),
                                  rows_per_tile_of<bf16_t, bf16_t>(n, width)});
    return size_t((n + per - 1) / per) * 2 * size_t(width) * 4;
}

template <class W, class O>
int lookup(const void *table, int64_t table_pitch, int64_t rows, int64_t width, int token_bits, const void *token,
           int64_t n, float scale, void *out, int64_t out_pitch, hipStream_t s) {
    constexpr int E = lane_elems<W, O>;
    int lanes_log2 = 0;
    while (lanes_log2 < 6 && (int64_t(E) << lanes_log2) < width) ++lanes_log2;
    const int64_t chunks = (width + (int64_t(E) << lanes_log2) - 1) / (int64_t(E) << lanes_log2);
    const int64_t items = ((n + (64 >> lanes_log2) - 1) >> (6 - lanes_log2)) * chunks;
    hipLaunchKernelGGL((k_lookup<W, O>), dim3(row_grid((items + 3) / 4)), dim3(256), 0, s,
                       static_cast<const W *>(table), table_pitch, rows, width, token, token_bits == 64, n, scale,
                       static_cast<O *>(out), out_pitch, lanes_log2, chunks, items);
    ESGD_HIP(hipGetLastError());
    return ESGD_SUCCESS;
}

template <class G, class W>
int row_sums(const void *grad, int64_t grad_pitch, int64_t n, int64_t width, const uint32_t *key,
             const uint32_t *place, int64_t rows, float scale, void *table, int accumulate, float *part,
             hipStream_t s) {
    constexpr int E = sum_elems<W>;
    const int64_t chunks = (width + 64 * E - 1) / (64 * E);
    const int per = rows_per_tile_of<G, W>(n, width);
    const int64_t tiles = (n + per - 1) / per, items = tiles * chunks;
    hipLaunchKernelGGL((k_row_sums<G, W>), dim3(unsigned((items + 3) / 4)), dim3(256), 0, s,
                       static_cast<const G *>(grad), grad_pitch, n, width, key, place, uint32_t(rows), per, scale,
                       static_cast<W *>(table), accumulate, part, chunks, items);
    ESGD_HIP(hipGetLastError());
    if (tiles > 1) {
        int lanes_log2 = 0;   // of 4 columns each
        while (lanes_log2 < 6 && (int64_t(4) << lanes_log2) < width) ++lanes_log2;
        const int64_t join_chunks = (width + 255) / 256;
        hipLaunchKernelGGL((k_row_join<W>), dim3(unsigned((tiles - 1) * join_chunks)), dim3(256), 0, s, key, n, width,
                           uint32_t(rows), per, scale, static_cast<W *>(table), accumulate, part, lanes_log2,
                           join_chunks);
        ESGD_HIP(hipGetLastError());
    }
    return ESGD_SUCCESS;
}

}  // namespace
}  // namespace esgd

using namespace esgd;

extern "C" {

int esgd_embedding(int table_type, const void *table, int64_t table_pitch, int64_t rows, int64_t width,
                   int token_bits, const void *token, int64_t n, float scale, int out_type, void *out,
                   int64_t out_pitch, void *stream) {
    ESGD_ARG(rows >= 0 && width >= 0 && n >= 0, "esgd_embedding: negative size");
    ESGD_ARG(token_bits == 32 || token_bits == 64, "esgd_embedding: tokens of %d bits", token_bits);
    ESGD_ARG(table_type == out_type || table_type == ESGD_FLOAT,
             "esgd_embedding: a table of type %d gives rows of its own type only", table_type);
    if (!n || !width) return ESGD_SUCCESS;
    ESGD_ARG(token && out && (table || !rows), "esgd_embedding: null pointer");
    ESGD_ARG(table_pitch >= 0 && out_pitch >= width, "esgd_embedding: rows of the output overlap");
    ESGD_ARG(width < (int64_t(1) << 28) && n < (int64_t(1) << 40), "esgd_embedding: too large");
    if (int rc = require_device()) return rc;
    hipStream_t s = as_stream(stream);
    return with_type(table_type, "esgd_embedding", [&](auto w) {
        using W = typename decltype(w)::type;
        return with_type(out_type, "esgd_embedding", [&](auto o) {
            using O = typename decltype(o)::type;
            if constexpr (std::is_same_v<W, O> || std::is_same_v<W, float>)
                return lookup<W, O>(table, table_pitch, rows, width, token_bits, token, n, scale, out, out_pitch, s);
            else
                return ESGD_INVALID_ARG;   // refused above
        });
    });
}

int esgd_embedding_grad_work(int64_t n, int64_t rows, int64_t width, size_t *bytes) {
    ESGD_ARG(bytes, "esgd_embedding_grad_work: null pointer");
    ESGD_ARG(n >= 0 && rows >= 0 && width >= 0, "esgd_embedding_grad_work: negative size");
    ESGD_ARG(n < (int64_t(1) << 31) - 65536 && rows < (int64_t(1) << 31) - 1 && width < (int64_t(1) << 28),
             "esgd_embedding_grad: too many tokens, rows or columns");
    *bytes = sort_work_bytes(n, rows) + part_bytes(n, width);
    return ESGD_SUCCESS;
}

int esgd_embedding_grad(int grad_type, const void *grad, int64_t grad_pitch, int64_t n, int64_t width,
                        int token_bits, const void *token, int64_t skip_token, float scale, int table_type,
                        void *grad_table, int64_t rows, int accumulate, void *work, size_t work_bytes,
                        void *stream) {
    size_t need = 0;
    if (int rc = esgd_embedding_grad_work(n, rows, width, &need)) return rc;
    ESGD_ARG(token_bits == 32 || token_bits == 64, "esgd_embedding_grad: tokens of %d bits", token_bits);
    ESGD_ARG(row_type_ok(grad_type) && row_type_ok(table_type), "esgd_embedding_grad: unsupported element type");
    ESGD_ARG(table_type == grad_type || table_type == ESGD_FLOAT,
             "esgd_embedding_grad: gradient rows of type %d give a table gradient of that type or FLOAT", grad_type);
    if (!rows || !width || (!n && accumulate)) return ESGD_SUCCESS;
    ESGD_ARG(grad_table && (!n || (grad && token)) && work, "esgd_embedding_grad: null pointer");
    ESGD_ARG(grad_pitch >= 0, "esgd_embedding_grad: negative pitch");
    ESGD_ARG(work_bytes >= need, "esgd_embedding_grad: %zu bytes of work memory, %zu needed", work_bytes, need);
    ESGD_ARG((reinterpret_cast<uintptr_t>(work) & 15) == 0, "esgd_embedding_grad: work memory off a 16-byte boundary");
    ESGD_ARG((n + 7) / 8 * ((width + 255) / 256) < (int64_t(1) << 24),
             "esgd_embedding_grad: too many gradient elements in one call");
    if (int rc = require_device()) return rc;
    hipStream_t s = as_stream(stream);
    const KeySource src{token, token_bits == 64, rows, skip_token};
    Fill fill{nullptr, 0};
    if (!accumulate) fill = Fill{grad_table, int64_t(rows * width * int64_t(row_type_size(table_type)))};
    const uint32_t *key, *place;
    if (int rc = sort_keys(src, n, fill, work, &key, &place, s)) return rc;
    if (!n) return ESGD_SUCCESS;
    float *part = reinterpret_cast<float *>(static_cast<char *>(work) + sort_work_bytes(n, rows));
    return with_type(grad_type, "esgd_embedding_grad", [&](auto g) {
        using G = typename decltype(g)::type;
        return with_type(table_type, "esgd_embedding_grad", [&](auto w) {
            using W = typename decltype(w)::type;
            if constexpr (std::is_same_v<W, G> || std::is_same_v<W, float>)
                return row_sums<G, W>(grad, grad_pitch, n, width, key, place, rows, scale, grad_table, accumulate,
                                      part, s);
            else
                return ESGD_INVALID_ARG;   // refused above
        });
    });
}

}  // extern "C"
