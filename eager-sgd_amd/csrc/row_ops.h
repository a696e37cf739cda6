// row_ops.h — what the row operators (include/esgd_ops.h) share: element types, 16-byte row
// accesses, wave reductions, and the stable sort of small integer keys behind the embedding's
// gradient and the experts' order.
#pragma once

#include <hip/hip_runtime.h>

#include <cstdint>
#include <type_traits>

#include "esgd_internal.h"
#include "esgd_ops.h"

namespace esgd {

// ---- elements: T is the storage type, arithmetic is float ----
using f32_t = float;
using bf16_t = __bf16;
using f16_t = _Float16;

// N elements of T in one access.  The alignment is the element's: gfx950 loads and stores 16
// bytes at any such address in one instruction, so rows of odd widths and odd pitches
// need no path of their own.
template <class T, int N>
using vec = T __attribute__((ext_vector_type(N), aligned(sizeof(T))));

template <class T, int N>
__device__ __forceinline__ vec<T, N> load_vec(const T *p) {
    return *reinterpret_cast<const vec<T, N> *>(p);
}
// Stores stream past the caches (nontemporal): the largest results do not fit there, and lines
// that wait to be written back hold up the next kernel's reads (16384 x 8 rows of 2048 bf16, out
// and back with gradients: 612 us of kernels with plain stores, 560 with these, though the way out
// alone takes 116 instead of 101).  Measured with these kernels one after the other; with a
// product that reads a few MB of rows in between it has not been.
template <class T, int N>
__device__ __forceinline__ void store_vec(T *p, vec<T, N> v) {
    __builtin_nontemporal_store(v, reinterpret_cast<vec<T, N> *>(p));
}

// The N elements from column c of a row of `width`, as they are stored (half the registers of
// floats where a kernel holds several): whole vectors inside, single elements at the row's end,
// zeros behind it.
template <class T, int N>
__device__ __forceinline__ vec<T, N> load_packed(const T *row, int64_t c, int64_t width) {
    if (c + N <= width) return load_vec<T, N>(row + c);
    vec<T, N> v{};
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (c + i < width) v[i] = row[c + i];
    return v;
}
template <class T, int N>
__device__ __forceinline__ void load_row(const T *row, int64_t c, int64_t width, float (&x)[N]) {
    const vec<T, N> v = load_packed<T, N>(row, c, width);
#pragma unroll
    for (int i = 0; i < N; ++i) x[i] = float(v[i]);
}
// KEEP: into the caches, for a kernel that follows at once
template <class T, int N, bool KEEP = false>
__device__ __forceinline__ void store_row(T *row, int64_t c, int64_t width, const float (&x)[N]) {
    if (c + N <= width) {
        vec<T, N> v;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = T(x[i]);   // one round to nearest even
        if (KEEP) *reinterpret_cast<vec<T, N> *>(row + c) = v;
        else store_vec<T, N>(row + c, v);
        return;
    }
#pragma unroll
    for (int i = 0; i < N; ++i)
        if (c + i < width) row[c + i] = T(x[i]);
}

// A lane whose N columns would pass the row's end takes the row's last N instead (where there are
// as many): the columns that it shares with its neighbour come out the same there and are stored
// twice with the same bits, and no lane goes through single elements.
template <int N>
__device__ __forceinline__ int64_t inside(int64_t c, int64_t width) {
    return c + N > width && c < width && width >= N ? width - N : c;
}

// Over the 64 lanes of a wave that are all active, the same order at every call; every lane has
// the result.  Four steps inside the rows of 16 lanes go through the register file's own lane
// permutes (DPP: pairs, quads, halves and rows mirrored), the four rows through scalars: a fifth of
// the latency of six shuffles through LDS, which counts where a row's work is short.
template <int CTRL>
__device__ __forceinline__ float lane_of(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xf, 0xf, true));
}
__device__ __forceinline__ float lane_at(float x, int lane) {
    return __builtin_bit_cast(float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, x), lane));
}
constexpr int kPairs = 0xb1, kQuads = 0x4e, kHalfMirror = 0x141, kMirror = 0x140;
__device__ __forceinline__ float wave_sum(float x) {
    x += lane_of<kPairs>(x);
    x += lane_of<kQuads>(x);
    x += lane_of<kHalfMirror>(x);
    x += lane_of<kMirror>(x);
    return (lane_at(x, 0) + lane_at(x, 16)) + (lane_at(x, 32) + lane_at(x, 48));
}
__device__ __forceinline__ float wave_max(float x) {
    x = fmaxf(x, lane_of<kPairs>(x));
    x = fmaxf(x, lane_of<kQuads>(x));
    x = fmaxf(x, lane_of<kHalfMirror>(x));
    x = fmaxf(x, lane_of<kMirror>(x));
    return fmaxf(fmaxf(lane_at(x, 0), lane_at(x, 16)), fmaxf(lane_at(x, 32), lane_at(x, 48)));
}

// ---- types of a call, as template arguments ----
template <class T>
struct type_tag { using type = T; };

template <class T>
constexpr int type_code = std::is_same_v<T, f32_t> ? ESGD_FLOAT : std::is_same_v<T, bf16_t> ? ESGD_BF16 : ESGD_HALF;

template <class F>
inline int with_type(int dtype, const char *who, F &&f) {
    switch (dtype) {
    case ESGD_FLOAT: return f(type_tag<f32_t>{});
    case ESGD_BF16: return f(type_tag<bf16_t>{});
    case ESGD_HALF: return f(type_tag<f16_t>{});
    default: break;
    }
    set_error("%s: unsupported element type %d (FLOAT, BF16, HALF)", who, dtype);
    return ESGD_INVALID_ARG;
}
inline bool row_type_ok(int dtype) { return dtype == ESGD_FLOAT || dtype == ESGD_BF16 || dtype == ESGD_HALF; }
inline size_t row_type_size(int dtype) { return dtype == ESGD_FLOAT ? 4 : 2; }

// workgroups of a launch whose waves stride over their items: enough to fill the chip many
// times over, well below the grid's limits
inline unsigned row_grid(int64_t blocks, int64_t most = int64_t(1) << 20) {
    return unsigned(blocks < 1 ? 1 : blocks < most ? blocks : most);
}

// ---- stable sort of keys ----
// key(i) = index[i] where 0 <= index[i] < limit and index[i] != skip, else `limit`: sorted last.
struct KeySource {
    const void *index;
    int wide;         // int64 / int32
    int64_t limit;
    int64_t skip;     // < 0: none
};
// memory to be zeroed by workgroups beside the sort's own (bytes: a multiple of 2)
struct Fill {
    void *ptr;
    int64_t bytes;
};
size_t sort_work_bytes(int64_t n, int64_t limit);
// keys, places: n each, inside `work`; set by the call
int sort_keys(const KeySource &src, int64_t n, Fill fill, void *work, const uint32_t **keys,
              const uint32_t **places, hipStream_t s);
// the same sort told per item: slots[i] = place, or -1 - place where the key is `limit`;
// offsets[k] = items with keys below k, for k in [0, limit]
int sort_slots(const KeySource &src, int64_t n, int32_t *offsets, int32_t *slots, void *work, hipStream_t s);

}  // namespace esgd
