// Attention over packed documents with a distance bias (gfx950).
//
// Query i of Sq stands at position p = i + Sk - Sq among the Sk keys; query
// head h reads key-value head g = h / (Hq / Hkv):
//
//   s_ij = scale q_i.k_j - slope_h |p - j|
//   P_ij = exp(s_ij - lse_i) where j is visible, 0 elsewhere
//   o_i  = sum_j P_ij v_j            lse_i = log sum over visible j of exp(s_ij)
//
//   delta_i = do_i.o_i               dS_ij = P_ij (do_i.v_j - delta_i)
//   dq_i = scale sum_j dS_ij k_j
//   dk_j = scale sum dS_ij q_i       dv_j = sum P_ij do_i    over i and g's heads h
//
// Key j is visible if its document is the query's and not negative (padding),
// and with `causal` if j <= p.  A row that sees nothing gives 0, with zero
// gradients.  Scores are kept in units of log2, so that exp is one exp2.

#include "lm_ops.h"

#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <hip/hip_runtime.h>
#include <algorithm>
#include <cmath>

namespace {

constexpr float LOG2E = 1.4426950408889634f;
constexpr int MOST_D = 128;

// [batch, length, heads, d] with strides in values, d contiguous
struct View {
    void* at;
    int64_t sb, ss, sh;
};

struct Args {
    View q, k, v, out, dout, dq, dk, dv;
    float* lse;              // [batch, hq, sq], in log2 units
    float* delta;            // [batch, hq, sq]
    const int* documents;    // [batch, sk] or none
    int64_t documents_sb;
    const float* slopes;     // [hq] or none
    int b, sq, sk, hq, hkv, d;
    int causal;
    float scale;
    float c;                 // the scores' factor in log2 units, not 0: hidden ones stay -inf
};

template <typename T>
__device__ __forceinline__ T* row(const View& x, int b, int s, int h) {
    return (T*)x.at + (int64_t)b * x.sb + (int64_t)s * x.ss + (int64_t)h * x.sh;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

__device__ __forceinline__ float wave_sum(float x) {
    for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
    return x;
}
__device__ __forceinline__ float wave_max(float x) {
    for (int m = 32; m; m >>= 1) x = fmaxf(x, __shfl_xor(x, m));
    return x;
}

__device__ __forceinline__ bool visible(const Args& a, int b, int pos, int j) {
    if (a.causal && j > pos) return false;
    if (a.documents) {
        const int* doc = a.documents + b * a.documents_sb;
        int dj = doc[j];
        return dj >= 0 && dj == doc[pos];
    }
    return true;
}

// rows start at 16-byte addresses and d is a multiple of 8
template <typename T>
__device__ __forceinline__ float dot(const T* x, const T* y, int d) {
    typedef T Vec __attribute__((ext_vector_type(16 / sizeof(T))));
    float s = 0;
#pragma unroll 4
    for (int i = 0; i < d; i += 16 / sizeof(T)) {
        const Vec u = *(const Vec*)(x + i), v = *(const Vec*)(y + i);
#pragma unroll
        for (int e = 0; e < (int)(16 / sizeof(T)); ++e) s = fmaf((float)u[e], (float)v[e], s);
    }
    return s;
}

// Rows of up to DP values, of which a lane reads 16 bytes and CHUNKS lanes all:
// 64 / CHUNKS rows at a time.  RowSum is a weighted sum of them.
template <typename T, int DP> struct Chunk {
    static constexpr int PER = 16 / sizeof(T), VECS = DP / PER;
    static constexpr int CHUNKS = VECS <= 4 ? 4 : VECS <= 8 ? 8 : VECS <= 16 ? 16 : 32;
    typedef T Vec __attribute__((ext_vector_type(PER)));
};
template <typename T, int DP> struct RowSum : Chunk<T, DP> {
    using Chunk<T, DP>::PER;
    using Chunk<T, DP>::CHUNKS;
    using typename Chunk<T, DP>::Vec;
    float x[PER] = {};

    // w of lane n times row_of(n) for the lanes n in `any`; others' rows are not read
    template <typename R>
    __device__ __forceinline__ void add(float w, uint64_t any, int d, R row_of) {
        const int lane = threadIdx.x & 63, c = (lane % CHUNKS) * PER;
#pragma unroll 4
        for (int n = 0; n < CHUNKS; ++n) {
            const int r = n * (64 / CHUNKS) + lane / CHUNKS;
            const float by = __shfl(w, r);
            if (!(any >> r & 1) || c >= d) continue;
            const Vec v = *(const Vec*)(row_of(r) + c);
#pragma unroll
            for (int e = 0; e < PER; ++e) x[e] = fmaf(by, (float)v[e], x[e]);
        }
    }
    __device__ __forceinline__ void store(T* to, int d, float scale) {
        const int lane = threadIdx.x & 63, c = (lane % CHUNKS) * PER;
        Vec v;
#pragma unroll
        for (int e = 0; e < PER; ++e) {
            for (int m = CHUNKS; m < 64; m <<= 1) x[e] += __shfl_xor(x[e], m);
            v[e] = (T)(x[e] * scale);
        }
        if (lane < CHUNKS && c < d) *(Vec*)(to + c) = v;
    }
};

__device__ __forceinline__ float slope_of(const Args& a, int h) {
    return a.slopes ? a.slopes[h] * LOG2E : 0.f;
}

// ---------------------------------------------------------------------------
// One wave for each row, lanes over keys (or queries) for the scores and over
// the head's values for the sums.  Pairs that are not visible are passed over,
// never multiplied by zero, so that an infinity or NaN behind the mask stays
// there.
// ---------------------------------------------------------------------------

template <typename T, int DP>
__device__ void forward_row(const Args& a, int b, int h, int i) {
    const int lane = threadIdx.x & 63, g = h / (a.hq / a.hkv), pos = i + a.sk - a.sq;
    const float slope = slope_of(a, h);
    const T* q = row<T>(a.q, b, i, h);
    const int end = a.causal ? pos + 1 : a.sk;
    auto score = [&](int j) {
        return dot(q, row<T>(a.k, b, j, g), a.d) * (a.scale * LOG2E) - slope * abs(pos - j);
    };
    // the sum first: with whole probabilities no partial result passes the
    // largest value
    float top = -INFINITY, total = 0;
    for (int j = lane; j < end; j += 64)
        if (visible(a, b, pos, j)) {
            float s = score(j), next = fmaxf(top, s);
            float base = next == -INFINITY ? 0.f : next;
            total = total * exp2_fast(top - base) + exp2_fast(s - base);
            top = next;
        }
    float base = wave_max(top);
    base = base == -INFINITY ? 0.f : base;
    total = wave_sum(total * exp2_fast(top - base));
    const float inv = total == 0.f ? 0.f : 1.f / total;
    RowSum<T, DP> o;
    for (int j0 = 0; j0 < end; j0 += 64) {
        int j = j0 + lane;
        bool seen = j < end && visible(a, b, pos, j);
        float p = seen ? exp2_fast(score(j) - base) * inv : 0.f;
        o.add(p, __ballot(seen), a.d, [&](int n) { return row<T>(a.v, b, j0 + n, g); });
    }
    o.store(row<T>(a.out, b, i, h), a.d, 1.f);
    if (lane == 0 && a.lse)
        a.lse[((int64_t)b * a.hq + h) * a.sq + i] = total == 0.f ? -INFINITY : base + log2f(total);
}

// also leaves the row's delta, from probabilities of 32 bits
template <typename T, int DP>
__device__ void dq_row(const Args& a, int b, int h, int i) {
    const int lane = threadIdx.x & 63, g = h / (a.hq / a.hkv), pos = i + a.sk - a.sq;
    const float slope = slope_of(a, h);
    const int64_t at = ((int64_t)b * a.hq + h) * a.sq + i;
    const float lse = a.lse[at];
    const T *q = row<T>(a.q, b, i, h), *dout = row<T>(a.dout, b, i, h);
    RowSum<T, DP> acc;
    float delta = 0;
    const int end = lse == -INFINITY ? 0 : a.causal ? pos + 1 : a.sk;
    auto p_of = [&](int j) {
        return exp2_fast(dot(q, row<T>(a.k, b, j, g), a.d) * (a.scale * LOG2E) -
                         slope * abs(pos - j) - lse);
    };
    for (int j = lane; j < end; j += 64)
        if (visible(a, b, pos, j))
            delta = fmaf(p_of(j), dot(dout, row<T>(a.v, b, j, g), a.d), delta);
    delta = wave_sum(delta);
    for (int j0 = 0; j0 < end; j0 += 64) {
        int j = j0 + lane;
        bool seen = j < end && visible(a, b, pos, j);
        float ds = seen ? p_of(j) * (dot(dout, row<T>(a.v, b, j, g), a.d) - delta) : 0.f;
        acc.add(ds, __ballot(seen), a.d, [&](int n) { return row<T>(a.k, b, j0 + n, g); });
    }
    acc.store(row<T>(a.dq, b, i, h), a.d, a.scale);
    if (lane == 0) a.delta[at] = delta;
}

template <typename T, int DP>
__device__ void dkv_row(const Args& a, int b, int g, int j) {
    const int lane = threadIdx.x & 63, group = a.hq / a.hkv;
    const T *k = row<T>(a.k, b, j, g), *v = row<T>(a.v, b, j, g);
    RowSum<T, DP> dk, dv;
    const int begin = a.causal ? max(0, j - (a.sk - a.sq)) : 0;
    for (int h = g * group; h < (g + 1) * group; ++h) {
        const float slope = slope_of(a, h);
        const int64_t at = ((int64_t)b * a.hq + h) * a.sq;
        for (int i0 = begin & ~63; i0 < a.sq; i0 += 64) {
            int i = i0 + lane, pos = i + a.sk - a.sq;
            bool seen = i < a.sq && visible(a, b, pos, j) && a.lse[at + i] != -INFINITY;
            uint64_t any = __ballot(seen);
            float p = 0, ds = 0;
            if (seen) {
                float s = dot(row<T>(a.q, b, i, h), k, a.d) * (a.scale * LOG2E) -
                          slope * abs(pos - j);
                p = exp2_fast(s - a.lse[at + i]);
                ds = p * (dot(row<T>(a.dout, b, i, h), v, a.d) - a.delta[at + i]);
            }
            dv.add(p, any, a.d, [&](int n) { return row<T>(a.dout, b, i0 + n, h); });
            dk.add(ds, any, a.d, [&](int n) { return row<T>(a.q, b, i0 + n, h); });
        }
    }
    dk.store(row<T>(a.dk, b, j, g), a.d, a.scale);
    dv.store(row<T>(a.dv, b, j, g), a.d, 1.f);
}

// ---------------------------------------------------------------------------
// Tiles on the matrix cores.  A fragment of a 32x32x16 product is 8 values a
// lane: lane l holds row (or column) l % 32, k = (l / 32) * 8 + 0..7; of the
// result it holds column l % 32 and rows 8 (i / 4) + 4 (l / 32) + i % 4.
//
// Scores are formed transposed, keys as rows and queries as columns.  A query
// then lies in one lane and its other half, so its maximum and sum need one
// exchange between lanes for a whole tile, and the lane's probabilities are,
// in the order they come, the right operand of the product with V: k index
// (l / 32) * 8 + j stands for key 8 (j / 4) + 4 (l / 32) + j % 4 on both
// sides.  The left operand is V transposed, which the transposing read of
// shared memory gives from rows as they lie in memory.
// ---------------------------------------------------------------------------

typedef float acc16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x8 __attribute__((ext_vector_type(8)));
typedef short short4v __attribute__((ext_vector_type(4)));
typedef float f32x4 __attribute__((ext_vector_type(4)));

template <typename T> struct FragOf;
template <> struct FragOf<__bf16> { typedef bf16x8 type; };
template <> struct FragOf<_Float16> { typedef f16x8 type; };
template <> struct FragOf<float> { typedef f32x8 type; };
template <typename T> using Frag = typename FragOf<T>::type;

__device__ __forceinline__ acc16 mma(bf16x8 a, bf16x8 b, acc16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ acc16 mma(f16x8 a, f16x8 b, acc16 c) {
    return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// 32-bit products have a k of 2, one value of each half of the wave: the 8
// values of a fragment take 8 of them
__device__ __forceinline__ acc16 mma(f32x8 a, f32x8 b, acc16 c) {
#pragma unroll
    for (int j = 0; j < 8; ++j) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[j], b[j], c, 0, 0, 0);
    return c;
}

constexpr int RANGE = 32;            // positions whose documents share a range
constexpr int NONE = 0x7fffffff;

// Rows of a tile in shared memory: chunks of 16 bytes, a power of two a row,
// at their number XOR a mirrored row number.  16 lanes that read one chunk of
// 16 rows, and 16 that read four chunks of 4 rows, then meet all banks.
template <typename T, int DP> struct Tile {
    static constexpr int PER = 16 / sizeof(T);
    static constexpr int VECS = DP / PER;
    static constexpr int CHUNKS = VECS <= 4 ? 4 : VECS <= 8 ? 8 : 16;
    // 32-bit columns are read one value a lane: a padded row serves them
    static constexpr int LD = sizeof(T) == 2 ? CHUNKS * PER : DP + PER;

    static __device__ __forceinline__ int mirrored(int row) {
        if constexpr (CHUNKS == 4) return (row >> 3 & 1) | (row >> 1 & 2);
        if constexpr (CHUNKS == 8) return (row >> 3 & 1) | (row >> 1 & 2) | (row << 1 & 4);
        return (row >> 3 & 1) | (row >> 1 & 2) | (row << 1 & 4) | (row << 3 & 8);
    }
    static __device__ __forceinline__ int at(int row, int x) {
        if constexpr (sizeof(T) == 4) return row * LD + x;
        return row * LD + ((x / PER) ^ mirrored(row)) * PER + x % PER;
    }
};

// Rows of one tile on their way from memory to shared memory, through
// registers so that they travel while the tile before is worked on.  Buffer
// loads take the tile's address from scalar registers and give zero behind
// its end, so a load costs no address and no comparison.
template <typename T, int DP, int ROWS, int THREADS> struct Stage {
    using G = Tile<T, DP>;
    static constexpr int N = ROWS * G::VECS / THREADS;
    static_assert(N * THREADS == ROWS * G::VECS, "threads share a tile's vectors evenly");
    typedef unsigned raw4 __attribute__((ext_vector_type(4)));
    raw4 r[N];
    int offset[N];   // of this thread's vectors, in bytes; the end for those behind d
    int row_bytes, d_bytes, tid;

    __device__ __forceinline__ Stage(int64_t stride, int d, int tid)
        : row_bytes((int)stride * (int)sizeof(T)), d_bytes(d * (int)sizeof(T)), tid(tid) {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            int v = tid + n * THREADS, y = v / G::VECS, x = (v % G::VECS) * G::PER;
            offset[n] = x < d ? y * row_bytes + x * (int)sizeof(T) : 0x7fffffff - 15;
        }
    }
    __device__ __forceinline__ void load(const T* base, int rows) {
        auto buffer = __builtin_amdgcn_make_buffer_rsrc(
            (void*)base, 0, (min(rows, ROWS) - 1) * row_bytes + d_bytes, 0x00027000);
#pragma unroll
        for (int n = 0; n < N; ++n)
            r[n] = __builtin_amdgcn_raw_buffer_load_b128(buffer, offset[n], 0, 0);
    }
    // rows that `there` does not say become zero
    template <typename F> __device__ __forceinline__ void keep(F there) {
#pragma unroll
        for (int n = 0; n < N; ++n)
            if (!there((tid + n * THREADS) / G::VECS)) r[n] = raw4{};
    }
    __device__ __forceinline__ void store(T* tile) const {
#pragma unroll
        for (int n = 0; n < N; ++n) {
            int v = tid + n * THREADS, y = v / G::VECS, x = (v % G::VECS) * G::PER;
            *(raw4*)(tile + G::at(y, x)) = r[n];
        }
    }
};

// rows y0 + l % 32 of a tile, values x0 + (l / 32) * 8 + 0..7
template <typename T, int DP>
__device__ __forceinline__ Frag<T> rows_of(const T* tile, int y0, int x0) {
    using G = Tile<T, DP>;
    const int lane = threadIdx.x & 63, y = lane & 31, x = x0 + (lane >> 5) * 8;
    Frag<T> f;
    tile += y0 * G::LD;
    if constexpr (sizeof(T) == 2) {
        f = *(const Frag<T>*)(tile + G::at(y, x));
    } else {
        const f32x4 lo = *(const f32x4*)(tile + G::at(y, x));
        const f32x4 hi = *(const f32x4*)(tile + G::at(y, x + 4));
        f = Frag<T>{lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
    }
    return f;
}

// columns x0 + l % 32, rows y0 + 8 (j / 4) + 4 (l / 32) + j % 4
template <typename T, int DP>
__device__ __forceinline__ Frag<T> columns_of(const T* tile, int y0, int x0) {
    using G = Tile<T, DP>;
    const int lane = threadIdx.x & 63;
    Frag<T> f;
    tile += y0 * G::LD;
    if constexpr (sizeof(T) == 2) {
        // 16 lanes read 4 rows of 16 values and get a column of 4 each
        const int y = (lane >> 5) * 4 + ((lane & 15) >> 2);
        const int x = x0 + ((lane >> 4) & 1) * 16 + (lane & 3) * 4;
        typedef __attribute__((address_space(3))) short4v* Shared;
        short4v lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Shared)(tile + G::at(y, x)));
        short4v hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((Shared)(tile + G::at(y + 8, x)));
        __builtin_memcpy(&f, &lo, 8);
        __builtin_memcpy((char*)&f + 8, &hi, 8);
    } else {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            f[j] = tile[G::at((lane >> 5) * 4 + 8 * (j >> 2) + (j & 3), x0 + (lane & 31))];
    }
    return f;
}

// 8 values of a row in memory, zero behind d or where there is no row
template <typename T>
__device__ __forceinline__ Frag<T> row_frag(const T* base, int x, int d, bool there) {
    Frag<T> f = {};
    if (there && x < d) f = *(const Frag<T>*)(base + x);
    return f;
}

template <typename T>
__device__ __forceinline__ Frag<T> to_frag(const acc16& c, int first) {
    Frag<T> f;
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = (T)c[first + j];
    return f;
}

// the other half of the wave's value for the same column
__device__ __forceinline__ float max_halves(float x) {
    auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(s[0]), __uint_as_float(s[1]));
}
__device__ __forceinline__ float add_halves(float x) {
    auto s = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(s[0]) + __uint_as_float(s[1]);
}

// sums += (rows y0 .. y0 + 32 of a tile) transposed * c.  In 32 bits the rows'
// own sum comes first: added one by one, tens of thousands of products would
// lose more bits than a product of matrices does.
template <typename T, int DP>
__device__ __forceinline__ void add_product(const T* tile, int y0, const acc16& c, acc16* sums) {
    const Frag<T> lo = to_frag<T>(c, 0), hi = to_frag<T>(c, 8);
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) {
        acc16 x = {};
        if constexpr (sizeof(T) == 2) x = sums[n];
        x = mma(columns_of<T, DP>(tile, y0, n * 32), lo, x);
        x = mma(columns_of<T, DP>(tile, y0 + 16, n * 32), hi, x);
        if constexpr (sizeof(T) == 4) x += sums[n];
        sums[n] = x;
    }
}

// The documents of some positions: x is the least of those that are not
// negative (NONE without one), with the top bit set if there are negative
// ones too, y the largest.
__device__ __forceinline__ bool meet(int2 a, int2 b) {
    return max(a.x & NONE, b.x & NONE) <= min(a.y, b.y);
}
// all positions of both hold one document, and it is the same
__device__ __forceinline__ bool one_document(int2 a, int2 b) {
    return a.x == a.y && b.x == b.y && a.x == b.x;
}
__device__ __forceinline__ int2 both(int2 a, int2 b) {
    return make_int2(min(a.x & NONE, b.x & NONE) | ((a.x | b.x) & INT_MIN), max(a.y, b.y));
}

// ranges of RANGE positions each, [batch, count], from position `first` on
struct Ranges {
    const int2* at;  // none without documents
    int count;

    __device__ __forceinline__ int2 of(int b, int n) const {
        return n < count ? at[(int64_t)b * count + n] : make_int2(-1, -1);
    }
};

__global__ __launch_bounds__(256) void ranges_kernel(const int* documents, int64_t sb, int first,
                                                     int end, int count, int64_t all,
                                                     int2* ranges) {
    int64_t n = (int64_t)blockIdx.x * (256 / RANGE) + threadIdx.x / RANGE;
    if (n >= all) return;
    int at = first + (int)(n % count) * RANGE + threadIdx.x % RANGE;
    int doc = at < end ? documents[n / count * sb + at] : -1;
    int2 r = make_int2(doc < 0 ? -1 : doc, doc);
    for (int m = RANGE / 2; m; m >>= 1)
        r = both(r, make_int2(__shfl_xor(r.x, m), __shfl_xor(r.y, m)));
    if (threadIdx.x % RANGE == 0) ranges[n] = r;
}

// The next 64 tiles, a bit each: `block` those that some position of the
// block may see, `wave` some of the wave, `whole` those that all of the wave
// see wholly as far as documents go.  Every wave looks at all 64, one each
// lane, so that nothing passes between waves.
struct Visits {
    uint64_t block, wave, whole;
};
template <int SIZE>
__device__ __forceinline__ Visits visits_of(const Ranges& r, int b, int first, int n, int2 block,
                                            int2 wave) {
    const uint64_t all = n >= 64 ? ~0ull : (1ull << n) - 1;
    if (!r.at) return {all, all, all};
    const int t = first + (threadIdx.x & 63);
    int2 x = r.of(b, t * (SIZE / RANGE));
#pragma unroll
    for (int m = 1; m < SIZE / RANGE; ++m) x = both(x, r.of(b, t * (SIZE / RANGE) + m));
    return {__ballot(meet(x, block)) & all, __ballot(meet(x, wave)) & all,
            __ballot(one_document(x, wave)) & all};
}

// A block of ROWS * SHARES waves: ROWS waves of 32 rows each share their tiles,
// and SHARES such groups take the block's tiles in turn, with a tile each at a
// time, and add their sums up at the end.  Shares put more waves on few rows.
__device__ __forceinline__ uint64_t bit_of(uint64_t bits, int n) {
    for (; n; --n) bits &= bits - 1;
    return bits & -bits;
}
template <int N> __device__ __forceinline__ uint64_t without(uint64_t bits) {
#pragma unroll
    for (int n = 0; n < N; ++n) bits &= bits - 1;
    return bits;
}

// With 4 shares a wave fetches its tile alone: 32 rows keep it in registers.
template <typename T, int SHARES>
constexpr int tile_rows = SHARES == 4 || sizeof(T) == 4 ? 32 : 64;

// the shares' tiles and, at the end, the sums they leave for the first
template <typename T, int DP, int N, int SHARES, int FLOATS> union Shared {
    alignas(256) T tiles[SHARES][2][N * Tile<T, DP>::LD];
    alignas(16) float boxes[FLOATS ? FLOATS : 4];
};

// a wave's sums for another: [32 DP / 64] floats a lane, lanes next to each other
template <int DP>
__device__ __forceinline__ void leave(float* box, const acc16* x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i) box[(n * 16 + i) * 64 + lane] = x[n][i];
}
template <int DP>
__device__ __forceinline__ void take(const float* box, float mine, float theirs, acc16* x) {
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
        for (int i = 0; i < 16; ++i)
            x[n][i] = fmaf(box[(n * 16 + i) * 64 + lane], theirs, x[n][i] * mine);
}

// Workgroups go round the 8 XCDs: neighbours in the order returned run on one
// XCD and share its L2.
__device__ __forceinline__ unsigned xcd_order(unsigned block, unsigned blocks) {
    unsigned each = blocks / 8, more = blocks % 8, x = block % 8;
    return x * each + min(x, more) + block / 8;
}

// The tile of queries (the last sees most keys) that the n-th block of a head
// takes where rows are causal.  Blocks go round the CUs: where all fit at once,
// every other head runs the other way and each CU gets long and short ones (24
// heads of 64, 4096 rows, 768 blocks, three a CU: forward 99 us for 118); where
// some wait for others, the longest go first (dq of the same, two a CU: 147 us
// for 170).
__device__ __forceinline__ int causal_order(int n, int tiles, int head, bool alternate) {
    return alternate && (head & 1) ? n : tiles - 1 - n;
}

// Waves a SIMD that the registers are shared out for: 2, 3 where they do for as
// many (the forward of heads of 64 and blocks of 4 waves), or 1 where two would
// spill (to 256 registers; 3 spill in the backward of heads of 64: dq 133 us for
// 72 on packed rows of 512).
template <typename T, int DP, int SHARES>
constexpr int forward_waves =
    (DP >= 96 && SHARES > 1) || (DP == 128 && sizeof(T) == 4) || SHARES == 4 ? 1
    : sizeof(T) == 2 && DP <= 64 && SHARES == 1                              ? 3
                                                                             : 2;
template <int DP, int SHARES> constexpr int dq_waves = DP >= 96 || SHARES > 1 ? 1 : 2;
template <typename T, int DP, int SHARES>
constexpr int dkv_waves = DP >= 96 || (DP == 64 && sizeof(T) == 4) || SHARES == 4 ? 1 : 2;

constexpr float HEADROOM = 3.f;  // how far (log2) a score may pass the reference maximum
constexpr float SHIFT = 12.f;    // probabilities carry a factor 2^12, at most 2^15 in all:
                                 // in fp16 the small ones keep their bits

// Scores (log2) that 32 bits hold to less than about 1: a probability that a
// product formed with them, and not its rounded score, could be anything.  Rows
// with such a maximum are formed pair by pair.
constexpr float FAR = 0x1p22f;

// x = -inf for the rows of other documents, of sub-tile t of 32 rows; docs of a
// tile's rows, with -1 behind the last
__device__ __forceinline__ void hide_documents(acc16& x, const int* docs, int t, int doc) {
    const int hf = (threadIdx.x & 63) >> 5;
#pragma unroll
    for (int r = 0; r < 4; ++r) {
        int4 d = *(const int4*)(docs + t * 32 + r * 8 + 4 * hf);
        x[r * 4] = d.x == doc ? x[r * 4] : -INFINITY;
        x[r * 4 + 1] = d.y == doc ? x[r * 4 + 1] : -INFINITY;
        x[r * 4 + 2] = d.z == doc ? x[r * 4 + 2] : -INFINITY;
        x[r * 4 + 3] = d.w == doc ? x[r * 4 + 3] : -INFINITY;
    }
}
// ... and for those past row `last` of the tile
__device__ __forceinline__ void hide_past(acc16& x, int t, int last) {
    const int l = last - t * 32 - 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 8 * (i >> 2) + (i & 3) > l ? -INFINITY : x[i];
}

// ... or before row `begin`
__device__ __forceinline__ void hide_before(acc16& x, int t, int begin) {
    const int l = begin - t * 32 - 4 * ((threadIdx.x & 63) >> 5);
#pragma unroll
    for (int i = 0; i < 16; ++i) x[i] = 8 * (i >> 2) + (i & 3) < l ? -INFINITY : x[i];
}

// products to the exponents of their probabilities; far: how far the query lies
// behind the tile's first key of this half
template <int KT>
__device__ __forceinline__ void exponents(acc16* s, float c, float off, float slope, float far) {
    if (slope != 0.f) {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i)
                s[t][i] = fmaf(s[t][i], c,
                               fmaf(-slope, fabsf(far - (float)(t * 32 + 8 * (i >> 2) + (i & 3))),
                                    -off));
    } else {
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) s[t][i] = fmaf(s[t][i], c, -off);
    }
}

// One wave's 32 queries against tiles of keys: the running softmax.
template <typename T, int DP> struct Forward {
    using G = Tile<T, DP>;
    Frag<T> q[DP / 16];
    acc16 o[DP / 32];
    float off, total;       // what exponents lose (the reference maximum less SHIFT), this
                            // half's sum
    bool fresh;             // nothing seen yet
    float c;                // score factor, in units of log2
    float slope;
    int doc;                // the lane's query's document, INT_MIN for none
    int pos;                // its position

    __device__ __forceinline__ void begin(const Args& a, const T* row, bool there, float slope_) {
        const int hf = (threadIdx.x & 63) >> 5;
        slope = slope_;
        c = a.c;
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
            q[n] = row_frag<T>(row, n * 16 + hf * 8, a.d, there);
            if (a.scale < 0) q[n] = -q[n];
        }
#pragma unroll
        for (int n = 0; n < DP / 32; ++n) o[n] = acc16{};
        fresh = true;
        off = 0;
        total = 0;
    }

    // keys key0 .. key0 + 32 KT, k(t, n) the fragments of their rows; some may
    // be hidden by their documents or lie past the query
    template <int KT, typename K>
    __device__ __forceinline__ void step(K k, const T* v, const int* docs, int key0,
                                         bool by_document, bool by_position) {
        const int hf = (threadIdx.x & 63) >> 5;
        acc16 s[KT];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            s[t] = acc16{};
#pragma unroll
            for (int n = 0; n < DP / 16; ++n) s[t] = mma(k(t, n), q[n], s[t]);
        }
        exponents<KT>(s, c, off, slope, (float)(pos - key0 - 4 * hf));
        if (by_document)
#pragma unroll
            for (int t = 0; t < KT; ++t) hide_documents(s[t], docs, t, doc);
        if (by_position)
#pragma unroll
            for (int t = 0; t < KT; ++t) hide_past(s[t], t, pos - key0);
        float most = -INFINITY;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 16; i += 2) most = fmaxf(most, fmaxf(s[t][i], s[t][i + 1]));
        most = max_halves(most);
        if (__any(most > (fresh ? -INFINITY : SHIFT + HEADROOM))) {
            // keys far below others to come, and rows of such keys alone, whose sum
            // will be 0, do not set the reference
            float by = fresh ? most == -INFINITY ? 0.f : fmaxf(most - SHIFT, -FAR)
                             : fmaxf(most - SHIFT, 0.f);
            const float next = off + by;
            by = next - off;  // as far as off really went
            const float keep = fresh ? 1.f : exp2_fast(-by);
            fresh = fresh && most == -INFINITY;
            off = next;
            total *= keep;
#pragma unroll
            for (int n = 0; n < DP / 32; ++n)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[n][i] *= keep;
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][i] -= by;
        }
        float sum = 0;  // a tile's first, so that long rows keep their bits
#pragma unroll
        for (int t = 0; t < KT; ++t) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[t][i] = exp2_fast(s[t][i]);
                sum += s[t][i];
            }
            add_product<T, DP>(v, t * 32, s[t], o);
        }
        total += sum;
    }

    // the sum of both halves, NaN if the row is to be formed pair by pair; the
    // reference maximum has only grown
    __device__ __forceinline__ float sum() const {
        const float x = add_halves(total);
        return off > FAR ? __builtin_nanf("") : x;
    }

    __device__ __forceinline__ bool finite() const {
        bool fine = true;
#pragma unroll
        for (int n = 0; n < DP / 32; ++n)
#pragma unroll
            for (int i = 0; i < 16; ++i) fine &= fabsf(o[n][i]) <= 3.4028235e38f;
        return fine;
    }
};

// ---------------------------------------------------------------------------
// Results that are not finite.  A hidden infinity or NaN times a probability
// of zero is NaN, and a scaled sum may pass the largest value: such rows are
// done again pair by pair, one after the other by their wave, which takes
// hundreds of times as long.  A row that its own inputs make so is left as it
// is, where that is certain, so that an overflowed step, an ordinary one under
// loss scaling, costs about what others do.  They make all of it NaN if a score
// is NaN or plus infinity, and a column not finite if a visible value is not,
// NaN for a NaN and an infinity for an infinity.  Forward and back of 2048 causal
// rows, 4 heads of 64, bf16, take 90 us, 105 with NaN all over, and 1.4 to 4.2 ms
// with one infinity, whose tiles are done again.
// ---------------------------------------------------------------------------

__device__ __forceinline__ uint32_t wave_or(uint32_t x, int from, int to) {
    for (int m = from; m < to; m <<= 1) x |= __shfl_xor(x, m);
    return x;
}

// columns of a head that hold NaN and infinities
template <int DP> struct Columns {
    static constexpr int N = DP / 32;
    uint32_t nan[N] = {}, inf[N] = {};

    static __device__ __forceinline__ uint32_t all(int n, int d) {
        return d - n * 32 >= 32 ? ~0u : (1u << (d - n * 32)) - 1;
    }
    // those of each lane's row, which lies in a result's registers
    __device__ __forceinline__ void of(const acc16* x, int d) {
        const int hf = (threadIdx.x & 63) >> 5;
#pragma unroll
        for (int n = 0; n < N; ++n) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const uint32_t bit = 1u << (8 * (i >> 2) + (i & 3));
                if (x[n][i] != x[n][i]) nan[n] |= bit;
                if (fabsf(x[n][i]) == INFINITY) inf[n] |= bit;
            }
            nan[n] = wave_or(nan[n] << (4 * hf), 32, 64) & all(n, d);
            inf[n] = wave_or(inf[n] << (4 * hf), 32, 64) & all(n, d);
        }
    }
    // those of any row among the lanes that `mine` says
    __device__ __forceinline__ Columns joined(bool mine) const {
        Columns c;
#pragma unroll
        for (int n = 0; n < N; ++n) {
            c.nan[n] = wave_or(mine ? nan[n] : 0, 1, 64);
            c.inf[n] = wave_or(mine ? inf[n] : 0, 1, 64);
        }
        return c;
    }
    __device__ __forceinline__ bool any() const {
        uint32_t x = 0;
#pragma unroll
        for (int n = 0; n < N; ++n) x |= nan[n] | inf[n];
        return x;
    }
    __device__ __forceinline__ bool all_nan(int d) const {
        bool yes = true;
#pragma unroll
        for (int n = 0; n < N; ++n) yes &= nan[n] == all(n, d);
        return yes;
    }
    // `seen` makes them so
    __device__ __forceinline__ bool within(const Columns& seen) const {
        uint32_t x = 0;
#pragma unroll
        for (int n = 0; n < N; ++n)
            x |= (nan[n] & ~seen.nan[n]) | (inf[n] & ~(seen.nan[n] | seen.inf[n]));
        return x == 0;
    }
};

// Adds to `seen` the columns of NaN and infinities in those of the rows first
// to end of a head of x that `sees` says, until it holds all of `need`.  The
// wave reads 64 rows at a time; all lanes get the same.
template <typename T, int DP, typename S>
__device__ __forceinline__ void look_for(const Columns<DP>& need, const View& x, int b, int h,
                                         int first, int end, int d, S sees, Columns<DP>& seen) {
    constexpr int PER = Chunk<T, DP>::PER, CHUNKS = Chunk<T, DP>::CHUNKS;
    typedef typename Chunk<T, DP>::Vec Vec;
    const int lane = threadIdx.x & 63, c = (lane % CHUNKS) * PER, y = lane / CHUNKS;
    auto part = [&](const uint32_t* words) {  // this lane's columns
        uint32_t w = 0;
#pragma unroll
        for (int n = 0; n < DP / 32; ++n) w = c / 32 == n ? words[n] : w;
        return w >> (c % 32) & ((1u << PER) - 1);
    };
    const uint32_t need_nan = part(need.nan), need_inf = part(need.inf);
    uint32_t nan = part(seen.nan), inf = part(seen.inf);
    for (int j0 = first; j0 < end; j0 += 64) {
        if (__all((need_nan & ~nan) == 0 && (need_inf & ~(nan | inf)) == 0)) break;
        const uint64_t rows = __ballot(j0 + lane < end && sees(j0 + lane));
        if (!rows) continue;
#pragma unroll 4
        for (int n = 0; n < CHUNKS; ++n) {
            const int r = n * (64 / CHUNKS) + y;
            if (!(rows >> r & 1) || c >= d) continue;
            const Vec v = *(const Vec*)(row<T>(x, b, j0 + r, h) + c);
#pragma unroll
            for (int e = 0; e < PER; ++e) {
                const float f = (float)v[e];
                if (f != f) nan |= 1u << e;
                if (fabsf(f) == INFINITY) inf |= 1u << e;
            }
        }
        nan = wave_or(nan, CHUNKS, 64);
        inf = wave_or(inf, CHUNKS, 64);
    }
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) {
        seen.nan[n] |= wave_or(c / 32 == n ? nan << (c % 32) : 0, 1, CHUNKS);
        seen.inf[n] |= wave_or(c / 32 == n ? inf << (c % 32) : 0, 1, CHUNKS);
    }
}

// Calls f with the document, the first row and all rows of each group of a
// wave's rows (a bit each) that are of one document.
template <typename F>
__device__ __forceinline__ void for_documents(uint32_t rows, int doc, F f) {
    while (rows) {
        const int lead = __builtin_ctz(rows), of = __shfl(doc, lead);
        const bool mine = (rows >> (threadIdx.x & 31) & 1) && doc == of;
        const uint32_t group = (uint32_t)__ballot(mine);
        rows &= ~group;
        f(of, mine, group);
    }
}

// Those of the wave's queries `rows` whose columns `lost` are not explained by
// the rows of x, V or K, that they see.  Keys of a probability of 0 times an
// infinity make NaN of K's (`zeros`).
template <typename T, int DP>
__device__ __forceinline__ uint32_t unexplained(const Args& a, const View& x, int b, int g,
                                                uint32_t rows, int doc, int pos, bool zeros,
                                                const Columns<DP>& lost) {
    uint32_t again = 0;
    for_documents(rows, doc, [&](int of, bool mine, uint32_t group) {
        bool fine = false;
        if (of >= 0) {  // others see nothing
            const int* doc_row = a.documents ? a.documents + b * a.documents_sb : nullptr;
            const int end = a.causal ? __shfl(pos, __builtin_ctz(group)) + 1 : a.sk;
            Columns<DP> need = lost.joined(mine), seen;
            if (zeros)
#pragma unroll
                for (int n = 0; n < DP / 32; ++n) need.inf[n] |= need.nan[n], need.nan[n] = 0;
            look_for<T, DP>(need, x, b, g, 0, end, a.d,
                            [&](int j) { return !doc_row || doc_row[j] == of; }, seen);
            if (zeros)
#pragma unroll
                for (int n = 0; n < DP / 32; ++n) seen.nan[n] |= seen.inf[n];
            fine = lost.within(seen);
        }
        again |= group & (uint32_t)__ballot(mine && !fine);
    });
    return again;
}

// those of the rows j0 + n, n a bit of `rows`, that hold a value that is not finite
template <typename T, int DP>
__device__ __forceinline__ uint64_t not_finite(const View& x, int b, int h, int j0, uint64_t rows,
                                               int d) {
    constexpr int PER = Chunk<T, DP>::PER, CHUNKS = Chunk<T, DP>::CHUNKS, EACH = 64 / CHUNKS;
    typedef typename Chunk<T, DP>::Vec Vec;
    const int lane = threadIdx.x & 63, c = (lane % CHUNKS) * PER;
    uint64_t bad = 0;
#pragma unroll 4
    for (int n = 0; n < CHUNKS; ++n) {
        const int r = n * EACH + lane / CHUNKS;
        bool fine = true;
        if ((rows >> r & 1) && c < d) {
            const Vec v = *(const Vec*)(row<T>(x, b, j0 + r, h) + c);
#pragma unroll
            for (int e = 0; e < PER; ++e) fine &= fabsf((float)v[e]) < INFINITY;
        }
        const uint64_t found = __ballot(!fine);
        for (int y = 0; y < EACH; ++y)
            if (found >> (y * CHUNKS) & ((1ull << CHUNKS) - 1)) bad |= 1ull << (n * EACH + y);
    }
    return bad;
}

// Calls f for blocks of 64 keys, from j0 on and a bit each, that all of some of
// the wave's queries see: those of document `of` (not negative) up to position
// `last` if rows are causal; until f returns true.
template <typename F>
__device__ __forceinline__ void for_keys(const Args& a, int b, int of, int last, F f) {
    const int lane = threadIdx.x & 63, end = a.causal ? last + 1 : a.sk;
    const int* doc_row = a.documents ? a.documents + b * a.documents_sb : nullptr;
    for (int j0 = 0; j0 < end; j0 += 64) {
        const int j = j0 + lane;
        const uint64_t keys = __ballot(j < end && (!doc_row || doc_row[j] == of));
        if (keys && f(j0, keys)) return;
    }
}

// Those of the wave's queries `rows`, i the lane's, that have a score of NaN or
// plus infinity with a key that is not finite, or by not being finite themselves.
template <typename T, int DP>
__device__ __forceinline__ uint32_t nan_scores(const Args& a, int b, int h, int i, uint32_t rows,
                                               int doc, int pos) {
    typedef typename Chunk<T, DP>::Vec Vec;
    const int g = h / (a.hq / a.hkv);
    const bool there = rows >> (threadIdx.x & 31) & 1;
    const T* q = row<T>(a.q, b, there ? i : 0, h);
    bool fine = true;
    for (int c = 0; c < a.d && there; c += Chunk<T, DP>::PER) {
        const Vec v = *(const Vec*)(q + c);
#pragma unroll
        for (int e = 0; e < Chunk<T, DP>::PER; ++e) fine &= fabsf((float)v[e]) < INFINITY;
    }
    uint32_t found = 0;
    for_documents(rows, doc, [&](int of, bool mine, uint32_t group) {
        if (of < 0) return;
        uint32_t left = group;
        for_keys(a, b, of, __shfl(pos, __builtin_ctz(group)), [&](int j0, uint64_t keys) {
            if (!(left & (uint32_t)__ballot(!fine)))
                keys = not_finite<T, DP>(a.k, b, g, j0, keys, a.d);
            for (; keys && left; keys &= keys - 1) {
                const T* k = row<T>(a.k, b, j0 + __builtin_ctzll(keys), g);
                const float x = mine ? dot(q, k, a.d) * (a.scale * LOG2E) : 0.f;
                left &= ~(uint32_t)__ballot(!(x < INFINITY));
            }
            return left == 0;
        });
        found |= group & ~left;
    });
    return found;
}

// Those of the wave's queries `rows` that see a row of V that is not finite.
template <typename T, int DP>
__device__ __forceinline__ uint32_t see_not_finite(const Args& a, int b, int g, uint32_t rows,
                                                   int doc, int pos) {
    uint32_t found = 0;
    for_documents(rows, doc, [&](int of, bool, uint32_t group) {
        if (of < 0) return;
        for_keys(a, b, of, __shfl(pos, __builtin_ctz(group)), [&](int j0, uint64_t keys) {
            if (!not_finite<T, DP>(a.v, b, g, j0, keys, a.d)) return false;
            found |= group;
            return true;
        });
    });
    return found;
}

// four values of a row, as they lie in a result's registers
template <typename T>
__device__ __forceinline__ void put4(T* at, float a, float b, float c, float d) {
    typedef T Four __attribute__((ext_vector_type(4)));
    *(Four*)at = Four{(T)a, (T)b, (T)c, (T)d};
}

// 32 queries for each wave, all heads and keys.  The block's waves share the
// tiles of K and V; block tiles of one head are neighbours on one XCD, whose
// L2 then serves the head's keys once.
//
// Vector and matrix unit work in turn more than side by side: for heads of 64
// the one is busy for 53 % of the cycles (a multiply-add, an exponential, a
// maximum, a sum and half a conversion for each pair), the other for 29 %.  2 x
// 16 heads, 4096 x 4096, bf16: 710 TFLOP/s at 64, 890 at 128; a large matrix
// product reaches 1373.  Tiles of 64 keys: passing over half a tile by its
// documents costs more than it saves (582 TFLOP/s for 640).
template <typename T, int DP, int ROWS, int SHARES>
__global__ __launch_bounds__(ROWS * SHARES * 64, (forward_waves<T, DP, SHARES>))
void forward_kernel(const Args a, const Ranges keys, const Ranges queries, int tiles_q,
                    bool alternate) {
    using G = Tile<T, DP>;
    constexpr int BOX = (DP / 2 + 2) * 64;  // o, off and total
    constexpr int THREADS = ROWS * 64, N = tile_rows<T, SHARES>;
    __shared__ Shared<T, DP, N, SHARES, (SHARES - 1) * ROWS * BOX> shared;
    __shared__ alignas(16) int tile_docs[SHARES][N];

    unsigned id = xcd_order(blockIdx.x, gridDim.x);
    int qt = id % tiles_q, h = id / tiles_q % a.hq, b = id / tiles_q / a.hq;
    if (a.causal) qt = causal_order(qt, tiles_q, h, alternate);
    const int g = h / (a.hq / a.hkv), lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % ROWS;
    const int share = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / ROWS;
    const int tid = threadIdx.x - share * THREADS;
    T *tile_k = shared.tiles[share][0], *tile_v = shared.tiles[share][1];
    int* docs = tile_docs[share];
    const int first = a.sk - a.sq, row0 = (qt * ROWS + wave) * 32;
    const int i = row0 + (lane & 31);
    const bool there = i < a.sq;
    const int* doc_row = a.documents ? a.documents + b * a.documents_sb : nullptr;

    Forward<T, DP> f;
    f.begin(a, row<T>(a.q, b, there ? i : 0, h), there, slope_of(a, h));
    f.pos = i + first;
    const int doc = there ? doc_row ? doc_row[f.pos] : 0 : -1;
    f.doc = doc < 0 ? INT_MIN : doc;
    int2 wave_docs{}, block_docs{};
    if (doc_row) {
        wave_docs = queries.of(b, qt * ROWS + wave);
        block_docs = queries.of(b, qt * ROWS);
        for (int w = 1; w < ROWS; ++w) block_docs = both(block_docs, queries.of(b, qt * ROWS + w));
    }
    const int wave_first = row0 + first, wave_last = min(row0 + 31, a.sq - 1) + first;
    int end = a.sk;
    if (a.causal) end = min(end, (qt + 1) * ROWS * 32 + first);
    const int tiles = (end + N - 1) / N;
    const T *k = row<T>(a.k, b, 0, g), *v = row<T>(a.v, b, 0, g);

    Stage<T, DP, N, THREADS> sk(a.k.ss, a.d, tid), sv(a.v.ss, a.d, tid);
    for (int chunk = 0; chunk < tiles; chunk += 64) {
        Visits visits = visits_of<N>(keys, b, chunk, tiles - chunk, block_docs, wave_docs);
        uint64_t mine = 0;
        int next = 0, key_doc = -1;
        auto fetch = [&] {
            mine = bit_of(visits.block, share);
            if (!mine) return;
            next = (chunk + __builtin_ctzll(mine)) * N;
            sk.load(k + (int64_t)next * a.k.ss, a.sk - next);
            sv.load(v + (int64_t)next * a.v.ss, a.sk - next);
            int j = next + tid;
            if (tid < N) key_doc = j < a.sk ? doc_row ? max(doc_row[j], -1) : 0 : -1;
        };
        if (visits.block) fetch();
        while (visits.block) {
            __syncthreads();
            sk.store(tile_k);
            sv.store(tile_v);
            if (tid < N) docs[tid] = key_doc;
            __syncthreads();
            const uint64_t bit = mine;
            const int at = next;
            visits.block = without<SHARES>(visits.block);
            if (visits.block) fetch();
            if (!(visits.wave & bit) || (a.causal && at > wave_last)) continue;
            f.template step<N / 32>(
                [&](int t, int n) { return rows_of<T, DP>(tile_k, t * 32, n * 16); }, tile_v,
                docs, at, !(visits.whole & bit) || at + N > a.sk,
                a.causal && at + N - 1 > wave_first);
        }
    }

    float total = f.sum();
    if constexpr (SHARES > 1) {
        float* box = shared.boxes + wave * BOX;
        __syncthreads();
        if (share) {
            float* to = box + (share - 1) * ROWS * BOX;
            leave<DP>(to, f.o);
            to[DP / 2 * 64 + lane] = f.off;
            to[(DP / 2 + 1) * 64 + lane] = total;
        }
        __syncthreads();
        if (share) return;
        for (int n = 0; n < SHARES - 1; ++n, box += ROWS * BOX) {
            const float off = box[DP / 2 * 64 + lane], sum = box[(DP / 2 + 1) * 64 + lane];
            const float top = total == 0.f ? off : sum == 0.f ? f.off : fmaxf(f.off, off);
            const float keep = total == 0.f ? 0.f : exp2_fast(f.off - top);
            const float add = sum == 0.f ? 0.f : exp2_fast(off - top);
            take<DP>(box, keep, add, f.o);
            total = total * keep + sum * add;
            f.off = top;
        }
    }
    const float inv = total == 0.f ? 0.f : 1.f / total;
    if (there) {
        T* out = row<T>(a.out, b, i, h);
#pragma unroll
        for (int n = 0; n < DP / 32; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                int d = n * 32 + r * 8 + (lane >> 5) * 4;
                if (d < a.d)
                    put4(out + d, f.o[n][r * 4] * inv, f.o[n][r * 4 + 1] * inv,
                         f.o[n][r * 4 + 2] * inv, f.o[n][r * 4 + 3] * inv);
            }
        if (a.lse && lane < 32)
            a.lse[((int64_t)b * a.hq + h) * a.sq + i] =
                total == 0.f ? -INFINITY : f.off + log2f(total);
    }
    const bool none = total == 0.f && f.doc >= 0;  // though a query sees itself
    if (__any(there && (!f.finite() || total != total || none))) {
        Columns<DP> lost;
        lost.of(f.o, a.d);
        const uint32_t rows = (uint32_t)__ballot(there && total == total && !none && lost.any());
        const uint32_t nan = (uint32_t)__ballot(there && total != total);
        uint32_t again = (uint32_t)__ballot(there && none);
        again |= unexplained<T, DP>(a, a.v, b, g, rows, f.doc, f.pos, false, lost);
        if (nan) again |= nan & ~nan_scores<T, DP>(a, b, h, i, nan, f.doc, f.pos);
        for (; again; again &= again - 1)
            forward_row<T, DP>(a, b, h, row0 + __builtin_ctz(again));
    }
}

// Few queries over many keys: bound by one read of what is visible of K and V.
// 8 requests of 32768 keys, 4 heads of 64, bf16: 268 MB in 42 us and 5 us the
// join (5.7 TB/s in all; reads alone reach 6.1); with 30 % of the keys hidden in
// front as long, 189 MB at 4.4 TB/s, since parts of hidden keys alone have nothing to do.
// A wave takes up to 32 columns, which are the queries of all heads of one
// key-value head, and one part of the keys; nothing is shared between waves.  K's fragments are
// rows as they lie in memory and go straight to registers, V passes through
// shared memory for its columns; both travel a tile ahead.  join_kernel adds
// the parts up, each with its own exponent.
template <typename T, int DP>
__global__ __launch_bounds__(64, DP >= 96 ? 1 : 2)
void split_kernel(const Args a, int parts, int keys_each, int column_tiles, float* part_o,
                  float2* part_state) {
    using G = Tile<T, DP>;
    constexpr int N = 32;
    __shared__ alignas(256) T tile_v[N * G::LD];
    __shared__ alignas(16) int docs[N];

    unsigned id = xcd_order(blockIdx.x, gridDim.x);
    const int part = id % parts, ct = id / parts % column_tiles;
    const int g = id / parts / column_tiles % a.hkv, b = id / parts / column_tiles / a.hkv;
    const int lane = threadIdx.x, hf = lane >> 5, group = a.hq / a.hkv, first = a.sk - a.sq;
    const int columns = group * a.sq, column = ct * 32 + (lane & 31);
    const bool there = column < columns;
    const int h = g * group + (there ? column / a.sq : 0), i = there ? column % a.sq : 0;
    const int* doc_row = a.documents ? a.documents + b * a.documents_sb : nullptr;

    Forward<T, DP> f;
    f.begin(a, row<T>(a.q, b, i, h), there, slope_of(a, h));
    f.pos = i + first;
    const int doc = there ? doc_row ? doc_row[f.pos] : 0 : -1;
    f.doc = doc < 0 ? INT_MIN : doc;
    int least = doc < 0 ? NONE : doc, largest = doc;
    for (int m = 16; m; m >>= 1) {
        least = min(least, __shfl_xor(least, m));
        largest = max(largest, __shfl_xor(largest, m));
    }
    int latest = there ? f.pos : 0, earliest = there ? f.pos : a.sk;
    for (int m = 32; m; m >>= 1) {
        latest = max(latest, __shfl_xor(latest, m));
        earliest = min(earliest, __shfl_xor(earliest, m));
    }
    int end = min(a.sk, (part + 1) * keys_each);
    if (a.causal) end = min(end, latest + 1);
    const T *k = row<T>(a.k, b, 0, g), *v = row<T>(a.v, b, 0, g);

    Frag<T> next_k[DP / 16];
    Stage<T, DP, N, 64> sv(a.v.ss, a.d, lane);
    for (int chunk = part * keys_each; chunk < end; chunk += 64 * N) {
        // tiles with a key that some query may see, of 64
        const int tiles = min(64, (end - chunk + N - 1) / N);
        uint64_t visits = tiles == 64 ? ~0ull : (1ull << tiles) - 1;
        uint64_t whole = visits;  // those that all their keys may be seen of
        if (doc_row) {
            visits = whole = 0;
            for (int t = 0; t < tiles; t += 2) {
                int j = chunk + t * N + lane, d = j < end ? doc_row[j] : -1;
                uint64_t met = __ballot(d >= least && d <= largest);
                if (met & 0xffffffffull) visits |= 1ull << t;
                if (met >> 32) visits |= 2ull << t;
                if ((met & 0xffffffffull) == 0xffffffffull) whole |= 1ull << t;
                if (met >> 32 == 0xffffffffull) whole |= 2ull << t;
            }
        }
        int key_doc = -1;
        auto fetch = [&](int at) {
            const bool row_there = at + (lane & 31) < a.sk;
            const T* kr = k + (int64_t)(row_there ? at + (lane & 31) : at) * a.k.ss;
#pragma unroll
            for (int n = 0; n < DP / 16; ++n)
                next_k[n] = row_frag<T>(kr, n * 16 + hf * 8, a.d, row_there);
            sv.load(v + (int64_t)at * a.v.ss, end - at);
            int j = at + lane;
            if (lane < N) key_doc = j < a.sk ? doc_row ? max(doc_row[j], -1) : 0 : -1;
        };
        int at = visits ? chunk + __builtin_ctzll(visits) * N : 0;
        if (visits) fetch(at);
        while (visits) {
            // what a cache holds where there is no sequence may be anything
            if (!(whole >> __builtin_ctzll(visits) & 1))
                sv.keep([&](int y) {
                    const int d = __shfl(key_doc, y);
                    return d >= least && d <= largest;
                });
            visits &= visits - 1;
            // one wave: its own reads and writes of shared memory keep order
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            sv.store(tile_v);
            if (lane < N) docs[lane] = key_doc;
            __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
            Frag<T> k_now[DP / 16];
#pragma unroll
            for (int n = 0; n < DP / 16; ++n) k_now[n] = next_k[n];
            const int now = at;
            if (visits) {
                at = chunk + __builtin_ctzll(visits) * N;
                fetch(at);
            }
            f.template step<1>([&](int, int n) { return k_now[n]; }, tile_v, docs, now,
                               doc_row || now + N > a.sk, a.causal && now + N - 1 > earliest);
        }
    }

    const float total = f.sum();
    if (!there) return;
    const int64_t at = (((int64_t)b * a.hkv + g) * columns + column) * parts + part;
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
        for (int r = 0; r < 4; ++r)
            put4(part_o + at * DP + n * 32 + r * 8 + hf * 4, f.o[n][r * 4], f.o[n][r * 4 + 1],
                 f.o[n][r * 4 + 2], f.o[n][r * 4 + 3]);
    if (hf == 0) part_state[at] = make_float2(f.off, total);
}

constexpr int MOST_PARTS = 256;

// One row a block: the parts' exponents and sums first, then their values in
// 256 / DP shares of the parts.
template <typename T, int DP>
__global__ __launch_bounds__(256, 6) void join_kernel(const Args a, int parts, const float* part_o,
                                                   const float2* part_state) {
    __shared__ float weight[MOST_PARTS], shared[8], values[256];
    __shared__ uint32_t lost[2][DP / 32], found[2][DP / 32];  // columns of NaN, of infinities
    const int group = a.hq / a.hkv, columns = group * a.sq;
    const int column = blockIdx.x % columns, g = blockIdx.x / columns % a.hkv;
    const int b = blockIdx.x / columns / a.hkv, h = g * group + column / a.sq, i = column % a.sq;
    const int tid = threadIdx.x, wave = tid >> 6;
    // the first parts' values travel while their weights are found
    constexpr int SHARES = 256 / DP, AHEAD = 16;
    const int d = tid % DP, share = tid / DP < SHARES ? tid / DP : parts;
    const float* from = part_o + (int64_t)blockIdx.x * parts * DP + d;
    float x[AHEAD];
    auto fetch = [&](int p0) {
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) {
            const int p = p0 + n * SHARES;
            x[n] = p < parts ? from[(int64_t)p * DP] : 0.f;
        }
    };
    fetch(share);
    const float2 state = tid < parts ? part_state[(int64_t)blockIdx.x * parts + tid]
                                     : make_float2(0.f, 0.f);
    const float exponent = state.y == 0.f ? -INFINITY : state.x;
    float most = wave_max(exponent);
    if ((tid & 63) == 0) shared[wave] = most;
    if (tid < 2 * (DP / 32)) lost[0][tid] = 0, found[0][tid] = 0;
    __syncthreads();
    most = fmaxf(fmaxf(shared[0], shared[1]), fmaxf(shared[2], shared[3]));
    const float w = state.y == 0.f ? 0.f : exp2_fast(exponent - most);
    float total = wave_sum(w * state.y);
    weight[tid] = w;
    if ((tid & 63) == 0) shared[4 + wave] = total;
    __syncthreads();
    total = shared[4] + shared[5] + shared[6] + shared[7];
    const float inv = total == 0.f ? 0.f : 1.f / total;

    float o = 0;
    for (int p0 = share; p0 < parts; p0 += AHEAD * SHARES) {
        if (p0 != share) fetch(p0);
#pragma unroll
        for (int n = 0; n < AHEAD; ++n) {
            const int p = p0 + n * SHARES;
            const float w = p < parts ? weight[p] : 0.f;
            o = w == 0.f ? o : fmaf(w, x[n], o);
        }
    }
    values[tid] = o;
    __syncthreads();
    if (tid < a.d) {
        o = 0;
        for (int n = 0; n < SHARES; ++n) o += values[n * DP + tid];
        o *= inv;
        row<T>(a.out, b, i, h)[tid] = (T)o;
        if (!(fabsf(o) <= 3.4028235e38f)) atomicOr(&lost[o == o][tid / 32], 1u << (tid % 32));
    }
    if (tid == 0 && a.lse)
        a.lse[((int64_t)b * a.hq + h) * a.sq + i] = total == 0.f ? -INFINITY : most + log2f(total);
    __syncthreads();
    // as in forward_kernel, a quarter of the keys each wave
    Columns<DP> need;
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) need.nan[n] = lost[0][n], need.inf[n] = lost[1][n];
    if (!need.any() && total != 0.f) return;
    const int pos = i + a.sk - a.sq, end = a.causal ? pos + 1 : a.sk;
    const int* doc_row = a.documents ? a.documents + b * a.documents_sb : nullptr;
    const int doc = doc_row ? doc_row[pos] : 0, each = (end + 255) / 256 * 64;
    if (total == 0.f) {
        if (wave == 0 && doc >= 0) forward_row<T, DP>(a, b, h, i);
        return;
    }
    if (total != total) {
        if (wave == 0 && !nan_scores<T, DP>(a, b, h, i, 1, doc, pos)) forward_row<T, DP>(a, b, h, i);
        return;
    }
    Columns<DP> seen;
    look_for<T, DP>(need, a.v, b, g, min(wave * each, end), min((wave + 1) * each, end), a.d,
                    [&](int j) { return !doc_row || doc_row[j] == doc; }, seen);
    if ((tid & 63) == 0)
#pragma unroll
        for (int n = 0; n < DP / 32; ++n) {
            atomicOr(&found[0][n], seen.nan[n]);
            atomicOr(&found[1][n], seen.inf[n]);
        }
    __syncthreads();
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) seen.nan[n] = found[0][n], seen.inf[n] = found[1][n];
    if (wave == 0 && !need.within(seen)) forward_row<T, DP>(a, b, h, i);
}

int padded(int d) { return (d + 31) / 32 * 32; }

// The shape of the blocks for `length` rows of each of `heads`: 4 waves of 32
// rows that share their tiles where that gives two blocks a CU; 1 wave of rows
// and 4 shares where that gives no more than one; else 2 and 2.  What counts
// for few rows is the number of blocks that a CU takes one after the other:
// 3 x 333 positions, 12 heads of 64 in 32 bits have 396 blocks of 1 x 4, two
// rounds, and 216 of 2 x 2, one (forward and back 101 and 85 us).
template <typename F>
void for_shape(int64_t heads, int length, F f) {
    auto blocks = [&](int rows) { return heads * ((length + rows - 1) / rows); };
    TORCH_CHECK(blocks(32) <= INT_MAX, "too many rows for one launch");
    auto go = [&](auto rows, auto shares) {
        const int each = 32 * decltype(rows)::value;
        f(rows, shares, (length + each - 1) / each, (unsigned)blocks(each));
    };
    if (blocks(128) >= 512)
        go(std::integral_constant<int, 4>{}, std::integral_constant<int, 1>{});
    else if (blocks(32) > 256)
        go(std::integral_constant<int, 2>{}, std::integral_constant<int, 2>{});
    else
        go(std::integral_constant<int, 1>{}, std::integral_constant<int, 4>{});
}

// Whether the forward pass is split over the keys, either
// - where 32 queries a block give fewer blocks than there are CUs, and the rows
//   to join are fewer than the keys: 12 heads of 64, bf16, split and not: 1
//   query of 2048 keys 9 and 22 us, 128 of 2048 19 and 22, 512 of 8192 55 and 73,
//   but 512 of 2048 36 and 23;
// - or where few queries of many requests leave most of a wave's 32 columns
//   empty, which the split fills with the heads that share keys.  A tile of 32
//   x 32 pairs that this saves pays for a row to join, 4096 for the second
//   launch.  One query, 12 heads on 4 of 64, bf16, split and not: 32 requests of
//   8192 keys 48 and 111 us, 64 of 2048 30 and 65, but 64 of 128 10 and 9; 16 on 1,
//   fp32, 32 of 32768 keys 116 and 4520; 16 queries, 16 on 1, bf16, 16 of 2048 29 and
//   23.
bool split_keys(const Args& a) {
    const int64_t heads = (int64_t)a.b * a.hq, rows = heads * a.sq;
    const int64_t blocks = heads * ((a.sq + 31) / 32);
    const int64_t packed =
        (int64_t)a.b * a.hkv * (((int64_t)(a.hq / a.hkv) * a.sq + 31) / 32);
    return (blocks < 256 && rows <= a.sk) || (blocks - packed) * a.sk / 32 > rows + 4096;
}

template <typename T, int DP>
void launch_split(const Args& a, const torch::Tensor& like, hipStream_t stream) {
    int64_t columns = (int64_t)(a.hq / a.hkv) * a.sq, tiles = (columns + 31) / 32;
    int64_t units = tiles * a.b * a.hkv, rows = (int64_t)a.b * a.hkv * columns;
    // 8 waves a CU, each with 2 tiles of 32 keys at least
    int64_t parts = std::min<int64_t>({std::max<int64_t>(1, 2048 / units),
                                       std::max<int64_t>(1, a.sk / 64), MOST_PARTS});
    int64_t each = ((a.sk + parts - 1) / parts + 31) / 32 * 32;
    parts = (a.sk + each - 1) / each;
    TORCH_CHECK(units * parts <= INT_MAX && rows <= INT_MAX, "too many rows for one launch");
    auto f32 = like.options().dtype(torch::kFloat32);
    auto part_o = torch::empty({rows, parts, DP}, f32), state = torch::empty({rows, parts, 2}, f32);
    hipLaunchKernelGGL((split_kernel<T, DP>), dim3((unsigned)(units * parts)), dim3(64), 0, stream,
                       a, (int)parts, (int)each, (int)tiles, part_o.data_ptr<float>(),
                       (float2*)state.data_ptr<float>());
    hipLaunchKernelGGL((join_kernel<T, DP>), dim3((unsigned)rows), dim3(256), 0, stream, a,
                       (int)parts, part_o.data_ptr<float>(),
                       (const float2*)state.data_ptr<float>());
}

template <typename T, int DP>
void launch_forward(const Args& a, const Ranges& keys, const Ranges& queries,
                    hipStream_t stream) {
    for_shape((int64_t)a.b * a.hq, a.sq, [&](auto rows, auto shares, int tiles, unsigned blocks) {
        constexpr int ROWS = decltype(rows)::value, SHARES = decltype(shares)::value;
        hipLaunchKernelGGL((forward_kernel<T, DP, ROWS, SHARES>), dim3(blocks),
                           dim3(ROWS * SHARES * 64), 0, stream, a, keys, queries, tiles,
                           blocks <= (DP <= 64 && sizeof(T) == 2 ? 768 : 512));
    });
}

// ---------------------------------------------------------------------------
// Backward.  First the queries' gradient, whose waves hold 32 queries as the
// forward's do, and their delta; then the keys' and values', whose waves hold
// 32 keys and go over the queries of all heads that share them.  Scores are
// formed again in both (7 products where 5 would do, and in 16 bits one more in
// dq for its correction), so that nothing is added across blocks: results repeat
// bit by bit and no buffer of gradients is needed.
//
// 2 x 16 heads, 4096 x 4096, bf16, four products each: dq 920 TFLOP/s and dkv 830
// with heads of 64 (298 and 331 us), 840 and 650 with heads of 128, whose sums
// leave one wave a SIMD: K and V in shared memory make room for two, but then its
// reads bound dkv (604 for 631).
// Packed rows of 512 (32 of them, 12 heads of 64: dq 77 us, dkv 82) are bound by
// their blocks' reads, in step with each other, and the masks of mixed tiles.
//
// dS is rounded to the inputs' type for its products.  In fp16 it first gets
// a factor, a power of two that puts the largest dout of its query near 2^-4
// and P's 2^12 with it, so that dq keeps its bits at any size of gradient.  For
// dk the queries of a tile share the least of their factors, and the sums go
// along with it from tile to tile (by no more than they have to: the scale may
// lie FACTOR_ROOM below the tile's), so that queries with large gradients cost
// others no bits unless they share a tile.  A query without a gradient has the
// largest factor, that of the least dout, and so takes nothing from its tile.
// ---------------------------------------------------------------------------

constexpr int FACTOR_ROWS = 32;
constexpr float MOST_FACTOR = 0x1p20f;  // 2^-4 over the least fp16
constexpr float FACTOR_ROOM = 16.f;

template <typename T> constexpr bool FACTORED = std::is_same<T, _Float16>::value;

// delta from 16-bit outputs is off by their roundings and those of their
// probabilities, which shows where few keys hold a row and do.v_j - delta
// nearly cancels.  The sum of P (do.v_j - delta), which would be 0, says by
// how much: dq is set right with the sum of P k, and dk takes the right delta.
template <typename T> constexpr bool CORRECTED = sizeof(T) == 2;

// Rows that saw nothing have probabilities of zero; those of far scores are made
// NaN, so that what they enter is formed pair by pair.
__device__ __forceinline__ float usable(float lse) {
    return lse == -INFINITY ? INFINITY : fabsf(lse) > FAR ? __builtin_nanf("") : lse;
}

template <typename T, int DP, int ROWS, int SHARES>
__global__ __launch_bounds__(ROWS * SHARES * 64, (dq_waves<DP, SHARES>))
void dq_kernel(const Args a, const Ranges keys, const Ranges queries, int tiles_q,
               bool alternate, float* factors, int factors_n) {
    using G = Tile<T, DP>;
    constexpr int BOX = (CORRECTED<T> ? DP + 1 : DP / 2) * 64;  // acc, mean and rest
    constexpr int THREADS = ROWS * 64, N = tile_rows<T, SHARES>;
    __shared__ Shared<T, DP, N, SHARES, (SHARES - 1) * ROWS * BOX> shared;
    __shared__ alignas(16) int tile_docs[SHARES][N];

    unsigned id = xcd_order(blockIdx.x, gridDim.x);
    int qt = id % tiles_q, h = id / tiles_q % a.hq, b = id / tiles_q / a.hq;
    if (a.causal) qt = causal_order(qt, tiles_q, h, alternate);
    const int g = h / (a.hq / a.hkv), lane = threadIdx.x & 63, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % ROWS;
    const int share = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / ROWS;
    const int tid = threadIdx.x - share * THREADS;
    T *tile_k = shared.tiles[share][0], *tile_v = shared.tiles[share][1];
    int* docs = tile_docs[share];
    const int first = a.sk - a.sq, row0 = (qt * ROWS + wave) * 32;
    const int i = row0 + (lane & 31), pos = i + first;
    const bool there = i < a.sq;
    const int* doc_row = a.documents ? a.documents + b * a.documents_sb : nullptr;
    const int64_t at_row = ((int64_t)b * a.hq + h) * a.sq + i;

    const float c = a.c, slope = slope_of(a, h);
    Frag<T> q[DP / 16], dout[DP / 16];
    float delta = 0, most = 0;
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) {
        q[n] = row_frag<T>(row<T>(a.q, b, there ? i : 0, h), n * 16 + hf * 8, a.d, there);
        dout[n] = row_frag<T>(row<T>(a.dout, b, there ? i : 0, h), n * 16 + hf * 8, a.d, there);
        const Frag<T> out =
            row_frag<T>(row<T>(a.out, b, there ? i : 0, h), n * 16 + hf * 8, a.d, there);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float x = (float)dout[n][e];
            delta = fmaf(x, (float)out[e], delta);
            if (FACTORED<T>) most = fabsf(x) < INFINITY ? fmaxf(most, fabsf(x)) : most;
        }
        if (a.scale < 0) q[n] = -q[n];
    }
    delta = add_halves(delta);
    acc16 acc[DP / 32], mean[DP / 32];  // mean: sum of P k
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) acc[n] = acc16{}, mean[n] = acc16{};
    float off = there ? usable(a.lse[at_row]) : INFINITY, rest = 0, factor = 1.f;
    if constexpr (FACTORED<T>) {
        const float largest = wave_max(most);
        auto factor_of = [](float x) {
            return x == 0.f ? MOST_FACTOR : exp2f(-4.f - ceilf(log2f(x)));
        };
        factor = factor_of(max_halves(most));
        off -= SHIFT;
        if (lane == 0 && row0 < a.sq)
            factors[((int64_t)b * a.hq + h) * factors_n + row0 / FACTOR_ROWS] =
                factor_of(largest);
    }

    const int seen = there ? doc_row ? doc_row[pos] : 0 : -1;
    const int doc = seen < 0 ? INT_MIN : seen;
    int2 wave_docs{}, block_docs{};
    if (doc_row) {
        wave_docs = queries.of(b, qt * ROWS + wave);
        block_docs = queries.of(b, qt * ROWS);
        for (int w = 1; w < ROWS; ++w) block_docs = both(block_docs, queries.of(b, qt * ROWS + w));
    }
    const int wave_first = row0 + first, wave_last = min(row0 + 31, a.sq - 1) + first;
    int end = a.sk;
    if (a.causal) end = min(end, (qt + 1) * ROWS * 32 + first);
    const int tiles = (end + N - 1) / N;
    const T *k = row<T>(a.k, b, 0, g), *v = row<T>(a.v, b, 0, g);

    Stage<T, DP, N, THREADS> sk(a.k.ss, a.d, tid), sv(a.v.ss, a.d, tid);
    for (int chunk = 0; chunk < tiles; chunk += 64) {
        Visits visits = visits_of<N>(keys, b, chunk, tiles - chunk, block_docs, wave_docs);
        uint64_t mine = 0;
        int next = 0, key_doc = -1;
        auto fetch = [&] {
            mine = bit_of(visits.block, share);
            if (!mine) return;
            next = (chunk + __builtin_ctzll(mine)) * N;
            sk.load(k + (int64_t)next * a.k.ss, a.sk - next);
            sv.load(v + (int64_t)next * a.v.ss, a.sk - next);
            int j = next + tid;
            if (tid < N) key_doc = j < a.sk ? doc_row ? max(doc_row[j], -1) : 0 : -1;
        };
        if (visits.block) fetch();
        while (visits.block) {
            __syncthreads();
            sk.store(tile_k);
            sv.store(tile_v);
            if (tid < N) docs[tid] = key_doc;
            __syncthreads();
            const uint64_t bit = mine;
            const int at = next;
            visits.block = without<SHARES>(visits.block);
            if (visits.block) fetch();
            if (!(visits.wave & bit) || (a.causal && at > wave_last)) continue;
            const bool by_document = !(visits.whole & bit) || at + N > a.sk;
            const bool by_position = a.causal && at + N - 1 > wave_first;
#pragma unroll
            for (int t = 0; t < N / 32; ++t) {
                acc16 s = {}, dp = {};
#pragma unroll
                for (int n = 0; n < DP / 16; ++n)
                    s = mma(rows_of<T, DP>(tile_k, t * 32, n * 16), q[n], s);
#pragma unroll
                for (int n = 0; n < DP / 16; ++n)
                    dp = mma(rows_of<T, DP>(tile_v, t * 32, n * 16), dout[n], dp);
                exponents<1>(&s, c, off, slope, (float)(pos - at - t * 32 - 4 * hf));
                if (by_document) hide_documents(s, docs, t, doc);
                if (by_position) hide_past(s, t, pos - at);
                float sum = 0;
#pragma unroll
                for (int e = 0; e < 16; ++e) {
                    s[e] = exp2_fast(s[e]);
                    if constexpr (FACTORED<T>)
                        dp[e] = s[e] * fmaf(dp[e], factor, -delta * factor);
                    else
                        dp[e] = s[e] * (dp[e] - delta);
                    sum += dp[e];
                }
                add_product<T, DP>(tile_k, t * 32, dp, acc);
                if constexpr (CORRECTED<T>) {
                    rest += sum;
                    add_product<T, DP>(tile_k, t * 32, s, mean);
                }
            }
        }
    }

    if constexpr (SHARES > 1) {
        float* box = shared.boxes + wave * BOX;
        __syncthreads();
        if (share) {
            float* to = box + (share - 1) * ROWS * BOX;
            leave<DP>(to, acc);
            if constexpr (CORRECTED<T>) {
                leave<DP>(to + DP / 2 * 64, mean);
                to[DP * 64 + lane] = rest;
            }
        }
        __syncthreads();
        if (share) return;
        for (int n = 0; n < SHARES - 1; ++n, box += ROWS * BOX) {
            take<DP>(box, 1.f, 1.f, acc);
            if constexpr (CORRECTED<T>) {
                take<DP>(box + DP / 2 * 64, 1.f, 1.f, mean);
                rest += box[DP * 64 + lane];
            }
        }
    }

    bool fine = true;
    float back = a.scale;
    if constexpr (FACTORED<T>) back *= exp2f(-SHIFT) / factor;
    if constexpr (CORRECTED<T>) {
        rest = add_halves(rest);
        fine = fabsf(rest) <= 3.4028235e38f;
        float by = FACTORED<T> ? rest * exp2f(-SHIFT) : rest;
#pragma unroll
        for (int n = 0; n < DP / 32; ++n)
#pragma unroll
            for (int e = 0; e < 16; ++e) acc[n][e] = fmaf(-by, mean[n][e], acc[n][e]);
        delta += FACTORED<T> ? by / factor : rest;
    } else {
        delta += delta - delta;  // an infinity is NaN here too
    }
    if (there && hf == 0) a.delta[at_row] = delta;
    if (there) {
        T* dq = row<T>(a.dq, b, i, h);
#pragma unroll
        for (int n = 0; n < DP / 32; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                int d = n * 32 + r * 8 + hf * 4;
                if (d < a.d)
                    put4(dq + d, acc[n][r * 4] * back, acc[n][r * 4 + 1] * back,
                         acc[n][r * 4 + 2] * back, acc[n][r * 4 + 3] * back);
#pragma unroll
                for (int e = 0; e < 4; ++e) fine &= fabsf(acc[n][r * 4 + e]) <= 3.4028235e38f;
            }
    }
    if (__any(there && !fine)) {
        Columns<DP> lost;
        lost.of(acc, a.d);
        // a row is NaN if a score is, if its output's gradient is not finite or
        // if a visible row of V is not, as its output then shows
        bool dout_fine = true, out_fine = true;
#pragma unroll
        for (int n = 0; n < DP / 16; ++n) {
            const Frag<T> o =
                row_frag<T>(row<T>(a.out, b, there ? i : 0, h), n * 16 + hf * 8, a.d, there);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                out_fine &= fabsf((float)o[e]) < INFINITY;
                dout_fine &= fabsf((float)dout[n][e]) < INFINITY;
            }
        }
        out_fine = !wave_or(!out_fine, 32, 64);
        dout_fine = !wave_or(!dout_fine, 32, 64);
        const float lse = there ? a.lse[at_row] : 0.f;
        // no key seen, whose gradient is 0, or far scores
        const bool apart = fabsf(lse) > FAR;
        bool stands = there && lost.all_nan(a.d) && !apart;
        const uint32_t by_v = (uint32_t)__ballot(stands && lse == lse && dout_fine && !out_fine);
        stands = stands && (lse != lse || !dout_fine ||
                            (see_not_finite<T, DP>(a, b, g, by_v, doc, pos) >> (lane & 31) & 1));
        const bool sum = fabsf(rest) <= 3.4028235e38f;
        uint32_t again = (uint32_t)__ballot(there && !stands && (!sum || apart));
        again |= unexplained<T, DP>(
            a, a.k, b, g, (uint32_t)__ballot(there && !stands && sum && !apart && lost.any()),
            doc, pos, true, lost);
        for (; again; again &= again - 1) dq_row<T, DP>(a, b, h, row0 + __builtin_ctz(again));
    }
}

template <typename T, int DP, int ROWS, int SHARES>
__global__ __launch_bounds__(ROWS * SHARES * 64, (dkv_waves<T, DP, SHARES>))
void dkv_kernel(const Args a, const Ranges keys, const Ranges queries, int tiles_k,
                bool alternate, const float* factors, int factors_n) {
    using G = Tile<T, DP>;
    constexpr int THREADS = ROWS * 64, N = tile_rows<T, SHARES>;  // queries a tile
    constexpr int BOX = DP * 64;  // dk and dv
    __shared__ Shared<T, DP, N, SHARES, (SHARES - 1) * ROWS * BOX> shared;
    __shared__ alignas(16) int tile_docs[SHARES][N];
    __shared__ alignas(16) float tile_lses[SHARES][N], tile_deltas[SHARES][N];

    unsigned id = xcd_order(blockIdx.x, gridDim.x);
    const int g = id / tiles_k % a.hkv, b = id / tiles_k / a.hkv;
    int kt = id % tiles_k;
    if (a.causal) kt = tiles_k - 1 - causal_order(kt, tiles_k, g, alternate);
    const int group = a.hq / a.hkv, lane = threadIdx.x & 63, hf = lane >> 5;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) % ROWS;
    const int share = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6) / ROWS;
    const int tid = threadIdx.x - share * THREADS;
    T *tile_q = shared.tiles[share][0], *tile_o = shared.tiles[share][1];
    int* docs = tile_docs[share];
    float *lses = tile_lses[share], *deltas = tile_deltas[share];
    const int first = a.sk - a.sq, block0 = kt * ROWS * 32;
    const int key0 = block0 + wave * 32, j = key0 + (lane & 31);
    const bool there = j < a.sk;
    const int* doc_row = a.documents ? a.documents + b * a.documents_sb : nullptr;

    const float c = a.c;
    Frag<T> k[DP / 16], v[DP / 16];
#pragma unroll
    for (int n = 0; n < DP / 16; ++n) {
        k[n] = row_frag<T>(row<T>(a.k, b, there ? j : 0, g), n * 16 + hf * 8, a.d, there);
        v[n] = row_frag<T>(row<T>(a.v, b, there ? j : 0, g), n * 16 + hf * 8, a.d, there);
        if (a.scale < 0) k[n] = -k[n];
    }
    acc16 dk[DP / 32], dv[DP / 32];
#pragma unroll
    for (int n = 0; n < DP / 32; ++n) dk[n] = acc16{}, dv[n] = acc16{};
    float factor = 0.f;  // what dk's sums have, 0 before the first tile

    const int seen = there ? doc_row ? doc_row[j] : 0 : -1;
    const int doc = seen < 0 ? INT_MIN : seen;
    int2 wave_docs{}, block_docs{};
    if (doc_row) {
        wave_docs = keys.of(b, kt * ROWS + wave);
        block_docs = keys.of(b, kt * ROWS);
        for (int w = 1; w < ROWS; ++w) block_docs = both(block_docs, keys.of(b, kt * ROWS + w));
    }
    const int wave_last = min(key0 + 31, a.sk - 1);
    const int tiles = (a.sq + N - 1) / N;
    const int begin = a.causal ? max(0, block0 - first) / N : 0;

    Stage<T, DP, N, THREADS> sq(a.q.ss, a.d, tid), so(a.dout.ss, a.d, tid);
    for (int chunk = begin; chunk < tiles; chunk += 64) {
        const Visits visits = visits_of<N>(queries, b, chunk, tiles - chunk, block_docs, wave_docs);
        if (!visits.block) continue;
        uint64_t left = visits.block, mine = 0;
        int next = 0, next_h = g * group, query_doc = -1;
        float lse = 0, delta = 0, next_factor = 1.f;
        auto fetch = [&] {
            mine = bit_of(left, share);
            if (!mine) return;
            next = (chunk + __builtin_ctzll(mine)) * N;
            sq.load(row<T>(a.q, b, next, next_h), a.sq - next);
            so.load(row<T>(a.dout, b, next, next_h), a.sq - next);
            if (tid < N) {
                int i = next + tid;
                int64_t at = ((int64_t)b * a.hq + next_h) * a.sq + i;
                lse = i < a.sq ? usable(a.lse[at]) - (FACTORED<T> ? SHIFT : 0.f) : INFINITY;
                delta = i < a.sq ? a.delta[at] : 0.f;
                query_doc = i < a.sq ? doc_row ? max(doc_row[i + first], -1) : 0 : -1;
            }
            if constexpr (FACTORED<T>) {
                const float* f = factors + ((int64_t)b * a.hq + next_h) * factors_n;
                next_factor = f[next / FACTOR_ROWS];
                for (int n = FACTOR_ROWS; n < N && next + n < a.sq; n += FACTOR_ROWS)
                    next_factor = fminf(next_factor, f[(next + n) / FACTOR_ROWS]);
            }
        };
        fetch();
        while (left) {
            __syncthreads();
            sq.store(tile_q);
            so.store(tile_o);
            if (tid < N) {
                docs[tid] = query_doc;
                lses[tid] = lse;
                deltas[tid] = delta;
            }
            __syncthreads();
            const uint64_t bit = mine;
            const int at = next, h = next_h;
            const float tile_factor = next_factor;
            left = without<SHARES>(left);
            if (!left && next_h + 1 < (g + 1) * group) {  // the next head of the group
                left = visits.block;
                ++next_h;
            }
            if (left) fetch();
            if (!(visits.wave & bit) || (a.causal && at + first + N - 1 < key0)) continue;
            const bool by_document = !(visits.whole & bit);
            const bool by_position = a.causal && at + first < wave_last;
            if constexpr (FACTORED<T>) {
                // dk's sums go to the factor of gradients of another size
                if (fminf(fmaxf(tile_factor, factor), factor * FACTOR_ROOM) != tile_factor) {
                    float by = factor == 0.f ? 1.f : tile_factor / factor;
#pragma unroll
                    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
                        for (int e = 0; e < 16; ++e) dk[n][e] *= by;
                    factor = tile_factor;
                }
            }
            const float slope = slope_of(a, h), far = (float)(at + first + 4 * hf - j);
            const float by_slope = slope / c;
#pragma unroll
            for (int t = 0; t < N / 32; ++t) {
                acc16 s = {}, dp = {};
#pragma unroll
                for (int n = 0; n < DP / 16; ++n)
                    s = mma(rows_of<T, DP>(tile_q, t * 32, n * 16), k[n], s);
#pragma unroll
                for (int n = 0; n < DP / 16; ++n)
                    dp = mma(rows_of<T, DP>(tile_o, t * 32, n * 16), v[n], dp);
                if (slope != 0.f)
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        s[e] = fmaf(-by_slope,
                                    fabsf(far + (float)(t * 32 + 8 * (e >> 2) + (e & 3))), s[e]);
                if (by_document) hide_documents(s, docs, t, doc);
                if (by_position) hide_before(s, t, j - at - first);
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const int i = t * 32 + r * 8 + 4 * hf;
                    const f32x4 l = *(const f32x4*)(lses + i), dl = *(const f32x4*)(deltas + i);
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int x = r * 4 + e;
                        s[x] = exp2_fast(fmaf(s[x], c, -l[e]));
                        if constexpr (FACTORED<T>)
                            dp[x] = s[x] * fmaf(dp[x], factor, -dl[e] * factor);
                        else
                            dp[x] = s[x] * (dp[x] - dl[e]);
                    }
                }
                add_product<T, DP>(tile_o, t * 32, s, dv);
                add_product<T, DP>(tile_q, t * 32, dp, dk);
            }
        }
    }

    float back_k = a.scale, back_v = 1.f;
    if constexpr (FACTORED<T>) {
        back_v = exp2f(-SHIFT);
        back_k *= factor == 0.f ? 0.f : back_v / factor;
    }
#pragma unroll
    for (int n = 0; n < DP / 32; ++n)
#pragma unroll
        for (int e = 0; e < 16; ++e) dk[n][e] *= back_k, dv[n][e] *= back_v;
    if constexpr (SHARES > 1) {
        float* box = shared.boxes + wave * BOX;
        __syncthreads();
        if (share) {
            leave<DP>(box + (share - 1) * ROWS * BOX, dk);
            leave<DP>(box + (share - 1) * ROWS * BOX + BOX / 2, dv);
        }
        __syncthreads();
        if (share) return;
        for (int n = 0; n < SHARES - 1; ++n, box += ROWS * BOX) {
            take<DP>(box, 1.f, 1.f, dk);
            take<DP>(box + BOX / 2, 1.f, 1.f, dv);
        }
    }
    bool fine = true;
    if (there) {
        T *to_k = row<T>(a.dk, b, j, g), *to_v = row<T>(a.dv, b, j, g);
#pragma unroll
        for (int n = 0; n < DP / 32; ++n)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                int d = n * 32 + r * 8 + hf * 4, e = r * 4;
                if (d < a.d) {
                    put4(to_k + d, dk[n][e], dk[n][e + 1], dk[n][e + 2], dk[n][e + 3]);
                    put4(to_v + d, dv[n][e], dv[n][e + 1], dv[n][e + 2], dv[n][e + 3]);
                }
#pragma unroll
                for (int x = e; x < e + 4; ++x)
                    fine &= fabsf(dk[n][x]) <= 3.4028235e38f && fabsf(dv[n][x]) <= 3.4028235e38f;
            }
    }
    if (__any(there && !fine)) {
        Columns<DP> lost_k, lost_v;
        lost_k.of(dk, a.d);
        lost_v.of(dv, a.d);
        uint32_t again = 0;
        for_documents((uint32_t)__ballot(there && (lost_k.any() || lost_v.any())), doc,
                      [&](int of, bool mine, uint32_t rows) {
            if (of < 0) {  // seen by no query
                again |= rows;
                return;
            }
            // queries that see all of these keys: a NaN among the scores of one
            // makes dk and dv NaN, one as its delta dk
            const int from = a.causal ? max(0, key0 + 31 - __builtin_clz(rows) - first) : 0;
            bool nan_score = false, nan_delta = false;
            auto sees = [&](int64_t at, int i) {
                return (!doc_row || doc_row[i + first] == of) && a.lse[at + i] != -INFINITY;
            };
            for (int h = g * group; h < (g + 1) * group && !nan_score; ++h) {
                const int64_t at = ((int64_t)b * a.hq + h) * a.sq;
                for (int i0 = from; i0 < a.sq && !nan_score; i0 += 64) {
                    const int i = i0 + lane;
                    const bool seen = i < a.sq && sees(at, i);
                    const float l = seen ? a.lse[at + i] : 0.f, x = seen ? a.delta[at + i] : 0.f;
                    nan_score = __any(l != l);
                    nan_delta |= __any(x != x);
                }
            }
            Columns<DP> seen;
            if (!nan_score) {
                const Columns<DP> need = lost_v.joined(mine);
                for (int h = g * group; h < (g + 1) * group && need.any(); ++h) {
                    const int64_t at = ((int64_t)b * a.hq + h) * a.sq;
                    look_for<T, DP>(need, a.dout, b, h, from, a.sq, a.d,
                                    [&](int i) { return sees(at, i); }, seen);
                }
            }
            const bool fine_k = !lost_k.any() || (lost_k.all_nan(a.d) && (nan_score || nan_delta));
            const bool fine_v = nan_score ? !lost_v.any() || lost_v.all_nan(a.d)
                                          : lost_v.within(seen);
            again |= rows & (uint32_t)__ballot(mine && !(fine_k && fine_v));
        });
        for (; again; again &= again - 1) dkv_row<T, DP>(a, b, g, key0 + __builtin_ctz(again));
    }
}

template <typename T, int DP>
void launch_backward(const Args& a, const Ranges& keys, const Ranges& queries, float* factors,
                     int factors_n, hipStream_t stream) {
    for_shape((int64_t)a.b * a.hq, a.sq, [&](auto rows, auto shares, int tiles, unsigned blocks) {
        constexpr int ROWS = decltype(rows)::value, SHARES = decltype(shares)::value;
        hipLaunchKernelGGL((dq_kernel<T, DP, ROWS, SHARES>), dim3(blocks),
                           dim3(ROWS * SHARES * 64), 0, stream, a, keys, queries, tiles,
                           DP <= 64 && blocks <= 512, factors, factors_n);
    });
    for_shape((int64_t)a.b * a.hkv, a.sk, [&](auto rows, auto shares, int tiles, unsigned blocks) {
        constexpr int ROWS = decltype(rows)::value, SHARES = decltype(shares)::value;
        hipLaunchKernelGGL((dkv_kernel<T, DP, ROWS, SHARES>), dim3(blocks),
                           dim3(ROWS * SHARES * 64), 0, stream, a, keys, queries, tiles,
                           DP <= 64 && blocks <= 512, factors, factors_n);
    });
}

// f of the head size, as the constant of its padded width
template <typename F>
void for_width(int d, F f) {
    switch (padded(d)) {
        case 32: f(std::integral_constant<int, 32>{}); break;
        case 64: f(std::integral_constant<int, 64>{}); break;
        case 96: f(std::integral_constant<int, 96>{}); break;
        default: f(std::integral_constant<int, 128>{}); break;
    }
}

// The ranges of the keys' documents and of the queries', which are the same
// where there are as many.
struct DocumentRanges {
    torch::Tensor buffer[2];
    Ranges keys{}, queries{};

    // `known`: those that the forward pass has left, or nothing
    DocumentRanges(const Args& a, const std::vector<torch::Tensor>& known,
                   const torch::Tensor& like, hipStream_t stream) {
        if (!a.documents) return;
        const int first = a.sk - a.sq;
        if (!known.empty()) {
            TORCH_CHECK(known.size() == (first ? 2 : 1), "ranges must be the forward's");
            keys = over(known[0], a, 0);
            queries = first ? over(known[1], a, first) : keys;
            return;
        }
        keys = fill(0, a, 0, like, stream);
        queries = first ? fill(1, a, first, like, stream) : keys;
    }
    static Ranges over(const torch::Tensor& t, const Args& a, int first) {
        const int count = (a.sk - first + RANGE - 1) / RANGE;
        TORCH_CHECK(t.is_cuda() && t.scalar_type() == torch::kInt32 && t.is_contiguous() &&
                        t.numel() == (int64_t)a.b * count * 2,
                    "ranges must be the forward's");
        return {(const int2*)t.data_ptr<int>(), count};
    }
    Ranges fill(int n, const Args& a, int first, const torch::Tensor& like, hipStream_t stream) {
        const int count = (a.sk - first + RANGE - 1) / RANGE;
        const int64_t all = (int64_t)a.b * count;
        buffer[n] = torch::empty({all, 2}, like.options().dtype(torch::kInt32));
        int2* at = (int2*)buffer[n].data_ptr<int>();
        constexpr int EACH = 256 / RANGE;
        hipLaunchKernelGGL(ranges_kernel, dim3((unsigned)((all + EACH - 1) / EACH)), dim3(256), 0,
                           stream, a.documents, a.documents_sb, first, a.sk, count, all, at);
        return {at, count};
    }
};

// ---------------------------------------------------------------------------

View view(const torch::Tensor& t) {
    return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

// d contiguous, every head at a 16-byte address and a tile of 64 rows within
// the 31 bits of a buffer load's offset, by a copy where it is not
torch::Tensor aligned(const torch::Tensor& t) {
    int64_t per = 16 / t.element_size();
    bool fine = (uintptr_t)t.data_ptr() % 16 == 0 && t.stride(3) == 1 &&
                t.stride(1) * t.element_size() < (1 << 24);
    for (int d = 0; d < 3; ++d) fine = fine && t.stride(d) % per == 0;
    return fine ? t : t.clone(at::MemoryFormat::Contiguous);
}

Args args_for(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
              const torch::Tensor& documents, const torch::Tensor& slopes, bool causal,
              double scale) {
    for (auto* t : {&q, &k, &v})
        TORCH_CHECK_VALUE(t->is_cuda() && t->dim() == 4 && t->device() == q.device() &&
                              t->scalar_type() == q.scalar_type(),
                          "attention: q, k and v must be [batch, length, heads, head size] of one "
                          "type on one device");
    Args a{};
    a.b = (int)q.size(0);
    a.sq = (int)q.size(1);
    a.hq = (int)q.size(2);
    a.d = (int)q.size(3);
    a.sk = (int)k.size(1);
    a.hkv = (int)k.size(2);
    TORCH_CHECK_VALUE(k.sizes() == v.sizes() && k.size(0) == a.b && k.size(3) == a.d,
                      "attention: q ", q.sizes(), ", k ", k.sizes(), " and v ", v.sizes(),
                      " do not fit");
    TORCH_CHECK_VALUE(a.d >= 8 && a.d <= MOST_D && a.d % 8 == 0,
                      "attention: the head size must be a multiple of 8 from 8 to 128, got ", a.d);
    TORCH_CHECK_VALUE(a.hkv >= 1 && a.hq % a.hkv == 0, "attention: ", a.hkv,
                      " key-value heads do not divide ", a.hq, " query heads");
    TORCH_CHECK_VALUE(q.size(1) <= k.size(1), "attention: ", q.size(1), " queries over ",
                      k.size(1), " keys; queries are the last positions");
    TORCH_CHECK_VALUE(k.size(1) < (1 << 30), "attention: too many keys");
    TORCH_CHECK_VALUE(std::isfinite((float)scale), "attention: scale must be finite");
    if (documents.defined()) {
        TORCH_CHECK_VALUE(documents.device() == q.device() &&
                              documents.scalar_type() == torch::kInt32 && documents.dim() == 2 &&
                              documents.size(0) == a.b && documents.size(1) == a.sk,
                          "attention: documents must be int32 [", a.b, ", ", a.sk,
                          "] on q's device");
        TORCH_CHECK(documents.stride(1) == 1 || a.sk <= 1, "documents have gaps");
        a.documents = documents.data_ptr<int>();
        a.documents_sb = documents.stride(0);
    }
    if (slopes.defined()) {
        TORCH_CHECK_VALUE(slopes.device() == q.device() &&
                              slopes.scalar_type() == torch::kFloat32 && slopes.dim() == 1 &&
                              slopes.size(0) == a.hq,
                          "attention: slopes must be float32 [", a.hq, "] on q's device");
        TORCH_CHECK_VALUE(!slopes.requires_grad(),
                          "attention: slopes are constants and get no gradient");
        TORCH_CHECK(slopes.is_contiguous(), "slopes have gaps");
        a.slopes = slopes.data_ptr<float>();
    }
    a.causal = causal;
    a.scale = (float)scale;
    a.c = std::max(std::fabs(a.scale) * LOG2E, 1e-30f);
    return a;
}

template <typename F>
void for_type(torch::ScalarType type, F f) {
    switch (type) {
        case torch::kFloat32: f((float*)nullptr); break;
        case torch::kBFloat16: f((__bf16*)nullptr); break;
        case torch::kFloat16: f((_Float16*)nullptr); break;
        default:
            TORCH_CHECK_VALUE(false, "attention: takes float32, bfloat16 or float16, got ", type);
    }
}

// out, the rows' sums if `want_lse`, and the ranges of documents if it made any
std::vector<torch::Tensor> attention_forward(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                                             const torch::Tensor& documents,
                                             const torch::Tensor& slopes, bool causal,
                                             double scale, bool want_lse) {
    Args a = args_for(q, k, v, documents, slopes, causal, scale);
    c10::DeviceGuard guard(q.device());
    q = aligned(q), k = aligned(k), v = aligned(v);
    auto out = torch::empty({a.b, a.sq, a.hq, a.d}, q.options());
    auto f32 = q.options().dtype(torch::kFloat32);
    auto lse = want_lse ? torch::empty({a.b, a.hq, a.sq}, f32) : torch::empty({0}, f32);
    a.q = view(q), a.k = view(k), a.v = view(v), a.out = view(out);
    a.lse = want_lse ? lse.data_ptr<float>() : nullptr;
    hipStream_t stream = at::hip::getCurrentHIPStream();
    if (out.numel() == 0) return {out, lse};
    std::vector<torch::Tensor> results = {out, lse};
    for_type(q.scalar_type(), [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        for_width(a.d, [&](auto width) {
            constexpr int DP = decltype(width)::value;
            if (split_keys(a)) {
                launch_split<T, DP>(a, q, stream);
            } else {
                DocumentRanges ranges(a, {}, q, stream);
                launch_forward<T, DP>(a, ranges.keys, ranges.queries, stream);
                for (auto& r : ranges.buffer)
                    if (r.defined()) results.push_back(r);
            }
        });
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
    return results;
}

std::vector<torch::Tensor> attention_backward(torch::Tensor dout, torch::Tensor q,
                                              torch::Tensor k, torch::Tensor v, torch::Tensor out,
                                              torch::Tensor lse,
                                              const std::vector<torch::Tensor>& known_ranges,
                                              const torch::Tensor& documents,
                                              const torch::Tensor& slopes, bool causal,
                                              double scale) {
    Args a = args_for(q, k, v, documents, slopes, causal, scale);
    c10::DeviceGuard guard(q.device());
    for (auto* t : {&dout, &out})
        TORCH_CHECK(t->is_cuda() && t->device() == q.device() && t->sizes() == q.sizes() &&
                        t->scalar_type() == q.scalar_type(),
                    "the output and its gradient must be like q");
    TORCH_CHECK(lse.is_cuda() && lse.device() == q.device() && lse.is_contiguous() &&
                    lse.scalar_type() == torch::kFloat32 &&
                    lse.numel() == (int64_t)a.b * a.hq * a.sq,
                "lse must be the forward's");
    q = aligned(q), k = aligned(k), v = aligned(v), out = aligned(out), dout = aligned(dout);
    auto dq = torch::empty(q.sizes(), q.options());
    auto dk = torch::empty(k.sizes(), k.options());
    auto dv = torch::empty(v.sizes(), v.options());
    auto delta = torch::empty(lse.sizes(), lse.options());
    a.q = view(q), a.k = view(k), a.v = view(v), a.out = view(out), a.dout = view(dout);
    a.dq = view(dq), a.dk = view(dk), a.dv = view(dv);
    a.lse = lse.data_ptr<float>();
    a.delta = delta.data_ptr<float>();
    hipStream_t stream = at::hip::getCurrentHIPStream();
    if (dq.numel() == 0) return {dq, dk.zero_(), dv.zero_()};
    const int factors_n = (a.sq + FACTOR_ROWS - 1) / FACTOR_ROWS;
    const bool factored = q.scalar_type() == torch::kFloat16;
    auto factors = torch::empty({factored ? (int64_t)a.b * a.hq * factors_n : 0}, lse.options());
    DocumentRanges ranges(a, known_ranges, q, stream);
    for_type(q.scalar_type(), [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        for_width(a.d, [&](auto width) {
            launch_backward<T, decltype(width)::value>(a, ranges.keys, ranges.queries,
                                                       factors.data_ptr<float>(), factors_n,
                                                       stream);
        });
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
    return {dq, dk, dv};
}

struct AttentionFunction : torch::autograd::Function<AttentionFunction> {
    static torch::Tensor forward(torch::autograd::AutogradContext* ctx, const torch::Tensor& q,
                                 const torch::Tensor& k, const torch::Tensor& v,
                                 const std::optional<torch::Tensor>& documents,
                                 const std::optional<torch::Tensor>& slopes, bool causal,
                                 double scale) {
        const torch::Tensor none, docs = documents.value_or(none), slope = slopes.value_or(none);
        auto r = attention_forward(q, k, v, docs, slope, causal, scale, true);
        torch::autograd::variable_list saved = {q, k, v, docs, slope};
        saved.insert(saved.end(), r.begin(), r.end());
        ctx->save_for_backward(saved);
        ctx->saved_data["causal"] = causal;
        ctx->saved_data["scale"] = scale;
        ctx->saved_data["elsewhere"] = held_elsewhere({q, k, v});
        return r[0];
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        const auto x = ctx->get_saved_variables();
        check_capture(ctx->saved_data["elsewhere"].toBool(), "attention");
        torch::autograd::variable_list d;
        {
            at::AutoGradMode no(false);
            d = attention_backward(grads[0].resolve_neg(), x[0], x[1], x[2], x[5], x[6],
                                   {x.begin() + 7, x.end()}, x[3], x[4],
                                   ctx->saved_data["causal"].toBool(),
                                   ctx->saved_data["scale"].toDouble());
        }
        d = once_differentiable(std::move(d), "attention");
        d.resize(7);
        return d;
    }
};

}  // namespace

torch::Tensor attention(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                        std::optional<torch::Tensor> documents,
                        std::optional<torch::Tensor> slopes, bool causal,
                        std::optional<double> scale) {
    TORCH_CHECK_VALUE(q.dim() == 4, "attention: q must be [batch, length, heads, head size]");
    if (documents && documents->dim() == 2 && documents->size(1) > 1 && documents->stride(1) != 1)
        documents = documents->contiguous();
    if (slopes) slopes = slopes->resolve_neg().contiguous();
    // views that torch negates when it reads them
    q = q.resolve_neg(), k = k.resolve_neg(), v = v.resolve_neg();
    const torch::Tensor none;
    check_seen({q, k, v, slopes.value_or(none)}, "attention");
    const double by = scale.value_or(1.0 / std::sqrt((double)q.size(3)));
    if (at::GradMode::is_enabled() &&
        (q.requires_grad() || k.requires_grad() || v.requires_grad()))
        return AttentionFunction::apply(q, k, v, documents, slopes, causal, by);
    return attention_forward(q, k, v, documents.value_or(none), slopes.value_or(none), causal, by,
                             false)[0];
}
