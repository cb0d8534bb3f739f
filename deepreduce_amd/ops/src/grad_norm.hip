// Global gradient norm over many tensors, and clipping (gfx950).
//
//   norm = sqrt(sum over all tensors of x^2)
//   y    = x * min(1, max_norm / norm)
//
// Squares are added in 64 bits: a float's square neither overflows nor
// vanishes there, so one exploding value gives the norm it has and not
// infinity, and the sum over 1e8 values keeps its 32-bit result exact to the
// last place or so.  The loads, not the 64-bit adds, bound both kernels (one
// multiply-add for 2 or 4 bytes): the norm of 2^28 values, 607 MB, takes 109 us
// (5.5 TB/s), clipping BERT-base's 435 MB into other buffers 260 us, of which
// 148 us are the second read and the write (5.9 TB/s: part of the read is
// still in the last-level cache).  Few small tensors are bound by the host:
// ResNet-20's 65 take 17 to 20 us a call, 9 us of it on the GPU.
//
// The tensors' addresses go to the kernel as its arguments (TABLE tensors a
// launch), so nothing is copied to the device and a captured graph replays
// on the same buffers.  Every block takes one chunk of one tensor and writes
// one partial sum; the partial sums are added in one fixed order, by every
// block of the clipping kernel for itself, so that results repeat bit by bit
// and no block waits for another.

#include "lm_ops.h"

#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <hip/hip_runtime.h>
#include <algorithm>

namespace {

constexpr int TABLE = 165;    // 24 bytes each, and the arguments stay under 4 KB
constexpr int THREADS = 256;
constexpr int WAVES = THREADS / 64;
constexpr int UNROLL = 4;     // 16-byte loads in flight for each thread
constexpr int BLOCKS = 4096;

enum Kind : uint8_t { F32 = 0, BF16 = 1, F16 = 2 };

struct Table {
    uint64_t in[TABLE];       // address | type << 56
    uint64_t out[TABLE];
    int first[TABLE];         // first chunk of each tensor, INT_MAX behind the last
    int tail[TABLE];          // values of its last chunk
    int blocks;               // chunks of all
    int chunks_before;        // partial sums of earlier launches
    int chunk;                // values of a chunk
};
static_assert(sizeof(Table) + 48 <= 4096, "kernel arguments are limited to 4 KB");

// 16 bytes at any element's address: buckets put tensors at odd offsets
typedef uint32_t raw4 __attribute__((ext_vector_type(4)));
struct __attribute__((packed, aligned(2))) Raw { raw4 v; };

template <int KIND> struct Type;
template <> struct Type<F32> {
    static constexpr int PER = 4;
    static __device__ float get(const uint32_t* w, int i) { return __uint_as_float(w[i]); }
    static __device__ float load(const void* p, int64_t i) { return ((const float*)p)[i]; }
};
template <> struct Type<BF16> {
    static constexpr int PER = 8;
    static __device__ float get(const uint32_t* w, int i) {
        return __uint_as_float((i & 1) ? (w[i >> 1] & 0xffff0000u) : (w[i >> 1] << 16));
    }
    static __device__ float load(const void* p, int64_t i) {
        return __uint_as_float((uint32_t)((const uint16_t*)p)[i] << 16);
    }
};
template <> struct Type<F16> {
    static constexpr int PER = 8;
    static __device__ float half(uint16_t b) {
        _Float16 h;
        __builtin_memcpy(&h, &b, 2);
        return (float)h;
    }
    static __device__ float get(const uint32_t* w, int i) {
        return half((uint16_t)(w[i >> 1] >> ((i & 1) * 16)));
    }
    static __device__ float load(const void* p, int64_t i) {
        return half(((const uint16_t*)p)[i]);
    }
};

__device__ __forceinline__ uint16_t to_bf16(float x) {
    __bf16 b = (__bf16)x;  // nearest even, NaN kept
    uint16_t r;
    __builtin_memcpy(&r, &b, 2);
    return r;
}

__device__ __forceinline__ int kind_size(int kind) { return kind == F32 ? 4 : 2; }

// What a block works on.  Each lane compares three starts: one memory latency
// for all where a binary search would take eight.
struct Chunk {
    const char* in;
    char* out;
    int n, from, to;
};
__device__ __forceinline__ Chunk chunk_of(const Table& t, int block) {
    const int lane = threadIdx.x & 63;
    int i = -1;
#pragma unroll
    for (int n = 0; n < TABLE; n += 64)
        i += __popcll(__ballot(n + lane < TABLE && t.first[min(n + lane, TABLE - 1)] <= block));
    i = __builtin_amdgcn_readfirstlane(i);
    const int end = i + 1 < TABLE ? min(t.first[i + 1], t.blocks) : t.blocks;
    const uint64_t mask = (1ull << 56) - 1;
    Chunk c;
    c.from = (int)(t.in[i] >> 56);
    c.to = (int)(t.out[i] >> 56);
    const int64_t start = (int64_t)(block - t.first[i]) * t.chunk;
    c.in = (const char*)(t.in[i] & mask) + start * kind_size(c.from);
    c.out = (char*)(t.out[i] & mask) + start * kind_size(c.to);
    c.n = block + 1 == end ? t.tail[i] : t.chunk;
    return c;
}

__device__ __forceinline__ double block_sum(double x, double* shared) {
    for (int m = 32; m; m >>= 1) x += __shfl_xor(x, m);
    if ((threadIdx.x & 63) == 0) shared[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0;
    for (int w = 0; w < (int)(blockDim.x >> 6); ++w) x += shared[w];
    __syncthreads();
    return x;
}

// values before the first 16-byte address
__device__ __forceinline__ int head_of(const void* at, int size, int n) {
    return min(n, (int)((16 - ((uintptr_t)at & 15)) & 15) / size);
}

template <int KIND>
__device__ double chunk_sum(const void* in, int n) {
    using T = Type<KIND>;
    constexpr int SIZE = KIND == F32 ? 4 : 2;
    double s = 0;
    const int head = head_of(in, SIZE, n);
    if ((int)threadIdx.x < head) {
        double x = T::load(in, threadIdx.x);
        s = x * x;
    }
    in = (const char*)in + head * SIZE;
    n -= head;
    const raw4* raw = (const raw4*)in;
    const int vecs = n / T::PER;
    int i = threadIdx.x;
    for (; i + (UNROLL - 1) * THREADS < vecs; i += UNROLL * THREADS) {
        raw4 r[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) r[u] = raw[i + u * THREADS];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int e = 0; e < T::PER; ++e) {
                double x = T::get((const uint32_t*)&r[u], e);
                s = fma(x, x, s);
            }
    }
    for (; i < vecs; i += THREADS) {
        raw4 r = raw[i];
#pragma unroll
        for (int e = 0; e < T::PER; ++e) {
            double x = T::get((const uint32_t*)&r, e);
            s = fma(x, x, s);
        }
    }
    for (i = vecs * T::PER + threadIdx.x; i < n; i += THREADS) {
        double x = T::load(in, i);
        s = fma(x, x, s);
    }
    return s;
}

__global__ __launch_bounds__(THREADS) void norm_partial_kernel(const Table t,
                                                               double* __restrict__ partial) {
    __shared__ double shared[WAVES];
    const Chunk c = chunk_of(t, blockIdx.x);
    double s = c.from == F32 ? chunk_sum<F32>(c.in, c.n)
             : c.from == BF16 ? chunk_sum<BF16>(c.in, c.n) : chunk_sum<F16>(c.in, c.n);
    s = block_sum(s, shared);
    if (threadIdx.x == 0) partial[t.chunks_before + blockIdx.x] = s;
}

__global__ __launch_bounds__(1024) void norm_join_kernel(const double* __restrict__ partial,
                                                         int n, float* __restrict__ norm) {
    __shared__ double shared[16];
    double s = 0;
    for (int i = threadIdx.x; i < n; i += 1024) s += partial[i];
    s = block_sum(s, shared);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// x * factor as OUT holds it: a 64-bit product (off by 2^-53), rounded.  For the
// 16-bit types a factor and a product of 32 bits serve, which add 2^-23 to half
// a step of 2^-8 or 2^-11, where the factor is a normal number (151 M values of
// fp16 take 173 us so, 254 with 64 bits).  Gradients near the largest value put
// it below 2^-126, 100 values of 3e38 cut to a norm of 1e-6 at 3e-46: then their
// products have 64 bits as well.
template <bool WIDE> __device__ __forceinline__ float scaled(float x, double factor) {
    return WIDE ? (float)((double)x * factor) : x * (float)factor;
}

template <int OUT, bool WIDE>
__device__ __forceinline__ void put(void* out, int64_t i, double factor, float x) {
    if (OUT == F32) {
        ((float*)out)[i] = scaled<true>(x, factor);
    } else if (OUT == BF16) {
        ((uint16_t*)out)[i] = to_bf16(scaled<WIDE>(x, factor));
    } else {
        ((_Float16*)out)[i] = (_Float16)scaled<WIDE>(x, factor);
    }
}

template <int IN, int OUT>
__device__ __forceinline__ void put_vec(Raw* out, int64_t i, double factor, raw4 r) {
    // IN values of one 16-byte load, as 32, 16 or 8 bytes of OUT
    constexpr int PER = Type<IN>::PER;
    if constexpr (OUT == F32) {
#pragma unroll
        for (int h = 0; h < PER / 4; ++h) {
            raw4 o;
#pragma unroll
            for (int e = 0; e < 4; ++e)
                o[e] = __float_as_uint(
                    scaled<true>(Type<IN>::get((const uint32_t*)&r, h * 4 + e), factor));
            out[i * (PER / 4) + h].v = o;
        }
    } else {
        uint32_t w[PER / 2];
#pragma unroll
        for (int e = 0; e < PER / 2; ++e) {
            const float a = scaled<false>(Type<IN>::get((const uint32_t*)&r, 2 * e), factor);
            const float b = scaled<false>(Type<IN>::get((const uint32_t*)&r, 2 * e + 1), factor);
            uint16_t u, v;
            if constexpr (OUT == BF16) {
                u = to_bf16(a), v = to_bf16(b);
            } else {
                _Float16 ha = (_Float16)a, hb = (_Float16)b;
                __builtin_memcpy(&u, &ha, 2);
                __builtin_memcpy(&v, &hb, 2);
            }
            w[e] = u | (uint32_t)v << 16;
        }
        if constexpr (PER == 8) {
            raw4 o = {w[0], w[1], w[2], w[3]};
            out[i].v = o;
        } else {
            struct __attribute__((packed, aligned(2))) Two { uint32_t a, b; };
            ((Two*)out)[i] = Two{w[0], w[1]};
        }
    }
}

template <int IN, int OUT>
__device__ void chunk_scale(const void* in, void* out, int n, double factor) {
    constexpr int PER = Type<IN>::PER, SIZE = IN == F32 ? 4 : 2, TO = OUT == F32 ? 4 : 2;
    const int head = head_of(out, TO, n);  // stores at 16-byte addresses, loads at any
    if ((int)threadIdx.x < head)
        put<OUT, OUT == F32>(out, threadIdx.x, factor, Type<IN>::load(in, threadIdx.x));
    in = (const char*)in + head * SIZE;
    out = (char*)out + head * TO;
    n -= head;
    const Raw* raw = (const Raw*)in;
    const int vecs = n / PER;
    int i = threadIdx.x;
    for (; i + (UNROLL - 1) * THREADS < vecs; i += UNROLL * THREADS) {
        raw4 r[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) r[u] = raw[i + u * THREADS].v;
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) put_vec<IN, OUT>((Raw*)out, i + u * THREADS, factor, r[u]);
    }
    for (; i < vecs; i += THREADS) put_vec<IN, OUT>((Raw*)out, i, factor, raw[i].v);
    for (i = vecs * PER + threadIdx.x; i < n; i += THREADS)
        put<OUT, OUT == F32>(out, i, factor, Type<IN>::load(in, i));
}

// value by value, in 64 bits
template <int IN, int OUT>
__device__ void chunk_scale_wide(const void* in, void* out, int n, double factor) {
#pragma unroll 1
    for (int i = threadIdx.x; i < n; i += THREADS)
        put<OUT, true>(out, i, factor, Type<IN>::load(in, i));
}

__global__ __launch_bounds__(THREADS) void clip_kernel(const Table t,
                                                       const double* __restrict__ partial, int n,
                                                       double max_norm,
                                                       float* __restrict__ norm) {
    __shared__ double shared[WAVES];
    const Chunk c = chunk_of(t, t.blocks - 1 - blockIdx.x);
    double s = 0;
    for (int i = threadIdx.x; i < n; i += THREADS) s += partial[i];
    double total = sqrt(block_sum(s, shared));
    if (blockIdx.x == 0 && t.chunks_before == 0 && threadIdx.x == 0) *norm = (float)total;
    // a NaN norm is no norm below the bound: it reaches every value
    double factor = total <= max_norm ? 1.0 : max_norm / total;
    if (c.in == c.out && factor == 1.0) return;  // in place and under the bound
    const bool wide = factor < 0x1p-126;
    auto scale = [&](auto in, auto out) {
        constexpr int IN = decltype(in)::value, OUT = decltype(out)::value;
        if (OUT != F32 && wide)
            chunk_scale_wide<IN, OUT>(c.in, c.out, c.n, factor);
        else
            chunk_scale<IN, OUT>(c.in, c.out, c.n, factor);
    };
    auto for_kind = [](int kind, auto f) {
        if (kind == F32) f(std::integral_constant<int, F32>{});
        else if (kind == BF16) f(std::integral_constant<int, BF16>{});
        else f(std::integral_constant<int, F16>{});
    };
    for_kind(c.from, [&](auto in) { for_kind(c.to, [&](auto out) { scale(in, out); }); });
}

Kind kind_of(const torch::Tensor& t) {
    switch (t.scalar_type()) {
        case torch::kFloat32: return F32;
        case torch::kBFloat16: return BF16;
        case torch::kFloat16: return F16;
        default:
            TORCH_CHECK_VALUE(false, "gradients must be float32, bfloat16 or float16, got ",
                              t.scalar_type());
    }
}

struct Plan {
    std::vector<Table> tables;
    int partials = 0;
};

// Chunks of a power of two, from 4096 values (a block's four loads of 16
// bytes a thread) up so that 4096 blocks, two rounds of the 8 that each of the
// 256 CUs holds, take all.
Plan plan_for(const std::vector<torch::Tensor>& ins, const std::vector<torch::Tensor>* outs) {
    Plan p;
    int64_t total = 0, chunk = 4096;
    for (auto& t : ins) total += t.numel();
    while (chunk * BLOCKS < total) chunk *= 2;
    TORCH_CHECK_VALUE(chunk < INT_MAX, "too many values");
    int used = TABLE;
    for (size_t i = 0; i < ins.size(); ++i) {
        int64_t n = ins[i].numel();
        if (n == 0) continue;
        if (used == TABLE) {
            p.tables.emplace_back();
            Table& t = p.tables.back();
            std::fill_n(t.first, TABLE, INT_MAX);
            t.blocks = 0;
            t.chunks_before = p.partials;
            t.chunk = (int)chunk;
            used = 0;
        }
        Table& t = p.tables.back();
        t.in[used] = (uint64_t)ins[i].data_ptr() | (uint64_t)kind_of(ins[i]) << 56;
        t.out[used] = outs ? (uint64_t)(*outs)[i].data_ptr() | (uint64_t)kind_of((*outs)[i]) << 56
                           : 0;
        t.first[used] = t.blocks;
        const int chunks = (int)((n + chunk - 1) / chunk);
        t.tail[used++] = (int)(n - (chunks - 1) * chunk);
        t.blocks += chunks;
        p.partials += chunks;
    }
    return p;
}

void check_grads(const std::vector<torch::Tensor>& grads) {
    for (auto& t : grads) {
        TORCH_CHECK_VALUE(t.layout() == torch::kStrided, "gradients must be dense tensors");
        TORCH_CHECK_VALUE(t.device() == grads[0].device(), "gradients must be on one device");
        kind_of(t);
    }
}

torch::Tensor partial_sums(const Plan& p, const torch::Tensor& like, hipStream_t stream) {
    auto partial = torch::empty({std::max(1, p.partials)}, like.options().dtype(torch::kFloat64));
    for (auto& t : p.tables)
        hipLaunchKernelGGL(norm_partial_kernel, dim3(t.blocks), dim3(THREADS), 0, stream, t,
                           partial.data_ptr<double>());
    return partial;
}

}  // namespace

torch::Tensor grad_norm(std::vector<torch::Tensor> grads) {
    TORCH_CHECK_VALUE(!grads.empty() && grads[0].is_cuda(), "grad_norm: needs GPU tensors");
    check_grads(grads);
    check_seen({}, "grad_norm");
    at::NoGradGuard no_grad;
    c10::DeviceGuard guard(grads[0].device());
    for (auto& t : grads)
        if (!t.is_non_overlapping_and_dense()) t = t.contiguous();
    Plan p = plan_for(grads, nullptr);
    hipStream_t stream = at::hip::getCurrentHIPStream();
    auto norm = torch::empty({}, grads[0].options().dtype(torch::kFloat32));
    auto partial = partial_sums(p, grads[0], stream);
    hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(1024), 0, stream,
                       partial.data_ptr<double>(), p.partials, norm.data_ptr<float>());
    C10_HIP_KERNEL_LAUNCH_CHECK();
    return norm;
}

// the new tensors, none where `out` takes the results, and the norm
std::pair<std::vector<torch::Tensor>, torch::Tensor> clip_grad_norm(
    std::vector<torch::Tensor> grads, double max_norm,
    std::optional<std::vector<torch::Tensor>> out, std::optional<torch::ScalarType> dtype) {
    TORCH_CHECK_VALUE(!grads.empty() && grads[0].is_cuda(), "clip_grad_norm: needs GPU tensors");
    TORCH_CHECK_VALUE(max_norm >= 0, "clip_grad_norm: max_norm must be 0 or more, got ", max_norm);
    TORCH_CHECK_VALUE(!out || !dtype, "clip_grad_norm: dtype is for new tensors, without out");
    check_grads(grads);
    check_seen({}, "clip_grad_norm");
    at::NoGradGuard no_grad;
    c10::DeviceGuard guard(grads[0].device());
    std::vector<torch::Tensor> outs;
    if (out) {
        outs = *out;
    } else {
        for (auto& t : grads)
            outs.push_back(
                torch::empty_like(t, t.options().dtype(dtype.value_or(t.scalar_type()))));
    }
    const std::vector<torch::Tensor> results = out ? std::vector<torch::Tensor>() : outs;
    TORCH_CHECK_VALUE(outs.size() == grads.size(), "clip_grad_norm: needs one output a gradient");
    check_grads(outs);
    TORCH_CHECK_VALUE(outs[0].device() == grads[0].device(),
                      "clip_grad_norm: outputs must be on the gradients' device");

    // Blocks read and write without an order between them: what is written
    // may be read only as the same values' own input.
    struct Range { const char *at, *end; size_t i; };
    std::vector<Range> ranges;
    auto range = [](const torch::Tensor& t, size_t i) {
        int64_t last = 0;
        for (int64_t d = 0; d < t.dim(); ++d) last += (t.size(d) - 1) * t.stride(d);
        const char* at = (const char*)t.data_ptr();
        return Range{at, at + (last + 1) * t.element_size(), i};
    };
    auto same_strides = [](const torch::Tensor& a, const torch::Tensor& b) {
        for (int64_t d = 0; d < a.dim(); ++d)
            if (a.size(d) > 1 && a.stride(d) != b.stride(d)) return false;
        return true;
    };
    auto same_order = [&](const torch::Tensor& a, const torch::Tensor& b) {
        return a.is_non_overlapping_and_dense() && same_strides(a, b);
    };
    for (size_t i = 0; i < outs.size(); ++i) {
        TORCH_CHECK_VALUE(outs[i].sizes() == grads[i].sizes(), "clip_grad_norm: output ", i,
                          " has another shape");
        for (int64_t d = 0; d < outs[i].dim(); ++d)
            TORCH_CHECK_VALUE(outs[i].size(d) < 2 || outs[i].stride(d), "clip_grad_norm: output ",
                              i, " is expanded");
        if (outs[i].numel()) ranges.push_back(range(outs[i], i));
    }
    std::sort(ranges.begin(), ranges.end(),
              [](const Range& a, const Range& b) { return a.at < b.at; });
    for (size_t i = 1; i < ranges.size(); ++i)
        TORCH_CHECK_VALUE(ranges[i].at >= ranges[i - 1].end, "clip_grad_norm: outputs ",
                          ranges[i - 1].i, " and ", ranges[i].i, " share memory");
    for (size_t i = 0; i < grads.size(); ++i) {
        if (!grads[i].numel()) continue;
        Range r = range(grads[i], i);
        auto it = std::upper_bound(ranges.begin(), ranges.end(), r.at,
                                   [](const char* a, const Range& b) { return a < b.end; });
        if (it == ranges.end() || it->at >= r.end) continue;
        TORCH_CHECK_VALUE(it->i == i && it->at == r.at && it->end == r.end &&
                              outs[i].scalar_type() == grads[i].scalar_type() &&
                              same_strides(outs[i], grads[i]),
                          "clip_grad_norm: gradient ", i, " shares memory with output ", it->i);
    }

    // other orders than dense ones go through copies, and so do views that torch
    // negates when it reads or writes them
    std::vector<std::pair<size_t, torch::Tensor>> copies;
    for (size_t i = 0; i < grads.size(); ++i) {
        if (same_order(grads[i], outs[i]) && grads[i].is_neg() == outs[i].is_neg()) continue;
        grads[i] = grads[i].resolve_neg().contiguous();
        if (!same_order(grads[i], outs[i]) || outs[i].is_neg()) {
            copies.emplace_back(i, outs[i]);
            outs[i] = torch::empty(grads[i].sizes(), outs[i].options());
        }
    }
    Plan p = plan_for(grads, &outs);
    hipStream_t stream = at::hip::getCurrentHIPStream();
    auto norm = torch::empty({}, grads[0].options().dtype(torch::kFloat32));
    auto partial = partial_sums(p, grads[0], stream);
    if (p.tables.empty())
        hipLaunchKernelGGL(norm_join_kernel, dim3(1), dim3(1024), 0, stream,
                           partial.data_ptr<double>(), 0, norm.data_ptr<float>());
    // last launch and last block first: what the sums read last is still in
    // the last-level cache (435 MB of BERT-base: 260 us, first block first 267)
    for (size_t i = p.tables.size(); i-- > 0;)
        hipLaunchKernelGGL(clip_kernel, dim3(p.tables[i].blocks), dim3(THREADS), 0, stream,
                           p.tables[i], partial.data_ptr<double>(), p.partials, max_norm,
                           norm.data_ptr<float>());
    C10_HIP_KERNEL_LAUNCH_CHECK();
    for (auto& c : copies) c.second.copy_(outs[c.first]);
    if (out)
        for (auto& t : *out) t.unsafeGetTensorImpl()->bump_version();
    return {results, norm};
}
