// Global gradient norm over many tensors, and clipping (gfx950).
//
//   norm = sqrt(sum over all tensors of x^2)
//   y    = x * min(1, max_norm / norm)
//
// Squares are added in 64 bits: a float's square neither overflows nor
// vanishes there, so one exploding value gives the norm it has and not
// infinity, and the sum over 1e8 values keeps its 32-bit result exact to the
// last place or so.  The loads, not the 64-bit adds, bound both kernels (one
// multiply-add for 2 or 4 bytes).
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
#include <hip/hip_runtime.h>
#include <algorithm>

namespace {

constexpr int TABLE = 128;    // 29 bytes each: the arguments stay under 4 KB
constexpr int THREADS = 256;
constexpr int WAVES = THREADS / 64;
constexpr int UNROLL = 4;     // 16-byte loads in flight for each thread

enum Kind : uint8_t { F32 = 0, BF16 = 1, F16 = 2 };

struct Table {
    const void* in[TABLE];
    void* out[TABLE];
    int64_t n[TABLE];
    int first[TABLE];         // first chunk of each tensor, INT_MAX behind the last
    uint8_t kind[TABLE];      // input type | output type << 4
    int chunks_before;        // partial sums of earlier launches
};
static_assert(sizeof(Table) + 64 <= 4096, "kernel arguments are limited to 4 KB");

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

// The block's tensor: each lane compares two starts, one memory latency for
// all of them where a binary search would take seven.
__device__ __forceinline__ int tensor_of(const Table& t, int block) {
    int lane = threadIdx.x & 63;
    uint64_t a = __ballot(t.first[lane] <= block), b = __ballot(t.first[lane + 64] <= block);
    return __popcll(a) + __popcll(b) - 1;
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

template <int KIND>
__device__ double chunk_sum(const void* in, int64_t n) {
    using T = Type<KIND>;
    const Raw* raw = (const Raw*)in;
    int64_t vecs = n / T::PER;
    double s = 0;
    int64_t i = threadIdx.x;
    for (; i + (UNROLL - 1) * THREADS < vecs; i += UNROLL * THREADS) {
        raw4 r[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) r[u] = raw[i + u * THREADS].v;
#pragma unroll
        for (int u = 0; u < UNROLL; ++u)
#pragma unroll
            for (int e = 0; e < T::PER; ++e) {
                double x = T::get((const uint32_t*)&r[u], e);
                s = fma(x, x, s);
            }
    }
    for (; i < vecs; i += THREADS) {
        raw4 r = raw[i].v;
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

__device__ __forceinline__ int kind_size(int kind) { return kind == F32 ? 4 : 2; }

__global__ __launch_bounds__(THREADS) void norm_partial_kernel(const Table t, int64_t chunk,
                                                               double* __restrict__ partial) {
    __shared__ double shared[WAVES];
    int block = blockIdx.x;
    int i = __builtin_amdgcn_readfirstlane(tensor_of(t, block));
    int64_t start = (int64_t)(block - t.first[i]) * chunk;
    int64_t n = min(chunk, t.n[i] - start);
    int kind = t.kind[i] & 15;
    const char* in = (const char*)t.in[i] + start * kind_size(kind);
    double s = kind == F32 ? chunk_sum<F32>(in, n)
             : kind == BF16 ? chunk_sum<BF16>(in, n) : chunk_sum<F16>(in, n);
    s = block_sum(s, shared);
    if (threadIdx.x == 0) partial[t.chunks_before + block] = s;
}

__global__ __launch_bounds__(1024) void norm_join_kernel(const double* __restrict__ partial,
                                                         int n, float* __restrict__ norm) {
    __shared__ double shared[16];
    double s = 0;
    for (int i = threadIdx.x; i < n; i += 1024) s += partial[i];
    s = block_sum(s, shared);
    if (threadIdx.x == 0) *norm = (float)sqrt(s);
}

// x * factor, rounded once: a 32-bit product of 64-bit factors is exact before
// its rounding; for the 16-bit types the factor's 32-bit rounding adds 2^-24
// to a step of 2^-8 or 2^-11.
template <int OUT>
__device__ __forceinline__ void put(void* out, int64_t i, double factor, float x) {
    if (OUT == F32) {
        ((float*)out)[i] = (float)((double)x * factor);
    } else if (OUT == BF16) {
        ((uint16_t*)out)[i] = to_bf16(x * (float)factor);
    } else {
        ((_Float16*)out)[i] = (_Float16)(x * (float)factor);
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
                    (float)((double)Type<IN>::get((const uint32_t*)&r, h * 4 + e) * factor));
            out[i * (PER / 4) + h].v = o;
        }
    } else {
        uint32_t w[PER / 2];
        float f = (float)factor;
#pragma unroll
        for (int e = 0; e < PER / 2; ++e) {
            float a = Type<IN>::get((const uint32_t*)&r, 2 * e) * f;
            float b = Type<IN>::get((const uint32_t*)&r, 2 * e + 1) * f;
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
__device__ void chunk_scale(const void* in, void* out, int64_t n, double factor) {
    constexpr int PER = Type<IN>::PER;
    const Raw* raw = (const Raw*)in;
    int64_t vecs = n / PER;
    int64_t i = threadIdx.x;
    for (; i + (UNROLL - 1) * THREADS < vecs; i += UNROLL * THREADS) {
        raw4 r[UNROLL];
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) r[u] = raw[i + u * THREADS].v;
#pragma unroll
        for (int u = 0; u < UNROLL; ++u) put_vec<IN, OUT>((Raw*)out, i + u * THREADS, factor, r[u]);
    }
    for (; i < vecs; i += THREADS) put_vec<IN, OUT>((Raw*)out, i, factor, raw[i].v);
    for (i = vecs * PER + threadIdx.x; i < n; i += THREADS)
        put<OUT>(out, i, factor, Type<IN>::load(in, i));
}

__global__ __launch_bounds__(THREADS) void clip_kernel(const Table t, int64_t chunk,
                                                       const double* __restrict__ partial, int n,
                                                       double max_norm,
                                                       float* __restrict__ norm) {
    __shared__ double shared[WAVES];
    double s = 0;
    for (int i = threadIdx.x; i < n; i += THREADS) s += partial[i];
    double total = sqrt(block_sum(s, shared));
    if (blockIdx.x == 0 && t.chunks_before == 0 && threadIdx.x == 0) *norm = (float)total;
    // a NaN norm is no norm below the bound: it reaches every value
    double factor = total <= max_norm ? 1.0 : max_norm / total;

    int block = gridDim.x - 1 - blockIdx.x;
    int i = __builtin_amdgcn_readfirstlane(tensor_of(t, block));
    int64_t start = (int64_t)(block - t.first[i]) * chunk;
    int64_t len = min(chunk, t.n[i] - start);
    int from = t.kind[i] & 15, to = t.kind[i] >> 4;
    const char* in = (const char*)t.in[i] + start * kind_size(from);
    char* out = (char*)t.out[i] + start * kind_size(to);
    if (in == out && factor == 1.0) return;  // in place and under the bound
    switch (from * 3 + to) {
        case 0: chunk_scale<F32, F32>(in, out, len, factor); break;
        case 1: chunk_scale<F32, BF16>(in, out, len, factor); break;
        case 2: chunk_scale<F32, F16>(in, out, len, factor); break;
        case 3: chunk_scale<BF16, F32>(in, out, len, factor); break;
        case 4: chunk_scale<BF16, BF16>(in, out, len, factor); break;
        case 5: chunk_scale<BF16, F16>(in, out, len, factor); break;
        case 6: chunk_scale<F16, F32>(in, out, len, factor); break;
        case 7: chunk_scale<F16, BF16>(in, out, len, factor); break;
        default: chunk_scale<F16, F16>(in, out, len, factor); break;
    }
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
    std::vector<int> blocks;
    int64_t chunk = 0;
    int partials = 0;
};

// Chunks of a power of two, from 4096 values (a block's four loads of 16
// bytes a thread) up so that 2048 blocks, 8 on each of the 256 CUs, hold all.
Plan plan_for(const std::vector<torch::Tensor>& ins, const std::vector<torch::Tensor>* outs) {
    Plan p;
    int64_t total = 0;
    for (auto& t : ins) total += t.numel();
    p.chunk = 4096;
    while (p.chunk * 2048 < total) p.chunk *= 2;
    int used = TABLE;
    for (size_t i = 0; i < ins.size(); ++i) {
        int64_t n = ins[i].numel();
        if (n == 0) continue;
        if (used == TABLE) {
            p.tables.emplace_back();
            p.blocks.push_back(0);
            std::fill_n(p.tables.back().first, TABLE, INT_MAX);
            p.tables.back().chunks_before = p.partials;
            used = 0;
        }
        Table& t = p.tables.back();
        t.in[used] = ins[i].data_ptr();
        t.out[used] = outs ? (*outs)[i].data_ptr() : nullptr;
        t.n[used] = n;
        t.kind[used] = kind_of(ins[i]) | (outs ? kind_of((*outs)[i]) << 4 : 0);
        t.first[used++] = p.blocks.back();
        int64_t chunks = (n + p.chunk - 1) / p.chunk;
        p.blocks.back() += (int)chunks;
        p.partials += (int)chunks;
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
    for (size_t i = 0; i < p.tables.size(); ++i)
        hipLaunchKernelGGL(norm_partial_kernel, dim3(p.blocks[i]), dim3(THREADS), 0, stream,
                           p.tables[i], p.chunk, partial.data_ptr<double>());
    return partial;
}

}  // namespace

torch::Tensor grad_norm(std::vector<torch::Tensor> grads) {
    TORCH_CHECK_VALUE(!grads.empty() && grads[0].is_cuda(), "grad_norm: needs GPU tensors");
    check_grads(grads);
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
    return norm;
}

std::pair<std::vector<torch::Tensor>, torch::Tensor> clip_grad_norm(
    std::vector<torch::Tensor> grads, double max_norm,
    std::optional<std::vector<torch::Tensor>> out, std::optional<torch::ScalarType> dtype) {
    TORCH_CHECK_VALUE(!grads.empty() && grads[0].is_cuda(), "clip_grad_norm: needs GPU tensors");
    TORCH_CHECK_VALUE(max_norm >= 0, "clip_grad_norm: max_norm must be 0 or more, got ", max_norm);
    TORCH_CHECK_VALUE(!out || !dtype, "clip_grad_norm: dtype is for new tensors, without out");
    check_grads(grads);
    at::NoGradGuard no_grad;
    c10::DeviceGuard guard(grads[0].device());
    std::vector<torch::Tensor> outs;
    if (out) {
        outs = *out;
    } else {
        for (auto& t : grads)
            outs.push_back(torch::empty_like(t, t.options().dtype(dtype.value_or(t.scalar_type()))));
    }
    const std::vector<torch::Tensor> results = outs;
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
        if (outs[i].numel()) ranges.push_back(range(outs[i], i));
    }
    std::sort(ranges.begin(), ranges.end(),
              [](const Range& a, const Range& b) { return a.at < b.at; });
    for (size_t i = 1; i < ranges.size(); ++i)
        TORCH_CHECK_VALUE(ranges[i].at >= ranges[i - 1].end, "clip_grad_norm: outputs ", ranges[i - 1].i, " and ",
                    ranges[i].i, " share memory");
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

    // other orders than dense ones go through copies
    std::vector<std::pair<size_t, torch::Tensor>> copies;
    for (size_t i = 0; i < grads.size(); ++i) {
        if (same_order(grads[i], outs[i])) continue;
        grads[i] = grads[i].contiguous();
        if (!same_order(grads[i], outs[i])) {
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
    // the last-level cache
    for (size_t i = p.tables.size(); i-- > 0;)
        hipLaunchKernelGGL(clip_kernel, dim3(p.blocks[i]), dim3(THREADS), 0, stream, p.tables[i],
                           p.chunk, partial.data_ptr<double>(), p.partials, max_norm,
                           norm.data_ptr<float>());
    for (auto& c : copies) c.second.copy_(outs[c.first]);
    if (out)
        for (auto& t : results) t.unsafeGetTensorImpl()->bump_version();
    return {results, norm};
}
