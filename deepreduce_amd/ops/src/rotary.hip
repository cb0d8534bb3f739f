// Rotary positions (gfx950): each pair (a, b) of a head's first `dim` values is
// turned by the angle position * frequency,
//
//   (a, b) -> (a cos t - b sin t, a sin t + b cos t),
//
// pairs being (i, i + dim / 2) or, interleaved, (2 i, 2 i + 1); the values
// behind `dim` are copied.  The gradient is the turn by -t.
//
// An angle depends on the token and the pair only, so a block computes the
// sines of its tokens once, into shared memory, and uses them for all heads
// of all tensors.  Angles are formed and reduced in 64 bits: position 1e6 has
// an angle that 32 bits hold to 0.06.  The kernel is bound by the one read and
// write of the heads: 2 x 8191 tokens, 20 heads of 128 in 32 bits, 69 us
// (4.9 TB/s; a large copy reaches 4.8 to 5.4), where one item at a time took 84.

#include "lm_ops.h"

#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>
#include <c10/hip/HIPException.h>
#include <hip/hip_runtime.h>
#include <algorithm>

namespace {

constexpr int THREADS = 256;
constexpr int MOST_PAIRS = 2048;  // (cos, sin) of a block: 16 KB
constexpr int MOST_TOKENS = 8;
constexpr int AHEAD = 4;          // work items that a thread has under way

struct Heads {
    const void* in;
    void* out;              // [batch, length, heads, d], contiguous
    int64_t sb, ss, sh;     // the input's strides, in values
    int heads;
};

template <typename T, int V> struct Vec {
    T v[V];
};
template <typename T, int V> struct alignas(sizeof(T) * V) Aligned : Vec<T, V> {};

struct Args {
    Heads x[2];
    int tensors;
    const void* positions;
    int64_t pb, ps;         // the positions' strides
    bool wide;              // positions are 64-bit
    const double* frequencies;
    int length, d, half;    // tokens of a row, head size, pairs
    int64_t tokens;
    int per_block;          // tokens of a block
    float sign;             // -1: the turn back
};

// One work item: V pairs (two vectors, or one with V / 2 pairs), or one vector
// behind them.
template <typename T, int V, bool INTERLEAVED> struct Item {
    Aligned<T, V> v, u;
    const T* in;
    T* out;
    const float2* w;
    bool turns;

    __device__ __forceinline__ void load(const T* from, T* to, const float2* turn, int half,
                                         int slot, int turned) {
        turns = slot < turned;
        const int at = turns ? slot * V : 2 * half + (slot - turned) * V;
        in = from + at;
        out = to + at;
        w = turn + (INTERLEAVED ? slot * (V / 2) : slot * V);
        v = *(const Aligned<T, V>*)in;
        if (!INTERLEAVED && turns) u = *(const Aligned<T, V>*)(in + half);
    }
    __device__ __forceinline__ void store(int half) {
        if (turns) {
            Aligned<T, V> o, r;
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int e = 0; e < V / 2; ++e) {
                    const float2 c = w[e];
                    const float p = (float)v.v[2 * e], q = (float)v.v[2 * e + 1];
                    o.v[2 * e] = (T)(p * c.x - q * c.y);
                    o.v[2 * e + 1] = (T)(p * c.y + q * c.x);
                }
            } else {
#pragma unroll
                for (int e = 0; e < V; ++e) {
                    const float2 c = w[e];
                    const float p = (float)v.v[e], q = (float)u.v[e];
                    o.v[e] = (T)(p * c.x - q * c.y);
                    r.v[e] = (T)(p * c.y + q * c.x);
                }
                *(Aligned<T, V>*)(out + half) = r;
            }
            *(Aligned<T, V>*)out = o;
        } else {
            *(Aligned<T, V>*)out = v;
        }
    }
};

template <typename T, int V, bool INTERLEAVED>
__global__ __launch_bounds__(THREADS) void rotary_kernel(const Args a) {
    __shared__ float2 turn[MOST_PAIRS];
    __shared__ double position[MOST_TOKENS];
    __shared__ int64_t from[2][MOST_TOKENS];  // the tokens' rows in the inputs
    const int64_t first = (int64_t)blockIdx.x * a.per_block;
    const int tokens = (int)min((int64_t)a.per_block, a.tokens - first);
    if ((int)threadIdx.x < tokens) {
        const int64_t token = first + threadIdx.x, b = token / a.length, s = token - b * a.length;
        const int64_t at = b * a.pb + s * a.ps;
        position[threadIdx.x] = a.wide ? (double)((const int64_t*)a.positions)[at]
                                       : (double)((const int*)a.positions)[at];
        for (int t = 0; t < a.tensors; ++t) from[t][threadIdx.x] = b * a.x[t].sb + s * a.x[t].ss;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < tokens * a.half; i += THREADS) {
        // quarters of a turn: what is left lies within an eighth of one
        const int tok = i / a.half;
        const double quarters = position[tok] * a.frequencies[i - tok * a.half] *
                                0.63661977236758134308;
        const double n = rint(quarters);
        float sn, cs;
        sincospif((float)(quarters - n) * 0.5f, &sn, &cs);
        const int q = (int)(n - 4.0 * floor(n * 0.25));
        if (q & 1) {
            float t = cs;
            cs = -sn;
            sn = t;
        }
        if (q & 2) cs = -cs, sn = -sn;
        turn[i] = make_float2(cs, sn * a.sign);
    }
    __syncthreads();

    const int turned = INTERLEAVED ? 2 * a.half / V : a.half / V;
    const int per_head = turned + (a.d - 2 * a.half) / V;
    for (int t = 0; t < a.tensors; ++t) {
        const Heads& x = a.x[t];
        const unsigned per_token = (unsigned)x.heads * per_head, all = tokens * per_token;
        T* to = (T*)x.out + first * x.heads * a.d;
        for (unsigned i0 = threadIdx.x; i0 < all; i0 += AHEAD * THREADS) {
            Item<T, V, INTERLEAVED> items[AHEAD];  // their loads travel together
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) {
                const unsigned i = i0 + n * THREADS;
                if (i >= all) break;
                const unsigned row = i / per_head, tok = row / x.heads;
                items[n].load((const T*)x.in + from[t][tok] + (row - tok * x.heads) * x.sh,
                              to + (int64_t)row * a.d, turn + tok * a.half, a.half,
                              i - row * per_head, turned);
            }
#pragma unroll
            for (int n = 0; n < AHEAD; ++n) {
                if (i0 + n * THREADS >= all) break;
                items[n].store(a.half);
            }
        }
    }
}

template <typename T, int V>
void launch(const Args& a, bool interleaved, int blocks, hipStream_t stream) {
    if (interleaved) {
        if constexpr (V > 1)
            hipLaunchKernelGGL((rotary_kernel<T, V, true>), dim3(blocks), dim3(THREADS), 0,
                               stream, a);
    } else {
        hipLaunchKernelGGL((rotary_kernel<T, V, false>), dim3(blocks), dim3(THREADS), 0, stream,
                           a);
    }
}

template <typename T>
void launch_vec(const Args& a, int v, bool interleaved, int blocks, hipStream_t stream) {
    switch (v) {
        case 8:
            if constexpr (sizeof(T) == 2) launch<T, 8>(a, interleaved, blocks, stream);
            break;
        case 4: launch<T, 4>(a, interleaved, blocks, stream); break;
        case 2: launch<T, 2>(a, interleaved, blocks, stream); break;
        default: launch<T, 1>(a, interleaved, blocks, stream); break;
    }
}

// xs [batch, length, heads, d], turned
torch::autograd::variable_list rotate(torch::autograd::variable_list xs,
                                      const torch::Tensor& positions,
                                      const torch::Tensor& frequencies, bool interleaved,
                                      bool inverse) {
    const torch::Tensor x0 = xs[0];
    c10::DeviceGuard guard(x0.device());
    Args a{};
    a.d = (int)x0.size(3);
    a.half = (int)frequencies.numel();
    a.length = (int)x0.size(1);
    a.tokens = x0.size(0) * x0.size(1);
    a.positions = positions.data_ptr();
    a.pb = positions.dim() == 2 ? positions.stride(0) : 0;
    a.ps = positions.stride(-1);
    a.wide = positions.scalar_type() == torch::kInt64;
    a.frequencies = frequencies.data_ptr<double>();
    a.sign = inverse ? -1.f : 1.f;
    a.tensors = (int)xs.size();

    // the widest vector that every address and extent is a multiple of
    int size = (int)x0.element_size();
    int v = 16 / size;
    torch::autograd::variable_list outs;
    int heads = 0;
    for (size_t t = 0; t < xs.size(); ++t) {
        auto& x = xs[t];
        x = x.resolve_neg();  // a view that torch negates when it reads it
        if (x.stride(3) != 1) x = x.contiguous();
        outs.push_back(torch::empty(x.sizes(), x.options()));
        a.x[t] = {x.data_ptr(), outs[t].data_ptr(), x.stride(0), x.stride(1), x.stride(2),
                  (int)x.size(2)};
        heads += a.x[t].heads;
        while (v > 1 && ((uintptr_t)x.data_ptr() % (v * size) || x.stride(0) % v ||
                         x.stride(1) % v || x.stride(2) % v))
            v /= 2;
    }
    while (v > 1 && (a.d % v || (interleaved ? 2 * a.half : a.half) % v)) v /= 2;
    if (interleaved && v == 1) {
        // pairs at odd addresses: a copy's are even
        for (size_t t = 0; t < xs.size(); ++t) {
            xs[t] = xs[t].clone(at::MemoryFormat::Contiguous);
            a.x[t].in = xs[t].data_ptr();
            a.x[t].sb = xs[t].stride(0);
            a.x[t].ss = xs[t].stride(1);
            a.x[t].sh = xs[t].stride(2);
        }
        v = 2;
    }
    if (a.tokens == 0 || heads == 0) return outs;

    // A block's sines serve all its tokens' heads; tokens are shared out so
    // that 8 blocks a CU have work first, and the sines fit.
    int64_t per = std::max<int64_t>(1, a.tokens / 2048);
    a.per_block =
        (int)std::min<int64_t>({per, (int64_t)MOST_TOKENS, (int64_t)(MOST_PAIRS / a.half)});
    int64_t blocks = (a.tokens + a.per_block - 1) / a.per_block;
    TORCH_CHECK_VALUE(blocks <= INT_MAX, "rotary: too many tokens for one launch");
    hipStream_t stream = at::hip::getCurrentHIPStream();
    switch (x0.scalar_type()) {
        case torch::kFloat32: launch_vec<float>(a, v, interleaved, (int)blocks, stream); break;
        case torch::kBFloat16: launch_vec<__bf16>(a, v, interleaved, (int)blocks, stream); break;
        default: launch_vec<_Float16>(a, v, interleaved, (int)blocks, stream); break;
    }
    C10_HIP_KERNEL_LAUNCH_CHECK();
    return outs;
}

struct RotaryFunction : torch::autograd::Function<RotaryFunction> {
    static torch::autograd::variable_list forward(torch::autograd::AutogradContext* ctx,
                                                  const torch::Tensor& q, const torch::Tensor& k,
                                                  const torch::Tensor& positions,
                                                  const torch::Tensor& frequencies,
                                                  bool interleaved) {
        ctx->save_for_backward({positions, frequencies});
        ctx->saved_data["interleaved"] = interleaved;
        ctx->saved_data["elsewhere"] = held_elsewhere({q, k});
        return rotate({q, k}, positions, frequencies, interleaved, false);
    }
    static torch::autograd::variable_list backward(torch::autograd::AutogradContext* ctx,
                                                   torch::autograd::variable_list grads) {
        const auto x = ctx->get_saved_variables();
        check_capture(ctx->saved_data["elsewhere"].toBool(), "rotary");
        torch::autograd::variable_list need, d(5);
        for (int n = 0; n < 2; ++n)
            if (ctx->needs_input_grad(n)) need.push_back(grads[n]);
        {
            at::AutoGradMode no(false);
            need = rotate(std::move(need), x[0], x[1], ctx->saved_data["interleaved"].toBool(),
                          true);
        }
        need = once_differentiable(std::move(need), "rotary");
        for (int n = 0, at = 0; n < 2; ++n)
            if (ctx->needs_input_grad(n)) d[n] = need[at++];
        return d;
    }
};

}  // namespace

std::vector<torch::Tensor> rotary(torch::Tensor q, torch::Tensor k, torch::Tensor positions,
                                  torch::Tensor frequencies, bool interleaved) {
    for (auto* x : {&q, &k})
        TORCH_CHECK_VALUE(x->is_cuda() && x->dim() == 4 && x->device() == q.device() &&
                              x->scalar_type() == q.scalar_type() && x->size(0) == q.size(0) &&
                              x->size(1) == q.size(1) && x->size(3) == q.size(3),
                          "rotary: q ", q.sizes(), " and k ", k.sizes(),
                          " must be [batch, length, heads, head size] with one batch, length and "
                          "head size, of one type on one device");
    const auto type = q.scalar_type();
    TORCH_CHECK_VALUE(type == torch::kFloat32 || type == torch::kBFloat16 ||
                          type == torch::kFloat16,
                      "rotary: takes float32, bfloat16 or float16, got ", type);
    const int64_t b = q.size(0), s = q.size(1), d = q.size(3);
    TORCH_CHECK_VALUE(d % 2 == 0 && d <= 1024,
                      "rotary: the head size must be even and at most 1024, got ", d);
    TORCH_CHECK_VALUE(positions.device() == q.device() &&
                          (positions.scalar_type() == torch::kInt64 ||
                           positions.scalar_type() == torch::kInt32) &&
                          (positions.sizes() == at::IntArrayRef({s}) ||
                           positions.sizes() == at::IntArrayRef({b, s})),
                      "rotary: positions must be int32 or int64, [", s, "] or [", b, ", ", s,
                      "], on q's device");
    TORCH_CHECK_VALUE(frequencies.device() == q.device() &&
                          frequencies.scalar_type() == torch::kFloat64 &&
                          frequencies.dim() == 1 && frequencies.numel() >= 1 &&
                          frequencies.numel() <= d / 2,
                      "rotary: frequencies must be float64 with 1 to ", d / 2,
                      " values on q's device");
    TORCH_CHECK_VALUE(!frequencies.requires_grad(),
                      "rotary: frequencies are constants and get no gradient");
    check_seen({q, k, frequencies}, "rotary");
    frequencies = frequencies.resolve_neg().contiguous();
    if (at::GradMode::is_enabled() && (q.requires_grad() || k.requires_grad()))
        return RotaryFunction::apply(q, k, positions, frequencies, interleaved);
    return rotate({q, k}, positions, frequencies, interleaved, false);
}
