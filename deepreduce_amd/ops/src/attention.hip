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
#include <hip/hip_runtime.h>
#include <algorithm>

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

template <typename T>
__device__ __forceinline__ float dot(const T* x, const T* y, int d) {
    float s = 0;
    for (int i = 0; i < d; ++i) s = fmaf((float)x[i], (float)y[i], s);
    return s;
}

__device__ __forceinline__ float slope_of(const Args& a, int h) {
    return a.slopes ? a.slopes[h] * LOG2E : 0.f;
}

// ---------------------------------------------------------------------------
// One wave for each row, lanes over keys (or queries) for the scores and over
// the head's values for the sums.  Pairs that are not visible are passed over,
// never multiplied by zero, so that an infinity or NaN behind the mask stays
// there.
// ---------------------------------------------------------------------------

template <typename T>
__device__ void forward_row(const Args& a, int b, int h, int i) {
    const int lane = threadIdx.x & 63, g = h / (a.hq / a.hkv), pos = i + a.sk - a.sq;
    const float slope = slope_of(a, h);
    const T* q = row<T>(a.q, b, i, h);
    float top = -INFINITY, total = 0, o[2] = {0, 0};
    const int end = a.causal ? pos + 1 : a.sk;
    for (int j0 = 0; j0 < end; j0 += 64) {
        int j = j0 + lane;
        bool seen = j < end && visible(a, b, pos, j);
        uint64_t any = __ballot(seen);
        if (!any) continue;
        float s = -INFINITY;
        if (seen)
            s = dot(q, row<T>(a.k, b, j, g), a.d) * (a.scale * LOG2E) - slope * abs(pos - j);
        float next = fmaxf(top, wave_max(s));
        float base = next == -INFINITY ? 0.f : next;
        float keep = exp2_fast(top - base), p = seen ? exp2_fast(s - base) : 0.f;
        top = next;
        total = total * keep + wave_sum(p);
        o[0] *= keep;
        o[1] *= keep;
        for (; any; any &= any - 1) {
            int n = __builtin_ctzll(any);
            float w = __shfl(p, n);
            const T* v = row<T>(a.v, b, j0 + n, g);
            if (lane < a.d) o[0] = fmaf(w, (float)v[lane], o[0]);
            if (lane + 64 < a.d) o[1] = fmaf(w, (float)v[lane + 64], o[1]);
        }
    }
    float inv = total == 0.f ? 0.f : 1.f / total;
    T* out = row<T>(a.out, b, i, h);
    if (lane < a.d) out[lane] = (T)(total == 0.f ? 0.f : o[0] * inv);
    if (lane + 64 < a.d) out[lane + 64] = (T)(total == 0.f ? 0.f : o[1] * inv);
    if (lane == 0 && a.lse)
        a.lse[((int64_t)b * a.hq + h) * a.sq + i] = total == 0.f ? -INFINITY : top + log2f(total);
}

template <typename T>
__device__ void dq_row(const Args& a, int b, int h, int i) {
    const int lane = threadIdx.x & 63, g = h / (a.hq / a.hkv), pos = i + a.sk - a.sq;
    const float slope = slope_of(a, h);
    const int64_t at = ((int64_t)b * a.hq + h) * a.sq + i;
    const float lse = a.lse[at], delta = a.delta[at];
    const T *q = row<T>(a.q, b, i, h), *dout = row<T>(a.dout, b, i, h);
    float acc[2] = {0, 0};
    const int end = a.causal ? pos + 1 : a.sk;
    if (lse != -INFINITY)
        for (int j0 = 0; j0 < end; j0 += 64) {
            int j = j0 + lane;
            bool seen = j < end && visible(a, b, pos, j);
            uint64_t any = __ballot(seen);
            float ds = 0;
            if (seen) {
                float s = dot(q, row<T>(a.k, b, j, g), a.d) * (a.scale * LOG2E) -
                          slope * abs(pos - j);
                ds = exp2_fast(s - lse) * (dot(dout, row<T>(a.v, b, j, g), a.d) - delta);
            }
            for (; any; any &= any - 1) {
                int n = __builtin_ctzll(any);
                float w = __shfl(ds, n);
                const T* k = row<T>(a.k, b, j0 + n, g);
                if (lane < a.d) acc[0] = fmaf(w, (float)k[lane], acc[0]);
                if (lane + 64 < a.d) acc[1] = fmaf(w, (float)k[lane + 64], acc[1]);
            }
        }
    T* dq = row<T>(a.dq, b, i, h);
    if (lane < a.d) dq[lane] = (T)(acc[0] * a.scale);
    if (lane + 64 < a.d) dq[lane + 64] = (T)(acc[1] * a.scale);
}

template <typename T>
__device__ void dkv_row(const Args& a, int b, int g, int j) {
    const int lane = threadIdx.x & 63, group = a.hq / a.hkv;
    const T *k = row<T>(a.k, b, j, g), *v = row<T>(a.v, b, j, g);
    float dk[2] = {0, 0}, dv[2] = {0, 0};
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
            for (; any; any &= any - 1) {
                int n = __builtin_ctzll(any);
                float w = __shfl(p, n), u = __shfl(ds, n);
                const T *dout = row<T>(a.dout, b, i0 + n, h), *q = row<T>(a.q, b, i0 + n, h);
                if (lane < a.d) {
                    dv[0] = fmaf(w, (float)dout[lane], dv[0]);
                    dk[0] = fmaf(u, (float)q[lane], dk[0]);
                }
                if (lane + 64 < a.d) {
                    dv[1] = fmaf(w, (float)dout[lane + 64], dv[1]);
                    dk[1] = fmaf(u, (float)q[lane + 64], dk[1]);
                }
            }
        }
    }
    T *to_k = row<T>(a.dk, b, j, g), *to_v = row<T>(a.dv, b, j, g);
    if (lane < a.d) to_k[lane] = (T)(dk[0] * a.scale), to_v[lane] = (T)dv[0];
    if (lane + 64 < a.d) to_k[lane + 64] = (T)(dk[1] * a.scale), to_v[lane + 64] = (T)dv[1];
}

enum Pass { FORWARD, DELTA, DQ, DKV };

template <typename T>
__device__ void delta_row(const Args& a, int b, int h, int i) {
    const int lane = threadIdx.x & 63;
    const T *x = row<T>(a.dout, b, i, h), *y = row<T>(a.out, b, i, h);
    float s = 0;
    for (int d = lane; d < a.d; d += 64) s = fmaf((float)x[d], (float)y[d], s);
    s = wave_sum(s);
    if (lane == 0) a.delta[((int64_t)b * a.hq + h) * a.sq + i] = s;
}

template <typename T, Pass PASS>
__global__ __launch_bounds__(256) void rows_kernel(const Args a, int64_t rows, int length,
                                                   int heads) {
    int64_t r = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (r >= rows) return;
    int i = (int)(r % length);
    int h = (int)(r / length % heads), b = (int)(r / length / heads);
    if constexpr (PASS == FORWARD) forward_row<T>(a, b, h, i);
    if constexpr (PASS == DELTA) delta_row<T>(a, b, h, i);
    if constexpr (PASS == DQ) dq_row<T>(a, b, h, i);
    if constexpr (PASS == DKV) dkv_row<T>(a, b, h, i);
}

template <typename T, Pass PASS>
void launch_rows(const Args& a, hipStream_t stream) {
    int length = PASS == DKV ? a.sk : a.sq, heads = PASS == DKV ? a.hkv : a.hq;
    int64_t rows = (int64_t)a.b * length * heads;
    if (rows == 0) return;
    int64_t blocks = (rows + 3) / 4;
    TORCH_CHECK(blocks <= INT_MAX, "too many rows for one launch");
    hipLaunchKernelGGL((rows_kernel<T, PASS>), dim3((unsigned)blocks), dim3(256), 0, stream, a,
                       rows, length, heads);
}

// ---------------------------------------------------------------------------

View view(const torch::Tensor& t) {
    return {t.data_ptr(), t.stride(0), t.stride(1), t.stride(2)};
}

// d contiguous and every head at a 16-byte address, by a copy where it is not
torch::Tensor aligned(const torch::Tensor& t) {
    int64_t per = 16 / t.element_size();
    bool fine = (uintptr_t)t.data_ptr() % 16 == 0 && t.stride(3) == 1;
    for (int d = 0; d < 3; ++d) fine = fine && t.stride(d) % per == 0;
    return fine ? t : t.clone(at::MemoryFormat::Contiguous);
}

Args args_for(const torch::Tensor& q, const torch::Tensor& k, const torch::Tensor& v,
              const std::optional<torch::Tensor>& documents,
              const std::optional<torch::Tensor>& slopes, bool causal, double scale) {
    for (auto* t : {&q, &k, &v})
        TORCH_CHECK(t->is_cuda() && t->dim() == 4 && t->device() == q.device() &&
                        t->scalar_type() == q.scalar_type(),
                    "q, k and v must be 4-D GPU tensors of one type and device");
    Args a{};
    a.b = (int)q.size(0);
    a.sq = (int)q.size(1);
    a.hq = (int)q.size(2);
    a.d = (int)q.size(3);
    a.sk = (int)k.size(1);
    a.hkv = (int)k.size(2);
    TORCH_CHECK(k.sizes() == v.sizes() && k.size(0) == a.b && k.size(3) == a.d,
                "k and v must be [batch, length, heads, d] like q");
    TORCH_CHECK(a.d >= 8 && a.d <= MOST_D && a.d % 8 == 0,
                "the head size must be a multiple of 8 from 8 to 128");
    TORCH_CHECK(a.hkv >= 1 && a.hq % a.hkv == 0, "kv heads must divide the query heads");
    TORCH_CHECK(a.sq <= a.sk, "there are more queries than keys");
    TORCH_CHECK(k.size(1) < (1 << 30), "too many keys");
    if (documents) {
        TORCH_CHECK(documents->is_cuda() && documents->device() == q.device() &&
                        documents->scalar_type() == torch::kInt32 && documents->dim() == 2 &&
                        documents->size(0) == a.b && documents->size(1) == a.sk &&
                        (documents->stride(1) == 1 || a.sk <= 1),
                    "documents must be int32 [batch, keys]");
        a.documents = documents->data_ptr<int>();
        a.documents_sb = documents->stride(0);
    }
    if (slopes) {
        TORCH_CHECK(slopes->is_cuda() && slopes->device() == q.device() &&
                        slopes->scalar_type() == torch::kFloat32 && slopes->dim() == 1 &&
                        slopes->size(0) == a.hq && slopes->is_contiguous(),
                    "slopes must be float32 [query heads]");
        a.slopes = slopes->data_ptr<float>();
    }
    a.causal = causal;
    a.scale = (float)scale;
    return a;
}

template <typename F>
void for_type(torch::ScalarType type, F f) {
    switch (type) {
        case torch::kFloat32: f((float*)nullptr); break;
        case torch::kBFloat16: f((__bf16*)nullptr); break;
        case torch::kFloat16: f((_Float16*)nullptr); break;
        default: TORCH_CHECK(false, "attention takes float32, bfloat16 or float16");
    }
}

}  // namespace

std::vector<torch::Tensor> attention_forward(torch::Tensor q, torch::Tensor k, torch::Tensor v,
                                             std::optional<torch::Tensor> documents,
                                             std::optional<torch::Tensor> slopes, bool causal,
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
    for_type(q.scalar_type(), [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        launch_rows<T, FORWARD>(a, stream);
    });
    return {out, lse};
}

std::vector<torch::Tensor> attention_backward(torch::Tensor dout, torch::Tensor q,
                                              torch::Tensor k, torch::Tensor v, torch::Tensor out,
                                              torch::Tensor lse,
                                              std::optional<torch::Tensor> documents,
                                              std::optional<torch::Tensor> slopes, bool causal,
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
    for_type(q.scalar_type(), [&](auto* t) {
        using T = std::remove_pointer_t<decltype(t)>;
        launch_rows<T, DELTA>(a, stream);
        launch_rows<T, DQ>(a, stream);
        launch_rows<T, DKV>(a, stream);
    });
    return {dq, dk, dv};
}
