// Distillation from a teacher's top logits on sm_100a: the loss of each row, its log-sum-exp, and the gradient.
//
// A block per row.  One pass over the logits keeps, in each thread, the largest value so far and the sum of exponentials
// against it (both in 32 bits, the exponentials to the base 2 with log2(e) / T as a factor of the difference, so that rows at the
// ends of the type's range do not overflow); a second pass writes the gradient.  The entries' own part of the gradient is written after a barrier, by the first thread that holds the id, with
// the probabilities of all entries of that id added in their order: no atomics, the same bits every time.
#include <algorithm>
#include <cmath>

#include "float_rows.cuh"

namespace aeonb
{
    namespace
    {
        constexpr int   THREADS = 256;
        constexpr int   ENTRIES = AEONB_DISTILL_MAX_ENTRIES;
        constexpr float LN2     = 0.693147180559945309417f;

        struct distill_launch
        {
            aeonb_distill_desc d;
            float              c;      // log2(e) / T
            float              factor; // T grad_scale
            float              tt;     // T^2
        };

        template <typename Op>
        __device__ __forceinline__ float block_reduce(float v, float* shared, Op op)
        {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
                v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
            __syncthreads();
            if ((threadIdx.x & 31) == 0)
                shared[threadIdx.x / 32] = v;
            __syncthreads();
            float r = shared[0];
            for (int i = 1; i < THREADS / 32; ++i)
                r = op(r, shared[i]);
            return r;
        }
        struct add
        {
            __device__ float operator()(float a, float b) const { return __fadd_rn(a, b); }
        };
        struct larger // NaN where one of the two is
        {
            __device__ float operator()(float a, float b) const { return a != a || b != b ? __uint_as_float(0x7fffffffu) : fmaxf(a, b); }
        };

        __device__ __forceinline__ float pow2(float x) { return exp2f(x); }

        template <typename T, bool WITH_LOSS>
        __global__ void __launch_bounds__(THREADS) distill_kernel(const distill_launch L)
        {
            __shared__ float shared[THREADS / 32];
            __shared__ int   ids[ENTRIES];
            __shared__ float probs[ENTRIES];
            const aeonb_distill_desc& d   = L.d;
            const int                 tid = threadIdx.x;
            const float               nan = __uint_as_float(0x7fffffffu), inf = __uint_as_float(0x7f800000u);
            for (int64_t row = blockIdx.x; row < d.rows; row += gridDim.x)
            {
                const T* s    = static_cast<const T*>(d.logits) + row * d.logits_stride;
                T*       grad = d.grad ? static_cast<T*>(d.grad) + row * d.grad_stride : nullptr;
                // the entries: thread i has entry i
                int   id = -1;
                float t  = -inf;
                if (tid < d.k)
                {
                    id = d.ids[row * d.entry_stride + tid];
                    t  = d.teacher[row * d.entry_stride + tid];
                    if (id < 0 || t == -inf)
                    {
                        id = -1;
                        t  = -inf;
                    }
                }
                __syncthreads();
                ids[tid]           = id;
                const bool  beyond = __syncthreads_or(id >= d.vocab);
                const float w      = d.weights ? d.weights[row] : 1.0f;
                const float tmax   = block_reduce(t, shared, larger());
                if (w == 0.0f || tmax == -inf)
                {
                    if (WITH_LOSS && tid == 0)
                    {
                        if (d.loss)
                            d.loss[row] = 0.0f;
                        if (d.lse)
                            d.lse[row] = 0.0f;
                    }
                    if (grad)
                        for (int64_t v = tid; v < d.vocab; v += THREADS)
                            grad[v] = from_float<T>(0.0f);
                    continue;
                }
                const float e    = id >= 0 ? pow2(__fmul_rn(__fsub_rn(t, tmax), L.c)) : 0.0f;
                const float esum = block_reduce(e, shared, add());
                const float p    = __fdiv_rn(e, esum);
                const float sid  = id >= 0 && !beyond ? to_float(s[id]) : 0.0f;
                probs[tid]       = p;

                float top, sum = 1.0f; // the largest logit (or lse times T), and the sum of exponentials against it
                float correct = 1.0f;  // factor that makes up for the rounding of lse times T
                bool  bad = beyond || !(tmax < inf);
                if (WITH_LOSS)
                {
                    float m = -inf, z = 0.0f;
                    bool  isnan = false;
                    if (!bad)
                        for (int64_t v = tid; v < d.vocab; v += THREADS)
                        {
                            const float x = to_float(s[v]);
                            isnan |= x != x;
                            if (x > m)
                            {
                                z = m == -inf ? 0.0f : __fmul_rn(z, pow2(__fmul_rn(__fsub_rn(m, x), L.c)));
                                m = x;
                            }
                            if (m > -inf)
                                z += pow2(__fmul_rn(__fsub_rn(x, m), L.c));
                        }
                    const float all = block_reduce(isnan ? nan : m, shared, larger());
                    bad |= !(fabsf(all) < inf);
                    top = all;
                    sum  = block_reduce(m > -inf && !bad ? __fmul_rn(z, pow2(__fmul_rn(__fsub_rn(m, all), L.c))) : 0.0f, shared, add());
                    // p (log p - s / T + lse), to the base 2
                    float term = 0.0f;
                    const float l2 = log2f(sum);
                    if (p > 0.0f)
                    {
                        const float logp = __fsub_rn(__fmul_rn(__fsub_rn(t, tmax), L.c), log2f(esum));
                        term             = __fmul_rn(p, __fadd_rn(logp, __fadd_rn(l2, __fmul_rn(__fsub_rn(all, sid), L.c))));
                    }
                    const float total = block_reduce(term, shared, add());
                    if (tid == 0)
                    {
                        if (d.loss)
                            d.loss[row] = bad ? nan : __fmul_rn(__fmul_rn(w, L.tt), __fmul_rn(total, LN2));
                        if (d.lse)
                            d.lse[row] = bad ? nan : __fadd_rn(__fdiv_rn(top, d.temperature), __fmul_rn(l2, LN2));
                    }
                    if (!grad)
                        continue;
                }
                else
                {
                    const float lse = d.lse[row];
                    bad |= !(fabsf(lse) < inf);
                    top     = __fmul_rn(lse, d.temperature);
                    correct = pow2(__fmul_rn(-__fmaf_rn(lse, d.temperature, -top), L.c));
                }
                float f = __fmul_rn(w, L.factor);
                if (d.upstream)
                    f = __fmul_rn(f, d.upstream[row]);
                if (bad)
                    f = nan;
                const float fq = WITH_LOSS ? __fdiv_rn(f, sum) : __fmul_rn(f, correct);
                for (int64_t v = tid; v < d.vocab; v += THREADS)
                    grad[v] = from_float<T>(__fmul_rn(fq, pow2(__fmul_rn(__fsub_rn(to_float(s[v]), top), L.c))));
                __syncthreads(); // the entries' logits have been read, and the row written
                if (!bad && id >= 0)
                {
                    float all   = 0.0f;
                    bool  first = true;
                    for (int i = 0; i < d.k; ++i)
                        if (ids[i] == id)
                        {
                            first &= i >= tid;
                            all = __fadd_rn(all, probs[i]);
                        }
                    if (first)
                        grad[id] = from_float<T>(__fsub_rn(__fmul_rn(fq, pow2(__fmul_rn(__fsub_rn(sid, top), L.c))), __fmul_rn(f, all)));
                }
            }
        }

        void check_distill(const aeonb_distill_desc& d, bool with_loss)
        {
            const int e = float_size(d.dtype);
            if (d.rows < 0 || d.rows > 0x7fffffff || d.vocab < 1)
                throw std::invalid_argument("the logits need between 0 and 2^31-1 rows of at least one value");
            if (d.k < 1 || d.k > ENTRIES)
                throw std::invalid_argument("a row has between 1 and 256 entries");
            if (!(d.temperature > 0.0f) || !std::isfinite(d.temperature) || !std::isfinite(1.4426950408889634 / d.temperature) ||
                !std::isfinite(d.temperature * d.temperature))
                throw std::invalid_argument("the temperature must be a positive number");
            if (d.rows == 0)
                return;
            if (!d.logits || !d.ids || !d.teacher)
                throw std::invalid_argument("NULL logits, ids or teacher's logits");
            if (with_loss ? !d.loss && !d.lse && !d.grad : !d.lse || !d.grad)
                throw std::invalid_argument(with_loss ? "nothing to compute: loss, lse and grad are NULL" : "NULL lse or grad");
            if (!aligned_to(d.logits, e) || !aligned_to(d.grad, e) || !aligned_to(d.ids, 4) || !aligned_to(d.teacher, 4) ||
                !aligned_to(d.weights, 4) || !aligned_to(d.loss, 4) || !aligned_to(d.lse, 4) || !aligned_to(d.upstream, 4))
                throw std::invalid_argument("a pointer is not aligned to its elements");
            if (d.rows > 1 && (d.logits_stride < 0 || d.entry_stride < 0))
                throw std::invalid_argument("negative stride");
            if (d.grad && d.rows > 1 && d.grad_stride < d.vocab)
                throw std::invalid_argument("the rows of the gradient overlap one another");
            if (d.grad == d.logits && d.rows > 1 && d.grad_stride != d.logits_stride)
                throw std::invalid_argument("a gradient in place of the logits needs their stride");
        }

        template <typename T>
        void launch_distill(const distill_launch& L, bool with_loss, unsigned blocks, cudaStream_t stream)
        {
            with_loss ? distill_kernel<T, true><<<blocks, THREADS, 0, stream>>>(L) : distill_kernel<T, false><<<blocks, THREADS, 0, stream>>>(L);
        }

        int run_distill(aeonb_ctx* ctx, const aeonb_distill_desc* desc, bool with_loss)
        {
            return guarded([&]() {
                if (!ctx || !desc)
                    throw std::invalid_argument(with_loss ? "aeonb_distill_loss: NULL argument" : "aeonb_distill_grad: NULL argument");
                check_distill(*desc, with_loss);
                if (desc->rows == 0)
                    return AEONB_OK;
                device_scope   scope(ctx->device);
                distill_launch L;
                L.d      = *desc;
                L.c      = (float)(1.4426950408889634074 / desc->temperature);
                L.factor = (float)((double)desc->temperature * desc->grad_scale);
                L.tt     = (float)((double)desc->temperature * desc->temperature);
                const int64_t  bytes  = desc->rows * ((int64_t)desc->vocab * float_size(desc->dtype) * (desc->grad ? 2 : 1) + desc->k * 8 + 8);
                const unsigned blocks = (unsigned)std::min<int64_t>(desc->rows, 1 << 20);
                launch_timer   timer(ctx, AEONB_KERNEL_OTHER, bytes);
                switch (desc->dtype)
                {
                case AEONB_F32: launch_distill<float>(L, with_loss, blocks, ctx->stream); break;
                case AEONB_F16: launch_distill<__half>(L, with_loss, blocks, ctx->stream); break;
                case AEONB_BF16: launch_distill<__nv_bfloat16>(L, with_loss, blocks, ctx->stream); break;
                }
                const cudaError_t e = cudaGetLastError();
                if (e != cudaSuccess)
                    throw error(AEONB_ERR_CUDA, cuda_message("distillation kernel launch", e));
                ctx->launches++;
                return AEONB_OK;
            });
        }
    }
}

extern "C" {

int aeonb_distill_loss(aeonb_ctx* ctx, const aeonb_distill_desc* desc)
{
    return aeonb::run_distill(ctx, desc, true);
}

int aeonb_distill_grad(aeonb_ctx* ctx, const aeonb_distill_desc* desc)
{
    return aeonb::run_distill(ctx, desc, false);
}

} // extern "C"
