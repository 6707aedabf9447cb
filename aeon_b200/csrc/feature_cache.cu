// The feature cache on sm_100a: rows of floats to 8-bit codes in pages, with a scale for each token and head, and back.
//
// A warp per group (token and head): it looks up the page, takes the largest magnitude of the group's values, and writes the
// codes.  The quotient x / scale is first formed as x times the reciprocal; where that lies so near to the middle between
// two codes that the roundings of the two operations could decide, the exact quotient does (in 64 bits: the numerator and
// denominator have 24 bits each, so a quotient that is not in the middle is at least 2^-25 of it away, and the division's
// own rounding cannot carry it there).
#include <cuda_fp8.h>

#include <algorithm>

#include "float_rows.cuh"

namespace aeonb
{
    namespace
    {
        constexpr uint32_t ABS_BITS = 0x7fffffffu, INF_BITS = 0x7f800000u, MINUS_INF = 0xff800000u;

        // Where a group's codes and scale lie; -1 for a token without a place.
        __device__ __forceinline__ int64_t group_place(const aeonb_cache_desc& d, int seq, int token, int head)
        {
            const int64_t at = (int64_t)token + (d.start ? d.start[seq] : 0);
            if (at < 0 || at >= (int64_t)d.table_pages * d.page_tokens)
                return -1;
            const int32_t page = d.table[seq * d.table_stride + at / d.page_tokens];
            if (page < 0 || page >= d.pages)
                return -1;
            return ((int64_t)page * d.page_tokens + at % d.page_tokens) * d.heads + head;
        }

        __device__ __forceinline__ int tokens_of(const aeonb_cache_desc& d, int seq)
        {
            return d.length ? min(max(d.length[seq], 0), d.tokens) : d.tokens;
        }

        // bits of |x| that count in the group's largest magnitude: none of -infinity, NaN and +infinity as they are
        __device__ __forceinline__ uint32_t magnitude(float x)
        {
            const uint32_t b = __float_as_uint(x);
            return b == MINUS_INF ? 0u : b & ABS_BITS;
        }

        template <int CODE>
        __device__ __forceinline__ float group_scale(uint32_t largest)
        {
            const float q = CODE == AEONB_CODE_INT8 ? 127.0f : 448.0f;
            if (largest >= INF_BITS)
                return __uint_as_float(0x7fffffffu);
            float s = fmaxf(__fdiv_rn(__uint_as_float(largest), q), 1.17549435e-38f);
            if (__fmul_rn(s, q) > 3.40282347e38f) // the largest code would read back as infinity
                s = __uint_as_float(__float_as_uint(s) - 1);
            return s;
        }

        template <int CODE>
        __device__ __forceinline__ uint8_t encode(float x, float scale, float inverse)
        {
            if (__float_as_uint(x) == MINUS_INF)
                return CODE == AEONB_CODE_INT8 ? 0x80 : 0xff;
            const float t = __fmul_rn(x, inverse); // off by 2^-23 of itself at most
            if (CODE == AEONB_CODE_INT8)
            {
                float q = rintf(t);
                if (fabsf(__fsub_rn(t, q)) > 0.5f - 0x1p-15f)
                    q = (float)rint(__ddiv_rn((double)x, (double)scale));
                return (uint8_t)(int8_t)(int)q;
            }
            const uint32_t low  = __float_as_uint(t) & 0xfffffu; // the bits behind the three that a normal e4m3 keeps
            float          odd  = t;
            if (low - 0x7fff8u <= 16u || (fabsf(t) < 0x1p-6f && t != 0.0f))
            {
                // the exact quotient, cut to float with its last bit set where bits were lost: rounds to e4m3 as it would itself
                const double q = __ddiv_rn((double)x, (double)scale);
                odd            = __double2float_rz(q);
                if ((double)odd != q)
                    odd = __uint_as_float(__float_as_uint(odd) | 1u);
            }
            return (uint8_t)__nv_cvt_float_to_fp8(odd, __NV_SATFINITE, __NV_E4M3);
        }

        template <int CODE>
        __device__ __forceinline__ float decode(uint8_t code, float scale)
        {
            if (CODE == AEONB_CODE_INT8)
                return code == 0x80 ? __uint_as_float(MINUS_INF) : __fmul_rn((float)(int8_t)code, scale);
            if (code == 0xff)
                return __uint_as_float(MINUS_INF);
            return __fmul_rn(__half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3))), scale);
        }

        template <typename T, int CODE>
        __global__ void __launch_bounds__(256) cache_write_kernel(const aeonb_cache_desc d)
        {
            const int64_t groups = (int64_t)d.seqs * d.tokens * d.heads;
            const int     lane   = threadIdx.x & 31;
            for (int64_t g = blockIdx.x * (int64_t)(blockDim.x / 32) + threadIdx.x / 32; g < groups; g += (int64_t)gridDim.x * (blockDim.x / 32))
            {
                const int head = (int)(g % d.heads), token = (int)(g / d.heads % d.tokens), seq = (int)(g / d.heads / d.tokens);
                if (token >= tokens_of(d, seq))
                    continue;
                const int64_t place = group_place(d, seq, token, head);
                if (place < 0)
                {
                    if (lane == 0 && d.status)
                        *d.status = 1;
                    continue;
                }
                const T* x = static_cast<const T*>(d.rows) + seq * d.row_stride_seq + token * d.row_stride_token + head * d.row_stride_head;
                T*       v = d.values ? static_cast<T*>(d.values) + seq * d.value_stride_seq + token * d.value_stride_token + head * d.value_stride_head
                                      : nullptr;
                uint32_t largest = 0;
                for (int i = lane; i < d.dim; i += 32)
                    largest = max(largest, magnitude(to_float(x[i])));
                largest           = __reduce_max_sync(0xffffffffu, largest);
                const float scale = group_scale<CODE>(largest), inverse = __frcp_rn(scale);
                uint8_t*    codes = static_cast<uint8_t*>(d.codes) + place * d.dim;
                if (lane == 0)
                    d.scales[place] = scale;
                for (int i = lane; i < d.dim; i += 32)
                {
                    const uint8_t q = scale == scale ? encode<CODE>(to_float(x[i]), scale, inverse) : (uint8_t)0;
                    codes[i]        = q;
                    if (v)
                        v[i] = from_float<T>(decode<CODE>(q, scale));
                }
            }
        }

        template <typename T, int CODE>
        __global__ void __launch_bounds__(256) cache_read_kernel(const aeonb_cache_desc d)
        {
            const int64_t groups = (int64_t)d.seqs * d.tokens * d.heads;
            const int     lane   = threadIdx.x & 31;
            for (int64_t g = blockIdx.x * (int64_t)(blockDim.x / 32) + threadIdx.x / 32; g < groups; g += (int64_t)gridDim.x * (blockDim.x / 32))
            {
                const int head = (int)(g % d.heads), token = (int)(g / d.heads % d.tokens), seq = (int)(g / d.heads / d.tokens);
                T*        v = static_cast<T*>(d.rows) + seq * d.row_stride_seq + token * d.row_stride_token + head * d.row_stride_head;
                if (token >= tokens_of(d, seq))
                {
                    for (int i = lane; i < d.dim; i += 32)
                        v[i] = from_float<T>(0.0f);
                    continue;
                }
                const int64_t place = group_place(d, seq, token, head);
                if (place < 0)
                {
                    if (lane == 0 && d.status)
                        *d.status = 1;
                    for (int i = lane; i < d.dim; i += 32)
                        v[i] = from_float<T>(__uint_as_float(0x7fffffffu));
                    continue;
                }
                const float    scale = d.scales[place];
                const uint8_t* codes = static_cast<const uint8_t*>(d.codes) + place * d.dim;
                for (int i = lane; i < d.dim; i += 32)
                    v[i] = from_float<T>(decode<CODE>(codes[i], scale));
            }
        }

        void check_cache(const aeonb_cache_desc& d, bool write)
        {
            const int e = float_size(d.dtype);
            if (d.code != AEONB_CODE_INT8 && d.code != AEONB_CODE_E4M3)
                throw std::invalid_argument("the code of a cache must be AEONB_CODE_INT8 or AEONB_CODE_E4M3");
            if (d.page_tokens <= 0 || d.heads <= 0 || d.dim <= 0 || d.pages < 0)
                throw std::invalid_argument("a cache needs page_tokens, heads and dim above 0");
            if (d.seqs < 0 || d.tokens < 0 || d.table_pages < 0)
                throw std::invalid_argument("negative number of sequences, tokens or table entries");
            if ((double)d.pages * d.page_tokens * d.heads * d.dim > 0x1p62 || (double)d.seqs * d.tokens * d.heads * d.dim > 0x1p62)
                throw std::invalid_argument("more values than 64-bit offsets reach");
            if (d.seqs == 0 || d.tokens == 0)
                return;
            if (!d.rows || (d.pages > 0 && (!d.codes || !d.scales)) || (d.table_pages > 0 && !d.table))
                throw std::invalid_argument("NULL rows, codes, scales or table");
            if (!aligned_to(d.rows, e) || (write && !aligned_to(d.values, e)) || !aligned_to(d.scales, 4) || !aligned_to(d.table, 4) ||
                !aligned_to(d.start, 4) || !aligned_to(d.length, 4) || !aligned_to(d.status, 4))
                throw std::invalid_argument("a pointer is not aligned to its elements");
            // two groups of a destination that share values would be written by two warps at once
            const auto overlap = [&](int64_t seq, int64_t token, int64_t head) {
                struct axis
                {
                    int64_t n, stride;
                } a[3] = {{d.seqs, seq}, {d.tokens, token}, {d.heads, head}};
                std::sort(a, a + 3, [](const axis& l, const axis& r) { return l.stride < r.stride; });
                int64_t reach = d.dim; // values that the axes so far span
                for (const axis& x : a)
                {
                    if (x.n <= 1)
                        continue;
                    if (x.stride < reach)
                        return true;
                    reach += (x.n - 1) * x.stride;
                }
                return false;
            };
            if (!write && overlap(d.row_stride_seq, d.row_stride_token, d.row_stride_head))
                throw std::invalid_argument("the rows that are read to overlap one another");
            if (write && d.values)
            {
                if (overlap(d.value_stride_seq, d.value_stride_token, d.value_stride_head))
                    throw std::invalid_argument("the rows of the values overlap one another");
                if (d.values == d.rows && (d.value_stride_seq != d.row_stride_seq || d.value_stride_token != d.row_stride_token ||
                                           d.value_stride_head != d.row_stride_head))
                    throw std::invalid_argument("values in place of the rows need the rows' strides");
            }
            if (write && (d.row_stride_seq < 0 || d.row_stride_token < 0 || d.row_stride_head < 0))
                throw std::invalid_argument("negative stride");
        }

        template <typename T>
        void launch_cache(const aeonb_cache_desc& d, bool write, unsigned blocks, cudaStream_t stream)
        {
            if (write)
                d.code == AEONB_CODE_INT8 ? cache_write_kernel<T, AEONB_CODE_INT8><<<blocks, 256, 0, stream>>>(d)
                                          : cache_write_kernel<T, AEONB_CODE_E4M3><<<blocks, 256, 0, stream>>>(d);
            else
                d.code == AEONB_CODE_INT8 ? cache_read_kernel<T, AEONB_CODE_INT8><<<blocks, 256, 0, stream>>>(d)
                                          : cache_read_kernel<T, AEONB_CODE_E4M3><<<blocks, 256, 0, stream>>>(d);
        }

        int run_cache(aeonb_ctx* ctx, const aeonb_cache_desc* desc, bool write)
        {
            return guarded([&]() {
                if (!ctx || !desc)
                    throw std::invalid_argument(write ? "aeonb_cache_write: NULL argument" : "aeonb_cache_read: NULL argument");
                const aeonb_cache_desc& d = *desc;
                check_cache(d, write);
                if (d.seqs == 0 || d.tokens == 0)
                    return AEONB_OK;
                device_scope   scope(ctx->device);
                const int64_t  groups = (int64_t)d.seqs * d.tokens * d.heads;
                const unsigned blocks = (unsigned)std::min<int64_t>((groups + 7) / 8, 148 * 64);
                const int64_t  values = groups * d.dim;
                const cudaStream_t stream = d.stream ? static_cast<cudaStream_t>(d.stream) : ctx->stream;
                launch_timer   timer(ctx, AEONB_KERNEL_OTHER, values * (float_size(d.dtype) * (d.values && write ? 2 : 1) + 1) + groups * 4, stream);
                switch (d.dtype)
                {
                case AEONB_F32: launch_cache<float>(d, write, blocks, stream); break;
                case AEONB_F16: launch_cache<__half>(d, write, blocks, stream); break;
                case AEONB_BF16: launch_cache<__nv_bfloat16>(d, write, blocks, stream); break;
                }
                const cudaError_t e = cudaGetLastError();
                if (e != cudaSuccess)
                    throw error(AEONB_ERR_CUDA, cuda_message("feature cache kernel launch", e));
                ctx->launches++;
                return AEONB_OK;
            });
        }
    }
}

extern "C" {

int aeonb_cache_write(aeonb_ctx* ctx, const aeonb_cache_desc* desc)
{
    return aeonb::run_cache(ctx, desc, true);
}

int aeonb_cache_read(aeonb_ctx* ctx, const aeonb_cache_desc* desc)
{
    return aeonb::run_cache(ctx, desc, false);
}

} // extern "C"
