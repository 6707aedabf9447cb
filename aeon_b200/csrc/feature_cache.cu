// The feature cache on sm_100a: rows of floats to 8-bit codes in pages, with a scale for each token and head, and back.
//
// A group (token and head) is read once: up to 32 lanes hold chunks of it, of 32 bytes of the rows where their place allows it, else 16,
// else four values that lie the group's lanes apart; several groups share a warp.  Its largest magnitude is that of the bit patterns without their sign; only where
// that is no finite number are infinities looked at one by one.  Floor: the bytes of rows, codes and scales.
//
// Measured on B200, 6.55 TB/s being what a copy reaches (events around a call, inputs not in L2): 64 x 4096 x 8 groups of 128 bf16 with
// values to e4m3 0.21 ms (6.5 TB/s), to int8 0.21 (6.5), read back 0.13 (6.3); of 64 floats 0.19 (6.5) and 0.11 (6.3); 2560 x 2000 of
// 40 floats 0.31 (5.9) and 0.17 (6.1); rows off 16 bytes less: 2560 x 200 of 161 floats 0.16 (4.7) and 0.10 (4.0), 5120 x 3330 of 13
// 0.91 (2.3) and 0.40 (2.9), which wait for the issue of instructions (whole runs of tokens through shared memory were slower).
//
// Codes are those of the exact quotient x / scale.  That is formed to 24 bits, the last one set where it is not exact, on the quotient's own
// side of every middle between two codes, so that it rounds as the quotient itself would (16-bit rows are full of quotients next to
// such a middle: ratios of small numbers, but for the rounding of the scale).
#include <cuda_fp8.h>

#include <algorithm>
#include <type_traits>

#include "float_rows.cuh"

namespace aeonb
{
    namespace
    {
        constexpr int      MAX_DIM  = 0x7fffffff - 1023;
        constexpr uint32_t ABS_BITS = 0x7fffffffu, INF_BITS = 0x7f800000u, MINUS_INF = 0xff800000u;

        // Division of numbers below 2^31 by one known to the host: the upper half of a product, shifted.
        struct fast_divisor
        {
            uint32_t by, factor, shift;
            fast_divisor() = default;
            explicit fast_divisor(uint32_t d) : by(d), factor(0), shift(0)
            {
                while (1ull << (shift + 1) < d)
                    ++shift;
                factor = (uint32_t)(((1ull << (32 + shift)) + d - 1) / d); // ceil(2^(32 + shift) / d), 2^shift < d <= 2^(shift + 1)
            }
            __device__ __forceinline__ uint32_t operator()(uint32_t n) const { return by == 1 ? n : __umulhi(n, factor) >> shift; }
        };

        struct cache_launch
        {
            aeonb_cache_desc d;
            int              lanes;  // of a group
            int              groups; // of a sequence
            fast_divisor     by_heads, by_page, by_lanes;
            int64_t          positions;      // that the table reaches
            int64_t          by_page_groups; // groups of a page
        };

        // a b, a not negative: two multiplications of 32 bits
        __device__ __forceinline__ int64_t times(int a, int64_t b) { return (int64_t)((uint64_t)(uint32_t)a * (uint64_t)b); }

        // Where a group's codes and scale lie; -1 for a token without a place.
        __device__ __forceinline__ int64_t group_place(const cache_launch& L, int seq, int token, int head)
        {
            const aeonb_cache_desc& d  = L.d;
            const int64_t           at = (int64_t)token + (d.start ? d.start[seq] : 0);
            if (at < 0 || at >= L.positions)
                return -1;
            const uint32_t page_of = at < 0x7fffffff ? L.by_page((uint32_t)at) : (uint32_t)at / (uint32_t)d.page_tokens; // (at is below 2^32)
            const int32_t  page    = d.table[times(seq, d.table_stride) + page_of];
            if (page < 0 || page >= d.pages)
                return -1;
            return times(page, L.by_page_groups) + times(d.heads, (uint32_t)at - page_of * (uint32_t)d.page_tokens) + head;
        }

        __device__ __forceinline__ int tokens_of(const aeonb_cache_desc& d, int seq)
        {
            return d.length ? min(max(d.length[seq], 0), d.tokens) : d.tokens;
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

        // The code of one value, whatever it is.  (In 64 bits: numerator and denominator have 24 bits each, so a quotient that is not in the
        // middle between two codes is at least 2^-25 of it away, and the division's own rounding cannot carry it there.)
        template <int CODE>
        __device__ __noinline__ uint32_t encode_exactly(float x, float scale)
        {
            if (!(scale == scale))
                return 0;
            if (__float_as_uint(x) == MINUS_INF)
                return CODE == AEONB_CODE_INT8 ? 0x80 : 0xff;
            const double q = __ddiv_rn((double)x, (double)scale);
            if (CODE == AEONB_CODE_INT8)
                return (uint32_t)(int)rint(q) & 0xff;
            // cut to float with the last bit set where bits were lost: rounds to e4m3 as the quotient itself would
            float odd = __double2float_rz(q);
            if ((double)odd != q)
                odd = __uint_as_float(__float_as_uint(odd) | 1u);
            return __nv_cvt_float_to_fp8(odd, __NV_SATFINITE, __NV_E4M3);
        }

        template <int CODE>
        __device__ __forceinline__ float decode(uint32_t code, float scale)
        {
            if (CODE == AEONB_CODE_INT8)
                return code == 0x80 ? __uint_as_float(MINUS_INF) : __fmul_rn((float)(int8_t)code, scale);
            if (code == 0xff)
                return __uint_as_float(MINUS_INF);
            return __fmul_rn(__half2float(__half(__nv_cvt_fp8_to_halfraw((__nv_fp8_storage_t)code, __NV_E4M3))), scale);
        }

        __device__ __forceinline__ float2 mul2(float2 a, float b)
        {
            float2 r;
            asm("{ .reg .b64 t, u;\n"
                "mov.b64 t, {%2, %3};\n"
                "mov.b64 u, {%4, %4};\n"
                "mul.rn.f32x2 t, t, u;\n"
                "mov.b64 {%0, %1}, t; }"
                : "=f"(r.x), "=f"(r.y)
                : "f"(a.x), "f"(a.y), "f"(b));
            return r;
        }
        __device__ __forceinline__ float2 add2(float2 a, float2 b)
        {
            float2 r;
            asm("{ .reg .b64 t, u;\n"
                "mov.b64 t, {%2, %3};\n"
                "mov.b64 u, {%4, %5};\n"
                "add.rn.f32x2 t, t, u;\n"
                "mov.b64 {%0, %1}, t; }"
                : "=f"(r.x), "=f"(r.y)
                : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
            return r;
        }

        // a b + c for two values at once, to nearest and cut
        __device__ __forceinline__ float2 fma2(float2 a, float b, float2 c)
        {
            float2 r;
            asm("{ .reg .b64 t, u, v;\n"
                "mov.b64 t, {%2, %3};\n"
                "mov.b64 u, {%4, %4};\n"
                "mov.b64 v, {%5, %6};\n"
                "fma.rn.f32x2 t, t, u, v;\n"
                "mov.b64 {%0, %1}, t; }"
                : "=f"(r.x), "=f"(r.y)
                : "f"(a.x), "f"(a.y), "f"(b), "f"(c.x), "f"(c.y));
            return r;
        }
        __device__ __forceinline__ float2 fma2_cut(float2 a, float b, float2 c)
        {
            float2 r;
            asm("{ .reg .b64 t, u, v;\n"
                "mov.b64 t, {%2, %3};\n"
                "mov.b64 u, {%4, %4};\n"
                "mov.b64 v, {%5, %6};\n"
                "fma.rz.f32x2 t, t, u, v;\n"
                "mov.b64 {%0, %1}, t; }"
                : "=f"(r.x), "=f"(r.y)
                : "f"(a.x), "f"(a.y), "f"(b), "f"(c.x), "f"(c.y));
            return r;
        }

        // What a group's values are divided with: minus the reciprocal of the scale, a little too small and a little too large (by three and
        // by four units of the last place of its nearest float).
        struct divisor
        {
            float scale, small, large;
            __device__ __forceinline__ explicit divisor(float s) : scale(s)
            {
                const uint32_t inverse = __float_as_uint(__frcp_rn(s));
                small                  = -__uint_as_float(inverse - 3);
                large                  = -__uint_as_float(inverse + 4);
            }
        };

        // -x / scale for two values, for rounding to a code.  The first guess t is not above the quotient q (in magnitude), eight units of
        // its last place below it at most.  The correction by its remainder, a little too large (2^-17 of those units at most), ends at q
        // or just above and is cut.  The last bit is set where the second remainder says that this is not q.
        // Why that rounds as q does: a middle M between two codes has at most eight bits, so the product of M and the scale has at most 32,
        // and x, unless it is that product, differs from it by 2^-32 of it or more; so q is M or at least 2^-9 units away from it, and
        // 2^-17 units do not carry it there.  Below M it is cut to the float below at most, which is odd; at M it is exact; above M it is
        // cut to M at least and made odd.  (Elsewhere it may end a unit above q: a quotient can lie 2^-24 units below a float.)
        // (Of this sign, the steps leave a zero's sign as it should be.)
        __device__ __forceinline__ float2 minus_quotient2(float2 x, const divisor& by)
        {
            const float2 t = mul2(x, by.small);
            const float2 y = fma2_cut(fma2(t, by.scale, x), by.large, t);
            const float2 r = fma2(y, by.scale, x);
            uint32_t a, b; // all ones where something was cut
            asm("set.ne.u32.f32 %0, %1, 0f00000000;" : "=r"(a) : "f"(r.x));
            asm("set.ne.u32.f32 %0, %1, 0f00000000;" : "=r"(b) : "f"(r.y));
            return make_float2(__uint_as_float(__float_as_uint(y.x) | (a & 1u)), __uint_as_float(__float_as_uint(y.y) | (b & 1u)));
        }

        // Codes of four finite values at once (in the order of the bytes); for int8 the values become the codes' numbers.
        template <int CODE>
        __device__ __forceinline__ uint32_t encode4(float2& a, float2& b, const divisor& by)
        {
            const float2 s = minus_quotient2(a, by), t = minus_quotient2(b, by);
            if (CODE == AEONB_CODE_INT8)
            {
                const float  magic = 12582912.0f; // 1.5 2^23: the difference's last bits are the nearest integer, the even one in the middle
                const float2 up = make_float2(magic, magic), down = make_float2(-magic, -magic);
                const float2 p = fma2(s, -1.0f, up), q = fma2(t, -1.0f, up);
                a = add2(p, down), b = add2(q, down);
                const uint32_t lo = __byte_perm(__float_as_uint(p.x), __float_as_uint(p.y), 0x0040),
                               hi = __byte_perm(__float_as_uint(q.x), __float_as_uint(q.y), 0x0040);
                return __byte_perm(lo, hi, 0x5410);
            }
            const uint32_t lo = __nv_cvt_float2_to_fp8x2(s, __NV_SATFINITE, __NV_E4M3), hi = __nv_cvt_float2_to_fp8x2(t, __NV_SATFINITE, __NV_E4M3);
            return (lo | hi << 16) ^ 0x80808080u;
        }

        // Whether one of four codes stands for no finite number.
        template <int CODE>
        __device__ __forceinline__ bool odd4(uint32_t w)
        {
            if (CODE == AEONB_CODE_INT8)
            {
                const uint32_t v = w ^ 0x80808080u; // a byte of 0?
                return ((v - 0x01010101u) & ~v & 0x80808080u) != 0;
            }
            return (((w & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) != 0;
        }

        // The numbers (not yet scaled) of four codes, all of them finite.
        template <int CODE>
        __device__ __forceinline__ void numbers4(uint32_t w, float2& a, float2& b)
        {
            if (CODE == AEONB_CODE_INT8)
            {
                w ^= 0x80808080u; // code + 128, as the last byte of 2^23 + code + 128
                const float2 bias = make_float2(-8388736.0f, -8388736.0f);
                a = add2(make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7540)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7541))), bias);
                b = add2(make_float2(__uint_as_float(__byte_perm(w, 0x4b000000u, 0x7542)), __uint_as_float(__byte_perm(w, 0x4b000000u, 0x7543))), bias);
                return;
            }
            a = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w & 0xffffu), __NV_E4M3)));
            b = __half22float2(__half2(__nv_cvt_fp8x2_to_halfraw2((__nv_fp8x2_storage_t)(w >> 16), __NV_E4M3)));
        }

        // V values of a row in one lane's registers, and how they and their codes get there and away.  `step` and `left` are for values apart:
        // how far they lie from one another, and how many of the group's come from the chunk's first one on.
        template <typename T, int V>
        struct chunk
        {
            static constexpr int  N = V, W = V * sizeof(T) / 4; // values, words
            static constexpr bool WIDE = sizeof(T) == 4;
            uint32_t              w[W];
            // where lane l of L finds its chunk j
            __device__ __forceinline__ static int place(int j, int l, int L) { return (j * L + l) * V; }
            __device__ __forceinline__ void load(const T* p, int, int)
            {
                if constexpr (W == 8)
                    asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                                 : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                                 : "l"(p)
                                 : "memory");
                else
                {
                    const uint4 q = *reinterpret_cast<const uint4*>(p);
                    w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
                }
            }
            __device__ __forceinline__ void store(T* p, int, int) const
            {
                if constexpr (W == 8)
                    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(p), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]),
                                 "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                                 : "memory");
                else
                    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
            }
            __device__ __forceinline__ void fill(float v)
            {
                const T one = from_float<T>(v);
                uint32_t bits;
                if constexpr (WIDE)
                    bits = *reinterpret_cast<const uint32_t*>(&one);
                else
                    bits = *reinterpret_cast<const uint16_t*>(&one) * 0x10001u;
#pragma unroll
                for (int i = 0; i < W; ++i)
                    w[i] = bits;
            }
            __device__ __forceinline__ float2 pair(int i) const
            {
                if constexpr (WIDE)
                    return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
                else if constexpr (std::is_same<T, __half>::value)
                    return __half22float2(*reinterpret_cast<const __half2*>(&w[i]));
                else
                    return make_float2(__uint_as_float(w[i] << 16), __uint_as_float(w[i] & 0xffff0000u));
            }
            __device__ __forceinline__ void set(int i, float2 v)
            {
                if constexpr (WIDE)
                    w[2 * i] = __float_as_uint(v.x), w[2 * i + 1] = __float_as_uint(v.y);
                else if constexpr (std::is_same<T, __half>::value)
                {
                    const __half2 h = __floats2half2_rn(v.x, v.y);
                    w[i]            = *reinterpret_cast<const uint32_t*>(&h);
                }
                else
                {
                    const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
                    w[i]                   = *reinterpret_cast<const uint32_t*>(&h);
                }
            }
            // bits of the largest magnitude as a float's, infinities and NaN among them
            __device__ __forceinline__ uint32_t largest() const
            {
                if constexpr (WIDE)
                {
                    uint32_t m = 0;
#pragma unroll
                    for (int i = 0; i < W; ++i)
                        m = max(m, w[i] & ABS_BITS);
                    return m;
                }
                else
                {
                    // (NaN stays; no sign, so the larger float has the larger bits)
                    if constexpr (std::is_same<T, __half>::value)
                    {
                        __half2 m = __habs2(*reinterpret_cast<const __half2*>(&w[0]));
#pragma unroll
                        for (int i = 1; i < W; ++i)
                            m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __half2*>(&w[i])));
                        const float2 v = __half22float2(m);
                        return max(__float_as_uint(v.x) & ABS_BITS, __float_as_uint(v.y) & ABS_BITS);
                    }
                    else
                    {
                        __nv_bfloat162 m = __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[0]));
#pragma unroll
                        for (int i = 1; i < W; ++i)
                            m = __hmax2_nan(m, __habs2(*reinterpret_cast<const __nv_bfloat162*>(&w[i])));
                        const uint32_t bits = *reinterpret_cast<const uint32_t*>(&m);
                        return max(bits << 16 & ABS_BITS, bits & 0x7fff0000u);
                    }
                }
            }
            __device__ __forceinline__ float value(int i) const
            {
                const float2 v = pair(i / 2);
                return i & 1 ? v.y : v.x;
            }
        };

        // Four values apart: rows that lie on no 16 bytes.
        constexpr int APART = -4;
        template <typename T>
        struct chunk<T, APART>
        {
            static constexpr int N = 4;
            float                v[4];
            __device__ __forceinline__ static int place(int j, int l, int L) { return j * 4 * L + l; }
            __device__ __forceinline__ void       load(const T* p, int step, int left)
            {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    v[i] = i * step < left ? to_float(p[i * step]) : 0.0f;
            }
            __device__ __forceinline__ void store(T* p, int step, int left) const
            {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    if (i * step < left)
                        p[i * step] = from_float<T>(v[i]);
            }
            __device__ __forceinline__ void     fill(float x) { v[0] = v[1] = v[2] = v[3] = x; }
            __device__ __forceinline__ float2   pair(int i) const { return make_float2(v[2 * i], v[2 * i + 1]); }
            __device__ __forceinline__ void     set(int i, float2 x) { v[2 * i] = x.x, v[2 * i + 1] = x.y; }
            __device__ __forceinline__ float    value(int i) const { return v[i]; }
            __device__ __forceinline__ uint32_t largest() const
            {
                return max(max(__float_as_uint(v[0]) & ABS_BITS, __float_as_uint(v[1]) & ABS_BITS),
                           max(__float_as_uint(v[2]) & ABS_BITS, __float_as_uint(v[3]) & ABS_BITS));
            }
        };

        // The codes of a chunk.
        template <int V>
        struct code_words
        {
            static constexpr int N = V == APART ? 4 : V;
            uint32_t             w[N / 4];
            __device__ __forceinline__ void load(const uint8_t* q, int step, int left)
            {
                if constexpr (V == 16)
                {
                    const uint4 u = __ldcs(reinterpret_cast<const uint4*>(q));
                    w[0] = u.x, w[1] = u.y, w[2] = u.z, w[3] = u.w;
                }
                else if constexpr (V == 8)
                {
                    const uint2 u = __ldcs(reinterpret_cast<const uint2*>(q));
                    w[0] = u.x, w[1] = u.y;
                }
                else if constexpr (V == 4)
                    w[0] = __ldcs(reinterpret_cast<const uint32_t*>(q));
                else
                {
                    uint32_t b[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        b[i] = i * step < left ? q[i * step] : 0;
                    w[0] = b[0] | b[1] << 8 | b[2] << 16 | b[3] << 24;
                }
            }
            __device__ __forceinline__ void store(uint8_t* q, int step, int left) const
            {
                if constexpr (V == 16)
                    *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
                else if constexpr (V == 8)
                    *reinterpret_cast<uint2*>(q) = make_uint2(w[0], w[1]);
                else if constexpr (V == 4)
                    *reinterpret_cast<uint32_t*>(q) = w[0];
                else
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (i * step < left)
                            q[i * step] = (uint8_t)(w[0] >> (8 * i));
            }
        };

        // The largest magnitude among a group's lanes, L of them from lane `base` on (any L: the largest of some values does not
        // mind which of them it has seen twice).
        template <int LANES>
        __device__ __forceinline__ uint32_t group_largest(uint32_t m, int L, int base, int l)
        {
            if constexpr (LANES > 0 && LANES < 32)
            {
#pragma unroll
                for (int o = LANES / 2; o > 0; o >>= 1)
                    m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
                return m;
            }
            if (L == 32)
                return __reduce_max_sync(0xffffffffu, m);
            for (int o = 1; o < L; o *= 2)
            {
                int from = l + o;
                from     = from >= L ? from - L : from;
                m        = max(m, __shfl_sync(0xffffffffu, m, base + from));
            }
            return m;
        }

        template <typename T, int CODE, int V>
        __device__ __forceinline__ void decode_chunk(chunk<T, V>& x, const code_words<V>& q, float scale)
        {
            bool odd = false;
#pragma unroll
            for (int i = 0; i < chunk<T, V>::N / 4; ++i)
            {
                float2 a, b;
                odd |= odd4<CODE>(q.w[i]);
                numbers4<CODE>(q.w[i], a, b);
                x.set(2 * i, mul2(a, scale));
                x.set(2 * i + 1, mul2(b, scale));
            }
            if (odd)
#pragma unroll
                for (int i = 0; i < chunk<T, V>::N / 4; ++i)
                {
                    x.set(2 * i, make_float2(decode<CODE>(q.w[i] & 0xff, scale), decode<CODE>(q.w[i] >> 8 & 0xff, scale)));
                    x.set(2 * i + 1, make_float2(decode<CODE>(q.w[i] >> 16 & 0xff, scale), decode<CODE>(q.w[i] >> 24, scale)));
                }
        }

        // Codes of a chunk of finite values, whose group has a scale so large that no remainder is lost below the smallest float (or nothing
        // but zeros); with `values` the chunk then holds the values that they stand for.
        template <typename T, int CODE, int V>
        __device__ __forceinline__ void encode_chunk(chunk<T, V>& x, code_words<V>& q, const divisor& by, bool values)
        {
#pragma unroll
            for (int i = 0; i < chunk<T, V>::N / 4; ++i)
            {
                float2 a = x.pair(2 * i), b = x.pair(2 * i + 1);
                q.w[i] = encode4<CODE>(a, b, by);
                if (values)
                {
                    if (CODE != AEONB_CODE_INT8)
                        numbers4<CODE>(q.w[i], a, b);
                    x.set(2 * i, mul2(a, by.scale));
                    x.set(2 * i + 1, mul2(b, by.scale));
                }
            }
        }

        // Any chunk: of a group with -infinities, or without a scale, or with one that small.
        template <typename T, int CODE, int V>
        __device__ __forceinline__ void encode_any_chunk(chunk<T, V>& x, code_words<V>& q, const divisor& by, bool tame)
        {
            constexpr int N    = chunk<T, V>::N;
            uint32_t      gone = 0; // a bit for each -infinity, which counts as 0 meanwhile
#pragma unroll
            for (int i = 0; i < N / 2; ++i)
            {
                const float2 v = x.pair(i);
                const bool   a = __float_as_uint(v.x) == MINUS_INF, b = __float_as_uint(v.y) == MINUS_INF;
                gone |= (a ? 1u : 0u) << (2 * i) | (b ? 2u : 0u) << (2 * i);
                x.set(i, make_float2(a ? 0.0f : v.x, b ? 0.0f : v.y));
            }
            if (tame)
                encode_chunk<T, CODE, V>(x, q, by, false);
            else
#pragma unroll
                for (int i = 0; i < N / 4; ++i)
                {
                    const float2 a = x.pair(2 * i), b = x.pair(2 * i + 1);
                    q.w[i] = encode_exactly<CODE>(a.x, by.scale) | encode_exactly<CODE>(a.y, by.scale) << 8 |
                             encode_exactly<CODE>(b.x, by.scale) << 16 | encode_exactly<CODE>(b.y, by.scale) << 24;
                }
            if (by.scale == by.scale)
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (gone >> i & 1)
                        q.w[i / 4] = (q.w[i / 4] & ~(0xffu << (8 * (i & 3)))) | (CODE == AEONB_CODE_INT8 ? 0x80u : 0xffu) << (8 * (i & 3));
            decode_chunk<T, CODE, V>(x, q, by.scale);
        }

        // Where a lane finds its group: 32 / L.lanes groups in a warp.  LANES: L.lanes where that is known when compiled, else 0.
        template <int LANES>
        struct spot
        {
            int  l, base, group, block_group; // lane of the group, its first lane, its number and that of the block's first one
            bool used;
            __device__ __forceinline__ explicit spot(const cache_launch& L)
            {
                const int lane = threadIdx.x & 31, at_once = LANES ? 32 / LANES : (int)L.by_lanes(32);
                const int mine = LANES ? lane / LANES : (int)L.by_lanes((uint32_t)lane);
                base        = mine * (LANES ? LANES : L.lanes);
                l           = lane - base;
                used        = LANES || mine < at_once;
                block_group = (int)(blockIdx.x * (blockDim.x / 32)) * at_once;
                group       = block_group + (int)(threadIdx.x / 32) * at_once + mine;
            }
        };

        template <typename T>
        __device__ __forceinline__ T* group_rows(void* p, int seq, int token, int head, int64_t by_seq, int64_t by_token, int64_t by_head)
        {
            return static_cast<T*>(p) + times(seq, by_seq) + times(token, by_token) + times(head, by_head);
        }

        // NC chunks a lane; NC = 0: as many as it takes, read a second time for their codes.
        template <typename T, int CODE, int V, int NC, int LANES>
        __global__ void __launch_bounds__(256, 4) cache_write_kernel(const cache_launch L)
        {
            typedef chunk<T, V>     C;
            const aeonb_cache_desc& d = L.d;
            const spot<LANES>       at(L);
            const int               lanes = LANES ? LANES : L.lanes;
            const int               token = (int)L.by_heads((uint32_t)at.group), head = at.group - token * d.heads;
            for (int seq = blockIdx.y; seq < d.seqs; seq += gridDim.y)
            {
                const int tokens = tokens_of(d, seq);
                if ((int)L.by_heads((uint32_t)at.block_group) >= tokens)
                    continue; // the block's first token lies behind the sequence
                const bool there = at.used && at.group < L.groups && token < tokens;
                const T*   x     = group_rows<T>(d.rows, seq, token, head, d.row_stride_seq, d.row_stride_token, d.row_stride_head);
                C          c[NC ? NC : 1];
                if constexpr (NC > 0)
                    if (there)
                    {
#pragma unroll
                        for (int j = 0; j < NC; ++j)
                            if (const int i = C::place(j, at.l, lanes); i < d.dim)
                                c[j].load(x + i, lanes, d.dim - i);
                    }
                const int64_t place = there ? group_place(L, seq, token, head) : -1;
                if (there && place < 0 && at.l == 0 && d.status)
                    *d.status = 1;
                uint32_t m = 0;
                if (place >= 0)
                {
                    if constexpr (NC > 0)
                    {
#pragma unroll
                        for (int j = 0; j < NC; ++j)
                            if (C::place(j, at.l, lanes) < d.dim)
                                m = max(m, c[j].largest());
                    }
                    else
                        for (int j = 0, i; (i = C::place(j, at.l, lanes)) < d.dim; ++j)
                        {
                            c[0].load(x + i, lanes, d.dim - i);
                            m = max(m, c[0].largest());
                        }
                }
                m                 = group_largest<LANES>(m, lanes, at.base, at.l);
                const bool finite = m < INF_BITS;
                if (__any_sync(0xffffffffu, !finite))
                {
                    // an infinity or NaN somewhere in the warp: the largest without -infinity
                    uint32_t   n   = 0;
                    const auto see = [&](float v) {
                        if (__float_as_uint(v) != MINUS_INF)
                            n = max(n, __float_as_uint(v) & ABS_BITS);
                    };
                    if (place >= 0)
                    {
                        if constexpr (NC > 0)
                        {
#pragma unroll
                            for (int j = 0; j < NC; ++j)
                                if (C::place(j, at.l, lanes) < d.dim)
#pragma unroll
                                    for (int i = 0; i < C::N; ++i)
                                        see(c[j].value(i));
                        }
                        else
                            for (int i = at.l; i < d.dim; i += lanes)
                                see(to_float(x[i]));
                    }
                    m = group_largest<LANES>(n, lanes, at.base, at.l);
                }
                if (place < 0)
                    continue;
                const float   scale = group_scale<CODE>(m);
                const divisor by(scale);
                const bool    tame = scale > 0x1p-90f || m == 0;
                if (at.l == 0)
                    d.scales[place] = scale;
                uint8_t*   codes = static_cast<uint8_t*>(d.codes) + times(d.dim, place);
                T*         v     = group_rows<T>(d.values, seq, token, head, d.value_stride_seq, d.value_stride_token, d.value_stride_head);
                const auto put   = [&](C& x, int i, bool usual) {
                    code_words<V> q;
                    if (usual)
                        encode_chunk<T, CODE, V>(x, q, by, d.values != nullptr);
                    else
                        encode_any_chunk<T, CODE, V>(x, q, by, tame);
                    q.store(codes + i, lanes, d.dim - i);
                    if (d.values)
                        x.store(v + i, lanes, d.dim - i);
                };
                if (finite && tame)
                {
                    if constexpr (NC > 0)
                    {
#pragma unroll
                        for (int j = 0; j < NC; ++j)
                            if (const int i = C::place(j, at.l, lanes); i < d.dim)
                                put(c[j], i, true);
                    }
                    else
                        for (int j = 0, i; (i = C::place(j, at.l, lanes)) < d.dim; ++j)
                        {
                            c[0].load(x + i, lanes, d.dim - i);
                            put(c[0], i, true);
                        }
                }
                else if constexpr (NC > 0)
                {
#pragma unroll
                    for (int j = 0; j < NC; ++j)
                        if (const int i = C::place(j, at.l, lanes); i < d.dim)
                            put(c[j], i, false);
                }
                else
                    for (int j = 0, i; (i = C::place(j, at.l, lanes)) < d.dim; ++j)
                    {
                        c[0].load(x + i, lanes, d.dim - i);
                        put(c[0], i, false);
                    }
            }
        }

        template <typename T, int CODE, int V, int NC, int LANES>
        __global__ void __launch_bounds__(256) cache_read_kernel(const cache_launch L)
        {
            typedef chunk<T, V>     C;
            const aeonb_cache_desc& d = L.d;
            const spot<LANES>       at(L);
            const int               lanes = LANES ? LANES : L.lanes;
            if (!at.used || at.group >= L.groups)
                return;
            const int token = (int)L.by_heads((uint32_t)at.group), head = at.group - token * d.heads;
            for (int seq = blockIdx.y; seq < d.seqs; seq += gridDim.y)
            {
                T*            v = group_rows<T>(d.rows, seq, token, head, d.row_stride_seq, d.row_stride_token, d.row_stride_head);
                code_words<V> q[NC ? NC : 1];
                int64_t       place = -1;
                float         scale = 0.0f; // of the group, or what it is filled with
                if (token < tokens_of(d, seq))
                {
                    place = group_place(L, seq, token, head);
                    scale = __uint_as_float(0x7fffffffu);
                    if (place < 0 && at.l == 0 && d.status)
                        *d.status = 1;
                }
                const uint8_t* codes = static_cast<const uint8_t*>(d.codes) + times(d.dim, place);
                if (place >= 0)
                {
                    scale = d.scales[place];
                    if constexpr (NC > 0)
                    {
#pragma unroll
                        for (int j = 0; j < NC; ++j)
                            if (const int i = C::place(j, at.l, lanes); i < d.dim)
                                q[j].load(codes + i, lanes, d.dim - i);
                    }
                }
                const auto put = [&](const code_words<V>& q, int i) {
                    C c;
                    if (place < 0)
                        c.fill(scale);
                    else
                        decode_chunk<T, CODE, V>(c, q, scale);
                    c.store(v + i, lanes, d.dim - i);
                };
                if constexpr (NC > 0)
                {
#pragma unroll
                    for (int j = 0; j < NC; ++j)
                        if (const int i = C::place(j, at.l, lanes); i < d.dim)
                            put(q[j], i);
                }
                else
                    for (int j = 0, i; (i = C::place(j, at.l, lanes)) < d.dim; ++j)
                    {
                        if (place >= 0)
                            q[0].load(codes + i, lanes, d.dim - i);
                        put(q[0], i);
                    }
            }
        }

        void check_cache(const aeonb_cache_desc& d, bool write)
        {
            const int e = float_size(d.dtype);
            if (d.code != AEONB_CODE_INT8 && d.code != AEONB_CODE_E4M3)
                throw std::invalid_argument("the code of a cache must be AEONB_CODE_INT8 or AEONB_CODE_E4M3");
            if (d.page_tokens <= 0 || d.heads <= 0 || d.dim <= 0 || d.pages < 0)
                throw std::invalid_argument("a cache needs page_tokens, heads and dim above 0");
            // lanes go through a group in steps of up to 512 values, in 32 bits: the step behind the last value has to fit as well
            if (d.dim > MAX_DIM)
                throw std::invalid_argument("the dim of a cache is at most 2^31 - 1024");
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

        template <typename T, int CODE, int V, int NC, int LANES = 0>
        void launch_lanes(cache_launch& L, bool write, cudaStream_t stream)
        {
            const int chunks  = (L.d.dim + chunk<T, V>::N - 1) / chunk<T, V>::N;
            L.lanes           = LANES ? LANES : NC ? (chunks + NC - 1) / NC : 32;
            L.by_lanes        = fast_divisor(L.lanes);
            const int at_once = 32 / L.lanes;
            const int warps   = (int)std::min<int64_t>(8, ((int64_t)L.groups + at_once - 1) / at_once);
            const int each    = warps * at_once;
            const dim3 grid((unsigned)(((int64_t)L.groups + each - 1) / each), (unsigned)std::min(L.d.seqs, 65535));
            if (write)
                cache_write_kernel<T, CODE, V, NC, LANES><<<grid, warps * 32, 0, stream>>>(L);
            else
                cache_read_kernel<T, CODE, V, NC, LANES><<<grid, warps * 32, 0, stream>>>(L);
        }

        // Values apart: lanes known when compiled, so that a lane's values lie at fixed distances, and few slots without a value.  2560 x 200
        // groups of 161 floats, lanes known when run / when compiled: written in 0.24 / 0.18 ms, read in 0.13 / 0.11; 64 x 1024 of 4100
        // bf16 written in 0.65 / 0.47.
        template <typename T, int CODE>
        void launch_apart(cache_launch& L, bool write, cudaStream_t stream)
        {
            const int dim = L.d.dim;
            if (dim <= 2 * 8)
                launch_lanes<T, CODE, APART, 2, 2>(L, write, stream);
            else if (dim <= 4 * 8)
                launch_lanes<T, CODE, APART, 2, 4>(L, write, stream);
            else if (dim <= 8 * 8)
                launch_lanes<T, CODE, APART, 2, 8>(L, write, stream);
            else if (dim <= 8 * 12)
                launch_lanes<T, CODE, APART, 3, 8>(L, write, stream);
            else if (dim <= 16 * 8)
                launch_lanes<T, CODE, APART, 2, 16>(L, write, stream);
            else if (dim <= 16 * 12)
                launch_lanes<T, CODE, APART, 3, 16>(L, write, stream);
            else if (dim <= 16 * 16)
                launch_lanes<T, CODE, APART, 4, 16>(L, write, stream);
            else if (dim <= 32 * 12)
                launch_lanes<T, CODE, APART, 3, 32>(L, write, stream);
            else
                launch_lanes<T, CODE, APART, 0, 32>(L, write, stream);
        }

        template <typename T, int CODE, int V>
        void launch_chunks(cache_launch& L, bool write, cudaStream_t stream)
        {
            const int chunks = L.d.dim / V;
            // Four chunks a lane where that leaves a thousand lanes to an SM, else two: what a lane finds out about its group serves them all.
            // 64 x 4096 x 8 groups of 128 bf16 with values, two / four: to e4m3 0.24 / 0.23 ms, to int8 0.24 / 0.22, read back
            // 0.13 / 0.13; 2560 x 2000 groups of 40 floats to int8 0.37 / 0.35, read back 0.20 / 0.18; 256 x 200 of them, half there,
            // 10.3 / 12.3 us.
            const bool many = (int64_t)L.d.seqs * L.groups * chunks / 4 >= 148 * 1024;
            if (chunks <= 32 * 2 && !(many && chunks >= 4))
                launch_lanes<T, CODE, V, 2>(L, write, stream);
            else if (chunks <= 32 * 4)
            {
                // (the usual sizes with the lanes known when compiled)
                if constexpr (V * sizeof(T) == 32)
                    switch (chunks)
                    {
                    case 4: return launch_lanes<T, CODE, V, 4, 1>(L, write, stream);
                    case 8: return launch_lanes<T, CODE, V, 4, 2>(L, write, stream);
                    case 16: return launch_lanes<T, CODE, V, 4, 4>(L, write, stream);
                    case 32: return launch_lanes<T, CODE, V, 4, 8>(L, write, stream);
                    }
                launch_lanes<T, CODE, V, 4>(L, write, stream);
            }
            else
                launch_lanes<T, CODE, V, 0>(L, write, stream);
        }

        // bytes that every group's first value lies on
        template <typename T>
        int rows_lie_on(const aeonb_cache_desc& d, bool write)
        {
            uintptr_t all = (uintptr_t)d.rows | (uintptr_t)d.dim * sizeof(T);
            if (d.seqs > 1)
                all |= (uintptr_t)d.row_stride_seq * sizeof(T);
            if (d.tokens > 1)
                all |= (uintptr_t)d.row_stride_token * sizeof(T);
            if (d.heads > 1)
                all |= (uintptr_t)d.row_stride_head * sizeof(T);
            if (write && d.values)
            {
                all |= (uintptr_t)d.values;
                if (d.seqs > 1)
                    all |= (uintptr_t)d.value_stride_seq * sizeof(T);
                if (d.tokens > 1)
                    all |= (uintptr_t)d.value_stride_token * sizeof(T);
                if (d.heads > 1)
                    all |= (uintptr_t)d.value_stride_head * sizeof(T);
            }
            // the codes of a chunk lie on as many bytes as it has values
            const uintptr_t codes = ((uintptr_t)d.codes | (uintptr_t)d.dim);
            if (all % 32 == 0 && codes % (32 / sizeof(T)) == 0)
                return 32;
            return all % 16 == 0 && codes % (16 / sizeof(T)) == 0 ? 16 : 1;
        }

        template <typename T, int CODE>
        void launch_code(cache_launch& L, bool write, cudaStream_t stream)
        {
            switch (rows_lie_on<T>(L.d, write))
            {
            case 32: launch_chunks<T, CODE, 32 / sizeof(T)>(L, write, stream); break;
            case 16: launch_chunks<T, CODE, 16 / sizeof(T)>(L, write, stream); break;
            default: launch_apart<T, CODE>(L, write, stream); break;
            }
        }

        template <typename T>
        void launch_cache(cache_launch& L, bool write, cudaStream_t stream)
        {
            L.d.code == AEONB_CODE_INT8 ? launch_code<T, AEONB_CODE_INT8>(L, write, stream) : launch_code<T, AEONB_CODE_E4M3>(L, write, stream);
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
                if ((int64_t)d.tokens * d.heads > 0x7ffff000)
                    throw error(AEONB_ERR_UNSUPPORTED, "more tokens and heads of a sequence than a launch takes");
                device_scope   scope(ctx->device);
                cache_launch   L{};
                L.d        = d;
                L.groups   = d.tokens * d.heads;
                L.by_heads = fast_divisor(d.heads);
                L.by_page  = fast_divisor(d.page_tokens);
                L.positions      = (int64_t)d.table_pages * d.page_tokens;
                L.by_page_groups = (int64_t)d.page_tokens * d.heads;
                const int64_t  groups = (int64_t)d.seqs * d.tokens * d.heads;
                const int64_t  values = groups * d.dim;
                const cudaStream_t stream = d.stream ? static_cast<cudaStream_t>(d.stream) : ctx->stream;
                launch_timer   timer(ctx, AEONB_KERNEL_OTHER, values * (float_size(d.dtype) * (d.values && write ? 2 : 1) + 1) + groups * 4, stream);
                switch (d.dtype)
                {
                case AEONB_F32: launch_cache<float>(L, write, stream); break;
                case AEONB_F16: launch_cache<__half>(L, write, stream); break;
                case AEONB_BF16: launch_cache<__nv_bfloat16>(L, write, stream); break;
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
