// Distillation from a teacher's top logits on sm_100a: the loss of each row, its log-sum-exp, and the gradient.
//
// A row's logits are read from memory once: the largest value and the sum of exponentials against it (to the base 2, with log2(e) / T as a
// factor of the difference, so that rows at the ends of the type's range do not overflow), then the gradient, which is written while
// the row is still on the chip.  Floor: the bytes of the row in, and out with the gradient.  Sums and exponentials are held in 32
// bits, sums of a thread's thousands of terms in 64; an exponential below 2^-126 of the row's largest counts as 0 (no type of the gradient keeps such a share of the sum).
//   * up to 128 values, or up to 256 vectors of 16 bytes, with up to 32 entries: 8, 16 or 32 lanes per row (distill_few_kernel; with
//     more entries distill_warp_kernel, a warp per row);
//   * longer: one to sixteen blocks of a cluster per row, persistent, the row in shared memory (distill_block_kernel);
//   * beyond what sixteen blocks hold (2^16 vectors), the loss: a block per row that reads it twice (distill_kernel).
// Vectors are whole ones that lie on 16 bytes; the up to seven values before the first and behind the last are a thread's each.
// The teacher's probabilities are formed while the row is on its way.  The entries' own part of the gradient is written behind a
// barrier, for each id by the first entry that has it, with the probabilities of all entries of that id added in their order: no
// atomics, the same bits every time.
//
// Measured on B200, 6.55 TB/s being what a copy reaches (events around a call, inputs not in L2): 8192 rows of 131072 bf16 logits with 64
// entries: with gradient 0.84 ms (5.1 TB/s), gradient alone 0.68 (6.3), loss alone 0.45 (4.8); 65536 rows of 16384: 0.75 (5.7), 0.74
// (5.8), 0.39 (5.5); 32768 rows of 16384 floats with gradient 0.69 (6.2); 131072 rows of 4096 bf16 0.41 (5.2), 65536 of 500 57 us (2.3);
// with 100 entries, which one warp of a block reads, 60000 rows of 3001 0.43 (1.7).  Above 131072 values blocks have 512 threads: 4096
// rows of 151936 with 20 entries and gradient 0.64 (3.9), 2048 of 256000 0.44 (4.7).
// Rows of 16-bit values wait for the issue of instructions and, where a row takes several blocks, for the other blocks' sums.
#include <algorithm>
#include <atomic>
#include <cmath>
#include <type_traits>

#include "float_rows.cuh"

namespace aeonb
{
    namespace
    {
        constexpr int   THREADS = 256; // of distill_kernel
        constexpr int   ENTRIES = AEONB_DISTILL_MAX_ENTRIES;
        constexpr int   BLOCK_VECTORS = 8; // vectors of 16 bytes that a thread of distill_block_kernel keeps
        constexpr float LN2     = 0.693147180559945309417f;

        enum distill_mode
        {
            LOSS,      // loss and lse
            LOSS_GRAD, // and the gradient
            GRAD       // the gradient from the lse
        };

        struct distill_launch
        {
            aeonb_distill_desc d;
            float              c;       // log2(e) / T
            float              factor;  // T grad_scale
            float              tt;      // T^2
            int                blocks;  // of a row
            int                vectors; // of a row's slice, for each of its blocks
            bool               together; // the gradient's rows lie in their 16 bytes as the logits' do
        };

        // 2^x; results below 2^-126 are 0 (a share of the sum that no type of the gradient holds to a useful precision)
        __device__ __forceinline__ float pow2(float x)
        {
            float r;
            asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
            return r;
        }

        struct add
        {
            __device__ float operator()(float a, float b) const { return __fadd_rn(a, b); }
        };
        struct add_wide
        {
            __device__ double operator()(double a, double b) const { return a + b; }
        };
        struct larger // a NaN only where both are
        {
            __device__ float operator()(float a, float b) const { return fmaxf(a, b); }
        };

        template <typename V, typename Op>
        __device__ __forceinline__ V warp_reduce(V v, Op op)
        {
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
                v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
            return v;
        }

        // The largest value of a warp, a NaN only where all are (as fmaxf), in one instruction.
        __device__ __forceinline__ float warp_reduce(float v, larger)
        {
            float r;
            asm volatile("redux.sync.max.f32 %0, %1, 0xffffffff;" : "=f"(r) : "f"(v));
            return r;
        }

        template <typename V, typename Op>
        __device__ __forceinline__ V block_reduce(V v, V* shared, Op op)
        {
            v = warp_reduce(v, op);
            __syncthreads();
            if ((threadIdx.x & 31) == 0)
                shared[threadIdx.x / 32] = v;
            __syncthreads();
            V r = shared[0];
            for (int i = 1; i < (int)blockDim.x / 32; ++i)
                r = op(r, shared[i]);
            return r;
        }

        // (x - m) c for two values at once
        __device__ __forceinline__ float2 scaled_difference(float2 x, float2 minus_m, float2 c)
        {
            float2 r;
            asm("{ .reg .b64 t, u;\n"
                "mov.b64 t, {%2, %3};\n"
                "mov.b64 u, {%4, %5};\n"
                "add.rn.f32x2 t, t, u;\n"
                "mov.b64 u, {%6, %7};\n"
                "mul.rn.f32x2 t, t, u;\n"
                "mov.b64 {%0, %1}, t; }"
                : "=f"(r.x), "=f"(r.y)
                : "f"(x.x), "f"(x.y), "f"(minus_m.x), "f"(minus_m.y), "f"(c.x), "f"(c.y));
            return r;
        }
        __device__ __forceinline__ float2 mul2(float2 a, float2 b)
        {
            float2 r;
            asm("{ .reg .b64 t, u;\n"
                "mov.b64 t, {%2, %3};\n"
                "mov.b64 u, {%4, %5};\n"
                "mul.rn.f32x2 t, t, u;\n"
                "mov.b64 {%0, %1}, t; }"
                : "=f"(r.x), "=f"(r.y)
                : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
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

        __device__ __forceinline__ float2 unpack(uint32_t w, __half)
        {
            return __half22float2(*reinterpret_cast<const __half2*>(&w));
        }
        __device__ __forceinline__ float2 unpack(uint32_t w, __nv_bfloat16)
        {
            return make_float2(__uint_as_float(w << 16), __uint_as_float(w & 0xffff0000u));
        }
        __device__ __forceinline__ uint32_t pack(float2 v, __half)
        {
            const __half2 h = __floats2half2_rn(v.x, v.y);
            return *reinterpret_cast<const uint32_t*>(&h);
        }
        __device__ __forceinline__ uint32_t pack(float2 v, __nv_bfloat16)
        {
            const __nv_bfloat162 h = __floats2bfloat162_rn(v.x, v.y);
            return *reinterpret_cast<const uint32_t*>(&h);
        }
        __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, __half)
        {
            const __half2 h = __hmax2(*reinterpret_cast<const __half2*>(&a), *reinterpret_cast<const __half2*>(&b));
            return *reinterpret_cast<const uint32_t*>(&h);
        }
        __device__ __forceinline__ uint32_t max2(uint32_t a, uint32_t b, __nv_bfloat16)
        {
            const __nv_bfloat162 h = __hmax2(*reinterpret_cast<const __nv_bfloat162*>(&a), *reinterpret_cast<const __nv_bfloat162*>(&b));
            return *reinterpret_cast<const uint32_t*>(&h);
        }

        // Sixteen bytes of a row.
        template <typename T>
        struct piece
        {
            static constexpr int  N    = 16 / sizeof(T);
            static constexpr bool WIDE = sizeof(T) == 4;
            uint32_t              w[4];
            __device__ __forceinline__ void load(const T* p)
            {
                const uint4 q = __ldcs(reinterpret_cast<const uint4*>(p));
                w[0] = q.x, w[1] = q.y, w[2] = q.z, w[3] = q.w;
            }
            __device__ __forceinline__ void clear() // -infinity
            {
#pragma unroll
                for (int i = 0; i < 4; ++i)
                    w[i] = WIDE ? 0xff800000u : std::is_same<T, __half>::value ? 0xfc00fc00u : 0xff80ff80u;
            }
            __device__ __forceinline__ float largest(float m) const
            {
                if constexpr (WIDE)
                    return fmaxf(fmaxf(m, fmaxf(__uint_as_float(w[0]), __uint_as_float(w[1]))), fmaxf(__uint_as_float(w[2]), __uint_as_float(w[3])));
                else
                {
                    const float2 v = unpack(max2(max2(w[0], w[1], T()), max2(w[2], w[3], T()), T()), T());
                    return fmaxf(m, fmaxf(v.x, v.y));
                }
            }
            __device__ __forceinline__ float2 pair(int i) const
            {
                if constexpr (WIDE)
                    return make_float2(__uint_as_float(w[2 * i]), __uint_as_float(w[2 * i + 1]));
                else
                    return unpack(w[i], T());
            }
            __device__ __forceinline__ float2 sum(float2 z, float m, float c) const
            {
#pragma unroll
                for (int i = 0; i < N / 2; ++i)
                {
                    const float2 x = scaled_difference(pair(i), make_float2(-m, -m), make_float2(c, c));
                    z              = add2(z, make_float2(pow2(x.x), pow2(x.y)));
                }
                return z;
            }
            __device__ __forceinline__ uint4 gradient(float m, float c, float f) const
            {
                uint32_t g[4];
#pragma unroll
                for (int i = 0; i < N / 2; ++i)
                {
                    const float2 x = scaled_difference(pair(i), make_float2(-m, -m), make_float2(c, c));
                    const float2 v = mul2(make_float2(pow2(x.x), pow2(x.y)), make_float2(f, f));
                    if constexpr (WIDE)
                        g[2 * i] = __float_as_uint(v.x), g[2 * i + 1] = __float_as_uint(v.y);
                    else
                        g[i] = pack(v, T());
                }
                return make_uint4(g[0], g[1], g[2], g[3]);
            }
        };

        // Writes a piece of the gradient, value by value where it does not lie on 16 bytes.
        template <typename T>
        __device__ __forceinline__ void store_piece(T* to, const uint4& q, bool whole)
        {
            if (whole)
            {
                __stcs(reinterpret_cast<uint4*>(to), q);
                return;
            }
            const uint32_t w[4] = {q.x, q.y, q.z, q.w};
#pragma unroll
            for (int i = 0; i < piece<T>::N; ++i)
                if constexpr (sizeof(T) == 4)
                    reinterpret_cast<uint32_t*>(to)[i] = w[i];
                else
                    reinterpret_cast<uint16_t*>(to)[i] = (uint16_t)(w[i / 2] >> (16 * (i & 1)));
        }

        // How a row lies in its 16-byte vectors: `head` values before the first whole one, `n` whole ones, `tail` values.
        template <typename T>
        struct cut
        {
            int head, n, tail;
            __device__ __forceinline__ cut(const T* s, int vocab)
            {
                head = min((int)((0u - (uint32_t)(uintptr_t)s) & 15u) / (int)sizeof(T), vocab);
                n    = (vocab - head) / piece<T>::N;
                tail = vocab - head - n * piece<T>::N;
            }
            // the value outside whole vectors that thread i takes (16 threads take one each), -1: none
            __device__ __forceinline__ int loose(int i, bool first, bool last) const
            {
                if (i < 8)
                    return first && i < head ? i : -1;
                return last && i - 8 < tail ? head + n * piece<T>::N + i - 8 : -1;
            }
        };

        __device__ __forceinline__ uint32_t shared_address(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }

        // ---- what the blocks of a cluster tell one another
        __device__ __forceinline__ void cluster_arrive() { asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory"); }
        __device__ __forceinline__ void cluster_wait() { asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory"); }
        // Sends v to the same place in another block's shared memory; that block's barrier (at the same place as this one's) counts the
        // eight bytes.  Unlike a store before the cluster's barrier it does not wait for the gradient's stores under way.
        __device__ __forceinline__ void cluster_send(float2* p, uint64_t* barrier, uint32_t rank, float2 v)
        {
            asm volatile("{ .reg .b32 to, at;\n"
                         "mapa.shared::cluster.u32 to, %0, %2;\n"
                         "mapa.shared::cluster.u32 at, %1, %2;\n"
                         "st.async.shared::cluster.mbarrier::complete_tx::bytes.v2.f32 [to], {%3, %4}, [at]; }" ::"r"(shared_address(p)),
                         "r"(shared_address(barrier)), "r"(rank), "f"(v.x), "f"(v.y)
                         : "memory");
        }
        __device__ __forceinline__ void barrier_init(uint64_t* barrier)
        {
            asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(shared_address(barrier)) : "memory");
        }
        __device__ __forceinline__ void barrier_expect(uint64_t* barrier, uint32_t bytes)
        {
            asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(shared_address(barrier)), "r"(bytes) : "memory");
        }
        // Waits until the barrier's phase of the given parity is complete; false when that takes beyond any reason (seconds).
        __device__ __forceinline__ bool barrier_wait(uint64_t* barrier, uint32_t parity)
        {
            for (int i = 0; i < 1 << 20; ++i)
            {
                uint32_t done;
                asm volatile("{ .reg .pred p;\n"
                             "mbarrier.try_wait.parity.acquire.cluster.shared::cta.b64 p, [%1], %2;\n"
                             "selp.u32 %0, 1, 0, p; }"
                             : "=r"(done)
                             : "r"(shared_address(barrier)), "r"(parity)
                             : "memory");
                if (done)
                    return true;
            }
            return false;
        }

        // The entries of a row, up to ROOM of them, in shared memory.
        template <int ROOM>
        struct entries
        {
            int   id[ROOM]; // -1: none
            float p[ROOM];  // teacher's probability
            float t[ROOM];  // (t - largest t) c
            float s[ROOM];  // the student's logit at id
        };

        // An entry: its id (-1 where it does not count) and the teacher's logit; true where the row is NaN for it.
        __device__ __forceinline__ bool read_entry(const aeonb_distill_desc& d, int64_t row, int k, int& id, float& t)
        {
            const float ninf = __uint_as_float(0xff800000u);
            id = d.ids[row * d.entry_stride + k];
            t  = d.teacher[row * d.entry_stride + k];
            if (id < 0 || t == ninf)
                id = -1, t = ninf;
            return id >= d.vocab || t != t;
        }

        // A warp reads a row's entries and forms their probabilities; returns the log2 of their sum.  found: whether there are any;
        // bad: an id outside the vocabulary, or teacher's logits without a finite largest one.
        template <typename T, int ROOM>
        __device__ __forceinline__ float read_entries(const distill_launch& L, int64_t row, const T* s, entries<ROOM>& e, bool& found, bool& bad)
        {
            const aeonb_distill_desc& d    = L.d;
            const int                 lane = threadIdx.x & 31;
            const float               ninf = __uint_as_float(0xff800000u);
            float                     top  = ninf;
            bool                      odd  = false;
            for (int k = lane; k < d.k; k += 32)
            {
                int   id;
                float t;
                odd |= read_entry(d, row, k, id, t);
                e.s[k]  = id >= 0 && id < d.vocab ? to_float(s[id]) : 0.0f;
                e.id[k] = id;
                e.t[k]  = t;
                top     = fmaxf(top, t);
            }
            top   = warp_reduce(top, larger());
            odd   = __any_sync(0xffffffffu, odd);
            found = odd || top != ninf;
            bad   = odd || !(top < __uint_as_float(0x7f800000u));
            float sum = 0.0f;
            for (int k = lane; k < d.k; k += 32)
            {
                const float t = __fmul_rn(__fsub_rn(e.t[k], top), L.c);
                const float p = e.id[k] >= 0 ? pow2(t) : 0.0f;
                e.t[k]        = t;
                e.p[k]        = p;
                sum           = __fadd_rn(sum, p);
            }
            sum = warp_reduce(sum, add());
            for (int k = lane; k < d.k; k += 32)
                e.p[k] = __fdiv_rn(e.p[k], sum);
            return log2f(sum);
        }

        // The loss of a row, by the warp that has read its entries.
        template <int ROOM>
        __device__ __forceinline__ float entries_loss(const distill_launch& L, const entries<ROOM>& e, float esum2, float top, float zsum2, float w)
        {
            float term = 0.0f; // p (log p - s / T + lse), to the base 2
            for (int k = threadIdx.x & 31; k < L.d.k; k += 32)
                if (e.p[k] > 0.0f)
                    term = __fadd_rn(term, __fmul_rn(e.p[k], __fadd_rn(__fsub_rn(e.t[k], esum2),
                                                                       __fadd_rn(zsum2, __fmul_rn(__fsub_rn(top, e.s[k]), L.c)))));
            return __fmul_rn(__fmul_rn(w, L.tt), __fmul_rn(warp_reduce(term, add()), LN2));
        }

        // The gradient at an entry's id, if it is the first entry that has it; the rest of the row has been written.
        template <typename T>
        __device__ __forceinline__ void entry_gradient(const distill_launch& L, const int* ids, const float* p, T* grad, int k, int id, float s,
                                                       float top, float f, float fq)
        {
            float all   = 0.0f;
            bool  first = true;
            for (int j = 0; j < L.d.k; ++j)
                if (ids[j] == id)
                {
                    first &= j >= k;
                    all = __fadd_rn(all, p[j]);
                }
            if (first)
                grad[id] = from_float<T>(__fsub_rn(__fmul_rn(fq, pow2(__fmul_rn(__fsub_rn(s, top), L.c))), __fmul_rn(f, all)));
        }

        // Whether an id in [from, to) occurs more than once among a row's entries: a warp compares them, or sets a bit for each in `bits`,
        // which has room for ROOM of them: all that are looked at (0), or a window of them at a time.  (60000 rows of 1500 floats with 100
        // entries each: 907 us where every entry was compared with every other one and blocks had 256 threads, 397 now.)
        template <int ROOM = 0>
        __device__ __forceinline__ bool repeats(const int* ids, uint32_t* bits, int k, int from, int to)
        {
            const int lane = threadIdx.x & 31;
            if (k <= 32)
            {
                const int      id   = lane < k ? ids[lane] : -1;
                const unsigned same = __match_any_sync(0xffffffffu, id); // (all lanes take part)
                return __any_sync(0xffffffffu, id >= from && id < to && __popc(same) > 1);
            }
            bool twice = false;
            do
            {
                const int end = ROOM ? min(to, from + ROOM) : to;
                for (int i = lane; i < (end - from + 31) / 32; i += 32)
                    bits[i] = 0;
                __syncwarp();
                for (int i = lane; i < k; i += 32)
                    if (const int id = ids[i]; id >= from && id < end)
                        twice |= (atomicOr(&bits[(id - from) / 32], 1u << ((id - from) & 31)) >> ((id - from) & 31) & 1) != 0;
                __syncwarp();
                from += ROOM;
            } while (ROOM && from < to);
            return __any_sync(0xffffffffu, twice);
        }

        __device__ __forceinline__ void write_loss(const aeonb_distill_desc& d, int64_t row, float loss, float lse)
        {
            if (d.loss)
                d.loss[row] = loss;
            if (d.lse)
                d.lse[row] = lse;
        }

        // lse times T, which stands for the largest logit where the lse is given, and the factor that makes up for its rounding
        __device__ __forceinline__ float2 against_lse(const distill_launch& L, float lse)
        {
            const float top = __fmul_rn(lse, L.d.temperature);
            return make_float2(top, pow2(__fmul_rn(-__fmaf_rn(lse, L.d.temperature, -top), L.c)));
        }

        // Rows of up to 128 values or 256 vectors with up to 32 entries: G lanes each, 32 / G rows to a warp, NV vectors a lane (VECTOR) or
        // values.  Every lane takes part in every step, whatever its row.
        struct few_entries
        {
            int   id[32];
            float p[32], t[32], s[32];
        };
        template <int G, typename V, typename Op>
        __device__ __forceinline__ V group_reduce(V v, Op op)
        {
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1)
                v = op(v, __shfl_xor_sync(0xffffffffu, v, o));
            return v;
        }

        template <typename T, int MODE, int G, int NV, bool VECTOR>
        __global__ void __launch_bounds__(256, 4) distill_few_kernel(const distill_launch L)
        {
            constexpr int N = piece<T>::N;
            __shared__ few_entries    all[256 / G];
            const aeonb_distill_desc& d   = L.d;
            const int                 l   = threadIdx.x & (G - 1);
            const int64_t             row = (int64_t)blockIdx.x * (256 / G) + threadIdx.x / G;
            const float               inf = __uint_as_float(0x7f800000u), nan = __uint_as_float(0x7fffffffu);
            few_entries&              e    = all[threadIdx.x / G];
            const bool                real = row < d.rows;
            const T*                  s    = static_cast<const T*>(d.logits) + row * d.logits_stride;
            const cut<T>              c(s, d.vocab);
            const float               w   = !real ? 0.0f : d.weights ? d.weights[row] : 1.0f; // (its row is read without waiting for it)
            piece<T>                  x[VECTOR ? NV : 1];
            float                     one[VECTOR ? 2 : NV]; // single values; of a row in vectors, one before them and one behind
            const auto at_one = [&](int j) { return !VECTOR ? (j * G + l < d.vocab ? j * G + l : -1)
                                                  : j == 0  ? (l < c.head ? l : -1)
                                                            : (l < c.tail ? c.head + c.n * N + l : -1); };
            constexpr int ONES = VECTOR ? 2 : NV;
#pragma unroll
            for (int j = 0; j < ONES; ++j)
                one[j] = real && at_one(j) >= 0 ? to_float(s[at_one(j)]) : -inf;
            if constexpr (VECTOR)
            {
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (real && j * G + l < c.n)
                        x[j].load(s + c.head + (j * G + l) * N);
                    else
                        x[j].clear();
            }
            float up = 1.0f, lse = 0.0f;
            if (real && MODE != LOSS && d.upstream)
                up = d.upstream[row];
            if (real && MODE == GRAD)
                lse = d.lse[row];
            // the largest entry and the largest value, then the two sums, then the gradient; the loss last
            float tmax = -inf, m = -inf;
            int   odd  = 0;
            for (int k = l; k < d.k; k += G)
            {
                int   id = -1;
                float t  = -inf;
                if (real)
                    odd |= read_entry(d, row, k, id, t);
                e.id[k] = id;
                e.t[k]  = t;
                e.s[k]  = id >= 0 && id < d.vocab ? to_float(s[id]) : 0.0f;
                tmax    = fmaxf(tmax, t);
            }
            if (MODE != GRAD)
            {
#pragma unroll
                for (int j = 0; j < ONES; ++j)
                    m = fmaxf(m, one[j]);
                if constexpr (VECTOR)
                {
#pragma unroll
                    for (int j = 0; j < NV; ++j)
                        m = x[j].largest(m);
                }
            }
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1)
            {
                const float a = __shfl_xor_sync(0xffffffffu, tmax, o), b = MODE != GRAD ? __shfl_xor_sync(0xffffffffu, m, o) : 0.0f;
                odd |= __shfl_xor_sync(0xffffffffu, odd, o);
                tmax = fmaxf(tmax, a);
                m    = fmaxf(m, b);
            }
            const bool found = w != 0.0f && (odd || tmax != -inf);
            bool       bad   = odd || !(tmax < inf);
            float      esum = 0.0f, sum = 0.0f, top = m;
            for (int k = l; k < d.k; k += G)
            {
                const float t = __fmul_rn(__fsub_rn(e.t[k], tmax), L.c);
                const float p = e.id[k] >= 0 ? pow2(t) : 0.0f;
                e.t[k]        = t;
                e.p[k]        = p;
                esum          = __fadd_rn(esum, p);
            }
            if (MODE != GRAD)
            {
                float2 z = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int j = 0; j < ONES; ++j)
                    z.x = __fadd_rn(z.x, pow2(__fmul_rn(__fsub_rn(one[j], top), L.c)));
                if constexpr (VECTOR)
                {
#pragma unroll
                    for (int j = 0; j < NV; ++j)
                        z = x[j].sum(z, top, L.c);
                }
                sum = __fadd_rn(z.x, z.y);
            }
#pragma unroll
            for (int o = G / 2; o > 0; o >>= 1)
            {
                const float a = __shfl_xor_sync(0xffffffffu, esum, o), b = MODE != GRAD ? __shfl_xor_sync(0xffffffffu, sum, o) : 0.0f;
                esum = __fadd_rn(esum, a);
                sum  = __fadd_rn(sum, b);
            }
            float fq, f = __fmul_rn(__fmul_rn(w, L.factor), up);
            if (MODE != GRAD)
            {
                bad |= !(fabsf(top) < inf) || sum != sum;
                fq = __fdiv_rn(f, sum);
            }
            else
            {
                const float2 at = against_lse(L, lse);
                bad |= !(fabsf(lse) < inf);
                top = at.x;
                fq  = __fmul_rn(f, at.y);
            }
            if (bad)
                fq = nan;
            const float share = __fdiv_rn(1.0f, esum);
            T*          grad  = static_cast<T*>(d.grad) + row * d.grad_stride;
            if (MODE != LOSS && real)
            {
#pragma unroll
                for (int j = 0; j < ONES; ++j)
                    if (at_one(j) >= 0)
                        grad[at_one(j)] = from_float<T>(found ? __fmul_rn(fq, pow2(__fmul_rn(__fsub_rn(one[j], top), L.c))) : 0.0f);
                if constexpr (VECTOR)
                {
#pragma unroll
                    for (int j = 0; j < NV; ++j)
                        if (j * G + l < c.n)
                            store_piece(grad + c.head + (j * G + l) * N, found ? x[j].gradient(top, L.c, fq) : make_uint4(0, 0, 0, 0), L.together);
                }
            }
            const float zsum2 = log2f(sum), esum2 = log2f(esum);
            float       term  = 0.0f; // p (log p - s / T + lse), to the base 2
            for (int k = l; k < d.k; k += G)
            {
                const float p = __fmul_rn(e.p[k], share);
                e.p[k]        = p;
                if (MODE != GRAD && p > 0.0f)
                    term = __fadd_rn(term, __fmul_rn(p, __fadd_rn(__fsub_rn(e.t[k], esum2),
                                                                  __fadd_rn(zsum2, __fmul_rn(__fsub_rn(top, e.s[k]), L.c)))));
            }
            if (MODE != GRAD)
            {
                term = group_reduce<G>(term, add());
                if (real && l == 0)
                {
                    const float loss  = __fmul_rn(__fmul_rn(w, L.tt), __fmul_rn(term, LN2));
                    const float whole = __fadd_rn(__fdiv_rn(top, d.temperature), __fmul_rn(zsum2, LN2));
                    write_loss(d, row, !found ? 0.0f : bad ? nan : loss, !found ? 0.0f : bad ? nan : whole);
                }
            }
            if (MODE == LOSS)
                return;
            __syncwarp();
            // (eight lanes have up to four entries each, and look through them all; those of a whole warp at most one)
            bool twice = true;
            if (G == 32)
                twice = repeats(e.id, nullptr, d.k, 0, d.vocab);
            if (found && !bad)
                for (int k = l; k < d.k; k += G)
                {
                    const int id = e.id[k];
                    if (id < 0)
                        continue;
                    if (twice)
                        entry_gradient(L, e.id, e.p, grad, k, id, e.s[k], top, f, fq);
                    else
                        grad[id] = from_float<T>(__fsub_rn(__fmul_rn(fq, pow2(__fmul_rn(__fsub_rn(e.s[k], top), L.c))), __fmul_rn(f, e.p[k])));
                }
        }

        // Rows of up to 128 values (a value per lane and step) or 256 vectors: a warp each.
        template <typename T, int MODE, int NT, int NV, bool VECTOR>
        __global__ void __launch_bounds__(NT) distill_warp_kernel(const distill_launch L)
        {
            extern __shared__ __align__(16) unsigned char dynamic[];
            const aeonb_distill_desc& d    = L.d;
            const int                 lane = threadIdx.x & 31;
            const int64_t             row  = (int64_t)blockIdx.x * (NT / 32) + threadIdx.x / 32;
            const float               inf = __uint_as_float(0x7f800000u), nan = __uint_as_float(0x7fffffffu);
            if (row >= d.rows)
                return;
            auto&    e    = reinterpret_cast<entries<ENTRIES>*>(dynamic)[threadIdx.x / 32];
            const T* s    = static_cast<const T*>(d.logits) + row * d.logits_stride;
            T*       grad = MODE == LOSS ? nullptr : static_cast<T*>(d.grad) + row * d.grad_stride;

            const float w   = d.weights ? d.weights[row] : 1.0f;
            bool        bad = false, found = false;
            float       esum2 = 0.0f;
            piece<T>    x[VECTOR ? NV : 1];
            float       one[VECTOR ? 1 : NV]; // single values
            const cut<T> c(s, d.vocab);
            const int   loose = VECTOR ? c.loose(lane, true, lane < 16) : -1;
            if (w != 0.0f)
            {
                if constexpr (VECTOR)
                {
                    one[0] = loose >= 0 ? to_float(s[loose]) : -inf;
#pragma unroll
                    for (int j = 0; j < NV; ++j)
                        if (j * 32 + lane < c.n)
                            x[j].load(s + c.head + (j * 32 + lane) * piece<T>::N);
                        else
                            x[j].clear();
                }
                else
                {
#pragma unroll
                    for (int j = 0; j < NV; ++j)
                        one[j] = j * 32 + lane < d.vocab ? to_float(s[j * 32 + lane]) : -inf;
                }
                esum2 = read_entries(L, row, s, e, found, bad);
            }
            if (!found)
            {
                if (MODE != GRAD && lane == 0)
                    write_loss(d, row, 0.0f, 0.0f);
                if (MODE != LOSS)
                    for (int i = lane; i < d.vocab; i += 32)
                        grad[i] = from_float<T>(0.0f);
                return;
            }
            float top, f, fq;
            if (MODE != GRAD)
            {
                float m = -inf;
#pragma unroll
                for (int j = 0; j < (VECTOR ? 1 : NV); ++j)
                    m = fmaxf(m, one[j]);
                if constexpr (VECTOR)
                {
#pragma unroll
                    for (int j = 0; j < NV; ++j)
                        m = x[j].largest(m);
                }
                top = warp_reduce(m, larger());
                bad |= !(fabsf(top) < inf);
                float2 z = make_float2(0.0f, 0.0f);
#pragma unroll
                for (int j = 0; j < (VECTOR ? 1 : NV); ++j)
                    z.x = __fadd_rn(z.x, pow2(__fmul_rn(__fsub_rn(one[j], top), L.c)));
                if constexpr (VECTOR)
                {
#pragma unroll
                    for (int j = 0; j < NV; ++j)
                        if (j * 32 < c.n)
                            z = x[j].sum(z, top, L.c);
                }
                const float sum   = warp_reduce(__fadd_rn(z.x, z.y), add());
                const float zsum2 = log2f(sum);
                bad |= sum != sum;
                const float loss = entries_loss(L, e, esum2, top, zsum2, w);
                if (lane == 0)
                    write_loss(d, row, bad ? nan : loss, bad ? nan : __fadd_rn(__fdiv_rn(top, d.temperature), __fmul_rn(zsum2, LN2)));
                if (MODE == LOSS)
                    return;
                f  = __fmul_rn(w, L.factor);
                fq = sum;
            }
            else
            {
                const float  lse = d.lse[row];
                const float2 at  = against_lse(L, lse);
                bad |= !(fabsf(lse) < inf);
                f   = __fmul_rn(w, L.factor);
                top = at.x;
                fq  = at.y;
            }
            if (d.upstream)
                f = __fmul_rn(f, d.upstream[row]);
            if (bad)
                f = nan;
            fq = MODE == GRAD ? __fmul_rn(f, fq) : __fdiv_rn(f, fq);
            if constexpr (VECTOR)
            {
                if (loose >= 0)
                    grad[loose] = from_float<T>(__fmul_rn(fq, pow2(__fmul_rn(__fsub_rn(one[0], top), L.c))));
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (j * 32 + lane < c.n)
                        store_piece(grad + c.head + (j * 32 + lane) * piece<T>::N, x[j].gradient(top, L.c, fq), L.together);
            }
            else
            {
#pragma unroll
                for (int j = 0; j < NV; ++j)
                    if (j * 32 + lane < d.vocab)
                        grad[j * 32 + lane] = from_float<T>(__fmul_rn(fq, pow2(__fmul_rn(__fsub_rn(one[j], top), L.c))));
            }
            __syncwarp();
            if (bad)
                return;
            // (nobody reads the entries' t any more; ids are below the vocabulary here, which is 2055 at most)
            const bool twice = repeats(e.id, reinterpret_cast<uint32_t*>(e.t), d.k, 0, d.vocab);
            for (int k = lane; k < d.k; k += 32)
            {
                const int id = e.id[k];
                if (id < 0)
                    continue;
                if (twice)
                    entry_gradient(L, e.id, e.p, grad, k, id, e.s[k], top, f, fq);
                else
                    grad[id] = from_float<T>(__fsub_rn(__fmul_rn(fq, pow2(__fmul_rn(__fsub_rn(e.s[k], top), L.c))), __fmul_rn(f, e.p[k])));
            }
        }

        // ---- named barriers of a block: those who wait, and those who only say that they have come
        __device__ __forceinline__ void bar_sync(int id, int threads) { asm volatile("bar.sync %0, %1;" ::"r"(id), "r"(threads) : "memory"); }
        __device__ __forceinline__ void bar_arrive(int id, int threads) { asm volatile("bar.arrive %0, %1;" ::"r"(id), "r"(threads) : "memory"); }

        // Waits until at most n groups of copies are under way (n known when unrolled).
        __device__ __forceinline__ void wait_copies(int n)
        {
            if (n == 0)
                asm volatile("cp.async.wait_group 0;" ::: "memory");
            else if (n == 1)
                asm volatile("cp.async.wait_group 1;" ::: "memory");
            else if (n == 2)
                asm volatile("cp.async.wait_group 2;" ::: "memory");
            else
                asm volatile("cp.async.wait_group 3;" ::: "memory");
        }

        // Longer rows: the blocks of a cluster (LOSS, LOSS_GRAD), or any number of blocks (GRAD).  A block keeps its part of a row, up to NV
        // vectors for each of NT threads, in shared memory, and goes from row to row: each thread copies its vectors of the next row into
        // the place of those that it has used for the last time, so that memory is never idle.  No other thread touches them.
        // The last warp has no vectors.  It reads the entries of the next row while the others work on this one, puts the warps' sums
        // (and the other blocks') together, hands out what the gradient needs, and writes the entries' own part when the rest is there.
        // So the others wait once in a row, from their last exponential to the first store.  (8192 rows of 131072 bf16 logits with gradient:
        // 1.30 ms with the row in registers and all threads at every barrier, 1.22 in shared memory, 0.91 with the warp of its own.)
        // Several blocks on an SM hide what one waits for: 3 to 15 by their size, at 32 to 40 registers a thread (of those with room for 256
        // entries, whose 8 KB leave less memory, 12 or 13 blocks of 64 threads, 10 of 96, 8 of 128 and 6 of 192).
        template <typename T, int MODE, int NT, int ROOM>
        __global__ void __launch_bounds__(NT + 32, NT == 512 ? 3 : NT == 256 ? 5 : NT == 192 ? 7 : NT == 128 ? 9 : NT == 96 ? 12 : 15) distill_block_kernel(const distill_launch L)
        {
            constexpr int NV = BLOCK_VECTORS, CHUNK = NT == 512 ? 2 : 4, CHUNKS = NV / CHUNK, WARPS = NT / 32, N = piece<T>::N, ALL = NT + 32;
            constexpr int SUMS = 1, RESULT = 2, WRITTEN = 3; // barriers
            struct outcome // of a row's sums
            {
                float top, fq; // the gradient at v is fq 2^((s[v] - top) c), less the entries' part
                int   found;   // 0: the row counts for nothing, the gradient is 0
                int   ahead;   // whether the row that is copied next is needed
            };
            // NV x NT vectors, on the 128 bytes that a copied line fills (131072 rows of 8192 bf16 with gradient: 905 us at another place, 757 there)
            extern __shared__ __align__(128) unsigned char row_part[];
            __shared__ float2   part[WARPS], theirs[2][16];
            __shared__ entries<ROOM> of_row[2]; // of this row and of the next one
            __shared__ outcome  result;
            // A bit for each value of this block's part; where 32768 of them would leave room for two blocks on an SM instead of three, for half
            // of it at a time (with gradient, two blocks / three: 2048 rows of 256000 bf16 logits with 20 entries 480 / 443 us, with 200 of
            // them 910 / 765; 4096 rows of 151936 with 100 entries 1.48 / 1.18 ms).
            constexpr int VALUES = NV * NT * N + 2 * N, SEEN = VALUES > 1 << 15 ? VALUES / 2 : VALUES;
            __shared__ uint32_t ids_seen[(SEEN + 31) / 32];
            __shared__ uint64_t arrived[2];
            static_assert(NT != 512 || 3 * (NV * NT * 16 + sizeof(of_row) + sizeof(ids_seen) + sizeof(part) + sizeof(theirs) + 256 + 1024) <= 228 * 1024,
                          "three blocks on an SM, each with the kilobyte that the system takes");
            const aeonb_distill_desc& d    = L.d;
            const int                 tid  = threadIdx.x, warp = tid / 32, lane = tid & 31;
            const int64_t             step = gridDim.x / (unsigned)L.blocks;
            const int                 rank = blockIdx.x % (unsigned)L.blocks;
            const bool                several = MODE != GRAD && L.blocks > 1, first = rank == 0, last = rank == L.blocks - 1;
            const float               inf = __uint_as_float(0x7f800000u), nan = __uint_as_float(0x7fffffffu), lowest = -3.40282347e38f;
            if (several)
            {
                if (tid == 0)
                {
                    barrier_init(&arrived[0]);
                    barrier_init(&arrived[1]);
                    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
                }
                cluster_arrive();
                cluster_wait(); // every block of the cluster has started and made its barriers: its memory may be written
            }
            const auto weight = [&](int64_t r) { return r >= d.rows ? 0.0f : d.weights ? __ldg(d.weights + r) : 1.0f; };
            int64_t    row    = blockIdx.x / (unsigned)L.blocks;
            const T*   s      = static_cast<const T*>(d.logits) + row * d.logits_stride;

            if (warp < WARPS)
            {
                const uint32_t vectors_at = shared_address(row_part) + tid * 16;
                // this block's part of a row
                struct share
                {
                    int at;    // this thread's first vector's first value
                    int left;  // vectors from there on
                    int loose; // the value outside the vectors that is this thread's; -1: none
                };
                const auto share_of = [&](const T* s) {
                    const cut<T> c(s, d.vocab);
                    const int    begin = min(rank * L.vectors, c.n);
                    return share{c.head + (begin + tid) * N, min(L.vectors, c.n - begin) - tid, c.loose(tid, first, last && tid < 16)};
                };
                const auto fetch = [&](const T* from, int left, int j) {
                    if (j * NT < left)
                        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(vectors_at + j * NT * 16), "l"(from + j * NT * N) : "memory");
                };
                const auto commit = [] { asm volatile("cp.async.commit_group;" ::: "memory"); };
                const auto vector = [&](piece<T>& x, int j) {
                    asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];"
                                 : "=r"(x.w[0]), "=r"(x.w[1]), "=r"(x.w[2]), "=r"(x.w[3])
                                 : "r"(vectors_at + j * NT * 16)
                                 : "memory");
                };

                bool  needed = weight(row) != 0.0f, needed_then = MODE == LOSS && weight(row + step) != 0.0f;
                share mine   = share_of(s);
#pragma unroll
                for (int j = 0; j < NV; ++j)
                {
                    fetch(s + mine.at, needed ? mine.left : 0, j);
                    if (j % CHUNK == CHUNK - 1)
                        commit();
                }
                for (; row < d.rows; row += step)
                {
                    const T*    s_then = s + step * d.logits_stride;
                    const share next   = share_of(s_then);
                    const float one    = needed && mine.loose >= 0 ? to_float(s[mine.loose]) : -inf;
                    if (MODE != GRAD)
                    {
                        // from the lowest finite value on: a row of nothing but -infinity has the sum 0
                        const int have = needed ? mine.left : 0, coming = needed_then ? next.left : 0;
                        float     m    = fmaxf(one, lowest);
                        float2    z    = make_float2(pow2(__fmul_rn(__fsub_rn(one, m), L.c)), 0.0f);
                        const auto first_pass = [&](auto all) {
                            constexpr bool whole = decltype(all)::value;
#pragma unroll
                            for (int q = 0; q < CHUNKS; ++q)
                            {
                                wait_copies(MODE == LOSS ? CHUNKS - 1 : CHUNKS - 1 - q);
                                if (whole || q * CHUNK * NT < have)
                                {
                                    piece<T> x[CHUNK];
                                    float    higher = m;
#pragma unroll
                                    for (int i = 0; i < CHUNK; ++i)
                                    {
                                        if (whole || (q * CHUNK + i) * NT < have)
                                            vector(x[i], q * CHUNK + i);
                                        else
                                            x[i].clear();
                                        higher = x[i].largest(higher);
                                    }
                                    const float scale = pow2(__fmul_rn(__fsub_rn(m, higher), L.c));
                                    m                 = higher;
                                    z                 = mul2(z, make_float2(scale, scale));
#pragma unroll
                                    for (int i = 0; i < CHUNK; ++i)
                                        z = x[i].sum(z, m, L.c);
                                }
                                if (MODE == LOSS)
                                {
#pragma unroll
                                    for (int i = 0; i < CHUNK; ++i)
                                        fetch(s_then + next.at, coming, q * CHUNK + i);
                                    commit();
                                }
                            }
                        };
                        // The loss alone looks at none of the numbers where a thread has all its vectors (65536 rows of 16384 bf16: 422 us else,
                        // now 396; with a gradient that costs the registers of a second copy: 32768 rows of 32000, 721 us as it is, 837 so).
                        if (MODE == LOSS && have > (NV - 1) * NT)
                            first_pass(std::true_type());
                        else
                            first_pass(std::false_type());
                        const float wm = warp_reduce(m, larger());
                        const float wz = warp_reduce(__fmul_rn(__fadd_rn(z.x, z.y), pow2(__fmul_rn(__fsub_rn(m, wm), L.c))), add());
                        if (lane == 0)
                            part[warp] = make_float2(wm, wz);
                        bar_arrive(SUMS, ALL);
                    }
                    bar_sync(RESULT, ALL);
                    const outcome o = result;
                    if (MODE == LOSS)
                    {
                        needed      = needed_then;
                        needed_then = o.ahead;
                    }
                    else
                    {
                        T*        grad   = static_cast<T*>(d.grad) + row * d.grad_stride;
                        T*        to     = grad + mine.at;
                        const int coming = o.ahead ? next.left : 0;
                        if (mine.loose >= 0)
                            grad[mine.loose] = from_float<T>(o.found ? __fmul_rn(o.fq, pow2(__fmul_rn(__fsub_rn(one, o.top), L.c))) : 0.0f);
                        if (o.found && L.together)
                        {
#pragma unroll
                            for (int j = 0; j < NV; ++j)
                            {
                                if (MODE == GRAD && j % CHUNK == 0)
                                    wait_copies(CHUNKS - 1);
                                if (j * NT < mine.left)
                                {
                                    piece<T> x;
                                    vector(x, j);
                                    __stcs(reinterpret_cast<uint4*>(to + j * NT * N), x.gradient(o.top, L.c, o.fq));
                                }
                                fetch(s_then + next.at, coming, j);
                                if (j % CHUNK == CHUNK - 1)
                                    commit();
                            }
                        }
                        else
                        {
                            asm volatile("cp.async.wait_all;" ::: "memory");
#pragma unroll 1
                            for (int j = 0; j < NV; ++j)
                            {
                                if (j * NT < mine.left)
                                {
                                    uint4 g = make_uint4(0, 0, 0, 0);
                                    if (o.found)
                                    {
                                        piece<T> x;
                                        vector(x, j);
                                        g = x.gradient(o.top, L.c, o.fq);
                                    }
                                    store_piece(to + j * NT * N, g, L.together);
                                }
                                fetch(s_then + next.at, coming, j);
                            }
                            for (int q = 0; q < CHUNKS; ++q) // all in the first one: the next row waits for as many as ever
                                commit();
                        }
                        bar_arrive(WRITTEN, ALL);
                        needed = o.ahead;
                    }
                    mine = next;
                    s    = s_then;
                }
            }
            else
            {
                // what this warp knows of a row
                struct facts
                {
                    float w, up, lse;
                    float esum2;
                    bool  found, bad;
                };
                const auto prepare = [&](int64_t r, float w, const T* s, entries<ROOM>& e) {
                    facts a{w, 1.0f, 0.0f, 0.0f, false, false};
                    if (w == 0.0f)
                        return a;
                    if (MODE != LOSS && d.upstream)
                        a.up = d.upstream[r];
                    if (MODE == GRAD)
                        a.lse = d.lse[r];
                    const cut<T> c(s, d.vocab);
                    const int    begin = min(rank * L.vectors, c.n), end = min(begin + L.vectors, c.n);
                    const int    from = first ? 0 : c.head + begin * N, to = last ? d.vocab : c.head + end * N;
                    float        top = -inf;
                    bool         odd = false;
#pragma unroll 4
                    for (int k = lane; k < d.k; k += 32)
                    {
                        int   id;
                        float t;
                        odd |= read_entry(d, r, k, id, t);
                        e.id[k] = id;
                        e.t[k]  = t;
                        top     = fmaxf(top, t);
                    }
#pragma unroll 4
                    for (int k = lane; k < d.k; k += 32)
                    {
                        const int  id   = e.id[k];
                        const bool here = id >= from && id < to;
                        e.s[k]          = here || (MODE != GRAD && first && id >= 0 && id < d.vocab) ? to_float(s[id]) : 0.0f;
                        if (!here && !(MODE != GRAD && first))
                            e.s[k] = 0.0f;
                    }
                    top     = warp_reduce(top, larger());
                    odd     = __any_sync(0xffffffffu, odd);
                    a.found = odd || top != -inf;
                    a.bad   = odd || !(top < inf);
                    float sum = 0.0f;
                    for (int k = lane; k < d.k; k += 32)
                    {
                        const float t = __fmul_rn(__fsub_rn(e.t[k], top), L.c);
                        const float p = e.id[k] >= 0 ? pow2(t) : 0.0f;
                        e.t[k]        = t;
                        e.p[k]        = p;
                        sum           = __fadd_rn(sum, p);
                    }
                    sum = warp_reduce(sum, add());
                    for (int k = lane; k < d.k; k += 32)
                        e.p[k] = __fdiv_rn(e.p[k], sum);
                    a.esum2 = log2f(sum);
                    return a;
                };
                float   w_then = weight(row + step);
                facts   now    = prepare(row, weight(row), s, of_row[0]);
                bool    lost   = false; // a wait for the other blocks has run out: rows are NaN from there on
                for (int turn = 0; row < d.rows; row += step, ++turn)
                {
                    const int      set = turn & 1;
                    const auto&    e   = of_row[set];
                    const float    w_after = weight(row + 2 * step);
                    float          top = 0.0f, z = 1.0f;
                    bool           bad = now.bad;
                    if (MODE != GRAD)
                    {
                        bar_sync(SUMS, ALL);
                        float2 o = lane < WARPS ? part[min(lane, WARPS - 1)] : make_float2(lowest, 0.0f);
                        if (MODE == LOSS)
                        {
                            __syncwarp();
                            if (lane == 0)
                                result.ahead = w_after != 0.0f;
                            __syncwarp();
                            bar_arrive(RESULT, ALL);
                        }
                        top = warp_reduce(o.x, larger());
                        z   = warp_reduce(__fmul_rn(o.y, pow2(__fmul_rn(__fsub_rn(o.x, top), L.c))), add());
                        if (several)
                        {
                            if (lane == 0)
                                barrier_expect(&arrived[set], L.blocks * 8);
                            __syncwarp();
                            if (lane < L.blocks)
                                cluster_send(&theirs[set][rank], &arrived[set], lane, make_float2(top, z));
                            lost = lost || !barrier_wait(&arrived[set], (turn >> 1) & 1);
                            bad |= __any_sync(0xffffffffu, lost);
                            o   = lane < L.blocks ? theirs[set][lane & 15] : make_float2(lowest, 0.0f);
                            top = warp_reduce(o.x, larger());
                            z   = warp_reduce(__fmul_rn(o.y, pow2(__fmul_rn(__fsub_rn(o.x, top), L.c))), add());
                        }
                        bad |= !(fabsf(top) < inf) || !(z > 0.0f);
                    }
                    float f = 0.0f, fq = 0.0f, high = top;
                    if (MODE != LOSS)
                    {
                        f = __fmul_rn(__fmul_rn(now.w, L.factor), now.up);
                        if (MODE == GRAD)
                        {
                            const float2 at = against_lse(L, now.lse);
                            bad |= !(fabsf(now.lse) < inf);
                            high = at.x;
                            fq   = __fmul_rn(f, at.y);
                        }
                        else
                            fq = __fdiv_rn(f, z);
                        if (bad)
                            fq = nan;
                        if (lane == 0)
                            result = outcome{high, fq, now.found, w_then != 0.0f};
                        __syncwarp();
                        bar_arrive(RESULT, ALL);
                    }
                    if (MODE != GRAD && first)
                    {
                        float loss = 0.0f, lse = 0.0f;
                        if (now.found)
                        {
                            const float zsum2 = log2f(z);
                            loss              = entries_loss(L, e, now.esum2, top, zsum2, now.w);
                            loss              = bad ? nan : loss;
                            lse               = bad ? nan : __fadd_rn(__fdiv_rn(top, d.temperature), __fmul_rn(zsum2, LN2));
                        }
                        if (lane == 0)
                            write_loss(d, row, loss, lse);
                    }
                    const facts here = now;
                    now              = prepare(row + step, w_then, s + step * d.logits_stride, of_row[set ^ 1]);
                    w_then           = w_after;
                    if (MODE != LOSS)
                    {
                        T*           grad = static_cast<T*>(d.grad) + row * d.grad_stride;
                        const cut<T> c(s, d.vocab);
                        const int    begin = min(rank * L.vectors, c.n), end = min(begin + L.vectors, c.n);
                        const int    from = first ? 0 : c.head + begin * N, to = last ? d.vocab : c.head + end * N;
                        const bool   twice = here.found && !bad && repeats<SEEN < VALUES ? SEEN : 0>(e.id, ids_seen, d.k, from, to);
                        bar_sync(WRITTEN, ALL);
                        if (here.found && !bad)
                            for (int k = lane; k < d.k; k += 32)
                            {
                                const int id = e.id[k];
                                if (id < from || id >= to)
                                    continue;
                                if (twice)
                                    entry_gradient(L, e.id, e.p, grad, k, id, e.s[k], high, f, fq);
                                else
                                    grad[id] = from_float<T>(__fsub_rn(__fmul_rn(fq, pow2(__fmul_rn(__fsub_rn(e.s[k], high), L.c))), __fmul_rn(f, e.p[k])));
                            }
                        __syncwarp();
                    }
                    s += step * d.logits_stride;
                }
            }
            if (several) // nothing is sent to a block that has left
            {
                cluster_arrive();
                cluster_wait();
            }
        }

        // The loss, and the gradient, of rows beyond what a cluster holds: a block per row, which reads it twice.
        template <typename T>
        __global__ void __launch_bounds__(THREADS) distill_kernel(const distill_launch L)
        {
            constexpr int RUN = 16;
            __shared__ float          shared[THREADS / 32];
            __shared__ double         wide[THREADS / 32];
            __shared__ entries<ENTRIES> e;
            __shared__ float          esum2_;
            __shared__ int            flags;
            const aeonb_distill_desc& d    = L.d;
            const int                 tid  = threadIdx.x;
            const float               nan  = __uint_as_float(0x7fffffffu), inf = __uint_as_float(0x7f800000u);
            const int64_t             row  = blockIdx.x;
            const T*                  s    = static_cast<const T*>(d.logits) + row * d.logits_stride;
            T*                        grad = d.grad ? static_cast<T*>(d.grad) + row * d.grad_stride : nullptr;
            const float               w    = d.weights ? d.weights[row] : 1.0f;
            if (tid < 32)
            {
                bool        found = false, bad = false;
                const float esum2 = w != 0.0f ? read_entries(L, row, s, e, found, bad) : 0.0f;
                if (tid == 0)
                {
                    esum2_ = esum2;
                    flags  = (found ? 1 : 0) | (bad ? 2 : 0);
                }
            }
            __syncthreads();
            if (!(flags & 1))
            {
                if (tid == 0)
                {
                    if (d.loss)
                        d.loss[row] = 0.0f;
                    if (d.lse)
                        d.lse[row] = 0.0f;
                }
                if (grad)
                    for (int64_t v = tid; v < d.vocab; v += THREADS)
                        grad[v] = from_float<T>(0.0f);
                return;
            }
            // The sum against a reference, which follows the largest value once that is 2^4 times as much: an exponential is 2^4 at most,
            // and few rescalings of a sum are of any weight.  Sixteen terms in 32 bits, then in 64: a thread may have millions.  (A row of
            // 2^26 bf16 logits, nearly alike: the lse off by 1.4e-3 with one 32-bit sum a thread, by 1.1e-6 so.  Sixteen loads at once: 16
            // rows of 4000001, loss alone 2.46 -> 1.76 ms.)
            float  m = -inf, ref = -inf;
            double total = 0.0;
            for (int64_t v0 = tid; v0 < d.vocab; v0 += RUN * THREADS)
            {
                float x[RUN], higher = m;
#pragma unroll
                for (int i = 0; i < RUN; ++i)
                {
                    const int64_t v = v0 + i * THREADS;
                    x[i]            = v < d.vocab ? to_float(s[v]) : -inf;
                    higher          = fmaxf(higher, x[i]); // (not NaN)
                }
                m = higher;
                if (__fmul_rn(__fsub_rn(m, ref), L.c) > 4.0f)
                {
                    total = ref == -inf ? total : total * pow2(__fmul_rn(__fsub_rn(ref, m), L.c));
                    ref   = m;
                }
                float z = 0.0f;
#pragma unroll
                for (int i = 0; i < RUN; ++i)
                    if (!(x[i] == -inf)) // a NaN stays in the sum
                        z = __fadd_rn(z, pow2(__fmul_rn(__fsub_rn(x[i], ref), L.c)));
                total += z;
            }
            const float top = block_reduce(m, shared, larger());
            // (a thread without a value has the sum 0, or NaN)
            const float sum = (float)block_reduce(ref == -inf ? total : total * exp2(((double)ref - top) * L.c), wide, add_wide());
            const bool  bad = (flags & 2) || !(fabsf(top) < inf) || sum != sum;
            if (tid < 32)
            {
                const float zsum2 = log2f(sum);
                const float loss  = entries_loss(L, e, esum2_, top, zsum2, w);
                if (tid == 0)
                {
                    if (d.loss)
                        d.loss[row] = bad ? nan : loss;
                    if (d.lse)
                        d.lse[row] = bad ? nan : __fadd_rn(__fdiv_rn(top, d.temperature), __fmul_rn(zsum2, LN2));
                }
            }
            if (!grad)
                return;
            float f = __fmul_rn(w, L.factor);
            if (d.upstream)
                f = __fmul_rn(f, d.upstream[row]);
            if (bad)
                f = nan;
            const float fq = __fdiv_rn(f, sum);
            for (int64_t v = tid; v < d.vocab; v += THREADS)
                grad[v] = from_float<T>(__fmul_rn(fq, pow2(__fmul_rn(__fsub_rn(to_float(s[v]), top), L.c))));
            __syncthreads();
            if (!bad)
                for (int k = tid; k < d.k; k += THREADS)
                    if (e.id[k] >= 0)
                        entry_gradient(L, e.id, e.p, grad, k, e.id[k], e.s[k], top, f, fq);
        }

        void check_distill(const aeonb_distill_desc& d, bool with_loss)
        {
            const int e = float_size(d.dtype);
            if (d.rows < 0 || d.rows > 0x7fffffff || d.vocab < 1 || d.vocab > 1 << 30)
                throw std::invalid_argument("the logits need between 0 and 2^31-1 rows of between 1 and 2^30 values");
            if (d.k < 1 || d.k > ENTRIES)
                throw std::invalid_argument("a row has between 1 and 256 entries");
            if (!(d.temperature >= 0x1p-40f && d.temperature <= 0x1p40f))
                throw std::invalid_argument("the temperature must be a number between 2^-40 and 2^40");
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

        template <typename T, int MODE, int NT, int NV, bool VECTOR>
        cudaError_t launch_warps(const distill_launch& L, cudaStream_t stream)
        {
            constexpr int ROWS   = NT / 32;
            const int64_t blocks = (L.d.rows + ROWS - 1) / ROWS;
            distill_warp_kernel<T, MODE, NT, NV, VECTOR><<<(unsigned)blocks, NT, sizeof(entries<ENTRIES>) * ROWS, stream>>>(L);
            return cudaGetLastError();
        }

        template <typename T, int MODE, int G, int NV, bool VECTOR>
        cudaError_t launch_few(const distill_launch& L, cudaStream_t stream)
        {
            constexpr int ROWS = 256 / G;
            distill_few_kernel<T, MODE, G, NV, VECTOR><<<(unsigned)((L.d.rows + ROWS - 1) / ROWS), 256, 0, stream>>>(L);
            return cudaGetLastError();
        }

        template <typename T, int MODE, int NT, int ROOM>
        cudaError_t launch_blocks(const distill_launch& L, cudaStream_t stream)
        {
            auto                kernel = distill_block_kernel<T, MODE, NT, ROOM>;
            cudaLaunchConfig_t  cfg    = {};
            cudaLaunchAttribute attr   = {};
            cfg.blockDim         = dim3(NT + 32);
            cfg.dynamicSmemBytes = BLOCK_VECTORS * NT * 16;
            cfg.stream           = stream;
            const bool cluster   = MODE != GRAD && L.blocks > 1;
            if (cluster)
            {
                attr.id               = cudaLaunchAttributeClusterDimension;
                attr.val.clusterDim.x = L.blocks;
                attr.val.clusterDim.y = attr.val.clusterDim.z = 1;
                cfg.attrs    = &attr;
                cfg.numAttrs = 1;
            }
            // rows at once: the groups of a row's blocks that find room together, asked for once per kernel, size and device
            static std::atomic<int> room[64][5];
            int                     size = 0; // log2 of the cluster's blocks
            while (cluster && 1 << size < L.blocks)
                ++size;
            int         device = 0, groups = 0;
            cudaError_t e = cudaGetDevice(&device);
            if (e != cudaSuccess)
                return e;
            if (device < 64)
                groups = room[device][size].load(std::memory_order_acquire);
            if (groups == 0)
            {
                if ((e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)cfg.dynamicSmemBytes)) != cudaSuccess ||
                    (e = cudaFuncSetAttribute(kernel, cudaFuncAttributeNonPortableClusterSizeAllowed, 1)) != cudaSuccess)
                    return e;
                cfg.gridDim = dim3(cluster ? L.blocks : 1);
                if (cluster)
                    e = cudaOccupancyMaxActiveClusters(&groups, kernel, &cfg);
                else
                {
                    int sms = 0;
                    e       = cudaOccupancyMaxActiveBlocksPerMultiprocessor(&groups, kernel, NT + 32, cfg.dynamicSmemBytes);
                    if (e == cudaSuccess)
                        e = cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, device);
                    groups *= sms;
                }
                if (e != cudaSuccess)
                    return e;
                if (groups < 1)
                    return cudaErrorInvalidConfiguration;
                if (device < 64)
                    room[device][size].store(groups, std::memory_order_release);
            }
            if (!cluster)
                groups = std::max(1, groups / L.blocks);
            cfg.gridDim = dim3((unsigned)(std::min<int64_t>(L.d.rows, groups) * L.blocks));
            return cudaLaunchKernelEx(&cfg, kernel, L);
        }

        // A row's part of up to 2048 vectors.  ROOM: its entries, at most.
        template <typename T, int MODE, int ROOM>
        cudaError_t launch_part(const distill_launch& L, cudaStream_t stream)
        {
            // Shorter parts: fewer threads and more blocks to an SM, unless all blocks have one to themselves.  131072 rows with gradient, always
            // 256 threads / by the part's length: 8192 bf16 logits 0.96 / 0.75 ms, 4096 0.80 / 0.41.  Between them, the next power of two / these:
            // 65536 rows of 6000 bf16 with gradient 344 / 291 us, loss alone 219 / 205, the gradient alone 289 / 313; 32768 rows of
            // 12000, loss alone 207 / 188, with gradient 328 / 330, the gradient alone 289 / 307.
            const bool alone = L.d.rows * L.blocks <= 148;
            if (L.vectors <= BLOCK_VECTORS * 64 && !alone)
                return launch_blocks<T, MODE, 64, ROOM>(L, stream);
            if constexpr (MODE != GRAD)
                if (L.vectors <= BLOCK_VECTORS * 96 && !alone)
                    return launch_blocks<T, MODE, 96, ROOM>(L, stream);
            if (L.vectors <= BLOCK_VECTORS * 128 && !alone)
                return launch_blocks<T, MODE, 128, ROOM>(L, stream);
            if constexpr (MODE == LOSS)
                if (L.vectors <= BLOCK_VECTORS * 192 && !alone)
                    return launch_blocks<T, MODE, 192, ROOM>(L, stream);
            return launch_blocks<T, MODE, 256, ROOM>(L, stream);
        }

        template <typename T, int MODE>
        cudaError_t launch_mode(distill_launch& L, cudaStream_t stream)
        {
            const int64_t vocab = L.d.vocab, vectors = vocab * (int64_t)sizeof(T) / 16; // whole ones, at most
            if (L.d.k <= 32 && (vocab <= 128 || vectors <= 32 * 8))
            {
                // Lanes of a row: as few as hold it with eight vectors each, so that what is done once a row is done for several rows at once.
                // A warp for each row / these, with gradient: 160000 rows of 29 floats 96 / 31 us, 65536 of 500 bf16 68 / 57, of 1000
                // floats 143 / 125.
                if (vocab <= 32)
                    return launch_few<T, MODE, 8, 4, false>(L, stream);
                if (vocab <= 64)
                    return launch_few<T, MODE, 8, 8, false>(L, stream);
                if (vocab <= 128)
                    return launch_few<T, MODE, 8, 16, false>(L, stream);
                if (vectors <= 8 * 4)
                    return launch_few<T, MODE, 8, 4, true>(L, stream);
                if (vectors <= 8 * 8)
                    return launch_few<T, MODE, 8, 8, true>(L, stream);
                if (vectors <= 16 * 8)
                    return launch_few<T, MODE, 16, 8, true>(L, stream);
                return launch_few<T, MODE, 32, 8, true>(L, stream);
            }
            if (vocab <= 128)
                return launch_warps<T, MODE, 256, 4, false>(L, stream);
            if (vectors <= 32 * 8)
                return launch_warps<T, MODE, 256, 8, true>(L, stream);
            // Threads of a block: 256 where there is a gradient and up to eight such blocks hold a row, else 512.  8192 rows of 131072 bf16
            // logits, 256 / 512: with gradient 0.86 / 0.91 ms, gradient alone 0.72 / 0.80, loss alone 0.51 / 0.47 (where nothing waits for
            // the other blocks, fewer of them cost less; one is enough for 65536 rows of 16384: 0.42 ms with 256).
            const bool    narrow = MODE == GRAD || (MODE == LOSS_GRAD && vectors <= 8 * BLOCK_VECTORS * 256);
            const int64_t most   = BLOCK_VECTORS * (narrow ? 256 : 512);
            // Blocks of a row: as many as hold it, and more while they do not fill the SMs and have 4 KB each.
            int64_t blocks = 1;
            while (blocks * most < vectors)
                blocks *= 2;
            while (blocks < 8 && L.d.rows * blocks < 148 && vectors / (blocks * 2) >= 256)
                blocks *= 2;
            if (MODE != GRAD && blocks > 16)
            {
                distill_kernel<T><<<(unsigned)L.d.rows, THREADS, 0, stream>>>(L);
                return cudaGetLastError();
            }
            L.blocks  = (int)blocks;
            L.vectors = (int)(((vectors + blocks - 1) / blocks + 7) / 8 * 8); // whole lines of 128 bytes
            if constexpr (MODE != GRAD)
                if (L.vectors > BLOCK_VECTORS * 256)
                    return launch_blocks<T, MODE, 512, ENTRIES>(L, stream);
            return L.d.k > 64 ? launch_part<T, MODE, ENTRIES>(L, stream) : launch_part<T, MODE, 64>(L, stream);
        }

        template <typename T>
        cudaError_t launch_distill(distill_launch& L, bool with_loss, cudaStream_t stream)
        {
            if (!with_loss)
                return launch_mode<T, GRAD>(L, stream);
            return L.d.grad ? launch_mode<T, LOSS_GRAD>(L, stream) : launch_mode<T, LOSS>(L, stream);
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
                const int      e = float_size(desc->dtype);
                L.d        = *desc;
                L.c        = (float)(1.4426950408889634074 / desc->temperature);
                L.factor   = (float)((double)desc->temperature * desc->grad_scale);
                L.tt       = (float)((double)desc->temperature * desc->temperature);
                L.together = (((uintptr_t)desc->logits ^ (uintptr_t)desc->grad) & 15) == 0 &&
                             (desc->rows == 1 || (desc->logits_stride - desc->grad_stride) * e % 16 == 0);
                const int64_t bytes = desc->rows * ((int64_t)desc->vocab * e * (desc->grad ? 2 : 1) + desc->k * 8 + 8);
                const cudaStream_t stream = desc->stream ? static_cast<cudaStream_t>(desc->stream) : ctx->stream;
                launch_timer  timer(ctx, AEONB_KERNEL_OTHER, bytes, stream);
                cudaError_t   err = cudaSuccess;
                switch (desc->dtype)
                {
                case AEONB_F32: err = launch_distill<float>(L, with_loss, stream); break;
                case AEONB_F16: err = launch_distill<__half>(L, with_loss, stream); break;
                case AEONB_BF16: err = launch_distill<__nv_bfloat16>(L, with_loss, stream); break;
                }
                if (err != cudaSuccess)
                    throw error(AEONB_ERR_CUDA, cuda_message("distillation kernel launch", err));
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
