// Distillation from a teacher's top logits: the teacher's half (the k largest logits of a row with the row's logsumexp)
// and the student's half (loss and gradient in one pass over the student's logits).
//
// Both work on one row per workgroup.  distill_kernel holds the row in registers, VPT 16-byte vectors per thread, and the
// second half of a wide one in LDS (VL vectors per thread), so the logits are read from memory once: at a few operations per
// byte it is bound by that read and by the store of the gradient.  Rows wider than both, or not made of whole vectors, are
// read a second time (VPT = 0).  Measured: 4096 x 131072 bf16 with both terms at T = 2 in 515 us, 4.2 TB/s read and written
// where a copy reaches 4.9, and at T = 3 in 602; 509 x 49999 fp32 in 47 us, 4.3 TB/s; 1536 x 1000 bf16 in 7 us, bound by the latency
// of its reductions.  Arithmetic is fp32, the teacher's listed mass 64-bit; the only rounding to fewer bits is the store of the
// gradient in the logits' own type.
#include "common.h"

#define DS_BF16 0
#define DS_FP16 1
#define DS_FP32 2
#define DS_MAX_K 512
#define DS_MAX_CLASSES 262144      // one bit per class in LDS: 32 KB
#define DS_ROWS (1 << 21)          // rows of one launch: the threads of a grid have to fit 32 bits (1024 a row: 2^22 - 1 rows)

typedef _Float16 f16;
typedef __attribute__((ext_vector_type(2))) _Float16 f16x2;
typedef __attribute__((ext_vector_type(2))) float f32x2;
// Rows of an odd width start at any multiple of the element size: global memory takes unaligned 16-byte accesses (the
// compiler needs to be told that the address has no more than the element's alignment, nothing else changes).
typedef u32x4 __attribute__((aligned(2))) u32x4_a2;

#define DS_LOG2E 1.44269504088896340736f

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

template <typename T> struct Pack;
template <> struct Pack<bf16> {
    static constexpr int E = 8;
    static constexpr unsigned FILL = 0xff80ff80u;                  // -inf, -inf
    static __device__ __forceinline__ void unpack(u32x4 r, float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f[2 * i] = __uint_as_float(r[i] << 16);
            f[2 * i + 1] = __uint_as_float(r[i] & 0xffff0000u);
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            bf16x2 p = __builtin_convertvector((f32x2){f[2 * i], f[2 * i + 1]}, bf16x2);
            r[i] = __builtin_bit_cast(unsigned, p);
        }
        return r;
    }
};
template <> struct Pack<f16> {
    static constexpr int E = 8;
    static constexpr unsigned FILL = 0xfc00fc00u;
    static __device__ __forceinline__ void unpack(u32x4 r, float (&f)[8]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f16x2 p = __builtin_bit_cast(f16x2, (unsigned)r[i]);
            f[2 * i] = (float)p[0];
            f[2 * i + 1] = (float)p[1];
        }
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[8]) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            f16x2 p = __builtin_convertvector((f32x2){f[2 * i], f[2 * i + 1]}, f16x2);
            r[i] = __builtin_bit_cast(unsigned, p);
        }
        return r;
    }
};
template <> struct Pack<float> {
    static constexpr int E = 4;
    static constexpr unsigned FILL = 0xff800000u;
    static __device__ __forceinline__ void unpack(u32x4 r, float (&f)[4]) {
#pragma unroll
        for (int i = 0; i < 4; ++i) f[i] = __uint_as_float(r[i]);
    }
    static __device__ __forceinline__ u32x4 pack(const float (&f)[4]) {
        u32x4 r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r[i] = __float_as_uint(f[i]);
        return r;
    }
};

// Vector v of a row covers E elements from class v * E on.  The vector that would run over the row's end is moved back to
// the row's last E elements instead (and so are the vectors behind it): every load is one unconditional 16-byte access
// inside the row, and drop_repeated() then sets what an earlier vector covers already to -inf, which takes part in nothing.
template <typename T>
__device__ __forceinline__ int first_class(int v, int N) {
    constexpr int E = Pack<T>::E;
    return min(v * E, max(N - E, 0));
}
template <typename T, bool NARROW>
__device__ __forceinline__ u32x4 ld_row(const T* __restrict__ src, int v, int N) {
    constexpr int E = Pack<T>::E;
    if (NARROW && N < E) {                                         // a row shorter than one vector
        float f[E];
#pragma unroll
        for (int e = 0; e < E; ++e) f[e] = e < N ? (float)src[e] : -INFINITY;
        return Pack<T>::pack(f);                                   // exact: every value is one of T
    }
    const unsigned at = (unsigned)first_class<T>(v, N) * (unsigned)sizeof(T);
    return *reinterpret_cast<const u32x4_a2*>(reinterpret_cast<const unsigned char*>(src) + at);
}
template <typename T>
__device__ __forceinline__ u32x4 drop_repeated(u32x4 r, int v, int N) {
    constexpr int E = Pack<T>::E;
    const int repeated = v * E - first_class<T>(v, N);
    float f[E];
    Pack<T>::unpack(r, f);
#pragma unroll
    for (int e = 0; e < E; ++e) f[e] = e < repeated ? -INFINITY : f[e];
    return Pack<T>::pack(f);
}

__device__ __forceinline__ float ld_as_float(const void* p, long long i, int type) {
    if (type == DS_BF16) return (float)static_cast<const bf16*>(p)[i];
    if (type == DS_FP16) return (float)static_cast<const f16*>(p)[i];
    return static_cast<const float*>(p)[i];
}

// Workgroup barrier that orders LDS but leaves global loads in flight (a __syncthreads would drain them).
__device__ __forceinline__ void lds_barrier() {
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
}

// Sum / maximum over a wave by DPP moves (a shuffle goes through LDS: at six of them per reduction and some ten reductions
// per row they were half of a narrow row's time).  The same order every time; every lane gets the result.
template <int CTRL, int ROWS>
__device__ __forceinline__ float dpp_or(float identity, float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(__float_as_int(identity), __float_as_int(v), CTRL, ROWS, 0xf, false));
}
template <typename Op>
__device__ __forceinline__ float wave_reduce(float v, float identity, Op op) {
    v = op(v, dpp_or<0x111, 0xf>(identity, v));                    // row_shr:1, 2, 4, 8 inside the rows of 16 lanes
    v = op(v, dpp_or<0x112, 0xf>(identity, v));
    v = op(v, dpp_or<0x114, 0xf>(identity, v));
    v = op(v, dpp_or<0x118, 0xf>(identity, v));
    v = op(v, dpp_or<0x142, 0xa>(identity, v));                    // row_bcast:15 into rows 1 and 3
    v = op(v, dpp_or<0x143, 0xc>(identity, v));                    // row_bcast:31 into rows 2 and 3
    return __int_as_float(__builtin_amdgcn_readlane(__float_as_int(v), 63));
}
__device__ __forceinline__ float wave_total(float v) {
    return wave_reduce(v, 0.0f, [](float a, float b) { return a + b; });
}
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_or_zero(double v) {
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = __builtin_amdgcn_update_dpp(0, (int)(unsigned)b, CTRL, ROWS, 0xf, false);
    const unsigned hi = __builtin_amdgcn_update_dpp(0, (int)(unsigned)(b >> 32), CTRL, ROWS, 0xf, false);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ double wave_total(double v) {
    v += dpp_or_zero<0x111, 0xf>(v);
    v += dpp_or_zero<0x112, 0xf>(v);
    v += dpp_or_zero<0x114, 0xf>(v);
    v += dpp_or_zero<0x118, 0xf>(v);
    v += dpp_or_zero<0x142, 0xa>(v);
    v += dpp_or_zero<0x143, 0xc>(v);
    const unsigned long long b = __builtin_bit_cast(unsigned long long, v);
    const unsigned lo = __builtin_amdgcn_readlane((int)(unsigned)b, 63), hi = __builtin_amdgcn_readlane((int)(unsigned)(b >> 32), 63);
    return __builtin_bit_cast(double, (unsigned long long)hi << 32 | lo);
}
__device__ __forceinline__ float wave_top(float v) {
    return wave_reduce(v, -INFINITY, [](float a, float b) { return fmaxf(a, b); });
}

// Ends one vector's share of a pass: the next pass unpacks the packed vector anew instead of keeping its fp32 values, and no
// vector's work is interleaved with the next one's: either would double the registers of a wide row and spill it.
__device__ __forceinline__ void hold(u32x4& r) {
    asm volatile("" : "+v"(r));
    __builtin_amdgcn_sched_barrier(0);
}

// The same number, but the compiler does not know: what it derives from it for every vector of one pass (offsets, columns)
// is then not kept in registers for the next.
__device__ __forceinline__ int anew(int x) {
    asm volatile("" : "+v"(x));
    return x;
}

__device__ __forceinline__ float finite_or_zero(float m) { return m == -INFINITY ? 0.0f : m; }

// (... which what was computed from it must not outlive unfinished: with the sums as operands they are complete here)
#define HOLD_STAT(r, s) asm volatile("" : "+v"(r), "+v"((s).m), "+v"((s).st), "+v"((s).s1)); __builtin_amdgcn_sched_barrier(0)

// How exp(z - m) of the hard term follows from exp((z - m) / T) of the soft one, e.  An exponential takes four issue slots of
// the vector unit, and with two of them per element and pass a wide row is bound by that unit, not by memory: the powers
// measured 4096 x 131072 in 515 us at T = 2 instead of the 602 of T = 3.
enum { EXP_ONE = 0,       // T = 1, or no hard term: one exponential
       EXP_TWO = 1,       // any T: a second one
       EXP_SQUARE = 2,    // T = 2: e^2
       EXP_FOURTH = 4 };  // T = 4: e^4
template <int MODE>
__device__ __forceinline__ float hard_exp(float e, float d) {
    if (MODE == EXP_TWO) return exp2_fast(d * DS_LOG2E);
    if (MODE == EXP_SQUARE) return e * e;
    if (MODE == EXP_FOURTH) return (e * e) * (e * e);
    return e;
}

// Running maximum with two sums of exponentials relative to it: st with factor kt = log2(e) / T, s1 with log2(e).
struct Stat {
    float m, st, s1;
};
template <int MODE>
__device__ __forceinline__ Stat merge(Stat a, Stat b, float kt) {
    Stat r;
    r.m = fmaxf(a.m, b.m);
    const float base = finite_or_zero(r.m), da = a.m - base, db = b.m - base;
    const float ea = exp2_fast(da * kt), eb = exp2_fast(db * kt);
    r.st = a.st * ea + b.st * eb;
    r.s1 = MODE ? a.s1 * hard_exp<MODE>(ea, da) + b.s1 * hard_exp<MODE>(eb, db) : r.st;
    return r;
}
template <int MODE>
__device__ __forceinline__ Stat wave_merge(Stat a, float kt) {
    const float m = wave_top(a.m), d = a.m - finite_or_zero(m), e = exp2_fast(d * kt);
    a.st = wave_total(a.st * e);
    a.s1 = MODE ? wave_total(a.s1 * hard_exp<MODE>(e, d)) : a.st;
    a.m = m;
    return a;
}
template <int MODE, int E>
__device__ __forceinline__ void accumulate(Stat& s, const float (&f)[E], float kt) {
    float vm = f[0];
#pragma unroll
    for (int e = 1; e < E; ++e) vm = fmaxf(vm, f[e]);
    const float m = fmaxf(s.m, vm), base = finite_or_zero(m);
    const float d0 = s.m - base, e0 = exp2_fast(d0 * kt);
    float st = s.st * e0, s1 = MODE ? s.s1 * hard_exp<MODE>(e0, d0) : 0.0f;
#pragma unroll
    for (int e = 0; e < E; ++e) {
        const float d = f[e] - base, x = exp2_fast(d * kt);
        st += x;
        if (MODE) s1 += hard_exp<MODE>(x, d);
    }
    s.m = m;
    s.st = st;
    s.s1 = MODE ? s1 : st;
}

// ------------------------------------------------------------------------------------------
// Loss and gradient.  With P the teacher's distribution over the listed classes, q = softmax(z / T) and w = grad_scale / B:
//   soft = sum_c P_c (log P_c - log q_c)  (+ the same term for the rest of both distributions when an lse is given)
//   hard = logsumexp(z) - z[label]
//   row loss = (1 - alpha) hard + alpha T^2 soft
//   d/dz_i = w (1 - alpha) (softmax(z)_i - [i = label]) + w alpha T (M q_i - P_i)              listed classes, or without an lse
//                                                       + w alpha T q_i (M q_r - P_r) / q_r    the others, q_r / P_r = the rests
// with M = sum P + P_r: 1, unless the lse is not that of the teacher's row, or the student has no rest to compare.
//
// Wave 0 reads the k slots while every wave's share of the row is on its way: it merges slots of one class (one bit per
// class in LDS finds them), and the bits also take the listed classes out of the sums of the rest: q_r is a sum of its
// own and never 1 - (a sum close to 1), relative to the rest's own maximum, so a student that is sure of the listed
// classes does not underflow it.  P_r has no such sum: it is 1 minus the listed mass, in 64 bits from the slots' exponents on (in
// fp32 a rest of 1e-5 was off by up to 6 %).  The main pass then writes c_T exp((z - m) / T) + c_1 exp(z - m) for every element, and
// after a barrier wave 0 rewrites the listed classes and the label (k + 1 elements).
// ------------------------------------------------------------------------------------------
#define DS_HEAD 256                 // bytes of the waves' statistics at the head of the LDS that is not row
typedef __attribute__((address_space(3))) void ds_lds_void_t;

struct DistillParams {
    const void* logits;
    const void* labels;
    const void* values;
    const void* indices;
    const float* lse;
    void* dlogits;
    float* row_loss;
    long long ld_in, ld_val, ld_idx, st_val, st_idx;
    int row0, N, k, ld_out;
    int label_bytes, index_bytes, value_type;
    float inv_t, w_soft_grad, w_hard_grad, w_soft_loss, w_hard_loss;
    double inv_t64;
};

template <typename T, int THREADS, int VPT, int VL, int MODE>
__global__ __launch_bounds__(THREADS) void distill_kernel(const DistillParams p) {
    constexpr int E = Pack<T>::E, W = THREADS / 64;
    // one array: next to a second one the compiler waits for the copies into LDS before it reads either
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];
    constexpr int HELD = VL * THREADS * 16;                        // the row's second part
    Stat* part = reinterpret_cast<Stat*>(lds + HELD);              // [W + 1]
    float* slot_sum = reinterpret_cast<float*>(part + W + 1);      // sum of P (negative: the row has no slots) and P_r
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = p.row0 + blockIdx.x, N = p.N, k = p.k;
    const int nv = (N + E - 1) / E;
    unsigned* bits = reinterpret_cast<unsigned*>(lds + HELD + DS_HEAD);
    const int words = ((N + 127) / 128) * 4;                       // a whole number of 16-byte stores
    int* s_idx = reinterpret_cast<int*>(bits + words);
    float* s_p = reinterpret_cast<float*>(s_idx + k);
    float* s_z = s_p + k;
    float* s_q = s_z + k;
    const T* src = static_cast<const T*>(p.logits) + (long long)row * p.ld_in;
    T* dst = static_cast<T*>(p.dlogits) + (long long)row * p.ld_out;
    const float kt = p.inv_t * DS_LOG2E;
    const bool rest = p.lse != nullptr;

    u32x4 r[VPT > 0 ? VPT : 1];
    auto load_row = [&]() {
        if (VPT > 0) {
#pragma unroll
            for (int j = 0; j < VPT; ++j) r[j] = ld_row<T, VPT == 1>(src, j * THREADS + tid, N);
        }
        if (VL > 0) {                                              // (rows of whole vectors: launcher)
            const __amdgpu_buffer_rsrc_t rsrc = make_rsrc(src, (unsigned)N * (unsigned)sizeof(T));
#pragma unroll
            for (int j = 0; j < VL; ++j)
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rsrc, (ds_lds_void_t*)(lds + (j * W + wave) * 1024), 16,
                                                         ((VPT + j) * THREADS + tid) * 16, 0, 0, 0);
        }
    };
    auto held = [&](int j) { return *reinterpret_cast<const u32x4*>(lds + (j * THREADS + tid) * 16); };

    // the slots (wave 0): classes, their bits, values
    int label = -1;
    float z_label = 0.0f, z_first = -INFINITY, tmax = -INFINITY;
    bool twice = false;
    auto load_slots = [&]() {
        for (int i = lane; i < words / 4; i += 64) reinterpret_cast<u32x4*>(bits)[i] = u32x4{0, 0, 0, 0};
        for (int s = lane; s < k; s += 64) {
            const long long oi = (long long)row * p.ld_idx + s * p.st_idx;
            const long long li = p.index_bytes == 8 ? static_cast<const long long*>(p.indices)[oi]
                                                    : (long long)static_cast<const int*>(p.indices)[oi];
            float t = ld_as_float(p.values, (long long)row * p.ld_val + s * p.st_val, p.value_type);
            const int i = li >= 0 && li < N && t != -INFINITY ? (int)li : -1;
            if (i < 0) t = -INFINITY;
            if (i >= 0) {
                twice |= (atomicOr(&bits[i >> 5], 1u << (i & 31)) >> (i & 31)) & 1u;
                if (s == lane) z_first = (float)src[i];            // (used after the pass over the row: nobody waits for it)
            }
            s_idx[s] = i;
            s_p[s] = t;
            tmax = t != t || tmax != tmax ? t + tmax : fmaxf(tmax, t);
        }
        if (label >= 0) z_label = (float)src[label];
    };
    if (p.labels) {
        const long long l = p.label_bytes == 8 ? static_cast<const long long*>(p.labels)[row]
                                               : (long long)static_cast<const int*>(p.labels)[row];
        label = l >= 0 && l < N ? (int)l : -1;
    }
    // loads return in order: the slots come first where the other waves wait for them and the row is long
    if (W > 1 && wave == 0) load_slots();
    load_row();
    if (W == 1) load_slots();
    if (rest) lds_barrier();                                       // the bits are complete
    if (wave == 0) {
        __builtin_amdgcn_wave_barrier();
        const bool any = __ballot(tmax != -INFINITY) != 0;         // a NaN counts: it shall reach the loss
        const float top = wave_top(tmax);
        const double base = rest ? (double)p.lse[row] : (double)top * p.inv_t64;
        double total = 0.0;
        for (int s = lane; s < k; s += 64) {
            const double e = s_idx[s] < 0 ? 0.0 : exp((double)s_p[s] * p.inv_t64 - base);
            s_p[s] = (float)e;
            total += e;
        }
        total = wave_total(total);
        if (!rest && any) {
            const float inv = 1.0f / (float)total;
            for (int s = lane; s < k; s += 64) s_p[s] *= inv;
            total = 1.0 + (total - total);                         // 1, or NaN
        }
        if (__ballot(twice)) {                                     // slots of one class: the first takes the sum, in slot order
            __builtin_amdgcn_wave_barrier();
            for (int s = lane; s < k; s += 64) {
                const int i = s_idx[s];
                float sum = 0.0f;
                bool first = i >= 0;
                for (int o = 0; o < k; ++o)
                    if (s_idx[o] == i) {
                        first &= o >= s;
                        sum += s_p[o];
                    }
                s_q[s] = first ? sum : -1.0f;
            }
            __builtin_amdgcn_wave_barrier();
            for (int s = lane; s < k; s += 64) {
                if (s_q[s] == -1.0f) s_idx[s] = -1;
                s_p[s] = s_q[s] == -1.0f ? 0.0f : s_q[s];
            }
        }
        if (lane == 0) slot_sum[0] = any ? (float)total : -1.0f, slot_sum[1] = (float)fmax(1.0 - total, 0.0);
    }

    Stat mine = {-INFINITY, 0.0f, 0.0f};
    // -inf for what this vector repeats of an earlier one and, with a rest, for the listed classes
    auto take_out = [&](u32x4 q, int v, bool whole) -> u32x4 {
        if (!whole) q = drop_repeated<T>(q, v, N);
        if (rest) {
            unsigned b;
            if (whole) {                                           // starts at a multiple of E: within one byte
                const unsigned c = (unsigned)v * E;
                b = reinterpret_cast<const unsigned char*>(bits)[c >> 3] >> (c & 7);
            } else {
                const int c = first_class<T>(v, N);
                b = bits[c >> 5] >> (c & 31);
                if ((c & 31) > 32 - E) b |= bits[(c >> 5) + 1] << (32 - (c & 31));
            }
            b &= (1u << E) - 1u;
            if (b) {
                float f[E];
                Pack<T>::unpack(q, f);
#pragma unroll
                for (int e = 0; e < E; ++e) f[e] = (b >> e) & 1u ? -INFINITY : f[e];
                q = Pack<T>::pack(f);
            }
        }
        return q;
    };
    if (VPT > 0) {
        const int t = anew(tid);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            r[j] = take_out(r[j], j * THREADS + t, (j + 1) * THREADS * E <= N);
            float f[E];
            Pack<T>::unpack(r[j], f);
            accumulate<MODE, E>(mine, f, kt);
            HOLD_STAT(r[j], mine);
        }
        if (VL > 0) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");       // what this wave copied into LDS is there: nobody else reads it
            for (int j = 0; j < VL; ++j) {
                const int v = (VPT + j) * THREADS + tid;
                if (v >= nv) break;
                const u32x4 q = take_out(held(j), v, true);
                if (rest) *reinterpret_cast<u32x4*>(lds + (j * THREADS + tid) * 16) = q;
                float f[E];
                Pack<T>::unpack(q, f);
                accumulate<MODE, E>(mine, f, kt);
            }
        }
    } else {
        for (int v = tid; v < nv; v += 4 * THREADS) {
            u32x4 q[4];
            const bool whole = (long long)(v - tid + 4 * THREADS) * E <= N;
#pragma unroll
            for (int u = 0; u < 4; ++u) q[u] = ld_row<T, false>(src, v + u * THREADS, N);
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                float f[E];
                Pack<T>::unpack(take_out(q[u], v + u * THREADS, whole), f);
                accumulate<MODE, E>(mine, f, kt);
            }
        }
    }
    if (wave == 0) {                                               // the listed classes' own logits and, with a rest, sums
        Stat own = {-INFINITY, 0.0f, 0.0f};
        for (int s = lane; s < k; s += 64) {
            const int i = s_idx[s];
            const float z = s == lane ? z_first : i >= 0 ? (float)src[i] : -INFINITY;
            s_z[s] = z;
            const float f[1] = {i >= 0 ? z : -INFINITY};
            if (rest) accumulate<MODE, 1>(own, f, kt);
        }
        own = wave_merge<MODE>(own, kt);
        if (lane == 0) part[W] = own;
    }
    mine = wave_merge<MODE>(mine, kt);
    if (lane == 0) part[wave] = mine;
    lds_barrier();

    // every wave works out the row's numbers for itself
    Stat a = part[0];
#pragma unroll
    for (int w = 1; w < W; ++w) a = merge<MODE>(a, part[w], kt);
    const Stat all = rest ? merge<MODE>(a, part[W], kt) : a;
    const float m = all.m;
    const bool some = m != -INFINITY || all.st != all.st;          // a row of -inf has no distribution: it counts for nothing
    const float sum_p = slot_sum[0], p_rest = slot_sum[1];
    const bool soft = some && !(sum_p < 0.0f) && p.w_soft_loss != 0.0f;
    const bool has_label = label >= 0 && some && p.w_hard_loss != 0.0f;
    const bool counts = __builtin_amdgcn_readfirstlane(soft || has_label);   // neither term: what the row holds reaches nothing
    const float base = finite_or_zero(a.m);
    const float inv_st = some ? 1.0f / all.st : 0.0f, inv_s1 = some ? 1.0f / all.s1 : 0.0f;
    const float q_rest = rest ? a.st * exp2_fast((a.m - m) * kt) * inv_st : 0.0f;
    const bool has_rest = rest && a.st > 0.0f;                     // nothing outside the list: no rest to compare
    const float mass = sum_p + (has_rest ? p_rest : 0.0f);
    float ct = 0.0f;
    if (soft) ct = rest ? (has_rest ? p.w_soft_grad * (mass * q_rest - p_rest) / a.st : 0.0f) : p.w_soft_grad * mass * inv_st;
    const float wh = has_label ? p.w_hard_grad : 0.0f;
    const float c1 = has_label ? wh * inv_s1 * (rest ? exp2_fast((a.m - m) * DS_LOG2E) : 1.0f) : 0.0f;   // (an empty row: m is -inf)
    const float cs = ct + c1;                                      // T = 1: one exponential serves both

    auto gradient = [&](u32x4 q, int v, bool whole) {
        float f[E], g[E];
        Pack<T>::unpack(q, f);
#pragma unroll
        for (int e = 0; e < E; ++e) {
            const float d = f[e] - base, x = exp2_fast(d * kt);
            if (MODE == EXP_TWO) g[e] = ct * x + c1 * exp2_fast(d * DS_LOG2E);
            else if (MODE == EXP_SQUARE) g[e] = x * (ct + c1 * x);
            else if (MODE == EXP_FOURTH) g[e] = x * (ct + (c1 * x) * (x * x));
            else g[e] = cs * x;
        }
        if (whole || (v + 1) * E <= N) {
            __builtin_nontemporal_store(Pack<T>::pack(g),
                                        reinterpret_cast<u32x4*>(reinterpret_cast<unsigned char*>(dst) + (unsigned)v * 16u));
        } else {
            const int c = first_class<T>(v, N), repeated = v * E - c;
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (e >= repeated && c + e < N) dst[c + e] = (T)g[e];
        }
    };
    if (!counts) {                                                 // zeros, not NaN times zero
        for (int c = tid * E; c < p.ld_out; c += THREADS * E) *reinterpret_cast<u32x4*>(dst + c) = u32x4{0, 0, 0, 0};
    } else if (VPT > 0) {
        const int t = anew(tid);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            gradient(r[j], j * THREADS + t, (j + 1) * THREADS * E <= N);
            hold(r[j]);
        }
        for (int j = 0; j < VL; ++j) {
            const int v = (VPT + j) * THREADS + tid;
            if (v >= nv) break;
            gradient(held(j), v, true);
        }
    } else {
        for (int v = tid; v < nv; v += 4 * THREADS) {
            u32x4 q[4];
            const bool whole = (long long)(v - tid + 4 * THREADS) * E <= N;
#pragma unroll
            for (int u = 0; u < 4; ++u) q[u] = ld_row<T, false>(src, v + u * THREADS, N);
#pragma unroll
            for (int u = 0; u < 4; ++u) gradient(take_out(q[u], v + u * THREADS, whole), v + u * THREADS, whole);
        }
    }
    for (int c = N + tid; c < p.ld_out; c += THREADS) dst[c] = (T)0.0f;   // the padding, whatever the row holds
    __syncthreads();                                               // the row is written: now the elements that differ
    if (wave != 0) return;
    float loss = 0.0f;
    const float log_st = some ? logf(all.st) : 0.0f;
    bool label_listed = false;
    for (int s = lane; s < k; s += 64) {
        const int i = s_idx[s];
        if (i < 0) continue;
        const float P = s_p[s], d = s_z[s] - finite_or_zero(m);
        if (soft && !(P == 0.0f)) loss += P * (logf(P) - (d * p.inv_t - log_st));
        float g = soft ? p.w_soft_grad * (mass * exp2_fast(d * kt) * inv_st - P) : 0.0f;
        if (has_label) g += wh * (exp2_fast(d * DS_LOG2E) * inv_s1 - (i == label ? 1.0f : 0.0f));
        dst[i] = (T)g;
        label_listed |= i == label;
    }
    loss = wave_total(loss);
    label_listed = __ballot(label_listed) != 0;
    if (lane == 0) {
        if (soft && has_rest && p_rest > 0.0f)
            loss += p_rest * (logf(p_rest) - ((a.m - m) * p.inv_t + logf(a.st) - log_st));
        loss *= p.w_soft_loss;
        if (has_label) {
            if (!label_listed) {
                const float d = z_label - base;
                const float g = ct * exp2_fast(d * kt) + wh * (exp2_fast((z_label - m) * DS_LOG2E) * inv_s1 - 1.0f);
                dst[label] = (T)g;
            }
            loss += p.w_hard_loss * (logf(all.s1) + (m - z_label));
        }
        p.row_loss[row] = loss;
    }
}

// Mean of the row losses in a fixed order: the same bits from run to run.
__global__ __launch_bounds__(256) void distill_mean_kernel(const float* __restrict__ v, float* __restrict__ out, int n) {
    __shared__ double red[256];
    double s = 0.0;
    for (long long i = threadIdx.x; i < n; i += 256) s += (double)v[i];
    red[threadIdx.x] = s;
    __syncthreads();
    for (int w = 128; w > 0; w >>= 1) {
        if (threadIdx.x < w) red[threadIdx.x] += red[threadIdx.x + w];
        __syncthreads();
    }
    if (threadIdx.x == 0) *out = n > 0 ? (float)(red[0] / (double)n) : 0.0f;
}

template <typename T, int MODE>
static void launch_distill(const DistillParams& p, int rows, hipStream_t s) {
    constexpr int NARROW = MODE == EXP_ONE ? EXP_ONE : EXP_TWO;    // (those are bound by latency, not by exponentials)
    constexpr int E = Pack<T>::E;
    const int nv = (p.N + E - 1) / E;
    const size_t shared = DS_HEAD + (size_t)((p.N + 127) / 128) * 16 + (size_t)p.k * 16;
    const dim3 grid(rows);
    // rows that start and end at 16-byte boundaries may be copied into LDS
    const bool whole = p.N % E == 0 && p.ld_in % E == 0 && ((unsigned long long)p.logits & 15) == 0;
#define DS_LAUNCH(TH, V, L, MD) \
    hipLaunchKernelGGL((distill_kernel<T, TH, V, L, MD>), grid, dim3(TH), shared + (size_t)L * TH * 16, s, p)
    if (nv <= 64) DS_LAUNCH(64, 1, 0, NARROW);
    else if (nv <= 128) DS_LAUNCH(64, 2, 0, NARROW);
    else if (nv <= 256) DS_LAUNCH(64, 4, 0, NARROW);
    else if (nv <= 1024) DS_LAUNCH(256, 4, 0, NARROW);
    else if (nv <= 4096) DS_LAUNCH(1024, 4, 0, MODE);
    else if (nv <= 8192 && whole) DS_LAUNCH(1024, 4, 4, MODE);
    else if (nv <= 8192) DS_LAUNCH(1024, 8, 0, MODE);
    else if (nv <= 16384 && whole) DS_LAUNCH(1024, 8, 8, MODE);
    else DS_LAUNCH(1024, 0, 0, MODE);
#undef DS_LAUNCH
}

template <typename T>
static void launch_distill(const DistillParams& p, int rows, int mode, hipStream_t s) {
    if (mode == EXP_ONE) launch_distill<T, EXP_ONE>(p, rows, s);
    else if (mode == EXP_SQUARE) launch_distill<T, EXP_SQUARE>(p, rows, s);
    else if (mode == EXP_FOURTH) launch_distill<T, EXP_FOURTH>(p, rows, s);
    else launch_distill<T, EXP_TWO>(p, rows, s);
}

// Status -1: an argument outside what the kernel is built for (nothing was launched).
PDT_API int pdt_distill_ce(const void* logits, const void* labels, const void* values, const void* indices, const void* lse,
                           void* dlogits, void* row_loss, void* loss, int B, int N, int k, long long ld_in, long long ld_val,
                           long long st_val, long long ld_idx, long long st_idx, int ld_out, int type, int value_type,
                           int label_bytes, int index_bytes, double temperature, float alpha, float grad_scale,
                           hipStream_t s) {
    if (B < 0 || N < 1 || N > DS_MAX_CLASSES || k < 1 || k > DS_MAX_K || ld_out < N || ld_out % 64 != 0) return -1;
    if (type < 0 || type > 2 || value_type < 0 || value_type > 2 || (label_bytes != 4 && label_bytes != 8)) return -1;
    if ((index_bytes != 4 && index_bytes != 8) || !(temperature > 0.0)) return -1;
    if (B > 0) {
        DistillParams p;
        p.logits = logits, p.labels = labels, p.values = values, p.indices = indices;
        p.lse = static_cast<const float*>(lse);
        p.dlogits = dlogits, p.row_loss = static_cast<float*>(row_loss);
        p.ld_in = ld_in, p.ld_val = ld_val, p.ld_idx = ld_idx, p.st_val = st_val, p.st_idx = st_idx;
        p.N = N, p.k = k, p.ld_out = ld_out;
        p.label_bytes = label_bytes, p.index_bytes = index_bytes, p.value_type = value_type;
        p.inv_t64 = 1.0 / temperature;
        p.inv_t = (float)p.inv_t64;
        p.w_soft_loss = (float)(alpha * temperature * temperature);
        p.w_hard_loss = labels ? 1.0f - alpha : 0.0f;
        p.w_soft_grad = (float)(alpha * temperature * grad_scale / B);
        p.w_hard_grad = p.w_hard_loss * grad_scale / (float)B;
        const int mode = p.w_hard_loss == 0.0f || temperature == 1.0 ? EXP_ONE
                         : temperature == 2.0                         ? EXP_SQUARE
                         : temperature == 4.0                         ? EXP_FOURTH
                                                                      : EXP_TWO;
        for (long long row = 0; row < B; row += DS_ROWS) {
            const int rows = (int)(B - row < DS_ROWS ? B - row : DS_ROWS);
            p.row0 = (int)row;
            if (type == DS_BF16) launch_distill<bf16>(p, rows, mode, s);
            else if (type == DS_FP16) launch_distill<f16>(p, rows, mode, s);
            else launch_distill<float>(p, rows, mode, s);
            const int rc = pdt_launch_status();
            if (rc != 0) return rc;
        }
    }
    hipLaunchKernelGGL(distill_mean_kernel, dim3(1), dim3(256), 0, s, (const float*)row_loss, (float*)loss, B);
    return pdt_launch_status();
}

// ------------------------------------------------------------------------------------------
// The k largest logits of a row in falling order (ties: lower class first; a NaN before every number; classes at -inf
// never) and the row's logsumexp at temperature T.
//
// A lower bound of the k-th largest comes from the threads' own maxima: with W waves, the smallest over the waves of the
// ceil(k / W)-th largest lane maximum has at least k elements at or above it, and for values in no particular order only
// a few times k.  Those candidates go to LDS as 64-bit keys (value, then class) and are sorted there; the keys differ, so
// the order in which the candidates arrive does not matter.  The bound is taken from the row's first chunk, which waits for it
// in registers, and again whenever twice as much has been read; the rest of the row streams past it: the row is read once.
// Rows on which the bound is too low (many equal values, sorted rows) or that hold a NaN or +inf are cut to exactly k
// candidates by bisecting the value and, among equals, the class: exact, some 50 more passes over the row.
// Measured: 2048 x 131072 bf16, k = 64, in 125 us, 4.3 TB/s; 1536 x 1000, k = 10, in 6.8 us; 3 x 50001 fp16, k = 100, in 16 us of
// latency, by the clock 17 % the first chunk and its bound, 16 % its candidates, 16 % the rest of the row, 20 % the statistics'
// merge and 30 % the sort of 264 to 382 candidates.
// ------------------------------------------------------------------------------------------
struct TopParams {
    const void* logits;
    void* values;
    int* indices;
    float* lse;
    long long ld_in;
    int row0, N, k;
    float inv_t;
    double inv_t64;
};

// unsigned order = float order; -0 = +0, NaN on top
__device__ __forceinline__ unsigned order_key(float f) {
    if (f != f) return 0xffffffffu;
    const unsigned u = __float_as_uint(f + 0.0f);
    return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ unsigned long long slot_key(float f, int c) {
    return (unsigned long long)order_key(f) << 32 | (unsigned)~c;
}
__device__ __forceinline__ unsigned long long shfl_xor_u64(unsigned long long v, int mask) {
    const unsigned lo = __shfl_xor((unsigned)v, mask, 64), hi = __shfl_xor((unsigned)(v >> 32), mask, 64);
    return (unsigned long long)hi << 32 | lo;
}

template <typename T, int THREADS, int VPT>
__global__ __launch_bounds__(THREADS) void top_logits_kernel(const TopParams p) {
    constexpr int E = Pack<T>::E, W = THREADS / 64, CAP = THREADS == 64 ? 512 : THREADS == 256 ? 2048 : 4096;
    __shared__ unsigned long long cand[CAP];
    __shared__ Stat part[W];
    __shared__ float bound[2][W];
    __shared__ int tally[W];
    __shared__ int count;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int row = p.row0 + blockIdx.x, N = p.N, k = p.k;
    const int nv = (N + E - 1) / E;
    const T* src = static_cast<const T*>(p.logits) + (long long)row * p.ld_in;
    const float kt = p.inv_t * DS_LOG2E;
    if (tid == 0) count = 0;                                       // (a barrier follows before the first use)

    auto keep = [&](float f, int c) {
        const int at = atomicAdd(&count, 1);
        if (at < CAP) cand[at] = slot_key(f, c);
    };
    Stat mine = {-INFINITY, 0.0f, 0.0f};
    int turn = 0;
    float floor_v = -INFINITY;
    const int rank = (k + W - 1) / W;                              // at most 64 (launcher)
    auto raise_floor = [&]() {                                     // (all threads)
        // the 16 leading bits of the rank-th largest maximum of the wave: bisected with ballots
        const unsigned key = order_key(mine.m);
        unsigned t = 0;
#pragma unroll
        for (int b = 31; b >= 16; --b) {
            const unsigned c = t | 1u << b;
            if (__popcll(__ballot(key >= c)) >= rank) t = c;
        }
        if (lane == 0) bound[turn][wave] = t <= 0x007fffffu ? -INFINITY : __uint_as_float(t & 0x80000000u ? t ^ 0x80000000u : ~t);
        lds_barrier();
        float f = bound[turn][0];
#pragma unroll
        for (int w = 1; w < W; ++w) f = fminf(f, bound[turn][w]);
        floor_v = f;
        turn ^= 1;                                                 // the next round writes the other set: one barrier each
    };
    auto collect = [&](const float (&f)[E], int v) {
        float m = f[0];
#pragma unroll
        for (int e = 1; e < E; ++e) m = fmaxf(m, f[e]);
        if (m >= floor_v) {
            const int c = first_class<T>(v, N);
#pragma unroll
            for (int e = 0; e < E; ++e)
                if (f[e] >= floor_v && f[e] != -INFINITY) keep(f[e], c + e);
        }
    };
    {
        u32x4 r[VPT];
#pragma unroll
        for (int j = 0; j < VPT; ++j) r[j] = ld_row<T, VPT == 1>(src, j * THREADS + tid, N);
        int t = anew(tid);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            if ((j + 1) * THREADS * E > N) r[j] = drop_repeated<T>(r[j], j * THREADS + t, N);
            float f[E];
            Pack<T>::unpack(r[j], f);
            accumulate<EXP_ONE, E>(mine, f, kt);
            HOLD_STAT(r[j], mine);
        }
        raise_floor();
        t = anew(tid);
#pragma unroll
        for (int j = 0; j < VPT; ++j) {
            float f[E];
            Pack<T>::unpack(r[j], f);
            collect(f, j * THREADS + t);
            hold(r[j]);
        }
    }
    // the rest, two vectors at a time with the next two on their way
    constexpr int U = 2;
    if (nv > VPT * THREADS) {
        u32x4 q[U];
#pragma unroll
        for (int u = 0; u < U; ++u) q[u] = ld_row<T, false>(src, VPT * THREADS + u * THREADS + tid, N);
        int raise_at = 2 * VPT * THREADS;                          // vectors read when the floor is raised next
        for (int v0 = VPT * THREADS; v0 < nv; v0 += U * THREADS) {
            u32x4 nx[U];
#pragma unroll
            for (int u = 0; u < U; ++u) nx[u] = ld_row<T, false>(src, v0 + (U + u) * THREADS + tid, N);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int v = v0 + u * THREADS + tid;
                if ((v0 + (u + 1) * THREADS) * E > N) q[u] = drop_repeated<T>(q[u], v, N);
                float f[E];
                Pack<T>::unpack(q[u], f);
                accumulate<EXP_ONE, E>(mine, f, kt);
                collect(f, v);
                HOLD_STAT(nx[u], mine);
                q[u] = nx[u];
            }
            if (v0 + U * THREADS == raise_at && raise_at < nv) {
                raise_floor();
                raise_at *= 2;
            }
        }
    }
    mine = wave_merge<EXP_ONE>(mine, kt);
    if (lane == 0) part[wave] = mine;
    lds_barrier();
    if (tid == 0) {
        Stat a = part[0];
        for (int w = 1; w < W; ++w) a = merge<EXP_ONE>(a, part[w], kt);
        // m / T in 64 bits: rounded with the sum, once (distill_ce subtracts it from values / T in 64 bits)
        p.lse[row] = (float)((double)finite_or_zero(a.m) * p.inv_t64 + (double)logf(a.st));
    }
    int n = count;
    bool plain = true;                                             // no NaN, no +inf: those make the sum NaN
#pragma unroll
    for (int w = 0; w < W; ++w) plain &= part[w].st == part[w].st;

    auto over_row = [&](auto&& fn) {                               // fn(values, first class) for every vector of this thread
        for (int v = tid; v < nv; v += THREADS) {
            float f[E];
            Pack<T>::unpack(drop_repeated<T>(ld_row<T, true>(src, v, N), v, N), f);
            fn(f, first_class<T>(v, N));
        }
    };
    if (n > CAP || !plain) {
        auto total = [&](int mine_n) {
            const int t = (int)wave_total((float)mine_n);            // below 2^24: exact
            lds_barrier();                                         // the last round's tallies have been read
            if (lane == 0) tally[wave] = t;
            lds_barrier();
            int s = 0;
#pragma unroll
            for (int w = 0; w < W; ++w) s += tally[w];
            return s;
        };
        int filled = 0, nans = 0;
        over_row([&](const float (&f)[E], int) {
#pragma unroll
            for (int e = 0; e < E; ++e) filled += f[e] != -INFINITY, nans += f[e] != f[e];
        });
        const int want = min(k, total(filled));
        if (!plain && total(nans) == 0 && tid == 0) p.lse[row] = INFINITY;   // +inf and no NaN
        unsigned t = 0;                                            // largest key that `want` elements reach
        for (int b = 31; b >= 0; --b) {
            const unsigned c = t | 1u << b;
            int m = 0;
            over_row([&](const float (&f)[E], int) {
#pragma unroll
                for (int e = 0; e < E; ++e) m += f[e] != -INFINITY && order_key(f[e]) >= c;
            });
            if (total(m) >= want) t = c;
        }
        int above = 0;
        over_row([&](const float (&f)[E], int) {
#pragma unroll
            for (int e = 0; e < E; ++e) above += f[e] != -INFINITY && order_key(f[e]) > t;
        });
        const int need = want - total(above);
        int lo = 0, hi = N - 1;                                    // smallest class up to which `need` elements equal the key
        while (lo < hi) {
            const int mid = lo + (hi - lo) / 2;
            int m = 0;
            over_row([&](const float (&f)[E], int c) {
#pragma unroll
                for (int e = 0; e < E; ++e) m += f[e] != -INFINITY && order_key(f[e]) == t && c + e <= mid;
            });
            if (total(m) >= need) hi = mid;
            else lo = mid + 1;
        }
        lds_barrier();
        if (tid == 0) count = 0;
        lds_barrier();
        over_row([&](const float (&f)[E], int c) {
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const unsigned key = order_key(f[e]);
                if (f[e] != -INFINITY && (key > t || (key == t && c + e <= lo))) keep(f[e], c + e);
            }
        });
        lds_barrier();
        n = count;
    }

    T* values = static_cast<T*>(p.values) + (long long)row * k;
    int* indices = p.indices + (long long)row * k;
    auto put = [&](int s, unsigned long long key, bool filled) {
        const int c = (int)~(unsigned)key;
        values[s] = filled ? src[c] : (T)-INFINITY;
        indices[s] = filled ? c : -1;
    };
    // bitonic sort, largest first.  Steps of 32 and less run in registers; those of 64 and more through LDS, with a barrier each
    // (all 55 steps of 1024 keys through LDS: 3 rows of 50001 with k = 100 take 20.8 us, with 45 in registers 15.9)
    auto wave_steps = [&](unsigned long long key, int i, int size, int step) {
        for (; step > 0; step >>= 1) {
            const unsigned long long o = shfl_xor_u64(key, step);
            const bool take_max = ((i & step) == 0) == ((i & size) == 0);
            key = (key > o) == take_max ? key : o;
        }
        return key;
    };
    if (n <= 64) {
        if (wave != 0) return;
        unsigned long long key = lane < n ? cand[lane] : 0ull;
        for (int size = 2; size < 2 * n; size <<= 1) key = wave_steps(key, lane, size, size >> 1);   // (lanes past the next power of two keep their zeros)
        for (int s = lane; s < k; s += 64) put(s, key, s == lane && s < n);
        return;
    }
    int size2 = 128;
    while (size2 < n) size2 <<= 1;
    for (int i = tid; i < size2; i += THREADS) {
        unsigned long long key = i < n ? cand[i] : 0ull;
        for (int size = 2; size <= 64; size <<= 1) key = wave_steps(key, i, size, size >> 1);
        cand[i] = key;
    }
    lds_barrier();
    for (int size = 128; size <= size2; size <<= 1) {
        for (int step = size >> 1; step >= 64; step >>= 1) {
            for (int i = tid; i < size2 / 2; i += THREADS) {
                const int a = 2 * i - (i & (step - 1)), b = a + step;
                const unsigned long long x = cand[a], y = cand[b];
                if ((x < y) == ((a & size) == 0)) {
                    cand[a] = y;
                    cand[b] = x;
                }
            }
            lds_barrier();
        }
        for (int i = tid; i < size2; i += THREADS) cand[i] = wave_steps(cand[i], i, size, 32);
        lds_barrier();
    }
    for (int s = tid; s < k; s += THREADS) put(s, cand[s], s < n);
}

template <typename T>
static void launch_top(const TopParams& p, int B, int rows, hipStream_t s) {
    const int nv = (p.N + Pack<T>::E - 1) / Pack<T>::E;
#define DS_LAUNCH(TH, V) hipLaunchKernelGGL((top_logits_kernel<T, TH, V>), dim3(rows), dim3(TH), 0, s, p)
    // at least two threads per wanted logit: with fewer the bound from the thread maxima lets too many candidates pass.
    // Wide rows: small workgroups where there are rows for several on every CU (one's loads run under another's sort)
    const bool many = B >= 4 * 256;
    if (nv <= 64 && p.k <= 32) DS_LAUNCH(64, 1);
    else if (nv <= 128 && p.k <= 32) DS_LAUNCH(64, 2);
    else if (nv <= 256 && p.k <= 32) DS_LAUNCH(64, 4);
    else if ((nv <= 1024 || many) && p.k <= 128) DS_LAUNCH(256, 4);
    else DS_LAUNCH(1024, 4);
#undef DS_LAUNCH
}

// Status -1: an argument outside what the kernel is built for (nothing was launched).
PDT_API int pdt_top_logits(const void* logits, void* values, void* indices, void* lse, int B, int N, int k, long long ld_in,
                           int type, double temperature, hipStream_t s) {
    if (B < 0 || N < 1 || k < 1 || k > DS_MAX_K || k > N || N > (1 << 24) || type < 0 || type > 2 || !(temperature > 0.0))
        return -1;
    if (B == 0) return 0;
    TopParams p;
    p.logits = logits, p.values = values, p.indices = static_cast<int*>(indices), p.lse = static_cast<float*>(lse);
    p.ld_in = ld_in, p.N = N, p.k = k, p.inv_t64 = 1.0 / temperature, p.inv_t = (float)p.inv_t64;
    for (long long row = 0; row < B; row += DS_ROWS) {
        const int rows = (int)(B - row < DS_ROWS ? B - row : DS_ROWS);
        p.row0 = (int)row;
        if (type == DS_BF16) launch_top<bf16>(p, B, rows, s);
        else if (type == DS_FP16) launch_top<f16>(p, B, rows, s);
        else launch_top<float>(p, B, rows, s);
        const int rc = pdt_launch_status();
        if (rc != 0) return rc;
    }
    return 0;
}
