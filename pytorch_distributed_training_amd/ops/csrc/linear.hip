// Matrix products of a classifier / MLP head with everything around them in the epilogue, bf16 in, fp32 accumulation on
// the matrix cores (v_mfma_f32_16x16x32_bf16), each result rounded to bf16 once:
//
//   forward     z = a w^T + bias,  y = act(z) + residual          a [M][K], w [N][K]
//   gradients   da = dz w,  dw = dz^T a,  dbias = column sums of dz,  dz = dy act'(z)
//
// One tile kernel serves the three products.  An operand is either K-contiguous (its reduction index is the fast one: a and w
// forward, dz for da) or K-strided (w for da, dz and a for dw); both are staged as they lie in memory by LDS-DMA
// (buffer_load ... lds, no staging registers) and differ in how fragments are read back: ds_read_b128 for the first,
// the transposing ds_read_b64_tr_b16 for the second.  No operand is ever transposed in memory.
//
// Sizes in this file are M x N x K of the layer or, at the cost rules, of one product: rows x columns x reduction (elsewhere in the
// repository a layer is rows x inner x outer, M x K x N).
//
// Bound by the matrix cores where the tiles fill the chip: 8192 x 4096 x 16384 forward with a residual in 808 us, 1360 TFLOP/s (the
// library's bare product: 695 us); both gradients and dbias of 4096 x 16384 x 4096 in 881 us, 1250 TFLOP/s (the library's two bare
// products: 884).  Smaller products are bound by the latency of one tile and by launches, so they get smaller tiles, a split K or
// one launch for both gradients, whichever the measured costs at plan_of() favour; up to 64 rows, by the weights' way through memory.
#include "common.h"
#include <type_traits>

#define LIN_NONE 0
#define LIN_RELU 1
#define LIN_GELU 2
#define LIN_SILU 3

#define OUT_BF16 0       // epilogue, bf16
#define OUT_ADD 1        // fp32, added to what is there (gradient buffers)
#define OUT_PART 2       // fp32 partial sums of one K range, joined by linear_join_kernel

typedef __attribute__((ext_vector_type(2))) float f32x2;
typedef __attribute__((ext_vector_type(2))) unsigned u32x2;
typedef u32x4 __attribute__((aligned(2))) u32x4_a2;           // global memory takes unaligned vector accesses
typedef u32x2 __attribute__((aligned(2))) u32x2_a2;
typedef __attribute__((address_space(3))) void lin_lds_void_t;

// ------------------------------------------------------------------------------------------ activations
// Phi(-|z|) of the normal distribution as exp(-z^2 / 2) / 2 times exp(x^2) erfc(x), x = |z| / sqrt(2): the second factor falls
// slowly, from 1 to 0.06 at |z| = 13, and is a polynomial in t = 1 / (1 + 0.375 x) (t^1 .. t^7, minimax fit of the relative error on
// 0 <= x <= 10: 6.4e-7).  So the tail has its digits relative to its own value: evaluated in fp32 it is off by 1.1e-6 up to
// |z| = 2 and 8e-6 up to 13, nearly all of it the rounded argument of the exponential, which also is the density that the
// derivative needs.  Below z = -13.2 the exponential is less than 2^-126 and taken as zero.  (The five-term approximation that is
// good to 7.5e-8 absolute was off by 0.2 % of the value at -5 and 3 % at -12, beyond bf16's half step of 0.4 %.)
__device__ __forceinline__ float normal_tail(float z, float& density) {
    const float t = __builtin_amdgcn_rcpf(1.0f + 0.26516503f * fabsf(z));
    const float e = __builtin_amdgcn_exp2f(z * z * -0.72134752044448170f);
    density = e * 0.39894228040143268f;
    return e * t * (0.10566973f + t * (0.10784456f + t * (0.083332427f + t * (0.14153039f + t * (-0.064798117f + t * (0.19396853f + t * -0.067547843f))))));
}
__device__ __forceinline__ float sigmoid(float z) {
    return __builtin_amdgcn_rcpf(1.0f + __builtin_amdgcn_exp2f(-1.44269504088896341f * z));
}
__device__ __forceinline__ float act_value(float z, int act) {
    if (act == LIN_RELU) return z < 0.0f ? 0.0f : z;          // a NaN stays one
    if (act == LIN_GELU) {
        float d;
        const float h = normal_tail(z, d);
        if (z == -INFINITY) return 0.0f;                       // (0 times infinity)
        return z > 0.0f ? z * (1.0f - h) : z * h;
    }
    if (act == LIN_SILU) return z == -INFINITY ? 0.0f : z * sigmoid(z);
    return z;
}
__device__ __forceinline__ float act_slope(float z, int act) {
    if (act == LIN_RELU) return z > 0.0f ? 1.0f : (z != z ? z : 0.0f);
    if (act == LIN_GELU) {
        float d;
        const float h = normal_tail(z, d);
        if (fabsf(z) == INFINITY) return z > 0.0f ? 1.0f : 0.0f;
        return (z > 0.0f ? 1.0f - h : h) + z * d;
    }
    if (act == LIN_SILU) {
        const float s = sigmoid(z);
        return z == -INFINITY ? 0.0f : (z == INFINITY ? 1.0f : s * (1.0f + z * (1.0f - s)));
    }
    return 1.0f;
}

// ------------------------------------------------------------------------------------------ epilogue
struct Epilogue {
    void* out;
    bf16* z;                   // pre-activation, or null
    const float* bias;         // [N], or null
    const bf16* res;           // [M][ldr], or null
    float* ws;                 // OUT_PART: slabs [splits][M][N]
    long long ldr;
    int ldo, n_pad;            // row stride of out and z; columns N .. n_pad - 1 are written as zeros
    int M, N, mode, act, vec;  // vec: rows of out (and z) allow stores of 8 values
};

__device__ __forceinline__ unsigned pack_bf16(float lo, float hi) {
    const bf16x2 p = __builtin_convertvector((f32x2){lo, hi}, bf16x2);
    return __builtin_bit_cast(unsigned, p);
}
__device__ __forceinline__ float lo_bf16(unsigned u) { return __uint_as_float(u << 16); }
__device__ __forceinline__ float hi_bf16(unsigned u) { return __uint_as_float(u & 0xffff0000u); }

template <int G>
__device__ __forceinline__ void st_group(bf16* p, const float (&v)[G]) {
    if (G == 8) {
        *reinterpret_cast<u32x4*>(p) = u32x4{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3]), pack_bf16(v[G - 4], v[G - 3]),
                                             pack_bf16(v[G - 2], v[G - 1])};
    } else {
        *reinterpret_cast<u32x2*>(p) = u32x2{pack_bf16(v[0], v[1]), pack_bf16(v[2], v[3])};
    }
}
template <int G>
__device__ __forceinline__ void ld_group(const bf16* p, float (&v)[G]) {
    if (G == 8) {
        const u32x4 u = *reinterpret_cast<const u32x4_a2*>(p);
#pragma unroll
        for (int i = 0; i < 4; ++i) v[(2 * i) % G] = lo_bf16(u[i]), v[(2 * i + 1) % G] = hi_bf16(u[i]);
    } else {
        const u32x2 u = *reinterpret_cast<const u32x2_a2*>(p);
        v[0] = lo_bf16(u[0]), v[1] = hi_bf16(u[0]), v[2] = lo_bf16(u[1]), v[3] = hi_bf16(u[1]);
    }
}

// G neighbouring columns n .. n+G-1 (n a multiple of G) of row m; b: their bias.
template <int G>
__device__ __forceinline__ void finish_bf16(const Epilogue& p, int m, int n, float (&v)[G], const float (&b)[G]) {
    if (m >= p.M || n >= p.n_pad) return;
    const long long o = (long long)m * p.ldo + n;
    const bool whole = n + G <= p.N;
    float r[G];
    if (p.res) {
        const bf16* src = p.res + (long long)m * p.ldr + n;
        if (whole) ld_group<G>(src, r);
        else {
#pragma unroll
            for (int e = 0; e < G; ++e) r[e] = n + e < p.N ? (float)src[e] : 0.0f;
        }
    }
#pragma unroll
    for (int e = 0; e < G; ++e) v[e] += b[e];
    if (!whole) {
#pragma unroll
        for (int e = 0; e < G; ++e) v[e] = n + e < p.N ? v[e] : 0.0f;
    }
    const bool wide = p.vec && n + G <= p.n_pad;
    if (p.z) {
        if (wide) st_group<G>(p.z + o, v);
        else {
#pragma unroll
            for (int e = 0; e < G; ++e)
                if (n + e < p.n_pad) p.z[o + e] = (bf16)v[e];
        }
    }
    if (p.act != LIN_NONE) {
#pragma unroll
        for (int e = 0; e < G; ++e) v[e] = act_value(v[e], p.act);
    }
    if (p.res) {
#pragma unroll
        for (int e = 0; e < G; ++e) v[e] += r[e];
    }
    bf16* out = static_cast<bf16*>(p.out) + o;
    if (wide) st_group<G>(out, v);
    else {
#pragma unroll
        for (int e = 0; e < G; ++e)
            if (n + e < p.n_pad) out[e] = (bf16)v[e];
    }
}
template <int G>
__device__ __forceinline__ void finish_add(const Epilogue& p, int m, int n, const float (&v)[G]) {
    if (m >= p.M) return;
    float* out = static_cast<float*>(p.out) + (long long)m * p.ldo + n;
    if (p.vec && n + G <= p.N) {                               // one writer per element
#pragma unroll
        for (int e = 0; e < G; e += 4) *reinterpret_cast<f32x4*>(out + e) += f32x4{v[e], v[e + 1], v[e + 2], v[e + 3]};
        return;
    }
#pragma unroll
    for (int e = 0; e < G; ++e)
        if (n + e < p.N) out[e] += v[e];
}
template <int G>
__device__ __forceinline__ void ld_bias(const Epilogue& p, int n, float (&b)[G]) {
#pragma unroll
    for (int e = 0; e < G; ++e) b[e] = p.bias && n + e < p.N ? p.bias[n + e] : 0.0f;
}

// Partial sums: [splits][M][slab_ld(N)], rows of whole 8-column groups.
__host__ __device__ __forceinline__ long long slab_ld(int N) { return (N + 7) / 8 * 8; }

// ------------------------------------------------------------------------------------------ tile kernel
struct GemmParams {
    const bf16* a;
    const bf16* b;
    unsigned long long a_bytes, b_bytes;
    int lda, ldb, K;                   // K: reduction length, a multiple of 8 where an operand is K-contiguous
    int splits, steps;                 // K ranges and 64-wide steps of one range
    int tiles_m, tiles_n;
    Epilogue ep;
};

#define LIN_BK 64

__device__ __forceinline__ bf16x8 lin_tr_pair(const unsigned char* lo, const unsigned char* hi) {
    typedef __attribute__((address_space(3))) s16x4 lds_s16x4;
    union { struct { s16x4 a, b; } s; bf16x8 v; } u;
    u.s.a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)lo);
    u.s.b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4*)hi);
    return u.v;
}

// One operand of the tile: how its DMA is addressed and its fragments are read.  TR: K-strided.  R: rows (columns of the
// memory image if TR) of the tile, NW: waves of the workgroup, PERM: fragment rows permuted (below).
//
// K-contiguous image: [R][64] bf16, 128-byte rows; LDS chunk c (16 bytes) of row r holds chunk c ^ key, key = (r >> 1) & 7,
// so that the 16 rows of a fragment read fall on different banks.
// K-strided image: [64][R], 2R-byte rows; a transposing read takes 4 k-rows x 16 columns per 16 lanes, and 32 lanes (rows
// {0-3, 8-11} or {4-7, 12-15} of a 16-row group) are served at once: chunk c of row r holds chunk c ^ 2 key with
// key = (r & 3) | (r >> 1 & 4), which puts those 8 rows on different banks.
// PERM: which row of the operand an MFMA row stands for is free.  Row 16 (x >> 2) + 4 j + (x & 3) for row x of block j leaves
// a lane with 16 neighbouring columns of the result; the key then follows x.
template <bool TR, int R, int NW, bool PERM>
struct Operand {
    static constexpr int BK = LIN_BK, BYTES = R * BK * 2, PER = BYTES / 1024 / NW;
    static_assert(PER >= 1, "every wave takes part in staging");
    static_assert(!(TR && PERM), "the permutation would put a transposing read's rows on the same banks");
    unsigned voff[PER];
    unsigned long long ptr;
    long long left;
    unsigned step;

    static __device__ __forceinline__ int key(int row) {
        if (PERM) row = ((row >> 4) & 3) * 4 + (row & 3);
        return (row >> 1) & 7;
    }
    __device__ __forceinline__ static int dma_row(int wave, int lane, int j) {
        return TR ? (wave * PER + j) * (512 / R) + lane / (R / 8) : (wave * PER + j) * 8 + lane / 8;
    }
    __device__ __forceinline__ static int dma_chunk(int lane, int row) {
        return TR ? (lane % (R / 8)) ^ (2 * ((row & 3) | (row >> 1 & 4))) : (lane % 8) ^ key(row);
    }
    __device__ __forceinline__ void init(const bf16* x, unsigned long long bytes, int ld, int row0, int k0, int wave, int lane) {
#pragma unroll
        for (int j = 0; j < PER; ++j) {
            const int row = dma_row(wave, lane, j);
            voff[j] = (unsigned)row * (unsigned)ld * 2u + (unsigned)dma_chunk(lane, row) * 16u;
        }
        const unsigned long long off = TR ? ((unsigned long long)k0 * (unsigned)ld + (unsigned)row0) * 2ull
                                          : ((unsigned long long)row0 * (unsigned)ld + (unsigned)k0) * 2ull;
        ptr = (unsigned long long)x + off;
        left = (long long)bytes - (long long)off;
        step = TR ? (unsigned)(BK * 2) * (unsigned)ld : BK * 2u;
    }
    __device__ __forceinline__ u32x4 desc() const {
        const unsigned n = left <= 0 ? 0u : (left < 0x7fff0000ll ? (unsigned)left : 0x7fff0000u);
        return u32x4{(unsigned)ptr, (unsigned)(ptr >> 32) & 0xffffu, n, 0x00020000u};
    }
    // piece j of this wave's share of a stage, to LDS offset m (moved on to the next piece's).  TAIL: `rem` may be less than a
    // stage: a K-contiguous row goes on behind K, those chunks are taken as zeros (a K-strided operand ends there, and the
    // range check returns zeros)
    template <bool TAIL>
    __device__ __forceinline__ void piece(u32x4 d, unsigned& m, int rem, int j, int wave, int lane) const {
        unsigned v = voff[j];
        if (TAIL && !TR) v = dma_chunk(lane, dma_row(wave, lane, j)) * 8 < rem ? v : PDT_OOB_OFFSET;
        asm volatile("s_mov_b32 m0, %0\n\ts_add_u32 %0, %0, 0x400\n\tbuffer_load_dwordx4 %1, %2, 0 offen lds"
                     : "+s"(m) : "v"(v), "s"(d) : "memory", "scc");
    }
    __device__ __forceinline__ void next() {
        ptr += step;
        left -= step;
    }
    // fragment of 16 rows (block f of the wave's rows, which start at row0) and 32 k (half kk)
    __device__ __forceinline__ static bf16x8 read(const unsigned char* lds, int row0, int f, int kk, int lane) {
        if (TR) {
            const int g = lane >> 4, q = (lane & 15) >> 2, pp = lane & 3;
            const int r = kk * 32 + 8 * g + q, k2 = 2 * (q | (g & 1) * 4);
            const int chunk = ((row0 + f * 16) / 8 + (pp >> 1)) ^ k2;
            const unsigned char* at = lds + r * (R * 2) + chunk * 16 + (pp & 1) * 8;
            return lin_tr_pair(at, at + 4 * (R * 2));
        }
        const int x = lane & 15;
        const int row = row0 + (PERM ? (f >> 2) * 64 + 16 * (x >> 2) + 4 * (f & 3) + (x & 3) : f * 16 + x);
        return *reinterpret_cast<const bf16x8*>(lds + row * (BK * 2) + (((kk * 4 + (lane >> 4)) ^ key(row)) << 4));
    }
};

// tile `block` of `p`; smem: RING slots
template <int BM, int BN, int RING, bool AT, bool BT>
__device__ __forceinline__ void gemm_tile(const GemmParams& p, const int block, unsigned char* smem) {
    constexpr int WM = 2, WN = 2, NW = WM * WN, BK = LIN_BK, WTM = BM / WM, WTN = BN / WN, MI = WTM / 16, NI = WTN / 16;
    static_assert(RING % 2 == 1 && RING >= 5 && BM <= BN, "the slots are filled by a and b in turn");
    constexpr bool PERM = !BT;
    typedef Operand<AT, BM, NW, false> A;
    typedef Operand<BT, BN, NW, PERM> B;
    constexpr int SLOT = B::BYTES;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int wm = wave / WN, wn = wave % WN;

    // ids 8 apart run on one XCD: each XCD gets a contiguous range of tiles, and tiles follow each other down columns of
    // GROUP rows, so what runs at a time on an XCD is about square and shares its panels in that XCD's L2
    constexpr int GROUP = 8;
    int m0, n0, split;
    {
        const int per = p.tiles_m * p.tiles_n, total = per * p.splits;
        const int xcd = block & 7, q = total >> 3, r = total & 7;
        int id = (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (block >> 3);
        split = id / per;
        id -= split * per;
        const int g = id / (GROUP * p.tiles_n), rows = min(GROUP, p.tiles_m - g * GROUP);
        id -= g * GROUP * p.tiles_n;
        m0 = (g * GROUP + id % rows) * BM;
        n0 = id / rows * BN;
    }
    const int k0 = split * p.steps * LIN_BK;
    const int nk = (min(p.steps * LIN_BK, p.K - k0) + BK - 1) / BK;   // stages, at least 1 (launcher)

    // (Nothing is in flight here.  The compiler does not know in the second of two tile codes of a kernel, and waited for it, and
    // so for every DMA, at the head of the loop: 512 x 4096 x 4096 58 us instead of 49.)
    __builtin_amdgcn_s_waitcnt(0x0f70);                        // vmcnt(0)
    A a;
    B b;
    a.init(p.a, p.a_bytes, p.lda, m0, k0, wave, lane);
    b.init(p.b, p.b_bytes, p.ldb, n0, k0, wave, lane);

    f32x4 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};

    // Operand stage n (of a: n = 2 ks, of b: 2 ks + 1) lives in slot n mod RING.  K step ks has two halves of 32 k: the first
    // multiplies the fragments read last, (ks, 0), reads (ks, 1) and stages n = 2 ks + RING - 1 (of a); a barrier, behind which
    // the slots of ks are free and those of ks + 1 have landed; the second multiplies (ks, 1), reads (ks + 1, 0) and stages
    // n = 2 ks + RING (of b).  Reads and DMA go out between the products at an even pace: a wave has its SIMD to itself (or
    // shares it with one of another workgroup), so whatever is issued in a clump stops the matrix cores.  The stages past the
    // end of K are staged too, as zeros: no conditions, and the number of DMA in flight is a constant.
    const unsigned lds_at = (unsigned)(unsigned long long)(lin_lds_void_t*)smem;
    const unsigned wave_a = lds_at + wave * (A::PER * 1024), wave_b = lds_at + wave * (B::PER * 1024);
    int rem_a = p.K - k0, rem_b = rem_a;                       // of K, from the stage that is staged next
    bf16x8 a0[MI], b0[NI], a1[MI], b1[NI];
    constexpr int GROUPS = MI * NI / 4, READS = (MI + NI) / (GROUPS / 2);
    static_assert(READS * GROUPS / 2 == MI + NI, "reads in the first half of the groups");
    auto half = [&](const bf16x8 (&ac)[MI], const bf16x8 (&bc)[NI], bf16x8 (&an)[MI], bf16x8 (&bn)[NI], int sa, int sb, int kk,
                    auto per, auto&& dma) {
        constexpr int PER = decltype(per)::value, PACE = PER < GROUPS ? GROUPS / PER : 1, EACH = PER * PACE / GROUPS;
        static_assert(EACH * GROUPS == PER * PACE, "DMA at an even pace");
        const unsigned char *as = smem + sa * SLOT, *bs = smem + sb * SLOT;
#pragma unroll
        for (int g = 0; g < GROUPS; ++g) {
            if (g < GROUPS / 2) {
#pragma unroll
                for (int r = g * READS; r < (g + 1) * READS; ++r) {
                    if (r < NI) bn[r % NI] = B::read(bs, wn * WTN, r % NI, kk, lane);
                    else an[(r - NI + MI) % MI] = A::read(as, wm * WTM, (r - NI + MI) % MI, kk, lane);
                }
            }
            if (g % PACE == 0) {
#pragma unroll
                for (int j = 0; j < EACH; ++j) dma(g / PACE * EACH + j);
            }
#pragma unroll
            for (int t = 4 * g; t < 4 * g + 4; ++t)            // (the compiler, left alone, moves half of the sums to VGPRs and spills)
                asm volatile("v_mfma_f32_16x16x32_bf16 %0, %1, %2, %0" : "+a"(acc[t / NI][t % NI]) : "v"(bc[t % NI]), "v"(ac[t / NI]));
            __builtin_amdgcn_sched_barrier(0);
        }
    };
    auto stage_a = [&](int slot) {
        const u32x4 d = a.desc();
        unsigned m = wave_a + slot * SLOT;
#pragma unroll
        for (int j = 0; j < A::PER; ++j) a.template piece<true>(d, m, rem_a, j, wave, lane);
        a.next();
        rem_a -= BK;
    };
    auto stage_b = [&](int slot) {
        const u32x4 d = b.desc();
        unsigned m = wave_b + slot * SLOT;
#pragma unroll
        for (int j = 0; j < B::PER; ++j) b.template piece<true>(d, m, rem_b, j, wave, lane);
        b.next();
        rem_b -= BK;
    };
#pragma unroll
    for (int n = 0; n < RING - 1; n += 2) {
        stage_a(n);
        stage_b(n + 1);
    }
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((RING - 3) / 2 * (A::PER + B::PER)) : "memory");
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
#pragma unroll
    for (int j = 0; j < NI; ++j) b0[j] = B::read(smem + SLOT, wn * WTN, j, 0, lane);
#pragma unroll
    for (int i = 0; i < MI; ++i) a0[i] = A::read(smem, wm * WTM, i, 0, lane);
    int sa = 0;                                                // slot of a's stage ks
    auto up = [](int s, int n) { return s + n >= RING ? s + n - RING : s + n; };
    auto k_step = [&](auto tail) {
        constexpr bool TAIL = decltype(tail)::value;
        {
            const u32x4 d = a.desc();
            unsigned m = wave_a + up(sa, RING - 1) * SLOT;
            half(a0, b0, a1, b1, sa, up(sa, 1), 1, std::integral_constant<int, A::PER>{}, [&](int j) { a.template piece<TAIL>(d, m, rem_a, j, wave, lane); });
            a.next();
            rem_a -= BK;
        }
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"((RING - 3) / 2 * A::PER + (RING - 5) / 2 * B::PER) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");
        {
            const u32x4 d = b.desc();
            unsigned m = wave_b + sa * SLOT;
            half(a1, b1, a0, b0, up(sa, 2), up(sa, 3), 0, std::integral_constant<int, B::PER>{}, [&](int j) { b.template piece<TAIL>(d, m, rem_b, j, wave, lane); });
            b.next();
            rem_b -= BK;
        }
        sa = up(sa, 2);
    };
    const int whole = min(rem_a / BK, nk);                     // steps that stage whole stages
    int ks = 0;
    for (; ks < whole; ++ks) k_step(std::integral_constant<bool, false>{});
    for (; ks < nk; ++ks) k_step(std::integral_constant<bool, true>{});
    // every DMA has landed, and the last products are through the pipeline before their sums are read
    asm volatile("s_waitcnt vmcnt(0)\n\ts_nop 15\n\ts_nop 15" ::: "memory");
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) asm volatile("" : "+a"(acc[i][j]));

    // The sums go through LDS: a lane holds row x = l & 15 of block i and, of block j, four neighbouring columns; out of LDS a
    // thread takes eight neighbouring columns of a row, so that whole rows are loaded (residual) and stored, and what is done to
    // them is one short loop.  (Straight from the accumulators, unrolled over them, this took 98 000 cycles of a 256 x 256
    // tile: as long as 40 K steps.)  16-byte chunk c of a row is kept at c ^ x: the 16 rows of a write fall on different banks.
    const Epilogue& ep = p.ep;
    constexpr int PI = MI < 4 ? MI : 4, ROWS = WM * PI * 16, NT = NW * 64, COLS8 = BN / 8;
    static_assert(ROWS * BN * 4 <= RING * SLOT, "a pass fits");
    const int x = lane & 15, fq = lane >> 4;
    const int n = n0 + (int)(threadIdx.x % COLS8) * 8;
    float bias[8];
    ld_bias<8>(ep, n, bias);
#pragma unroll
    for (int h = 0; h < MI / PI; ++h) {
        __syncthreads();                                       // what was in LDS has been read (and every DMA has landed)
#pragma unroll
        for (int i = 0; i < PI; ++i)
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                const int row = (wm * PI + i) * 16 + x;
                const int chunk = (wn * WTN + (PERM ? (j >> 2) * 64 + 16 * fq + 4 * (j & 3) : 16 * j + 4 * fq)) / 4;
                *reinterpret_cast<f32x4*>(smem + row * (BN * 4) + ((chunk ^ x) << 4)) = acc[h * PI + i][j];
            }
        __syncthreads();
        for (int row = threadIdx.x / COLS8; row < ROWS; row += NT / COLS8) {
            const int m = m0 + row / (PI * 16) * WTM + h * PI * 16 + row % (PI * 16);
            const int chunk = (threadIdx.x % COLS8) * 2, key = row & 15;
            const f32x4 lo = *reinterpret_cast<const f32x4*>(smem + row * (BN * 4) + ((chunk ^ key) << 4));
            const f32x4 hi = *reinterpret_cast<const f32x4*>(smem + row * (BN * 4) + (((chunk + 1) ^ key) << 4));
            float v[8] = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
            if (ep.mode == OUT_BF16) finish_bf16<8>(ep, m, n, v, bias);
            else if (ep.mode == OUT_ADD) finish_add<8>(ep, m, n, v);
            else if (m < ep.M && n < ep.N) {
                float* slab = ep.ws + ((long long)split * ep.M + m) * slab_ld(ep.N) + n;
                *reinterpret_cast<f32x4*>(slab) = lo;
                *reinterpret_cast<f32x4*>(slab + 4) = hi;
            }
        }
    }
}

template <int BM, int BN, int RING, bool AT, bool BT>
__global__ __launch_bounds__(256, BN* RING <= 128 * 5 ? 2 : 1) void linear_gemm_kernel(const GemmParams p) {
    __shared__ __attribute__((aligned(1024))) unsigned char smem[RING * BN * LIN_BK * 2];
    gemm_tile<BM, BN, RING, AT, BT>(p, blockIdx.x, smem);
}

struct SumsJob {
    const float* part;
    float* out;
    int N, parts, add, blocks;
};
// 64 columns a block, its four waves share the parts; the waves' sums are added in order
__device__ __forceinline__ void join_sums(const SumsJob& p, int block, float (*red)[64]) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = block * 64 + lane;
    float t = 0.0f;
    if (c < p.N) {
#pragma unroll 8
        for (int i = wave; i < p.parts; i += 4) t += p.part[(long long)i * p.N + c];
    }
    red[wave][lane] = t;
    __syncthreads();
    if (wave == 0 && c < p.N) {
        t = ((red[0][lane] + red[1][lane]) + red[2][lane]) + red[3][lane];
        p.out[c] = p.add ? p.out[c] + t : t;
    }
}
__global__ __launch_bounds__(256) void linear_sums_kernel(const SumsJob p) {
    __shared__ float red[4][64];
    join_sums(p, blockIdx.x, red);
}

// Both gradients of a layer in one launch, dw = dz^T a and da = dz w, that with more steps first, and dbias in the last
// blocks.  Each alone would leave CUs idle, at its end at least, or pay for a split of its K.
__global__ __launch_bounds__(256, 2) void linear_pair_kernel(const GemmParams dw, const GemmParams da, int dw_first,
                                                             int first, int sums_at, const SumsJob sums) {
    __shared__ __attribute__((aligned(1024))) unsigned char smem[5 * 128 * LIN_BK * 2];
    const int block = blockIdx.x;
    if (block >= sums_at) return join_sums(sums, block - sums_at, reinterpret_cast<float(*)[64]>(smem));
    const int id = block < first ? block : block - first;
    if ((block < first) == (dw_first != 0)) gemm_tile<128, 128, 5, true, true>(dw, id, smem);
    else gemm_tile<128, 128, 5, false, true>(da, id, smem);
}

// Joins the partial sums of a product whose K range was split (too few tiles for the chip), in slab order, and does what the
// tile kernel's epilogue does.  mode: that of the result.
__global__ __launch_bounds__(256) void linear_join_kernel(const Epilogue p, int splits) {
    const int groups = (p.n_pad + 7) / 8;                      // (n_pad: N where the result has no padding)
    const long long t = (long long)blockIdx.x * 256 + threadIdx.x;
    const int m = (int)(t / groups), n = (int)(t % groups) * 8;
    if (m >= p.M) return;
    float v[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    if (n < p.N) {
        const float* slab = p.ws + m * slab_ld(p.N) + n;
#pragma unroll 8
        for (int s = 0; s < splits; ++s, slab += p.M * slab_ld(p.N)) {
            const f32x4 lo = *reinterpret_cast<const f32x4*>(slab), hi = *reinterpret_cast<const f32x4*>(slab + 4);
#pragma unroll
            for (int e = 0; e < 4; ++e) v[e] += lo[e], v[4 + e] += hi[e];
        }
    }
    if (p.mode == OUT_ADD) finish_add<8>(p, m, n, v);
    else {
        float bias[8];
        ld_bias<8>(p, n, bias);
        finish_bf16<8>(p, m, n, v, bias);
    }
}

// ------------------------------------------------------------------------------------------ few rows
// Up to 16 * MT rows of a: bound by reading w once.  A wave takes 16 rows of w and a share of K and multiplies them with all
// rows of a on the matrix cores, operands straight from memory (every element of w is used by one wave only, so LDS would
// add nothing); the waves' sums meet in LDS.  Rows may start anywhere: unaligned 16-byte loads.
template <int MT, int NW>
__global__ __launch_bounds__(NW * 64) void linear_rows_kernel(const bf16* __restrict__ a, const bf16* __restrict__ w,
                                                              long long lda, long long ldw, int K, const Epilogue ep) {
    __shared__ f32x4 part[NW][MT][64];
    const int lane = threadIdx.x & 63;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);   // matrix instructions run under any exec mask: branches
    const int x = lane & 15, g = lane >> 4, n0 = blockIdx.x * 16;        // around them have to be scalar
    const bf16* wr = w + (long long)min(n0 + x, ep.N - 1) * ldw;       // rows past the end: computed and dropped
    const bf16* ar[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) ar[t] = a + (long long)min(t * 16 + x, ep.M - 1) * lda;
    f32x4 acc[MT];
#pragma unroll
    for (int t = 0; t < MT; ++t) acc[t] = f32x4{0.f, 0.f, 0.f, 0.f};
    auto load = [&](const bf16* p, int k) -> bf16x8 { return __builtin_bit_cast(bf16x8, *reinterpret_cast<const u32x4_a2*>(p + k)); };
    // U fragments of w at a time, the next U on their way while these are multiplied
    constexpr int U = 4;
    const int steps = K / 32;
    bf16x8 w0[U], a0[MT][U], w1[U], a1[MT][U];
    auto fetch = [&](bf16x8 (&wf)[U], bf16x8 (&af)[MT][U], int r) {
        if (r >= steps) return;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int k = min(r + u, steps - 1) * 32 + g * 8;          // past the last step: loaded again, not multiplied
            wf[u] = load(wr, k);
#pragma unroll
            for (int t = 0; t < MT; ++t) af[t][u] = load(ar[t], k);
        }
    };
    auto multiply = [&](const bf16x8 (&wf)[U], const bf16x8 (&af)[MT][U], int r) {
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (r + u < steps) {
#pragma unroll
                for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf[u], af[t][u], acc[t], 0, 0, 0);
            }
    };
    int r = wave * U;
    fetch(w0, a0, r);
    for (; r < steps; r += 2 * NW * U) {
        fetch(w1, a1, r + NW * U);
        multiply(w0, a0, r);
        fetch(w0, a0, r + 2 * NW * U);
        multiply(w1, a1, r + NW * U);
    }
    if (wave == NW - 1 && steps * 32 < K) {                            // the last, partial step
        const int k = steps * 32 + g * 8;
        auto load_part = [&](const bf16* p) -> bf16x8 {
            if (k + 8 <= K) return load(p, k);
            bf16x8 f;
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = k + e < K ? p[k + e] : (bf16)0.0f;
            return f;
        };
        const bf16x8 wf = load_part(wr);
#pragma unroll
        for (int t = 0; t < MT; ++t) acc[t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(wf, load_part(ar[t]), acc[t], 0, 0, 0);
    }
#pragma unroll
    for (int t = 0; t < MT; ++t) part[wave][t][lane] = acc[t];
    __syncthreads();
    for (int t = wave; t < MT; t += NW) {
        f32x4 s = part[0][t][lane];
#pragma unroll
        for (int v = 1; v < NW; ++v) s += part[v][t][lane];
        float v[4] = {s[0], s[1], s[2], s[3]}, bias[4];
        const int n = n0 + 4 * g;
        ld_bias<4>(ep, n, bias);
        finish_bf16<4>(ep, t * 16 + x, n, v, bias);
    }
    // columns of the padding that no 16-column block covers
    const int done = gridDim.x * 16;
    if (blockIdx.x == gridDim.x - 1)
        for (int i = threadIdx.x; i < ep.M * (ep.n_pad - done); i += NW * 64) {
            const long long o = (long long)(i / (ep.n_pad - done)) * ep.ldo + done + i % (ep.n_pad - done);
            static_cast<bf16*>(ep.out)[o] = (bf16)0.0f;
            if (ep.z) ep.z[o] = (bf16)0.0f;
        }
}

// ------------------------------------------------------------------------------------------ backward of the activation
// dz = dy * act'(z) in bf16 (rows padded with zeros to ldz columns: it is the next products' operand) and the column sums of
// the unrounded dz, rows_per rows per block; partial sums of several row blocks are joined in order.
// act == none: only the sums (dz == null) or also a padded copy of dy.
// dz is rounded because the matrix cores multiply bf16: unrounded it would be two operands, a high and a low part, and twice the
// matrix instructions of both products.  The rounding is half a step of each dz, as where a framework keeps the gradient of an
// activation in the compute type: 4096 x 16384 x 4096 gelu is 0.0023 off in the 2-norm, 0.0017 of it the results' own rounding.
// dy without an activation is taken as it is.  4096 x 16384 in 80 us, 5.0 TB/s.
__global__ __launch_bounds__(256) void linear_dz_kernel(const bf16* __restrict__ dy, const bf16* __restrict__ z,
                                                        bf16* __restrict__ dz, float* __restrict__ sums, long long ldy,
                                                        long long ldzin, int ldz, int M, int N, int act, int rows_per, int add) {
    __shared__ float red[8][32][8];
    const int cv = threadIdx.x & 31, rr = threadIdx.x >> 5;
    const int n = (blockIdx.x * 32 + cv) * 8;
    const int r0 = blockIdx.y * rows_per, r1 = r0 + min(rows_per, M - r0);   // (r0 + rows_per may pass 2^31)
    float s[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    const bool whole = n + 8 <= N;
    for (int m = r0 + rr; m < r1; m += 8) {
        float g[8], x[8];
        const bf16* src = dy + (long long)m * ldy + n;
        const bf16* zs = z ? z + (long long)m * ldzin + n : nullptr;
        if (whole) {
            ld_group<8>(src, g);
            if (zs) ld_group<8>(zs, x);
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                g[e] = n + e < N ? (float)src[e] : 0.0f;
                x[e] = zs && n + e < N ? (float)zs[e] : 0.0f;
            }
        }
        if (zs) {
#pragma unroll
            for (int e = 0; e < 8; ++e) g[e] = n + e < N ? g[e] * act_slope(x[e], act) : 0.0f;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) s[e] += g[e];
        if (dz && n < ldz) st_group<8>(dz + (long long)m * ldz + n, g);
    }
#pragma unroll
    for (int e = 0; e < 8; ++e) red[rr][cv][e] = s[e];
    __syncthreads();
    const int c = blockIdx.x * 256 + threadIdx.x;
    if (c >= N) return;
    float t = 0.0f;
#pragma unroll
    for (int r = 0; r < 8; ++r) t += red[r][threadIdx.x >> 3][threadIdx.x & 7];
    float* out = sums + (long long)blockIdx.y * N + c;
    *out = add ? *out + t : t;
}

// rows of any stride and alignment -> rows of ldp columns (a multiple of 8), zeros behind the last one; one or two matrices
struct PackJob {
    const bf16* src;
    bf16* dst;
    long long ld;
    int ldp, rows, cols, blocks;
};
__global__ __launch_bounds__(256) void linear_pack_kernel(const PackJob j0, const PackJob j1) {
    const bool second = (int)blockIdx.x >= j0.blocks;
    const PackJob& j = second ? j1 : j0;
    const int vecs = j.ldp / 8;
    const long long first = (long long)(blockIdx.x - (second ? j0.blocks : 0)) * 256 + threadIdx.x;
    for (long long t = first; t < (long long)j.rows * vecs; t += (long long)j.blocks * 256) {
        const long long row = t / vecs;
        const int c = (int)(t % vecs) * 8;
        const bf16* s = j.src + row * j.ld + c;
        u32x4 v;
        if (c + 8 <= j.cols) v = *reinterpret_cast<const u32x4_a2*>(s);
        else {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = c + e < j.cols ? (float)s[e] : 0.0f;
            v = u32x4{pack_bf16(f[0], f[1]), pack_bf16(f[2], f[3]), pack_bf16(f[4], f[5]), pack_bf16(f[6], f[7])};
        }
        *reinterpret_cast<u32x4*>(j.dst + row * j.ldp + c) = v;
    }
}

// ------------------------------------------------------------------------------------------ launchers
#define LIN_MAX_LD (1 << 22)           // 256 rows of an operand stay below 2 GiB of 32-bit offsets
#define LIN_CUS 256
#define LIN_MAX_BLOCKS 0xffffffll                              // of 256 threads: those of a launch have to fit 32 bits

// How a product is cut up.  Costs are in units of 10 ns.
struct Plan {
    int rows, splits, steps, tiles_m, tiles_n;                   // rows of a tile: 256, 128 or 64
    long long cost;
    long long blocks() const { return (long long)tiles_m * tiles_n * splits; }
};
static void cut(Plan& q, int rows, long long M, long long N, int nk, int splits) {
    q.rows = rows, q.tiles_m = cdiv(M, rows), q.tiles_n = cdiv(N, rows == 256 ? 256 : 128);
    q.steps = cdiv(nk, splits), q.splits = cdiv(nk, q.steps);
}
// joining partial sums: 4 us, 0.08 us a slab and their way through memory at 4.5 TB/s
static long long join_cost(long long M, long long N, int splits) {
    return splits > 1 ? 400 + splits * 8 + splits * M * N * 8 / 45000 : 0;
}

// thin: 64 x 128 tiles are built for this product (the forward one)
static Plan plan_of(long long M, long long N, long long K, bool thin) {
    Plan q;
    const int nk = cdiv(K, LIN_BK);
    // 256 x 256 tiles run one to a CU and take about 16 us plus 1.45 us a step of 64 each (most of the 16 us: nothing covers
    // their prologue and their 64 Ki results); 128 x 128 tiles run two to a CU and take 2.8 + 0.43 us per tile and CU.
    // 4096 x 16384 x 4096: 418 us against 580; x 1024: 156 / 152; x 128: 75 / 56; 2048 x 4096 x 4096 (128 tiles of 256): 91 / 63.
    const long long big = (long long)cdiv((long long)cdiv(M, 256) * cdiv(N, 256), LIN_CUS) * (1600 + 145ll * nk);
    // A lone 128 x 128 workgroup takes 0.56 us a step; K is split while one workgroup per CU holds the ranges (1000 x 2048 x 1536,
    // 128 tiles: one range 19 us, two 24; 64 x 4096 x 4096, 32 tiles: one 40 us, eight 16).
    const long long tiles = (long long)cdiv(M, 128) * cdiv(N, 128), two = (long long)cdiv(tiles, LIN_CUS) * (275 + 43ll * nk);
    const long long lone = 275 + 56ll * nk, small = two > lone ? two : lone;
    int rows = big < small ? 256 : 128, splits = 1;
    q.cost = big < small ? big : small;
    if (rows == 128) {
        for (int s = 2; s <= LIN_CUS / tiles && s <= nk / 2; ++s) {
            const long long cost = 275 + 56ll * cdiv(nk, s) + join_cost(M, N, s);
            if (cost < q.cost) q.cost = cost, splits = s;
        }
    }
    // 64 x 128 tiles: 2.2 us and 0.34 us a step, no less with two on a CU.  Twice as many workgroups where there are few:
    // 1536 x 1000 x 2048 16.0 us against 21.5 with 128 x 128, 128 x 4096 x 4096 15.6 / 18.2; 4096 x 4096 x 512 33.4 / 27.8.
    if (thin && rows != 256) {
        const long long t = (long long)cdiv(M, 64) * cdiv(N, 128), turns = cdiv(t, LIN_CUS);
        for (int s = 1; s == 1 || (s <= LIN_CUS / t && s <= nk / 2); ++s) {
            const long long cost = turns * (220 + 34ll * cdiv(nk, s)) + join_cost(M, N, s);
            if (cost < q.cost) q.cost = cost, splits = s, rows = 64;
        }
    }
    cut(q, rows, M, N, nk, splits);
    return q;
}

// Whether dw (N x K over M) and da (M x K over N) go in one launch, and how they are cut then: unless both take the large
// tiles.  Two workgroups on a CU take 0.75 us a step where the chip is not full, and 0.43 us per tile and CU where it is.
// One launch / two, with dbias: 1536 x 1000 x 2048 28.0 / 44.0 us, 64 x 4096 x 4096 30.2 / 37.1, 1024 x 4096 x 4096 77.5 / 94.7;
// where one would take large tiles 1500 x 16384 x 4096 423 / 453, 2048 x 4096 x 4096 136 / 138; both: 4096 x 4096 x 4096 261 / 231.
static bool plan_pair(long long M, long long N, long long K, Plan& dw, Plan& da) {
    dw = plan_of(N, K, M, false), da = plan_of(M, K, N, false);
    if (dw.rows == 256 && da.rows == 256) return false;
    const long long tw = (long long)cdiv(N, 128) * cdiv(K, 128), ta = (long long)cdiv(M, 128) * cdiv(K, 128);
    const int nw = cdiv(M, LIN_BK), na = cdiv(N, LIN_BK);
    long long best = -1;
    int best_w = 1, best_a = 1;
    for (int sw = 1; sw == 1 || (sw <= 16 && sw <= nw / 2 && sw * tw <= 2 * LIN_CUS); ++sw)
        for (int sa = 1; sa == 1 || (sa <= 16 && sa <= na / 2 && sa * ta <= 2 * LIN_CUS); ++sa) {
            const int kw = cdiv(nw, sw), ka = cdiv(na, sa), k = kw > ka ? kw : ka;
            const long long blocks = tw * sw + ta * sa;
            const long long work = (tw * sw * (275 + 43ll * kw) + ta * sa * (275 + 43ll * ka)) / LIN_CUS;
            const long long one = 275 + (blocks <= LIN_CUS ? 56ll : 75ll) * k, rounds = blocks > 2 * LIN_CUS ? work + one / 2 : 0;
            long long cost = work > one ? work : one;
            cost = (cost > rounds ? cost : rounds) + join_cost(N, K, sw) + join_cost(M, K, sa);
            if (best < 0 || cost < best) best = cost, best_w = sw, best_a = sa;
        }
    cut(dw, 128, N, K, nw, best_w), cut(da, 128, M, K, na, best_a);
    return true;
}

static bool aligned16(const void* p) { return ((unsigned long long)p & 15) == 0; }
static int pad8(int n) { return (n + 7) / 8 * 8; }
static int pad64(int n) { return (n + 63) / 64 * 64; }
static bool widths(int N, int K) { return N > 0 && K > 0 && N <= LIN_MAX_LD - 64 && K <= LIN_MAX_LD - 64; }   // (padded: still an operand)

// An operand of the tile kernel: rows start at 16-byte boundaries and hold a multiple of 8 columns (zeros behind the last
// one; a descriptor that ended inside a 4-byte word would return that word's valid half as zero too).
struct Matrix {
    const bf16* p;
    long long ld;
    int rows, cols;
    bool fits() const { return cols % 8 == 0 && ld % 8 == 0 && ld >= cols && ld < LIN_MAX_LD && aligned16(p); }
    unsigned long long bytes() const {
        return ((unsigned long long)(rows - 1) * (unsigned long long)ld + (unsigned long long)pad8(cols)) * 2ull;
    }
};

// Regions of a call's workspace, one behind the other; without memory (null) it only adds up what is needed.
struct Arena {
    unsigned char* base;
    unsigned long long used = 0;
    void* take(unsigned long long bytes) {
        void* p = base ? base + used : nullptr;
        used += (bytes + 255) / 256 * 256;
        return p;
    }
};

// ``m`` itself, or the place of its padded copy; the copies are made by one launch
static Matrix operand(const Matrix& m, Arena& ws, PackJob& job) {
    job.blocks = 0;
    if (m.fits()) return m;
    const int ldp = pad8(m.cols);
    bf16* dst = static_cast<bf16*>(ws.take((unsigned long long)m.rows * ldp * 2));
    job.src = m.p, job.dst = dst, job.ld = m.ld, job.ldp = ldp, job.rows = m.rows, job.cols = m.cols;
    const long long blocks = ((long long)m.rows * (ldp / 8) + 255) / 256;
    job.blocks = (int)(blocks < LIN_MAX_BLOCKS / 4 ? blocks : LIN_MAX_BLOCKS / 4);   // (beyond, a thread copies several vectors)
    return Matrix{dst, ldp, m.rows, m.cols};
}
static void launch_pack(const PackJob& j0, const PackJob& j1, hipStream_t s) {
    if (j0.blocks + j1.blocks > 0)
        hipLaunchKernelGGL(linear_pack_kernel, dim3(j0.blocks + j1.blocks), dim3(256), 0, s, j0, j1);
}

static unsigned long long slab_bytes(const Plan& q, long long M, int N) {
    return q.splits > 1 ? (unsigned long long)q.splits * M * slab_ld(N) * 4ull : 0ull;
}

static GemmParams gemm_params(const Plan& q, const Matrix& a, const Matrix& b, int K, const Epilogue& ep, float* slabs) {
    GemmParams p;
    p.a = a.p, p.b = b.p, p.a_bytes = a.bytes(), p.b_bytes = b.bytes(), p.lda = (int)a.ld, p.ldb = (int)b.ld, p.K = K;
    p.splits = q.splits, p.steps = q.steps, p.tiles_m = q.tiles_m, p.tiles_n = q.tiles_n;
    p.ep = ep;
    if (q.splits > 1) p.ep.mode = OUT_PART, p.ep.ws = slabs;
    return p;
}
static void launch_join(const GemmParams& p, int mode, hipStream_t s) {
    if (p.splits < 2) return;
    Epilogue e = p.ep;
    e.mode = mode;
    hipLaunchKernelGGL(linear_join_kernel, dim3(cdiv((long long)((e.n_pad + 7) / 8) * e.M, 256)), dim3(256), 0, s, e, p.splits);
}
template <bool T>
static void launch_gemm(const Plan& q, const GemmParams& p, int mode, hipStream_t s) {
    const dim3 grid((unsigned)q.blocks());
    // 128 columns: two workgroups of 80 KB on a CU where there are that many, else one with a deeper ring
    if constexpr (!T) {
        if (q.rows == 64) {
            if (grid.x <= LIN_CUS) hipLaunchKernelGGL((linear_gemm_kernel<64, 128, 9, T, T>), grid, dim3(256), 0, s, p);
            else hipLaunchKernelGGL((linear_gemm_kernel<64, 128, 5, T, T>), grid, dim3(256), 0, s, p);
            return launch_join(p, mode, s);
        }
    }
    if (q.rows == 256) hipLaunchKernelGGL((linear_gemm_kernel<256, 256, 5, T, T>), grid, dim3(256), 0, s, p);
    else if (grid.x <= LIN_CUS) hipLaunchKernelGGL((linear_gemm_kernel<128, 128, 9, T, T>), grid, dim3(256), 0, s, p);
    else hipLaunchKernelGGL((linear_gemm_kernel<128, 128, 5, T, T>), grid, dim3(256), 0, s, p);
    launch_join(p, mode, s);
}

static Epilogue plain_epilogue(void* out, int mode, int M, int N, long long ldo) {
    Epilogue e;
    e.out = out, e.z = nullptr, e.bias = nullptr, e.res = nullptr, e.ws = nullptr, e.ldr = 0;
    e.ldo = (int)ldo, e.n_pad = N, e.M = M, e.N = N, e.mode = mode, e.act = LIN_NONE;
    e.vec = ldo % 8 == 0 && aligned16(out);
    return e;
}

// Whether a forward product goes to the kernel for few rows.  It reads w at 4.9 TB/s and, once for every 16 rows of w, a out of
// the caches at 7 TB/s; where there is little of both, 1024 columns of K take a wave 0.9 us and 0.05 us per row of a.  Tiles
// are bound by w's way through memory at least, and pay for copies of what is not laid out for them.  Measured, few rows / tiles:
// 4096 x 4096 with 1 row 8.3 / 14.0 us, with 64 rows 21.4 / 15.9; 16384 x 4096 with 4 rows 26 / 38, with 32 rows 54 / 39;
// 276 x 7928 with 4 rows 10.2 / 11.0, with 64 rows 30 / 13.2; 777 x 1021 with 16 rows 6.4 / 12.4.  Where the two are close the rule
// is off by up to 17 %: 1000 x 2048 with 64 rows takes 11.4 and could take 9.8, 4096 x 16384 with 16 rows 40.1 and 37.3.
static bool few_rows(const Matrix& a, const Matrix& w, const Plan& tiles) {
    if (a.rows > 64) return false;
    const long long M = a.rows, N = w.rows, K = a.cols;
    const long long trips = cdiv(K, 1024) * (90 + 5 * M) + 220, bytes = N * K * 2 / 49000 + M * K * 2 * cdiv(N, 16) / 70000;
    long long copies = 0;
    if (!a.fits()) copies += M * K * 4;
    if (!w.fits()) copies += N * K * 4;
    const long long floor = 500 + N * K * 2 / 49000, cost = (tiles.cost > floor ? tiles.cost : floor) + 150;
    return (trips > bytes ? trips : bytes) < cost + (copies > 0 ? 250 + copies / 49000 : 0);
}
struct FwdPlan {
    Matrix a, w;
    PackJob ja, jw;
    Plan plan;
    float* slabs;
    bool few;
    unsigned long long bytes;
};
static FwdPlan plan_fwd(const void* a, const void* w, void* ws, int M, int N, int K, long long lda, long long ldw) {
    FwdPlan f;
    f.a = Matrix{static_cast<const bf16*>(a), lda, M, K}, f.w = Matrix{static_cast<const bf16*>(w), ldw, N, K};
    f.plan = plan_of(M, N, pad8(K), true);
    f.few = few_rows(f.a, f.w, f.plan);
    f.slabs = nullptr, f.ja.blocks = f.jw.blocks = 0;
    Arena mem{static_cast<unsigned char*>(ws)};
    if (!f.few) {
        f.a = operand(f.a, mem, f.ja), f.w = operand(f.w, mem, f.jw);
        f.slabs = static_cast<float*>(mem.take(slab_bytes(f.plan, M, N)));
    }
    f.bytes = mem.used;
    return f;
}

// Rows of the tiles that the cost rules give the products of a layer a [M][K], w [N][K]: forward (0), da (1), dw (2).  (Whether
// a forward product of up to 64 rows is cut into tiles at all also depends on its operands' layout.)
PDT_API int pdt_linear_tile_rows(int M, int N, int K, int product) {
    if (M < 1 || !widths(N, K) || product < 0 || product > 2) return -1;
    if (product == 0) return plan_of(M, N, pad8(K), true).rows;
    Plan pw, pa;
    plan_pair(M, N, K, pw, pa);
    return product == 1 ? pa.rows : pw.rows;
}

// bytes of workspace that pdt_linear_fwd needs for these operands
PDT_API long long pdt_linear_fwd_workspace(const void* a, const void* w, int M, int N, int K, long long lda, long long ldw) {
    if (M < 1 || !widths(N, K)) return 0;
    return (long long)plan_fwd(a, w, nullptr, M, N, K, lda, ldw).bytes;
}

// Status -1: sizes (or more tiles than a launch has blocks), -3: a workspace is needed (nothing was launched).  y and z: rows of ldo = N rounded up to 64 columns.
PDT_API int pdt_linear_fwd(const void* a, const void* w, const void* bias, const void* res, void* y, void* z, void* ws, int M, int N,
                           int K, long long lda, long long ldw, long long ldr, int ldo, int act, hipStream_t s) {
    if (M < 0 || !widths(N, K) || ldo != pad64(N) || act < 0 || act > LIN_SILU) return -1;
    if (M == 0) return 0;
    const FwdPlan f = plan_fwd(a, w, ws, M, N, K, lda, ldw);
    if (f.bytes > 0 && !ws) return -3;
    Epilogue e = plain_epilogue(y, OUT_BF16, M, N, ldo);
    e.z = static_cast<bf16*>(z), e.bias = static_cast<const float*>(bias), e.res = static_cast<const bf16*>(res);
    e.ldr = ldr, e.act = act, e.n_pad = ldo;
    if (f.few) {
        const dim3 grid(cdiv(N, 16));
        if (M <= 16) hipLaunchKernelGGL((linear_rows_kernel<1, 8>), grid, dim3(512), 0, s, f.a.p, f.w.p, lda, ldw, K, e);
        else if (M <= 32) hipLaunchKernelGGL((linear_rows_kernel<2, 8>), grid, dim3(512), 0, s, f.a.p, f.w.p, lda, ldw, K, e);
        else hipLaunchKernelGGL((linear_rows_kernel<4, 8>), grid, dim3(512), 0, s, f.a.p, f.w.p, lda, ldw, K, e);
        return pdt_launch_status();
    }
    if (f.plan.blocks() > LIN_MAX_BLOCKS) return -1;
    launch_pack(f.ja, f.jw, s);
    launch_gemm<false>(f.plan, gemm_params(f.plan, f.a, f.w, pad8(K), e, f.slabs), OUT_BF16, s);
    return pdt_launch_status();
}

struct BwdPlan {
    Matrix dz, a, w;
    PackJob ja, jw;
    bf16* dz_out;             // where dz is written, or null: dy is the operand as it is
    float *parts, *slabs_w, *slabs_a;
    int n_parts;
    Plan pw, pa;
    bool pair;
    unsigned long long bytes;
};
static BwdPlan plan_bwd(const void* dy, const void* a, const void* w, void* ws, int M, int N, int K, long long lddy, long long lda,
                        long long ldw, int act, int need_da) {
    BwdPlan f;
    Arena mem{static_cast<unsigned char*>(ws)};
    f.dz = Matrix{static_cast<const bf16*>(dy), lddy, M, N}, f.dz_out = nullptr;
    if (act != LIN_NONE || !f.dz.fits()) {
        f.dz_out = static_cast<bf16*>(mem.take((unsigned long long)M * pad64(N) * 2));
        f.dz = Matrix{f.dz_out, pad64(N), M, N};
    }
    f.a = operand(Matrix{static_cast<const bf16*>(a), lda, M, K}, mem, f.ja);
    f.jw.blocks = 0;
    if (need_da) f.w = operand(Matrix{static_cast<const bf16*>(w), ldw, N, K}, mem, f.jw);
    // row blocks of the bias gradient: about four workgroups per CU, each with at least 32 rows
    const int cap = 1024 * 256 / pad64(N);
    f.n_parts = cdiv(M, 32) < cap ? cdiv(M, 32) : (cap > 0 ? cap : 1);
    f.parts = f.n_parts > 1 ? static_cast<float*>(mem.take((unsigned long long)f.n_parts * N * 4)) : nullptr;
    f.pair = need_da && plan_pair(M, N, K, f.pw, f.pa);
    if (!need_da) f.pw = plan_of(N, K, M, false);
    f.slabs_w = static_cast<float*>(mem.take(slab_bytes(f.pw, N, K)));
    f.slabs_a = static_cast<float*>(mem.take(f.pair ? slab_bytes(f.pa, M, K) : 0ull));
    f.bytes = mem.used;
    return f;
}

PDT_API long long pdt_linear_bwd_workspace(const void* dy, const void* a, const void* w, int M, int N, int K, long long lddy,
                                           long long lda, long long ldw, int act, int need_da) {
    if (M < 1 || !widths(N, K)) return 0;
    return (long long)plan_bwd(dy, a, w, nullptr, M, N, K, lddy, lda, ldw, act, need_da).bytes;
}

// dz = dy act'(z);  dbias (+)= its column sums;  da = dz w (da null: not wanted);  dw (bf16, or fp32 added to) = dz^T a.
// Status as above.
PDT_API int pdt_linear_bwd(const void* dy, const void* z, const void* a, const void* w, void* da, void* dw, void* dbias, void* ws,
                           int M, int N, int K, long long lddy, long long ldz, long long lda, long long ldw, long long lddw, int act,
                           int add_w, int add_b, hipStream_t s) {
    if (M < 1 || !widths(N, K) || lddw < K || lddw > 0x7fffffffll || act < 0 || act > LIN_SILU || (act != LIN_NONE && !z)) return -1;
    const BwdPlan f = plan_bwd(dy, a, w, ws, M, N, K, lddy, lda, ldw, act, da != nullptr);
    if (f.pw.blocks() + (da ? f.pa.blocks() : 0) + cdiv(N, 64) > LIN_MAX_BLOCKS) return -1;
    if (f.bytes > 0 && !ws) return -3;
    const int cols = f.dz_out ? pad64(N) : N;
    hipLaunchKernelGGL(linear_dz_kernel, dim3(cdiv(cols, 256), f.n_parts), dim3(256), 0, s, static_cast<const bf16*>(dy),
                       act == LIN_NONE ? nullptr : static_cast<const bf16*>(z), f.dz_out,
                       f.n_parts > 1 ? f.parts : static_cast<float*>(dbias), lddy, ldz, (int)f.dz.ld, M, N, act, cdiv(M, f.n_parts),
                       f.n_parts > 1 ? 0 : add_b);
    const SumsJob sums = {f.parts, static_cast<float*>(dbias), N, f.n_parts, add_b, f.n_parts > 1 ? cdiv(N, 64) : 0};
    if (sums.blocks > 0 && !f.pair) hipLaunchKernelGGL(linear_sums_kernel, dim3(sums.blocks), dim3(256), 0, s, sums);
    launch_pack(f.ja, f.jw, s);
    const int mode = add_w ? OUT_ADD : OUT_BF16;
    const GemmParams pw = gemm_params(f.pw, f.dz, f.a, M, plain_epilogue(dw, mode, N, K, lddw), f.slabs_w);
    GemmParams pa;
    if (da) pa = gemm_params(f.pa, f.dz, f.w, pad8(N), plain_epilogue(da, OUT_BF16, M, K, K), f.slabs_a);
    if (f.pair) {
        const int nw = (int)f.pw.blocks(), na = (int)f.pa.blocks();
        const int dw_first = f.pw.steps >= f.pa.steps;
        hipLaunchKernelGGL(linear_pair_kernel, dim3(nw + na + sums.blocks), dim3(256), 0, s, pw, pa, dw_first, dw_first ? nw : na,
                           nw + na, sums);
        launch_join(pw, mode, s);
        launch_join(pa, OUT_BF16, s);
        return pdt_launch_status();
    }
    if (da)                                                    // (alone only with the large tiles)
        hipLaunchKernelGGL((linear_gemm_kernel<256, 256, 5, false, true>), dim3((unsigned)f.pa.blocks()), dim3(256), 0, s, pa);
    launch_gemm<true>(f.pw, pw, mode, s);
    return pdt_launch_status();
}
