// Writing keys and values into a cache of 4 bits a number (packed_kv.cuh says what is held), and reading them back.
//
// Append: a thread takes 8 neighbouring entries of a token's keys and the same 8 of its values; the G / 8 threads of a group find its least
// and largest number by shuffles (that a number is NaN goes along).  A quotient rounds by the addition of 1.5 · 2^23, whose sum's low bits are the
// code; where one lies within 10^-5 of the border half way between two codes, and is no tie, the thread does its eight again by exact remainders, so the
// codes are those of the exact quotients, and another implementation in more bits agrees with them one by one.  Read: two pieces a thread, their loads
// together.
// Their bytes: 2 · dh · (2 or 4) read a token and head and dh + 8 · dh / G written, or the reverse.  Append is held up by its instructions (issue slots 63 %
// busy, a quotient, its rounding and the look at its border for every number): 2,619 tokens of 25 heads of 64 in bfloat16 10.7 us, 2.0 TB/s; read by the
// latency of a thread's two loads: 8,191 tokens of 8 heads of 128 into bfloat16 12.4 us, 3.5 TB/s.
#include "common.cuh"
#include "packed_kv.cuh"

namespace {
constexpr int PK_THREADS = 256;
constexpr float PK_SURE = 0.49999f;                          // quotients this near a whole number round to it, whatever float32 makes of them

// n / d for n < 2^31 and a d ≥ 2 by a multiplication (m = ⌊2^(31 + l) / d⌋ + 1 with l = ⌈log2 d⌉)
struct Divide {
    unsigned d, m, shift;
    __host__ static Divide by(unsigned d) {
        unsigned l = 0;
        while ((1ull << l) < d) ++l;
        return {d, (unsigned)((1ull << (31 + l)) / d + 1), l - 1};
    }
    __device__ __forceinline__ unsigned operator()(unsigned n) const { return __umulhi(n, m) >> shift; }
};

// Eight neighbouring numbers of a row.  VEC: they lie on 16 bytes.
template <typename ET> struct Eight;
template <> struct Eight<float> {
    float x[8];
    template <bool VEC> __device__ __forceinline__ void load(const float* p) {
        if (VEC) {
            const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
            x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = p[i];
        }
    }
    __device__ __forceinline__ float at(int i) const { return x[i]; }
    // least and largest of the PIECES threads of a group; NaN if any is
    template <int PIECES> __device__ __forceinline__ void range(float& lo, float& hi) const {
        lo = hi = x[0];
#pragma unroll
        for (int i = 1; i < 8; ++i) {
            asm("min.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(x[i]));
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(x[i]));
        }
#pragma unroll
        for (int o = 1; o < PIECES; o <<= 1) {
            asm("min.NaN.f32 %0, %0, %1;" : "+f"(lo) : "f"(__shfl_xor_sync(0xffffffffu, lo, o)));
            asm("max.NaN.f32 %0, %0, %1;" : "+f"(hi) : "f"(__shfl_xor_sync(0xffffffffu, hi, o)));
        }
    }
};
__device__ __forceinline__ uint32_t min2_nan(uint32_t a, uint32_t b) {
    asm("min.NaN.bf16x2 %0, %0, %1;" : "+r"(a) : "r"(b));
    return a;
}
template <> struct Eight<__nv_bfloat16> {
    uint32_t w[4];
    template <bool VEC> __device__ __forceinline__ void load(const __nv_bfloat16* p) {
        if (VEC) {
            const uint4 a = *reinterpret_cast<const uint4*>(p);
            w[0] = a.x; w[1] = a.y; w[2] = a.z; w[3] = a.w;
        } else {
            const unsigned short* u = reinterpret_cast<const unsigned short*>(p);
#pragma unroll
            for (int i = 0; i < 4; ++i) w[i] = u[2 * i] | (uint32_t)u[2 * i + 1] << 16;
        }
    }
    __device__ __forceinline__ float at(int i) const { return __uint_as_float((i & 1) ? w[i / 2] & 0xffff0000u : w[i / 2] << 16); }
    template <int PIECES> __device__ __forceinline__ void range(float& lo, float& hi) const {
        constexpr uint32_t MINUS = 0x80008000u;              // (the largest is the least of the negated, so one word holds both)
        const uint32_t a = min2_nan(min2_nan(w[0], w[1]), min2_nan(w[2], w[3]));
        const uint32_t b = min2_nan(min2_nan(w[0] ^ MINUS, w[1] ^ MINUS), min2_nan(w[2] ^ MINUS, w[3] ^ MINUS));
        uint32_t m = min2_nan(__byte_perm(a, b, 0x5410), __byte_perm(a, b, 0x7632));
#pragma unroll
        for (int o = 1; o < PIECES; o <<= 1) m = min2_nan(m, __shfl_xor_sync(0xffffffffu, m, o));
        lo = __uint_as_float(m << 16);
        hi = -__uint_as_float(m & 0xffff0000u);
    }
};

// The sum a − b = d + e exactly (d its rounding); b = −a's partner of any size.
__device__ __forceinline__ float sub_rest(float a, float b, float d) {
    const float bb = a - d;
    return (a - (d + bb)) + (bb - b);
}

// (step, zero) of a group from its least and largest number
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi) {
    const float zero = __bfloat162float(__float2bfloat16_rn(lo));
    const float range = hi - zero, q = __fdiv_rn(range, 15.f);
    if (!(fabsf(range) < INFINITY) || !(fabsf(zero) < INFINITY)) return 0x7fff7fffu;         // (a number, or the range, is not finite)
    uint32_t bits = __float_as_uint(fmaxf(q, 0.f));
    uint32_t up = (bits & 0xffffu) > 0x8000u || ((bits & 0xffffu) == 0x8000u && (bits & 0x10000u)) ? 1u : 0u;
    if ((bits & 0xffffu) == 0x8000u) {                       // on the border in float32: which side is the exact quotient on?
        const float rest = fmaf(-15.f, q, range) + sub_rest(hi, zero, range);
        if (rest > 0.f) up = 1u;
        if (rest < 0.f) up = 0u;
    }
    const uint32_t step = (bits >> 16) + up;                 // (15 times the largest finite step is beyond any range: no overflow)
    return step | (__float_as_uint(zero) & 0xffff0000u);
}

__device__ __forceinline__ uint32_t pack_code(float x, float zero, float step, float inv) {
    const float d = x - zero;
    float k = floorf(d * inv);                               // (an approximation: beside a whole number it may be one off)
    k = fminf(fmaxf(k, 0.f), 15.f);
    const float over = fmaf(-step, k + 0.5f, d);             // exact where it is small: step · (k + ½) has 13 bits
    const float rest = over + sub_rest(x, zero, d);
    const bool up = rest > 0.f || (rest == 0.f && ((int)k & 1));
    return (uint32_t)fminf(k + (up ? 1.f : 0.f), 15.f);
}

// (out of line: hardly ever gone)
__device__ __noinline__ uint32_t pack_word_exact(float x0, float x1, float x2, float x3, float x4, float x5, float x6, float x7, float zero, float step) {
    // (a step so small that its inverse, or half of it, leaves float32: all three by 2^100, which changes no quotient)
    const float by = step < 1e-30f ? 0x1p100f : 1.f, inv = 1.f / (step * by), x[8] = {x0, x1, x2, x3, x4, x5, x6, x7};
    uint32_t word = 0;
#pragma unroll
    for (int j = 0; j < 8; ++j) word |= pack_code(x[j] * by, zero * by, step * by, inv) << (4 * j);
    return word;
}

__device__ __forceinline__ uint64_t two(float lo, float hi) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(lo), "f"(hi));
    return d;
}
__device__ __forceinline__ void apart(uint64_t v, float& lo, float& hi) { asm("mov.b64 {%0, %1}, %2;" : "=f"(lo), "=f"(hi) : "l"(v)); }
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}

// eight codes, and whether float32 could say them for sure; CLAMP: zero may lie above the least number (it was rounded)
template <bool CLAMP, typename E> __device__ __forceinline__ uint32_t pack_word(const E& e, uint32_t pair, bool& sure) {
    const float zero = pair_zero(pair);
    float step = pair_step(pair);
    const bool flat = !(step > 0.f);                         // (0, or NaN: codes are 0)
    step = flat ? 1.f : step;
    const float inv = 1.f / step;
    float worst = 0.f;
    uint32_t word = 0;
    // quotients to half a unit of float32's last place (exact where they are float32 numbers, as ties are), and 15.06 at most
    auto quotient = [&](int j) {
        const float d = e.at(j) - zero, q = d * inv;
        return fmaf(fmaf(-step, q, d), inv, q);
    };
    auto from_whole = [](float q) { return fabsf(q - ((q + 12582912.f) - 12582912.f)); };
    // (two at a time in one instruction; sm_100)
    const uint64_t less = two(-zero, -zero), inv2 = two(inv, inv), step2 = two(-step, -step), up = two(12582912.f, 12582912.f), down = two(-12582912.f, -12582912.f);
#pragma unroll
    for (int j = 6; j >= 0; j -= 2) {
        const uint64_t d = add2(two(e.at(j), e.at(j + 1)), less), q0 = mul2(d, inv2);
        uint64_t q = fma2(fma2(step2, q0, d), inv2, q0);
        float a, b, ya, yb, ra, rb;
        if (CLAMP) {
            apart(q, a, b);
            q = two(fmaxf(a, 0.f), fmaxf(b, 0.f));
        }
        const uint64_t y = add2(q, up);
        apart(add2(y, down), ra, rb);
        apart(add2(q, two(-ra, -rb)), a, b);
        apart(y, ya, yb);
        worst = fmaxf(worst, fmaxf(fabsf(a), fabsf(b)));
        word = (word * 16u + __float_as_uint(yb)) * 16u + __float_as_uint(ya);
    }
    word -= 0x4b400000u * 0x11111111u;                       // (the bits of 1.5 · 2^23, eight times)
    sure = flat || (worst < PK_SURE && step >= 1e-30f);
    if (!sure && step >= 1e-30f) {
        // A tie is one if nothing is left of the difference, nor of its rounding, as is nearly always so for bfloat16 numbers, whose ties are many (1.5 % of
        // the words of normal numbers; these eight looks cost a fifth of the kernel's time, and going the exact way for them would cost more).
        sure = true;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            const float q = CLAMP ? fmaxf(quotient(j), 0.f) : quotient(j), off = from_whole(q), d = e.at(j) - zero;
            sure = sure && (off < PK_SURE || (off == 0.5f && fmaf(-step, q, d) == 0.f && sub_rest(e.at(j), zero, d) == 0.f));
        }
    }
    return flat ? 0u : word;
}

// PIECES: threads of a group (8 entries each)
template <typename ET, bool VEC, int PIECES>
__global__ void __launch_bounds__(PK_THREADS)
packed_append_kernel(const ET* __restrict__ qkv, int ld, int k_off, int v_off, uint32_t* __restrict__ Kq, uint32_t* __restrict__ Kp,
                     uint32_t* __restrict__ Vq, uint32_t* __restrict__ Vp, int n_blocks, const int* __restrict__ block_table, int max_blocks,
                     const int* __restrict__ tok_slot, const int* __restrict__ tok_pos, unsigned total, Divide per_token, Divide per_head, int Hkv,
                     int BT, int* __restrict__ dev_err) {
    pdl_wait();                 // chained launch: nothing is read before the kernels ahead have finished
    pdl_launch_dependents();
    const unsigned i = min(blockIdx.x * (unsigned)PK_THREADS + threadIdx.x, total - 1);      // (threads behind the last repeat it: they shuffle too)
    const bool mine = blockIdx.x * (unsigned)PK_THREADS + threadIdx.x < total;
    const unsigned t = per_token(i), c = i - t * per_token.d;
    const int slot = tok_slot[t], pos = tok_pos[t];
    const ET* src = qkv + (size_t)t * ld + (size_t)c * 8;
    Eight<ET> x[2];
    x[0].template load<VEC>(src + k_off);
    x[1].template load<VEC>(src + v_off);
    const int blk = slot < 0 ? -1 : packed_block(block_table + (size_t)max(slot, 0) * max_blocks, max_blocks, n_blocks, pos >= 0 ? pos / BT : -1);
    if (mine && slot >= 0 && blk < 0 && c == 0) atomicOr(dev_err, VLRF_DEVERR_NO_BLOCK);
    const unsigned h = per_head(c), piece = c - h * per_head.d;
    const size_t row = ((size_t)max(blk, 0) * Hkv + h) * BT + (pos >= 0 ? pos % BT : 0);
    uint32_t pair[2], word[2];
    bool sure[2];
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        float lo, hi;
        x[s].template range<PIECES>(lo, hi);
        pair[s] = pack_pair(lo, hi);
        word[s] = pack_word<sizeof(ET) == 4>(x[s], pair[s], sure[s]);
    }
    if (!(sure[0] && sure[1])) {
#pragma unroll
        for (int s = 0; s < 2; ++s)
            if (!sure[s])
                word[s] = pack_word_exact(x[s].at(0), x[s].at(1), x[s].at(2), x[s].at(3), x[s].at(4), x[s].at(5), x[s].at(6), x[s].at(7), pair_zero(pair[s]),
                                          pair_step(pair[s]));
    }
    if (mine && blk >= 0) {
        Kq[row * per_head.d + piece] = word[0];
        Vq[row * per_head.d + piece] = word[1];
        if (piece % PIECES == 0) {
            Kp[row * (per_head.d / PIECES) + piece / PIECES] = pair[0];
            Vp[row * (per_head.d / PIECES) + piece / PIECES] = pair[1];
        }
    }
}

// VEC 0: anywhere; 1: on 16 bytes; 2: on the 32 bytes that eight float32 take
template <int VEC> __device__ __forceinline__ void store8(float* p, const float (&x)[8]) {
    if (VEC == 2) {
        const uint32_t w[8] = {__float_as_uint(x[0]), __float_as_uint(x[1]), __float_as_uint(x[2]), __float_as_uint(x[3]),
                               __float_as_uint(x[4]), __float_as_uint(x[5]), __float_as_uint(x[6]), __float_as_uint(x[7])};
        st_global_32B(p, w);
    } else if (VEC == 1) {
        *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
        *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = x[i];
    }
}
template <int VEC> __device__ __forceinline__ void store8(__nv_bfloat16* p, const float (&x)[8]) {
    if (VEC) {
        uint32_t w[4];
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
            w[i] = *reinterpret_cast<const uint32_t*>(&v);
        }
        *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) p[i] = __float2bfloat16_rn(x[i]);
    }
}

constexpr int PK_READ = 2;                                   // pieces of 8 entries (of keys and of values) a thread reads
template <typename ET, int VEC, int PIECES>
__global__ void __launch_bounds__(PK_THREADS)
packed_read_kernel(const uint32_t* __restrict__ Kq, const uint32_t* __restrict__ Kp, const uint32_t* __restrict__ Vq, const uint32_t* __restrict__ Vp,
                   int n_blocks, const int* __restrict__ block_table, int max_blocks, const int* __restrict__ tok_slot, const int* __restrict__ tok_pos,
                   ET* __restrict__ out_k, int ld_k, ET* __restrict__ out_v, int ld_v, unsigned total, Divide per_token, Divide per_head, int Hkv,
                   int BT, int* __restrict__ dev_err) {
    pdl_wait();
    pdl_launch_dependents();
    const unsigned first = blockIdx.x * (unsigned)(PK_THREADS * PK_READ) + threadIdx.x;
    unsigned t[PK_READ], c[PK_READ];
    int slot[PK_READ], pos[PK_READ], blk[PK_READ];
    uint32_t word[PK_READ][2], pair[PK_READ][2];
#pragma unroll
    for (int u = 0; u < PK_READ; ++u) {
        const unsigned i = min(first + u * PK_THREADS, total - 1);
        t[u] = per_token(i);
        c[u] = i - t[u] * per_token.d;
        slot[u] = tok_slot[t[u]];
        pos[u] = tok_pos[t[u]];
    }
#pragma unroll
    for (int u = 0; u < PK_READ; ++u)
        blk[u] = slot[u] < 0 ? -1 : packed_block(block_table + (size_t)max(slot[u], 0) * max_blocks, max_blocks, n_blocks, pos[u] >= 0 ? pos[u] / BT : -1);
#pragma unroll
    for (int u = 0; u < PK_READ; ++u) {
        word[u][0] = word[u][1] = pair[u][0] = pair[u][1] = 0u;             // padding rows, and tokens without a block: zeros
        if (blk[u] >= 0) {
            const unsigned h = per_head(c[u]), piece = c[u] - h * per_head.d;
            const size_t row = ((size_t)blk[u] * Hkv + h) * BT + pos[u] % BT;
            const size_t at = row * per_head.d + piece, at_pair = row * (per_head.d / PIECES) + piece / PIECES;
            word[u][0] = Kq[at];
            word[u][1] = Vq[at];
            pair[u][0] = Kp[at_pair];
            pair[u][1] = Vp[at_pair];
        }
    }
#pragma unroll
    for (int u = 0; u < PK_READ; ++u) {
        if (first + u * PK_THREADS >= total) break;
        if (slot[u] >= 0 && blk[u] < 0 && c[u] == 0) atomicOr(dev_err, VLRF_DEVERR_NO_BLOCK);
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            float x[8];
#pragma unroll
            for (int j = 0; j < 8; ++j) {
                const float code = __uint_as_float(((word[u][s] >> (4 * j)) & 15u) | 0x4b000000u) - 8388608.f;      // (2^23 and the code, less 2^23)
                x[j] = fmaf(pair_step(pair[u][s]), code, pair_zero(pair[u][s]));
            }
            store8<VEC>((s == 0 ? out_k + (size_t)t[u] * ld_k : out_v + (size_t)t[u] * ld_v) + (size_t)c[u] * 8, x);
        }
    }
}

bool on16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }
}  // namespace

extern "C" int vlrf_packed_group(int dh) { return packed_group(dh); }

extern "C" int vlrf_packed_append(const void* qkv, int dtype, int ld, int k_off, int v_off, void* Kq, void* Kp, void* Vq, void* Vp, int n_blocks,
                                  const int* block_table, int max_blocks, const int* tok_slot, const int* tok_pos, int T, int Hkv, int dh, int BT,
                                  int* dev_err, cudaStream_t stream) {
    const int G = packed_group(dh);
    VLRF_REQUIRE(G > 0, "packed_append: head size %d is not a multiple of 16 up to 256", dh);
    VLRF_REQUIRE(T >= 0 && Hkv > 0 && BT > 0 && max_blocks > 0 && n_blocks >= 0, "packed_append: bad sizes");
    VLRF_REQUIRE(dev_err != nullptr, "packed_append: needs the device error word");
    VLRF_REQUIRE(dtype == VLRF_F32 || dtype == VLRF_BF16, "packed_append: unknown dtype %d", dtype);
    const long long per_token = (long long)Hkv * dh / 8, total = per_token * T;
    VLRF_REQUIRE(total < (1ll << 31), "packed_append: %d tokens of %d heads of %d are too many for one launch", T, Hkv, dh);
    if (T == 0) return VLRF_OK;
    const int el = dtype == VLRF_F32 ? 4 : 2;
    const bool vec = on16(qkv) && (ld * (long long)el) % 16 == 0 && (k_off * (long long)el) % 16 == 0 && (v_off * (long long)el) % 16 == 0;
    const dim3 grid((unsigned)((total + PK_THREADS - 1) / PK_THREADS));
#define GO(ET, VEC, P) launch_chained(packed_append_kernel<ET, VEC, P>, grid, dim3(PK_THREADS), (size_t)0, stream, (const ET*)qkv, ld, k_off, v_off, \
                                      (uint32_t*)Kq, (uint32_t*)Kp, (uint32_t*)Vq, (uint32_t*)Vp, n_blocks, block_table, max_blocks, tok_slot, tok_pos, \
                                      (unsigned)total, Divide::by((unsigned)per_token), Divide::by((unsigned)(dh / 8)), Hkv, BT, dev_err)
#define GO_P(ET, VEC) do { if (G == 64) GO(ET, VEC, 8); else if (G == 32) GO(ET, VEC, 4); else GO(ET, VEC, 2); } while (0)
    if (dtype == VLRF_F32) { if (vec) GO_P(float, true); else GO_P(float, false); }
    else { if (vec) GO_P(__nv_bfloat16, true); else GO_P(__nv_bfloat16, false); }
#undef GO
    return vlrf_check_launch("packed_append");
}

extern "C" int vlrf_packed_read(const void* Kq, const void* Kp, const void* Vq, const void* Vp, int n_blocks, const int* block_table, int max_blocks,
                                const int* tok_slot, const int* tok_pos, void* out_k, int ld_k, void* out_v, int ld_v, int dtype, int T, int Hkv,
                                int dh, int BT, int* dev_err, cudaStream_t stream) {
    const int G = packed_group(dh);
    VLRF_REQUIRE(G > 0, "packed_read: head size %d is not a multiple of 16 up to 256", dh);
    VLRF_REQUIRE(T >= 0 && Hkv > 0 && BT > 0 && max_blocks > 0 && n_blocks >= 0, "packed_read: bad sizes");
    VLRF_REQUIRE(dev_err != nullptr, "packed_read: needs the device error word");
    VLRF_REQUIRE(dtype == VLRF_F32 || dtype == VLRF_BF16, "packed_read: unknown dtype %d", dtype);
    const long long per_token = (long long)Hkv * dh / 8, total = per_token * T;
    VLRF_REQUIRE(total < (1ll << 31), "packed_read: %d tokens of %d heads of %d are too many for one launch", T, Hkv, dh);
    if (T == 0) return VLRF_OK;
    const int el = dtype == VLRF_F32 ? 4 : 2;
    const long long where = (long long)(reinterpret_cast<uintptr_t>(out_k) | reinterpret_cast<uintptr_t>(out_v)) | ld_k * (long long)el | ld_v * (long long)el;
    const int vec = where % 32 == 0 ? 2 : where % 16 == 0 ? 1 : 0;
    const dim3 grid((unsigned)((total + PK_THREADS * PK_READ - 1) / (PK_THREADS * PK_READ)));
#define GO(ET, VEC, P) launch_chained(packed_read_kernel<ET, VEC, P>, grid, dim3(PK_THREADS), (size_t)0, stream, (const uint32_t*)Kq, (const uint32_t*)Kp, \
                                      (const uint32_t*)Vq, (const uint32_t*)Vp, n_blocks, block_table, max_blocks, tok_slot, tok_pos, (ET*)out_k, ld_k, \
                                      (ET*)out_v, ld_v, (unsigned)total, Divide::by((unsigned)per_token), Divide::by((unsigned)(dh / 8)), Hkv, BT, dev_err)
    if (dtype == VLRF_F32) { if (vec == 2) GO_P(float, 2); else if (vec) GO_P(float, 1); else GO_P(float, 0); }
    else { if (vec) GO_P(__nv_bfloat16, 1); else GO_P(__nv_bfloat16, 0); }
#undef GO
#undef GO_P
    return vlrf_check_launch("packed_read");
}
