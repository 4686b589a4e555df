// Writing keys and values into a cache of 4 bits a number (packed_kv.cuh says what is held), and reading them back.
//
// Append: a thread takes 8 neighbouring entries of a token's keys and the same 8 of its values, the G / 8 threads of a group find
// its least and largest number by shuffles.  The roundings are those of the exact quotients, whatever the input type: the
// candidate from float32 arithmetic is compared with the border half way to its neighbour by an exact remainder, so another
// implementation in more bits agrees code by code.
// Both are bound by their bytes: reading 2 · dh · (2 or 4) bytes a token and head and writing dh + 8 · dh / G of them, or the reverse.
#include "common.cuh"
#include "packed_kv.cuh"

namespace {
constexpr int PK_THREADS = 256;

// eight neighbouring numbers; VEC: they lie on 16 bytes
template <typename ET, bool VEC> __device__ __forceinline__ void load8(const ET* p, float (&x)[8]);
template <> __device__ __forceinline__ void load8<float, true>(const float* p, float (&x)[8]) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w; x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16, true>(const __nv_bfloat16* p, float (&x)[8]) {
    const uint4 a = *reinterpret_cast<const uint4*>(p);
    const uint32_t w[4] = {a.x, a.y, a.z, a.w};
#pragma unroll
    for (int i = 0; i < 4; ++i) { x[2 * i] = __uint_as_float(w[i] << 16); x[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u); }
}
template <> __device__ __forceinline__ void load8<float, false>(const float* p, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = p[i];
}
template <> __device__ __forceinline__ void load8<__nv_bfloat16, false>(const __nv_bfloat16* p, float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) x[i] = __bfloat162float(p[i]);
}

// The sum a − b = d + e exactly (d its rounding); b = −a's partner of any size.
__device__ __forceinline__ float sub_rest(float a, float b, float d) {
    const float bb = a - d;
    return (a - (d + bb)) + (bb - b);
}

// (step, zero) of a group from its least and largest number
__device__ __forceinline__ uint32_t pack_pair(float lo, float hi, bool finite) {
    const float zero = __bfloat162float(__float2bfloat16_rn(lo));
    const float range = hi - zero, q = __fdiv_rn(range, 15.f);
    // (`finite` speaks of the numbers; zero and the range may still overflow)
    if (!finite || !(fabsf(range) < INFINITY) || !(fabsf(zero) < INFINITY)) return 0x7fff7fffu;
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

// PIECES: threads of a group (8 entries each)
template <typename ET, bool VEC, int PIECES>
__global__ void __launch_bounds__(PK_THREADS)
packed_append_kernel(const ET* __restrict__ qkv, int ld, int k_off, int v_off, uint32_t* __restrict__ Kq, uint32_t* __restrict__ Kp,
                     uint32_t* __restrict__ Vq, uint32_t* __restrict__ Vp, int n_blocks, const int* __restrict__ block_table, int max_blocks,
                     const int* __restrict__ tok_slot, const int* __restrict__ tok_pos, unsigned total, unsigned per_token, unsigned per_head, int Hkv,
                     int BT, int* __restrict__ dev_err) {
    pdl_wait();                 // chained launch: nothing is read before the kernels ahead have finished
    pdl_launch_dependents();
    const unsigned i = min(blockIdx.x * (unsigned)PK_THREADS + threadIdx.x, total - 1);      // (threads behind the last repeat it: they shuffle too)
    const bool mine = blockIdx.x * (unsigned)PK_THREADS + threadIdx.x < total;
    const unsigned t = i / per_token, c = i - t * per_token;
    const int slot = tok_slot[t], pos = tok_pos[t];
    const ET* src = qkv + (size_t)t * ld + (size_t)c * 8;
    float x[2][8];
    load8<ET, VEC>(src + k_off, x[0]);
    load8<ET, VEC>(src + v_off, x[1]);
    const int blk = slot < 0 ? -1 : packed_block(block_table + (size_t)max(slot, 0) * max_blocks, max_blocks, n_blocks, pos >= 0 ? pos / BT : -1);
    if (mine && slot >= 0 && blk < 0 && c == 0) atomicOr(dev_err, VLRF_DEVERR_NO_BLOCK);
    const unsigned h = c / per_head, piece = c - h * per_head;
    const size_t row = ((size_t)max(blk, 0) * Hkv + h) * BT + (pos >= 0 ? pos % BT : 0);
#pragma unroll
    for (int s = 0; s < 2; ++s) {
        float lo = x[s][0], hi = x[s][0], sum = 0.f;         // sum: 0 · x, which is NaN where any x is not finite
#pragma unroll
        for (int j = 0; j < 8; ++j) {
            lo = fminf(lo, x[s][j]);
            hi = fmaxf(hi, x[s][j]);
            sum = fmaf(0.f, x[s][j], sum);
        }
#pragma unroll
        for (int o = 1; o < PIECES; o <<= 1) {
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            sum += __shfl_xor_sync(0xffffffffu, sum, o);
        }
        const uint32_t pair = pack_pair(lo, hi, sum == 0.f);
        const float step = pair_step(pair), zero = pair_zero(pair);
        uint32_t word = 0;
        if (step > 0.f) {
            // (a step so small that its inverse, or half of it, leaves float32: all three by 2^100, which changes no quotient)
            const float by = step < 1e-30f ? 0x1p100f : 1.f, inv = 1.f / (step * by);
#pragma unroll
            for (int j = 0; j < 8; ++j) word |= pack_code(x[s][j] * by, zero * by, step * by, inv) << (4 * j);
        }
        if (mine && blk >= 0) {
            (s == 0 ? Kq : Vq)[row * per_head + piece] = word;
            if (piece % PIECES == 0) (s == 0 ? Kp : Vp)[row * (per_head / PIECES) + piece / PIECES] = pair;
        }
    }
}

template <typename ET, bool VEC> __device__ __forceinline__ void store8(ET* p, const float (&x)[8]);
template <> __device__ __forceinline__ void store8<float, true>(float* p, const float (&x)[8]) {
    *reinterpret_cast<float4*>(p) = make_float4(x[0], x[1], x[2], x[3]);
    *reinterpret_cast<float4*>(p + 4) = make_float4(x[4], x[5], x[6], x[7]);
}
template <> __device__ __forceinline__ void store8<__nv_bfloat16, true>(__nv_bfloat16* p, const float (&x)[8]) {
    uint32_t w[4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const __nv_bfloat162 v = __floats2bfloat162_rn(x[2 * i], x[2 * i + 1]);
        w[i] = *reinterpret_cast<const uint32_t*>(&v);
    }
    *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
}
template <> __device__ __forceinline__ void store8<float, false>(float* p, const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = x[i];
}
template <> __device__ __forceinline__ void store8<__nv_bfloat16, false>(__nv_bfloat16* p, const float (&x)[8]) {
#pragma unroll
    for (int i = 0; i < 8; ++i) p[i] = __float2bfloat16_rn(x[i]);
}

template <typename ET, bool VEC, int PIECES>
__global__ void __launch_bounds__(PK_THREADS)
packed_read_kernel(const uint32_t* __restrict__ Kq, const uint32_t* __restrict__ Kp, const uint32_t* __restrict__ Vq, const uint32_t* __restrict__ Vp,
                   int n_blocks, const int* __restrict__ block_table, int max_blocks, const int* __restrict__ tok_slot, const int* __restrict__ tok_pos,
                   ET* __restrict__ out_k, int ld_k, ET* __restrict__ out_v, int ld_v, unsigned total, unsigned per_token, unsigned per_head, int Hkv,
                   int BT, int* __restrict__ dev_err) {
    pdl_wait();
    pdl_launch_dependents();
    const unsigned i = blockIdx.x * (unsigned)PK_THREADS + threadIdx.x;
    if (i >= total) return;
    const unsigned t = i / per_token, c = i - t * per_token;
    const int slot = tok_slot[t], pos = tok_pos[t];
    const int blk = slot < 0 ? -1 : packed_block(block_table + (size_t)slot * max_blocks, max_blocks, n_blocks, pos >= 0 ? pos / BT : -1);
    float x[2][8];
    if (blk >= 0) {
        const unsigned h = c / per_head, piece = c - h * per_head;
        const size_t row = ((size_t)blk * Hkv + h) * BT + pos % BT;
        const size_t at = row * per_head + piece, at_pair = row * (per_head / PIECES) + piece / PIECES;
        const uint32_t word[2] = {Kq[at], Vq[at]}, pair[2] = {Kp[at_pair], Vp[at_pair]};
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[s][j] = fmaf(pair_step(pair[s]), (float)((word[s] >> (4 * j)) & 15u), pair_zero(pair[s]));
    } else {                                               // padding rows, and tokens without a block: zeros
        if (slot >= 0 && c == 0) atomicOr(dev_err, VLRF_DEVERR_NO_BLOCK);
#pragma unroll
        for (int s = 0; s < 2; ++s)
#pragma unroll
            for (int j = 0; j < 8; ++j) x[s][j] = 0.f;
    }
    store8<ET, VEC>(out_k + (size_t)t * ld_k + (size_t)c * 8, x[0]);
    store8<ET, VEC>(out_v + (size_t)t * ld_v + (size_t)c * 8, x[1]);
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
                                      (unsigned)total, (unsigned)per_token, (unsigned)(dh / 8), Hkv, BT, dev_err)
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
    const bool vec = on16(out_k) && on16(out_v) && (ld_k * (long long)el) % 16 == 0 && (ld_v * (long long)el) % 16 == 0;
    const dim3 grid((unsigned)((total + PK_THREADS - 1) / PK_THREADS));
#define GO(ET, VEC, P) launch_chained(packed_read_kernel<ET, VEC, P>, grid, dim3(PK_THREADS), (size_t)0, stream, (const uint32_t*)Kq, (const uint32_t*)Kp, \
                                      (const uint32_t*)Vq, (const uint32_t*)Vp, n_blocks, block_table, max_blocks, tok_slot, tok_pos, (ET*)out_k, ld_k, \
                                      (ET*)out_v, ld_v, (unsigned)total, (unsigned)per_token, (unsigned)(dh / 8), Hkv, BT, dev_err)
    if (dtype == VLRF_F32) { if (vec) GO_P(float, true); else GO_P(float, false); }
    else { if (vec) GO_P(__nv_bfloat16, true); else GO_P(__nv_bfloat16, false); }
#undef GO
#undef GO_P
    return vlrf_check_launch("packed_read");
}
