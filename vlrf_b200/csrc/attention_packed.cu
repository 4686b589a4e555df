// Attention over a cache of keys and values in 4 bits (packed_kv.cuh), for any mix of tokens, float32 or bfloat16, every head size
// that is a multiple of 16 up to 256, any number of heads and groups, with or without a window: what the tensor-core kernels do not take.
//
// With k_j = zero_j + step_j · c_j in every group of a row, q · k_j = Σ over groups of step_j (q · c_j) + zero_j Σ q, and
// Σ_j p_j v_j = Σ_j p_j (step_j c_j + zero_j): codes are used as they are.  A warp takes one (token, head) and walks the visible keys in
// chunks of 32, a key a lane for the scores, a byte of the row (two entries) a lane for the values; the softmax runs online in float32.
// Bound by the instructions that take codes apart, one at a time, and, for few rows, by a context's chain, which one warp walks alone; the 32-bit engine, odd
// head sizes and prompts with heads of 192 and 256 come here.  Measured: one row of 1,001 tokens of 12 heads of 64 in float32 347 us, 32 such rows 484; two prompts of
// 1,024 tokens of them 1,459; bfloat16: 8 rows of 1,001 tokens of 12 heads of 80 446, a prompt of 512 tokens of them 292, of 8 heads of 256 over 2 492.
#include "common.cuh"
#include "packed_kv.cuh"

namespace {
constexpr int AP_WARPS = 4, AP_MAX_DH = 256;

// G: entries of a group
template <typename ET, int G>
__global__ void __launch_bounds__(AP_WARPS * 32)
attn_packed_kernel(const ET* __restrict__ qkv, int ld, int q_off, const unsigned char* __restrict__ Kq, const uint32_t* __restrict__ Kp,
                   const unsigned char* __restrict__ Vq, const uint32_t* __restrict__ Vp, int n_blocks, const int* __restrict__ block_table, int max_blocks,
                   const int* __restrict__ tok_slot, const int* __restrict__ tok_pos, ET* __restrict__ out, int ld_out, int H, int Hkv, int dh, int BT,
                   float scale, int window, int* __restrict__ dev_err) {
    extern __shared__ __align__(16) float ap_sm[];               // [AP_WARPS][dh] queries, then [AP_WARPS][16] their sums per group
    pdl_wait();                 // chained launch: nothing is read before the kernels ahead have finished
    pdl_launch_dependents();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int t = blockIdx.x, h = blockIdx.y * AP_WARPS + warp;
    const int slot = tok_slot[t];
    if (h >= H || slot < 0) return;                              // whole warps leave; no block-wide barrier below
    const int pos = tok_pos[t], hk = h / (H / Hkv), NG = dh / G;
    float* q = ap_sm + warp * dh;
    float* qsum = ap_sm + AP_WARPS * dh + warp * 16;
    const ET* qsrc = qkv + (size_t)t * ld + q_off + (size_t)h * dh;
    for (int i = lane; i < dh; i += 32) q[i] = ElemIO<ET>::load(qsrc + i) * scale;
    __syncwarp();
    if (lane < NG) {
        float s = 0.f;
        for (int i = 0; i < G; ++i) s += q[lane * G + i];
        qsum[lane] = s;
    }
    __syncwarp();

    constexpr int NB = AP_MAX_DH / 64;                           // bytes of a value row that a lane takes: lane, lane + 32, …
    float acc[2 * NB];
#pragma unroll
    for (int i = 0; i < 2 * NB; ++i) acc[i] = 0.f;
    float m = -INFINITY, l = 0.f;
    const int first = window > 0 ? max(0, pos - window + 1) : 0;
    const int* table = block_table + (size_t)slot * max_blocks;
    bool lost = false;
    for (int k0 = (first / 32) * 32; k0 <= pos; k0 += 32) {
        const int blk = packed_block(table, max_blocks, n_blocks, k0 / BT);
        if (blk < 0) { lost = true; break; }
        const size_t row0 = ((size_t)blk * Hkv + hk) * BT + k0 % BT;
        const int key = k0 + lane;
        const bool valid = key >= first && key <= pos;
        float s = -INFINITY;
        if (valid) {
            const uint2* codes = reinterpret_cast<const uint2*>(Kq + (row0 + lane) * (dh / 2));
            const uint32_t* pairs = Kp + (row0 + lane) * NG;
            s = 0.f;
            for (int g = 0; g < NG; ++g) {
                const uint32_t pair = pairs[g];
                float dot = 0.f;
#pragma unroll
                for (int c = 0; c < G / 16; ++c) {
                    const uint2 w = codes[g * (G / 16) + c];
                    const float* qq = q + g * G + c * 16;
#pragma unroll
                    for (int i = 0; i < 8; ++i) {
                        dot = fmaf(qq[i], (float)((w.x >> (4 * i)) & 15u), dot);
                        dot = fmaf(qq[8 + i], (float)((w.y >> (4 * i)) & 15u), dot);
                    }
                }
                s += fmaf(pair_step(pair), dot, pair_zero(pair) * qsum[g]);
            }
        }
        const float m_new = fmaxf(m, warp_max(s));               // at least one key of the chunk is valid
        const float m_use = m_new == -INFINITY ? 0.f : m_new;    // (all scores −inf: every weight is 0)
        const float p = valid ? expf(s - m_use) : 0.f;
        const float corr = (m == -INFINITY) ? 0.f : expf(m - m_use);
        l = l * corr + warp_sum(p);
#pragma unroll
        for (int i = 0; i < 2 * NB; ++i) acc[i] *= corr;
        const int from = max(first - k0, 0), n_here = min(32, pos - k0 + 1);
        for (int j = from; j < n_here; ++j) {                    // (hidden keys are not read: what lies there may be anything)
            const float pj = __shfl_sync(0xffffffffu, p, j);
            const unsigned char* codes = Vq + (row0 + j) * (dh / 2);
            const uint32_t* pairs = Vp + (row0 + j) * NG;
#pragma unroll
            for (int i = 0; i < NB; ++i) {
                const int b = i * 32 + lane;
                if (b < dh / 2) {
                    const uint32_t byte = codes[b], pair = pairs[2 * b / G];
                    acc[2 * i] = fmaf(pj, fmaf(pair_step(pair), (float)(byte & 15u), pair_zero(pair)), acc[2 * i]);
                    acc[2 * i + 1] = fmaf(pj, fmaf(pair_step(pair), (float)(byte >> 4), pair_zero(pair)), acc[2 * i + 1]);
                }
            }
        }
        m = m_new;
    }
    if (lost && lane == 0) atomicOr(dev_err, VLRF_DEVERR_NO_BLOCK);
    const float inv = (l > 0.f || l != l) ? 1.f / l : 0.f;       // (a sum that is NaN shows in the result; a row that sees nothing is 0)
    ET* dst = out + (size_t)t * ld_out + (size_t)h * dh;
#pragma unroll
    for (int i = 0; i < NB; ++i) {
        const int b = i * 32 + lane;
        if (b < dh / 2) {
            ElemIO<ET>::store(dst + 2 * b, acc[2 * i] * inv);
            ElemIO<ET>::store(dst + 2 * b + 1, acc[2 * i + 1] * inv);
        }
    }
}
}  // namespace

extern "C" int vlrf_attn_packed(const void* qkv, int dtype, int ld, int q_off, const void* Kq, const void* Kp, const void* Vq, const void* Vp,
                                int n_blocks, const int* block_table, int max_blocks, const int* tok_slot, const int* tok_pos, void* out, int ld_out,
                                int T, int H, int Hkv, int dh, int BT, float scale, int window, int* dev_err, cudaStream_t stream) {
    const int G = packed_group(dh);
    VLRF_REQUIRE(G > 0, "attn_packed: head size %d is not a multiple of 16 up to %d", dh, AP_MAX_DH);
    VLRF_REQUIRE(T >= 0 && H > 0 && Hkv > 0 && max_blocks > 0 && n_blocks >= 0, "attn_packed: bad sizes");
    VLRF_REQUIRE(H % Hkv == 0, "attn_packed: %d heads cannot share %d key/value heads", H, Hkv);
    VLRF_REQUIRE((H + AP_WARPS - 1) / AP_WARPS <= 65535, "attn_packed: %d heads are too many for one launch", H);
    VLRF_REQUIRE(BT > 0 && BT % 32 == 0, "attn_packed: cache blocks of %d tokens are not a multiple of 32", BT);
    VLRF_REQUIRE(window >= 0, "attn_packed: negative window");
    VLRF_REQUIRE(dev_err != nullptr, "attn_packed: needs the device error word");
    VLRF_REQUIRE(dtype == VLRF_F32 || dtype == VLRF_BF16, "attn_packed: unknown dtype %d", dtype);
    if (T == 0) return VLRF_OK;
    const dim3 grid(T, (H + AP_WARPS - 1) / AP_WARPS);
    const size_t smem = (size_t)AP_WARPS * (dh + 16) * sizeof(float);
#define GO(ET, GV) launch_chained(attn_packed_kernel<ET, GV>, grid, dim3(AP_WARPS * 32), smem, stream, (const ET*)qkv, ld, q_off, \
                                  (const unsigned char*)Kq, (const uint32_t*)Kp, (const unsigned char*)Vq, (const uint32_t*)Vp, n_blocks, block_table, \
                                  max_blocks, tok_slot, tok_pos, (ET*)out, ld_out, H, Hkv, dh, BT, scale, window, dev_err)
    if (dtype == VLRF_F32) { if (G == 64) GO(float, 64); else if (G == 32) GO(float, 32); else GO(float, 16); }
    else { if (G == 64) GO(__nv_bfloat16, 64); else if (G == 32) GO(__nv_bfloat16, 32); else GO(__nv_bfloat16, 16); }
#undef GO
    return vlrf_check_launch("attn_packed");
}
