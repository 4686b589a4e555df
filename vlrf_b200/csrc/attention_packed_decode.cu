// Decode attention over a cache of keys and values in 4 bits (packed_kv.cuh): one query a row and head, bfloat16, head sizes 64, 128,
// 192 and 256, any number of query heads to a key/value head.
//
// A CTA takes one row, one key/value head, up to NT · 8 of its query heads and one of n_split parts of the context; each of its warps
// walks tiles of 64 tokens (a cache block) of its own, which arrive in a ring of stages by bulk copies: codes and pairs of a block and head
// are contiguous.  In tensor-core products the codes are the 16-row operand as they lie in the cache, masked but not converted
// (packed_kv.cuh), and the queries the 8 columns:
//     Sᵀ [16 tokens × 8 queries]:  q · k_j = Σ over groups of step_j (q · c_j) + zero_j Σ q
//     Oᵀ [16 entries × 8 queries] += c [entries × 16 tokens] · (p_j step_j) [16 tokens × queries],   and Σ p_j zero_j beside it
// The order of entries inside a product is free, so each lane takes its keys' codes in pieces of eight bytes, and its values' entries
// pairwise from two tokens' words.  Weights change from the layout of a result to that of an operand by `movmatrix`.  Weights times steps
// are rounded to bfloat16 (each by up to 2^-8 of itself, as in the library's other bfloat16 attention); scores, sums, zeros and results stay
// in float32, and code products are exact.  Scales that keep code · 2^-133 in float32's range: queries by 2^90 (so |q| < 2^37), weights by 2^80 (steps of
// values below 2^47).
//
// The warps of a CTA merge their sums in shared memory, the parts of a context in that of their cluster's first CTA; no scratch.
#include "common.cuh"
#include "packed_kv.cuh"

namespace {
constexpr int PD_WARPS = 4, PD_TOKENS = 64, PD_MAX_SPLIT = 16;
constexpr uint32_t PD_WAIT_LIMIT = 1u << 21;
constexpr float PD_Q_UP = 0x1p90f, PD_P_UP = 0x1p80f;

__device__ __forceinline__ uint32_t pd_sm(const void* p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ bool pd_try_wait(uint64_t* bar, uint32_t parity) {
    uint32_t ok;
    asm volatile("{\n.reg .pred p;\nmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\nselp.u32 %0, 1, 0, p;\n}\n"
                 : "=r"(ok) : "r"(pd_sm(bar)), "r"(parity) : "memory");
    return ok != 0;
}
// the whole warp waits, with one answer
__device__ __forceinline__ bool pd_wait(uint64_t* bar, uint32_t parity) {
    for (uint32_t i = 0; i < PD_WAIT_LIMIT; ++i)
        if (__all_sync(0xffffffffu, pd_try_wait(bar, parity))) return true;
    return false;
}
__device__ __forceinline__ void pd_copy(void* dst, const void* src, uint32_t bytes, uint64_t* bar) {
    asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];"
                 ::"r"(pd_sm(dst)), "l"(src), "r"(bytes), "r"(pd_sm(bar)) : "memory");
}
__device__ __forceinline__ void pd_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};\n"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t pd_transpose(uint32_t v) {      // an 8 × 8 matrix of 16-bit numbers, a row a quad of lanes
    uint32_t r;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(v));
    return r;
}
__device__ __forceinline__ uint32_t pd_pack(float lo, float hi) {
    const __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<const uint32_t*>(&v);
}
__device__ __forceinline__ float pd_exp2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

template <int NG> struct PdTile {                                   // a tile in shared memory
    static constexpr int CODES = PD_TOKENS * NG * 32, PAIRS = PD_TOKENS * NG * 4, BYTES = 2 * (CODES + PAIRS);
};
__host__ __device__ constexpr int pd_stages(int NG) { return NG == 1 ? 4 : NG == 2 ? 3 : 2; }

// NG: groups of 64 entries of a head; NT: query heads in eights
template <int NG, int NT>
__global__ void __launch_bounds__(PD_WARPS * 32)
attn_packed_decode_kernel(const __nv_bfloat16* __restrict__ qkv, int ld, int q_off, const unsigned char* __restrict__ Kq, const unsigned char* __restrict__ Kp,
                          const unsigned char* __restrict__ Vq, const unsigned char* __restrict__ Vp, int n_blocks, const int* __restrict__ block_table,
                          int max_blocks, const int* __restrict__ tok_slot, const int* __restrict__ tok_pos, __nv_bfloat16* __restrict__ out, int ld_out, int R,
                          int Hkv, int q_tiles, float scale, int window, int n_split, int* __restrict__ dev_err) {
    constexpr int DH = NG * 64, ST = pd_stages(NG), NQ = NT * 8;
    typedef PdTile<NG> Tile;
    extern __shared__ __align__(128) unsigned char pd_raw[];
    __shared__ __align__(8) uint64_t full_all[PD_WARPS][ST];
    __shared__ float w_max[PD_WARPS][NQ], w_sum[PD_WARPS][NQ];
    __shared__ float c_max[NQ], c_sum[NQ];                          // the CTA's
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int hk = blockIdx.x / q_tiles, q0 = (blockIdx.x % q_tiles) * NQ, row = blockIdx.y, part = blockIdx.z;
    const int n_q = min(NQ, R - q0);                                // query heads of this CTA
    uint64_t* full = full_all[warp];
    unsigned char* ring = pd_raw + (size_t)warp * ST * Tile::BYTES;
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < ST; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(pd_sm(&full[i])));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    pdl_wait();
    pdl_launch_dependents();
    const int slot = tok_slot[row];
    if (slot < 0) return;                                           // padding: the whole cluster leaves
    const int pos = tok_pos[row];
    const int first = window > 0 ? max(0, pos - window + 1) : 0;
    const int tile0 = first / PD_TOKENS, n_tiles = pos >= 0 ? pos / PD_TOKENS - tile0 + 1 : 0;
    const int step_tiles = PD_WARPS * n_split, mine0 = part * PD_WARPS + warp;
    const int n_mine = n_tiles > mine0 ? (n_tiles - mine0 + step_tiles - 1) / step_tiles : 0;
    const int* table = block_table + (size_t)slot * max_blocks;

    // tile number i of this warp into stage i % ST; the blocks of 32 tiles at a time lie a lane each
    int held = -1;
    auto issue = [&](int i) {
        if ((i & 31) == 0) {
            const int j = i + lane;
            held = j < n_mine ? packed_block(table, max_blocks, n_blocks, tile0 + mine0 + j * step_tiles) : -1;
        }
        const int blk = __shfl_sync(0xffffffffu, held, i & 31);
        if (lane == 0) {
            uint64_t* bar = &full[i % ST];
            unsigned char* dst = ring + (i % ST) * Tile::BYTES;
            if (blk < 0) {
                atomicOr(dev_err, VLRF_DEVERR_NO_BLOCK);
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(pd_sm(bar)) : "memory");
            } else {
                const int tile = tile0 + mine0 + i * step_tiles;
                const uint32_t rows = (uint32_t)min(PD_TOKENS, (pos - tile * PD_TOKENS + 4) & ~3);   // tokens that exist, in fours (16 bytes of pairs)
                const size_t at = ((size_t)blk * Hkv + hk) * PD_TOKENS;
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(pd_sm(bar)), "r"(rows * (2 * NG * 36)) : "memory");
                pd_copy(dst, Kq + at * (NG * 32), rows * (NG * 32), bar);
                pd_copy(dst + 2 * Tile::CODES, Kp + at * (NG * 4), rows * (NG * 4), bar);
                pd_copy(dst + Tile::CODES, Vq + at * (NG * 32), rows * (NG * 32), bar);
                pd_copy(dst + 2 * Tile::CODES + Tile::PAIRS, Vp + at * (NG * 4), rows * (NG * 4), bar);
            }
        }
        return blk >= 0;
    };
    uint32_t there = 0;                                             // bit i % 32: tile i has a block
    auto ask = [&](int i) { if (i < n_mine) { const bool b = issue(i); there = (there & ~(1u << (i & 31))) | (b ? 1u << (i & 31) : 0u); } };
#pragma unroll
    for (int i = 0; i < ST; ++i) ask(i);

    // queries as the 16 × 8 operand: lane (g, t) holds query g's entries (2t + w) · 8 …; the codes of odd entries come sixteenfold
    uint32_t qf[NT][NG][4][2];
    float qs[NT][NG][2];                                            // Σ q of queries 2t and 2t + 1, times scale · log2 e
    const float sl2 = scale * 1.4426950408889634f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int a = 0; a < NG; ++a) {
            const int qi = n * 8 + g;
            float sum = 0.f;
#pragma unroll
            for (int w = 0; w < 2; ++w) {
                float e[8];
                const __nv_bfloat16* src = qkv + (size_t)row * ld + q_off + (size_t)(hk * R + q0 + qi) * DH + a * 64 + (2 * t + w) * 8;
                if (qi < n_q) {
                    const uint4 v = *reinterpret_cast<const uint4*>(src);
                    const uint32_t u[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
                    for (int i = 0; i < 4; ++i) { e[2 * i] = __uint_as_float(u[i] << 16); e[2 * i + 1] = __uint_as_float(u[i] & 0xffff0000u); }
                } else {
#pragma unroll
                    for (int i = 0; i < 8; ++i) e[i] = 0.f;
                }
#pragma unroll
                for (int i = 0; i < 8; ++i) sum += e[i];
#pragma unroll
                for (int j = 0; j < 2; ++j) {
                    qf[n][a][2 * w + j][0] = pd_pack(e[2 * j] * PD_Q_UP, e[2 * j + 4] * PD_Q_UP);
                    qf[n][a][2 * w + j][1] = pd_pack(e[2 * j + 1] * (PD_Q_UP / 16.f), e[2 * j + 5] * (PD_Q_UP / 16.f));
                }
            }
            sum += __shfl_xor_sync(0xffffffffu, sum, 1);
            sum += __shfl_xor_sync(0xffffffffu, sum, 2);
            qs[n][a][0] = __shfl_sync(0xffffffffu, sum, 8 * t) * sl2;
            qs[n][a][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4) * sl2;
        }
    const float up_k = (0x1p100f / PD_Q_UP) * 0x1p33f * sl2;        // 2^133 / 2^90 · scale · log2 e, times a step

    float o[NT][NG][4][4], z[NT][NG][2], m_run[NT][2], l_run[NT][2];
#pragma unroll
    for (int n = 0; n < NT; ++n) {
        m_run[n][0] = m_run[n][1] = -INFINITY;
        l_run[n][0] = l_run[n][1] = 0.f;
#pragma unroll
        for (int a = 0; a < NG; ++a) {
            z[n][a][0] = z[n][a][1] = 0.f;
#pragma unroll
            for (int i = 0; i < 4; ++i) o[n][a][i][0] = o[n][a][i][1] = o[n][a][i][2] = o[n][a][i][3] = 0.f;
        }
    }

    int done = 0;
    for (; done < n_mine; ++done) {
        const int i = done;
        if (!pd_wait(&full[i % ST], (uint32_t)((i / ST) & 1))) break;
        if ((there >> (i & 31)) & 1u) {
            const unsigned char* kc = ring + (i % ST) * Tile::BYTES;
            const unsigned char* vc = kc + Tile::CODES;
            const uint32_t* kp = reinterpret_cast<const uint32_t*>(kc + 2 * Tile::CODES);
            const uint32_t* vp = reinterpret_cast<const uint32_t*>(kc + 2 * Tile::CODES + Tile::PAIRS);
            const int k0 = (tile0 + mine0 + i * step_tiles) * PD_TOKENS;
            float s[4][NT][4];
#pragma unroll
            for (int u = 0; u < 4; ++u) {                           // 16 tokens: rows g and g + 8
#pragma unroll
                for (int n = 0; n < NT; ++n) s[u][n][0] = s[u][n][1] = s[u][n][2] = s[u][n][3] = 0.f;
#pragma unroll
                for (int a = 0; a < NG; ++a) {
                    const int r0 = u * 16 + g;
                    const uint2 w0 = *reinterpret_cast<const uint2*>(kc + r0 * (NG * 32) + a * 32 + t * 8);
                    const uint2 w1 = *reinterpret_cast<const uint2*>(kc + (r0 + 8) * (NG * 32) + a * 32 + t * 8);
                    float acc[NT][4];
#pragma unroll
                    for (int n = 0; n < NT; ++n) acc[n][0] = acc[n][1] = acc[n][2] = acc[n][3] = 0.f;
#pragma unroll
                    for (int w = 0; w < 2; ++w) {
                        const uint32_t x0 = w ? w0.y : w0.x, x1 = w ? w1.y : w1.x, y0 = x0 >> 8, y1 = x1 >> 8;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            pd_mma(acc[n], x0 & PK_LOW, x1 & PK_LOW, x0 & PK_HIGH, x1 & PK_HIGH, qf[n][a][2 * w][0], qf[n][a][2 * w][1]);
                            pd_mma(acc[n], y0 & PK_LOW, y1 & PK_LOW, y0 & PK_HIGH, y1 & PK_HIGH, qf[n][a][2 * w + 1][0], qf[n][a][2 * w + 1][1]);
                        }
                    }
                    const uint32_t p0 = kp[r0 * NG + a], p1 = kp[(r0 + 8) * NG + a];
                    const float st0 = pair_step(p0) * up_k, st1 = pair_step(p1) * up_k, ze0 = pair_zero(p0), ze1 = pair_zero(p1);
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        s[u][n][0] += fmaf(acc[n][0], st0, ze0 * qs[n][a][0]);
                        s[u][n][1] += fmaf(acc[n][1], st0, ze0 * qs[n][a][1]);
                        s[u][n][2] += fmaf(acc[n][2], st1, ze1 * qs[n][a][0]);
                        s[u][n][3] += fmaf(acc[n][3], st1, ze1 * qs[n][a][1]);
                    }
                }
            }
            const bool edge = k0 + PD_TOKENS - 1 > pos || k0 < first;
            if (edge) {                                             // (what lies behind the sequence's last token may be anything)
#pragma unroll
                for (int u = 0; u < 4; ++u)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = k0 + u * 16 + g + (e >> 1) * 8;
                        if (key > pos || key < first) {
#pragma unroll
                            for (int n = 0; n < NT; ++n) s[u][n][e] = -INFINITY;
                        }
                    }
            }
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int c = 0; c < 2; ++c) {
                    float mx = m_run[n][c];
#pragma unroll
                    for (int u = 0; u < 4; ++u) mx = fmaxf(mx, fmaxf(s[u][n][c], s[u][n][c + 2]));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                    mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                    const float use = mx == -INFINITY ? 0.f : mx;   // (nothing but −inf so far: every weight is 0)
                    const float corr = m_run[n][c] == -INFINITY ? 0.f : pd_exp2(m_run[n][c] - use);
                    m_run[n][c] = mx;
                    l_run[n][c] *= corr;
#pragma unroll
                    for (int a = 0; a < NG; ++a) {
                        z[n][a][c] *= corr;
#pragma unroll
                        for (int b = 0; b < 4; ++b) { o[n][a][b][c] *= corr; o[n][a][b][c + 2] *= corr; }
                    }
#pragma unroll
                    for (int u = 0; u < 4; ++u)
#pragma unroll
                        for (int e = c; e < 4; e += 2) {
                            s[u][n][e] = pd_exp2(s[u][n][e] - use);
                            l_run[n][c] += s[u][n][e];
                        }
                }
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int r0 = u * 16 + g;
                const bool gone0 = edge && (k0 + r0 > pos || k0 + r0 < first), gone1 = edge && (k0 + r0 + 8 > pos || k0 + r0 + 8 < first);
#pragma unroll
                for (int a = 0; a < NG; ++a) {
                    const uint32_t p0 = gone0 ? 0u : vp[r0 * NG + a], p1 = gone1 ? 0u : vp[(r0 + 8) * NG + a];
                    const float st0 = pair_step(p0) * PD_P_UP, st1 = pair_step(p1) * PD_P_UP, ze0 = pair_zero(p0), ze1 = pair_zero(p1);
                    uint32_t b[NT][2];
#pragma unroll
                    for (int n = 0; n < NT; ++n) {
                        z[n][a][0] = fmaf(s[u][n][0], ze0, fmaf(s[u][n][2], ze1, z[n][a][0]));
                        z[n][a][1] = fmaf(s[u][n][1], ze0, fmaf(s[u][n][3], ze1, z[n][a][1]));
                        b[n][0] = pd_transpose(pd_pack(s[u][n][0] * st0, s[u][n][1] * st0));
                        b[n][1] = pd_transpose(pd_pack(s[u][n][2] * st1, s[u][n][3] * st1));
                    }
                    const unsigned char* vrow = vc + (u * 16 + 2 * t) * (NG * 32) + a * 32 + g * 4;
                    const uint32_t v0 = *reinterpret_cast<const uint32_t*>(vrow), v1 = *reinterpret_cast<const uint32_t*>(vrow + NG * 32);
                    const uint32_t v8 = *reinterpret_cast<const uint32_t*>(vrow + 8 * NG * 32), v9 = *reinterpret_cast<const uint32_t*>(vrow + 9 * NG * 32);
#pragma unroll
                    for (int half = 0; half < 2; ++half) {          // entries 8g … + 3, then 8g + 4 … + 7
                        const uint32_t x = __byte_perm(v0, v1, half ? 0x7632 : 0x5410), y = __byte_perm(v8, v9, half ? 0x7632 : 0x5410);
                        const uint32_t x8 = x >> 8, y8 = y >> 8;
#pragma unroll
                        for (int n = 0; n < NT; ++n) {
                            pd_mma(o[n][a][2 * half], x & PK_LOW, x8 & PK_LOW, y & PK_LOW, y8 & PK_LOW, b[n][0], b[n][1]);
                            pd_mma(o[n][a][2 * half + 1], x & PK_HIGH, x8 & PK_HIGH, y & PK_HIGH, y8 & PK_HIGH, b[n][0], b[n][1]);
                        }
                    }
                }
            }
        }
        __syncwarp();                                               // the stage has been read
        ask(i + ST);
    }
    if (done < n_mine) {                                            // gave up: copies under way land in this CTA's shared memory, so wait for them (bounded)
        if (lane == 0) atomicOr(dev_err, VLRF_DEVERR_WAIT_TIMEOUT);
        for (int j = done; j < min(n_mine, done + ST); ++j) pd_wait(&full[j % ST], (uint32_t)((j / ST) & 1));
    }
    __syncthreads();                                                // every warp is done with its ring: the sums go there
    // the warp's sums: [warp][query][DH] float32 (a ring holds them: 8 queries of 64 numbers are less than a stage)
    float* sums = reinterpret_cast<float*>(pd_raw) + (size_t)warp * NQ * DH;
    const float down = (0x1p100f / PD_P_UP) * 0x1p33f;
#pragma unroll
    for (int n = 0; n < NT; ++n)
#pragma unroll
        for (int c = 0; c < 2; ++c) {
            float l = l_run[n][c];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
            const int qi = n * 8 + 2 * t + c;
            if (g == 0) { w_max[warp][qi] = m_run[n][c]; w_sum[warp][qi] = l; }
#pragma unroll
            for (int a = 0; a < NG; ++a) {
                float zz = z[n][a][c];
#pragma unroll
                for (int x = 4; x < 32; x <<= 1) zz += __shfl_xor_sync(0xffffffffu, zz, x);
                if (qi < n_q) {
                    float* dst = sums + (size_t)qi * DH + a * 64 + g * 8;
                    // products 0 … 3 hold entries (0, 2), (1, 3), (4, 6), (5, 7); the odd ones sixteenfold
                    *reinterpret_cast<float4*>(dst) = make_float4(fmaf(o[n][a][0][c], down, zz), fmaf(o[n][a][1][c], down / 16.f, zz),
                                                                  fmaf(o[n][a][0][c + 2], down, zz), fmaf(o[n][a][1][c + 2], down / 16.f, zz));
                    *reinterpret_cast<float4*>(dst + 4) = make_float4(fmaf(o[n][a][2][c], down, zz), fmaf(o[n][a][3][c], down / 16.f, zz),
                                                                      fmaf(o[n][a][2][c + 2], down, zz), fmaf(o[n][a][3][c + 2], down / 16.f, zz));
                }
            }
        }
    __syncthreads();
    // the CTA's sums, into the place of warp 0's
    float* all = reinterpret_cast<float*>(pd_raw);
    for (int idx = threadIdx.x; idx < n_q * (DH / 4); idx += PD_WARPS * 32) {
        const int qi = idx / (DH / 4), c4 = idx % (DH / 4);
        float M = -INFINITY;
#pragma unroll
        for (int w = 0; w < PD_WARPS; ++w) M = fmaxf(M, w_max[w][qi]);
        const float use = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < PD_WARPS; ++w) {
            const float f = pd_exp2(w_max[w][qi] - use);            // (−inf gives 0; the sums of such a warp are 0, or NaN as they should be)
            const float4 v = *reinterpret_cast<const float4*>(all + ((size_t)w * NQ + qi) * DH + c4 * 4);
            L = fmaf(w_sum[w][qi], f, L);
            acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
        }
        if (n_split == 1) {
            const float inv = (L > 0.f || L != L) ? 1.f / L : 0.f;
            *reinterpret_cast<uint2*>(out + (size_t)row * ld_out + (size_t)(hk * R + q0 + qi) * DH + c4 * 4) =
                make_uint2(pd_pack(acc.x * inv, acc.y * inv), pd_pack(acc.z * inv, acc.w * inv));
        } else {
            *reinterpret_cast<float4*>(all + (size_t)qi * DH + c4 * 4) = acc;
            if (c4 == 0) { c_max[qi] = M; c_sum[qi] = L; }
        }
    }
    if (n_split == 1) return;
    cluster_sync_all();                                             // every part's sums are in its CTA's shared memory
    // every CTA of the cluster finishes a share of the numbers
    const int n4 = n_q * (DH / 4);
    for (int idx = part * (PD_WARPS * 32) + threadIdx.x; idx < n4; idx += n_split * PD_WARPS * 32) {
        const int qi = idx / (DH / 4), c4 = idx % (DH / 4);
        float M = -INFINITY, L = 0.f;
        for (int p = 0; p < n_split; ++p) M = fmaxf(M, ld_cluster_f32(pd_sm(&c_max[qi]), (uint32_t)p));
        const float use = M == -INFINITY ? 0.f : M;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int p = 0; p < n_split; ++p) {
            const float f = pd_exp2(ld_cluster_f32(pd_sm(&c_max[qi]), (uint32_t)p) - use);
            const float4 v = ld_cluster_f32x4(pd_sm(all + (size_t)qi * DH + c4 * 4), (uint32_t)p);
            L = fmaf(ld_cluster_f32(pd_sm(&c_sum[qi]), (uint32_t)p), f, L);
            acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
        }
        const float inv = (L > 0.f || L != L) ? 1.f / L : 0.f;
        *reinterpret_cast<uint2*>(out + (size_t)row * ld_out + (size_t)(hk * R + q0 + qi) * DH + c4 * 4) =
            make_uint2(pd_pack(acc.x * inv, acc.y * inv), pd_pack(acc.z * inv, acc.w * inv));
    }
    cluster_sync_relaxed();                                         // nobody leaves while its shared memory is being read
}

template <int NG, int NT> int pd_launch(const void* qkv, int ld, int q_off, const void* Kq, const void* Kp, const void* Vq, const void* Vp, int n_blocks,
                                        const int* block_table, int max_blocks, const int* tok_slot, const int* tok_pos, void* out, int ld_out, int rows,
                                        int H, int Hkv, float scale, int window, int n_split, int* dev_err, cudaStream_t stream) {
    const int R = H / Hkv, q_tiles = (R + NT * 8 - 1) / (NT * 8);
    size_t smem = (size_t)PD_WARPS * pd_stages(NG) * PdTile<NG>::BYTES;
    const size_t sums = (size_t)PD_WARPS * NT * 8 * NG * 64 * sizeof(float);
    if (sums > smem) smem = sums;
    static DeviceMarks marks;
    static DeviceMarks wide;
    auto kern = attn_packed_decode_kernel<NG, NT>;
    cudaError_t e = allow_shared_memory(marks, kern, smem);
    int device = 0;
    if (e == cudaSuccess) e = cudaGetDevice(&device);
    if (e == cudaSuccess) e = (cudaError_t)wide.once(device, [&] { return (int)cudaFuncSetAttribute(kern, cudaFuncAttributeNonPortableClusterSizeAllowed, 1); });
    if (e != cudaSuccess) return vlrf_fail(VLRF_ERR_CUDA, "attn_packed_decode: %zu bytes of shared memory, clusters: %s", smem, cudaGetErrorString(e));
    const dim3 grid(Hkv * q_tiles, rows, n_split), block(PD_WARPS * 32);
#define ARGS (const __nv_bfloat16*)qkv, ld, q_off, (const unsigned char*)Kq, (const unsigned char*)Kp, (const unsigned char*)Vq, (const unsigned char*)Vp, n_blocks, \
             block_table, max_blocks, tok_slot, tok_pos, (__nv_bfloat16*)out, ld_out, R, Hkv, q_tiles, scale, window, n_split, dev_err
    e = n_split > 1 ? launch_chained_cluster(kern, grid, block, smem, dim3(1, 1, n_split), stream, ARGS) : launch_chained(kern, grid, block, smem, stream, ARGS);
#undef ARGS
    if (e != cudaSuccess) return vlrf_fail(VLRF_ERR_CUDA, "attn_packed_decode: %s", cudaGetErrorString(e));
    return vlrf_check_launch("attn_packed_decode");
}
}  // namespace

extern "C" int vlrf_attn_packed_decode_takes(int H, int Hkv, int dh, int BT, int ld, int q_off, int ld_out) {
    return H > 0 && Hkv > 0 && H % Hkv == 0 && dh > 0 && dh % 64 == 0 && dh <= 256 && BT == PD_TOKENS && ld % 8 == 0 && q_off % 8 == 0 && ld_out % 8 == 0;
}

extern "C" int vlrf_attn_packed_decode(const void* qkv, int ld, int q_off, const void* Kq, const void* Kp, const void* Vq, const void* Vp, int n_blocks,
                                       const int* block_table, int max_blocks, const int* tok_slot, const int* tok_pos, void* out, int ld_out, int rows,
                                       int H, int Hkv, int dh, int BT, float scale, int window, int n_split, int* dev_err, cudaStream_t stream) {
    VLRF_REQUIRE(vlrf_attn_packed_decode_takes(H, Hkv, dh, BT, ld, q_off, ld_out),
                 "attn_packed_decode: %d heads over %d of %d, blocks of %d, row strides %d and %d are not taken", H, Hkv, dh, BT, ld, ld_out);
    VLRF_REQUIRE(rows >= 0 && rows <= 65535 && max_blocks > 0 && n_blocks >= 0 && window >= 0 && dev_err != nullptr, "attn_packed_decode: bad arguments");
    VLRF_REQUIRE(n_split >= 1 && n_split <= PD_MAX_SPLIT, "attn_packed_decode: %d parts (1 to %d)", n_split, PD_MAX_SPLIT);
    for (const void* p : {qkv, Kq, Kp, Vq, Vp, (const void*)out})
        VLRF_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0, "attn_packed_decode: tensors begin on 16 bytes");
    if (rows == 0) return VLRF_OK;
#define GO(NG, NT) pd_launch<NG, NT>(qkv, ld, q_off, Kq, Kp, Vq, Vp, n_blocks, block_table, max_blocks, tok_slot, tok_pos, out, ld_out, rows, H, Hkv, scale, window, \
                                     n_split, dev_err, stream)
    const int R = H / Hkv;
    if (dh == 64) return R <= 8 ? GO(1, 1) : GO(1, 2);
    if (dh == 128) return R <= 8 ? GO(2, 1) : GO(2, 2);
    return dh == 192 ? GO(3, 1) : GO(4, 1);
#undef GO
}
