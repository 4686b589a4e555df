// Decode attention over a cache of keys and values in 4 bits (packed_kv.cuh): one query a row and head, bfloat16, head sizes 64, 128,
// 192 and 256, any number of query heads to a key/value head.
//
// A CTA takes one row, one key/value head, up to RC (2, 4 or 8) of its query heads and one of the parts into which a long context is cut; each of
// its warps walks tiles of 64 tokens (a cache block) of its own, which arrive in a ring of two stages by bulk copies: codes and pairs of a block and
// head are contiguous.  In tensor-core products the codes are the 16-row operand as they lie in the cache, masked but not converted
// (packed_kv.cuh), and the queries the 8 columns, 8 / RC sub-steps of 16 tokens side by side:
//     Sᵀ [16 tokens × columns]:  q · k_j = Σ over groups of step_j (q · c_j) + zero_j Σ q
//     Oᵀ [16 entries × columns] += c [entries × 16 tokens] · (p_j step_j) [16 tokens × columns],   and Σ p_j zero_j beside it
// The order of entries inside a product is free, so each lane takes its keys' codes in pieces of eight bytes, and its values' entries
// pairwise from two tokens' words.  Weights change from the layout of a result to that of an operand by `movmatrix`.  Weights times steps
// are rounded to bfloat16 (each by up to 2^-8 of itself, as in the library's other bfloat16 attention); scores, sums, zeros and results stay
// in float32, and code products are exact.  (As two bfloat16 numbers each they would leave results as near to 64 bits as the plain form, 0.0017 of them against 0.0019
// to 0.0024, for 4 to 7 % of the time.)  Scales that keep code · 2^-133 in float32's range: queries by 2^90 (so |q| < 2^37), weights by 2^80 (steps of
// values below 2^47; a weight times a step below 2^-73 is nothing).
//
// The warps of a CTA merge their sums in shared memory; the parts of a context leave theirs in scratch, and the CTA that comes last merges them
// in their order.  (A cluster a context, its CTAs merging in distributed shared memory, left SMs empty: 16 CTAs of one an SM found no room together.)
//
// Bound by taking codes apart and by latency rather than by bytes: 131,071 tokens of 8 heads of 128 for 32 queries (151 MB) 40 us, 3.8 TB/s, with the
// integer pipe 47 % and the tensor pipe 23 % busy; the copies alone take 31 us, the arithmetic alone 30.  16 rows of 1 to 8,116 tokens: 27 us, 2.7 TB/s;
// 32 rows of 300 to 1,013 tokens of 25 heads of 64: 15.6 us, 2.4 TB/s; one row of 701 tokens of 12 heads: 5.3 us, a chain of latencies.  A window of 512, 32 rows
// of 8 heads of 128 for 32 queries: 11.1 us, 1.7 TB/s; heads of 192 and 256 (8 over 2, 16 rows of 2,001 tokens): 12.8 and 20.6 us, 1.1 and 0.9 TB/s (two CTAs of four
// warps an SM are what 192 to 239 registers leave).
#include "common.cuh"
#include "packed_kv.cuh"

namespace {
constexpr int PD_TOKENS = 64, PD_MAX_SPLIT = 64;
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
// (not volatile: products of different sums change places, so that one does not wait for the other)
__device__ __forceinline__ void pd_mma(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm(
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

constexpr __host__ __device__ int pd_tile_codes(int NG) { return PD_TOKENS * NG * 32; }    // bytes of a tile's keys (or values)
constexpr __host__ __device__ int pd_tile_pairs(int NG) { return PD_TOKENS * NG * 4; }
constexpr __host__ __device__ int pd_tile_bytes(int NG) { return 2 * (pd_tile_codes(NG) + pd_tile_pairs(NG)); }
// FEW: a CTA an SM with as many warps as shared memory has rings for; else CTAs of four warps, several an SM.
constexpr int PD_STAGES = 2;
constexpr __host__ __device__ int pd_warps(int NG, bool FEW) { return !FEW ? 4 : NG == 1 ? 24 : NG == 2 ? 12 : NG == 3 ? 8 : 6; }
constexpr __host__ __device__ int pd_smem(int NG, bool FEW) { return pd_warps(NG, FEW) * PD_STAGES * pd_tile_bytes(NG); }
constexpr __host__ __device__ int pd_ctas(int NG, bool FEW) { return FEW ? 1 : NG == 1 ? 6 : NG == 2 ? 3 : 2; }

// NG: groups of 64 entries of a head.  RC: columns that the queries of a sub-step of 16 tokens take (2, 4 or 8): a product's 8 columns
// hold 8 / RC sub-steps side by side.
template <int NG, int RC, bool FEW>
__global__ void __launch_bounds__(pd_warps(NG, FEW) * 32, pd_ctas(NG, FEW))
attn_packed_decode_kernel(const __nv_bfloat16* __restrict__ qkv, int ld, int q_off, const unsigned char* __restrict__ Kq, const unsigned char* __restrict__ Kp,
                          const unsigned char* __restrict__ Vq, const unsigned char* __restrict__ Vp, int n_blocks, const int* __restrict__ block_table,
                          int max_blocks, const int* __restrict__ tok_slot, const int* __restrict__ tok_pos, const int* __restrict__ row_of, __nv_bfloat16* __restrict__ out, int ld_out, int R,
                          int Hkv, int q_tiles, float scale, int window, int part_tiles, float* __restrict__ partials, int* __restrict__ counters, int* __restrict__ dev_err) {
    constexpr int DH = NG * 64, WARPS = pd_warps(NG, FEW), ST = PD_STAGES, CODES = pd_tile_codes(NG), PAIRS = pd_tile_pairs(NG), BYTES = pd_tile_bytes(NG);
    constexpr int CP = 8 / RC, NP = 4 / CP;                         // sub-steps side by side; products one after another for a tile's four sub-steps
    extern __shared__ __align__(128) unsigned char pd_raw[];
    __shared__ __align__(8) uint64_t full_all[WARPS][ST];
    __shared__ float w_max[WARPS][8], w_sum[WARPS][8];
    __shared__ int s_last;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
    const int hk = blockIdx.x / q_tiles, q0 = (blockIdx.x % q_tiles) * RC, row = blockIdx.y, part = blockIdx.z;
    const int n_q = min(RC, R - q0);                                // query heads of this CTA
    uint64_t* full = full_all[warp];
    unsigned char* ring = pd_raw + (size_t)warp * ST * BYTES;
    if (lane == 0) {
#pragma unroll
        for (int i = 0; i < ST; ++i) asm volatile("mbarrier.init.shared::cta.b64 [%0], 1;" ::"r"(pd_sm(&full[i])));
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    pdl_wait();
    // (A large grid lets the next kernel's CTAs in when its own are done with their tiles: taken in beside them they sit on the places that are free then,
    // three on one SM and one on another, and so they run when their turn comes.  256 CTAs of 1,983 tokens of 128, the same kernel again and again:
    // 27.5 us, now 24.2.)
    const bool small = gridDim.x * gridDim.y * gridDim.z <= 64u;
    if (small) pdl_launch_dependents();
    const int slot = tok_slot[row], pos = tok_pos[row];
    // (with row_of, an entry stands for the rows row_of[i] … row_of[i + 1] − 1, and only those of one row are looked at)
    const int at_row = row_of == nullptr ? row : row_of[row];
    if (slot < 0 || (row_of != nullptr && row_of[row + 1] - at_row != 1)) return;            // padding
    const int first = window > 0 ? max(0, pos - window + 1) : 0;
    const int tile0 = first / PD_TOKENS, n_tiles = pos >= 0 ? pos / PD_TOKENS - tile0 + 1 : 0;
    // a context takes as many parts as it needs for at most part_tiles tiles each (a longer one than was said: all there are), about equally long
    const int parts = max(1, min((int)gridDim.z, (n_tiles + part_tiles - 1) / part_tiles));
    if (part >= parts) return;
    const int part_first = (int)((long long)part * n_tiles / parts), part_n = (int)((long long)(part + 1) * n_tiles / parts) - part_first;
    constexpr int step_tiles = WARPS;
    const int mine0 = part_first + warp, n_mine = (part_n - warp + WARPS - 1) / WARPS;     // (none or less where the part has fewer tiles than warps)
    const int* table = block_table + (size_t)slot * max_blocks;

    // tile number i of this warp into stage i % ST; the blocks of 32 tiles at a time lie a lane each
    int held = -1;
    uint32_t there = 0;                                             // bit i % 32: tile i has a block
    auto ask = [&](int i) {
        if (i >= n_mine) return;
        if ((i & 31) == 0) {
            const int j = i + lane;
            held = j < n_mine ? packed_block(table, max_blocks, n_blocks, tile0 + mine0 + j * step_tiles) : -1;
        }
        const int blk = __shfl_sync(0xffffffffu, held, i & 31);
        there = (there & ~(1u << (i & 31))) | (blk >= 0 ? 1u << (i & 31) : 0u);
        if (lane == 0) {
            uint64_t* bar = &full[i % ST];
            if (blk < 0) {
                atomicOr(dev_err, VLRF_DEVERR_NO_BLOCK);
                asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(pd_sm(bar)) : "memory");
            } else {
                unsigned char* dst = ring + (i % ST) * BYTES;
                const int tile = tile0 + mine0 + i * step_tiles;
                const uint32_t rows = (uint32_t)min(PD_TOKENS, (pos - tile * PD_TOKENS + 4) & ~3);   // tokens that exist, in fours (16 bytes of pairs)
                const size_t at = ((size_t)blk * Hkv + hk) * PD_TOKENS;
                asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(pd_sm(bar)), "r"(rows * (2 * NG * 36)) : "memory");
                pd_copy(dst, Kq + at * (NG * 32), rows * (NG * 32), bar);
                pd_copy(dst + 2 * CODES, Kp + at * (NG * 4), rows * (NG * 4), bar);
                pd_copy(dst + CODES, Vq + at * (NG * 32), rows * (NG * 32), bar);
                pd_copy(dst + 2 * CODES + PAIRS, Vp + at * (NG * 4), rows * (NG * 4), bar);
            }
        }
    };
#pragma unroll
    for (int i = 0; i < ST; ++i) ask(i);

    // queries as the 16 × 8 operand, column n query n % RC: lane (g, t) holds entries (2t + w) · 8 … of column g; the codes of odd entries
    // come sixteenfold
    uint32_t qf[NG][4][2];
    float qs[NG][2];                                                // Σ q of columns 2t and 2t + 1, times scale · log2 e
    const float sl2 = scale * 1.4426950408889634f;
#pragma unroll
    for (int a = 0; a < NG; ++a) {
        const int qi = g % RC;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < 2; ++w) {
            float e[8];
            const __nv_bfloat16* src = qkv + (size_t)at_row * ld + q_off + (size_t)(hk * R + q0 + qi) * DH + a * 64 + (2 * t + w) * 8;
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
                qf[a][2 * w + j][0] = pd_pack(e[2 * j] * PD_Q_UP, e[2 * j + 4] * PD_Q_UP);
                qf[a][2 * w + j][1] = pd_pack(e[2 * j + 1] * (PD_Q_UP / 16.f), e[2 * j + 5] * (PD_Q_UP / 16.f));
            }
        }
        sum += __shfl_xor_sync(0xffffffffu, sum, 1);
        sum += __shfl_xor_sync(0xffffffffu, sum, 2);
        qs[a][0] = __shfl_sync(0xffffffffu, sum, 8 * t) * sl2;
        qs[a][1] = __shfl_sync(0xffffffffu, sum, 8 * t + 4) * sl2;
    }
    const float up_k = (0x1p100f / PD_Q_UP) * 0x1p33f * sl2;        // 2^133 / 2^90 · scale · log2 e, times a step

    // a column's sums: of a query over the sub-steps that its column stands for
    float o[NG][4][4], z[NG][2], m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
#pragma unroll
    for (int a = 0; a < NG; ++a) {
        z[a][0] = z[a][1] = 0.f;
#pragma unroll
        for (int i = 0; i < 4; ++i) o[a][i][0] = o[a][i][1] = o[a][i][2] = o[a][i][3] = 0.f;
    }
    const int my_sub = 2 * t / RC;                                  // the sub-step (of those side by side) of this lane's two columns of a result
    int done = 0;
    for (; done < n_mine; ++done) {
        const int i = done;
        if (!pd_wait(&full[i % ST], (uint32_t)((i / ST) & 1))) break;
        if ((there >> (i & 31)) & 1u) {
            const unsigned char* kc = ring + (i % ST) * BYTES;
            const unsigned char* vc = kc + CODES;
            const uint32_t* kp = reinterpret_cast<const uint32_t*>(kc + 2 * CODES);
            const uint32_t* vp = reinterpret_cast<const uint32_t*>(kc + 2 * CODES + PAIRS);
            const int k0 = (tile0 + mine0 + i * step_tiles) * PD_TOKENS;
            const bool edge = k0 + PD_TOKENS - 1 > pos || k0 < first;
            float s[NP][4];
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                float acc[NG][CP][4];
#pragma unroll
                for (int a = 0; a < NG; ++a)
#pragma unroll
                    for (int c = 0; c < CP; ++c) {
                        const int r0 = (n * CP + c) * 16 + g;       // tokens r0 and r0 + 8
                        const uint2 w0 = *reinterpret_cast<const uint2*>(kc + r0 * (NG * 32) + a * 32 + t * 8);
                        const uint2 w1 = *reinterpret_cast<const uint2*>(kc + (r0 + 8) * (NG * 32) + a * 32 + t * 8);
                        acc[a][c][0] = acc[a][c][1] = acc[a][c][2] = acc[a][c][3] = 0.f;
#pragma unroll
                        for (int w = 0; w < 2; ++w) {
                            const uint32_t x0 = w ? w0.y : w0.x, x1 = w ? w1.y : w1.x, y0 = x0 >> 8, y1 = x1 >> 8;
                            pd_mma(acc[a][c], x0 & PK_LOW, x1 & PK_LOW, x0 & PK_HIGH, x1 & PK_HIGH, qf[a][2 * w][0], qf[a][2 * w][1]);
                            pd_mma(acc[a][c], y0 & PK_LOW, y1 & PK_LOW, y0 & PK_HIGH, y1 & PK_HIGH, qf[a][2 * w + 1][0], qf[a][2 * w + 1][1]);
                        }
                    }
#pragma unroll
                for (int a = 0; a < NG; ++a) {
                    // every column of a sub-step's result holds its query's score; this lane's columns take those of their own sub-step
                    float x[4];
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        x[e] = acc[a][0][e];
#pragma unroll
                        for (int c = 1; c < CP; ++c) x[e] = my_sub == c ? acc[a][c][e] : x[e];
                    }
                    const int r0 = (n * CP + my_sub) * 16 + g;
                    const uint32_t p0 = kp[r0 * NG + a], p1 = kp[(r0 + 8) * NG + a];
                    const float st0 = pair_step(p0) * up_k, st1 = pair_step(p1) * up_k, ze0 = pair_zero(p0), ze1 = pair_zero(p1);
                    x[0] = fmaf(x[0], st0, ze0 * qs[a][0]);
                    x[1] = fmaf(x[1], st0, ze0 * qs[a][1]);
                    x[2] = fmaf(x[2], st1, ze1 * qs[a][0]);
                    x[3] = fmaf(x[3], st1, ze1 * qs[a][1]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[n][e] = a == 0 ? x[e] : s[n][e] + x[e];
                }
                if (edge) {                                         // (what lies behind the sequence's last token may be anything)
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = k0 + (n * CP + my_sub) * 16 + g + (e >> 1) * 8;
                        if (key > pos || key < first) s[n][e] = -INFINITY;
                    }
                }
            }
#pragma unroll
            for (int c = 0; c < 2; ++c) {
                float mx = m_run[c];
#pragma unroll
                for (int n = 0; n < NP; ++n) mx = fmaxf(mx, fmaxf(s[n][c], s[n][c + 2]));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
                mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
                const float use = mx == -INFINITY ? 0.f : mx;       // (nothing but −inf so far: every weight is 0)
                const float corr = m_run[c] == -INFINITY ? 0.f : pd_exp2(m_run[c] - use);
                m_run[c] = mx;
                l_run[c] *= corr;
#pragma unroll
                for (int a = 0; a < NG; ++a) {
                    z[a][c] *= corr;
#pragma unroll
                    for (int b = 0; b < 4; ++b) { o[a][b][c] *= corr; o[a][b][c + 2] *= corr; }
                }
#pragma unroll
                for (int n = 0; n < NP; ++n)
#pragma unroll
                    for (int e = c; e < 4; e += 2) {
                        s[n][e] = pd_exp2(s[n][e] - use);
                        l_run[c] += s[n][e];
                    }
            }
#pragma unroll
            for (int n = 0; n < NP; ++n) {
                const int mine = (n * CP + my_sub) * 16 + g;
                const bool gone0 = edge && (k0 + mine > pos || k0 + mine < first), gone1 = edge && (k0 + mine + 8 > pos || k0 + mine + 8 < first);
#pragma unroll
                for (int a = 0; a < NG; ++a) {
                    const uint32_t p0 = gone0 ? 0u : vp[mine * NG + a], p1 = gone1 ? 0u : vp[(mine + 8) * NG + a];
                    const float st0 = pair_step(p0) * PD_P_UP, st1 = pair_step(p1) * PD_P_UP, ze0 = pair_zero(p0), ze1 = pair_zero(p1);
                    z[a][0] = fmaf(s[n][0], ze0, fmaf(s[n][2], ze1, z[a][0]));
                    z[a][1] = fmaf(s[n][1], ze0, fmaf(s[n][3], ze1, z[a][1]));
                    const uint32_t b0 = pd_transpose(pd_pack(s[n][0] * st0, s[n][1] * st0)), b1 = pd_transpose(pd_pack(s[n][2] * st1, s[n][3] * st1));
#pragma unroll
                    for (int c = 0; c < CP; ++c) {
                        const uint32_t bc0 = CP == 1 || g / RC == c ? b0 : 0u, bc1 = CP == 1 || g / RC == c ? b1 : 0u;      // the columns of sub-step c
                        const unsigned char* vrow = vc + ((n * CP + c) * 16 + 2 * t) * (NG * 32) + a * 32 + g * 4;
                        const uint32_t v0 = *reinterpret_cast<const uint32_t*>(vrow), v1 = *reinterpret_cast<const uint32_t*>(vrow + NG * 32);
                        const uint32_t v8 = *reinterpret_cast<const uint32_t*>(vrow + 8 * NG * 32), v9 = *reinterpret_cast<const uint32_t*>(vrow + 9 * NG * 32);
#pragma unroll
                        for (int half = 0; half < 2; ++half) {      // entries 8g … + 3, then 8g + 4 … + 7
                            const uint32_t x = __byte_perm(v0, v1, half ? 0x7632 : 0x5410), y = __byte_perm(v8, v9, half ? 0x7632 : 0x5410);
                            const uint32_t x8 = x >> 8, y8 = y >> 8;
                            pd_mma(o[a][2 * half], x & PK_LOW, x8 & PK_LOW, y & PK_LOW, y8 & PK_LOW, bc0, bc1);
                            pd_mma(o[a][2 * half + 1], x & PK_HIGH, x8 & PK_HIGH, y & PK_HIGH, y8 & PK_HIGH, bc0, bc1);
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
    if (!small) pdl_launch_dependents();
    __syncthreads();                                                // every warp is done with its ring: the sums go there
    // the warp's sums: [warp][column][DH] float32 (8 columns of DH numbers are less than a warp's ring)
    float* all = reinterpret_cast<float*>(pd_raw);
    const float down = (0x1p100f / PD_P_UP) * 0x1p33f;
#pragma unroll
    for (int c = 0; c < 2; ++c) {
        float l = l_run[c];
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) l += __shfl_xor_sync(0xffffffffu, l, x);
        const int col = 2 * t + c;
        if (g == 0) { w_max[warp][col] = m_run[c]; w_sum[warp][col] = l; }
#pragma unroll
        for (int a = 0; a < NG; ++a) {
            float zz = z[a][c];
#pragma unroll
            for (int x = 4; x < 32; x <<= 1) zz += __shfl_xor_sync(0xffffffffu, zz, x);
            if (col % RC < n_q) {
                float* dst = all + ((size_t)warp * 8 + col) * DH + a * 64 + g * 8;
                // products 0 … 3 hold entries (0, 2), (1, 3), (4, 6), (5, 7); the odd ones sixteenfold
                *reinterpret_cast<float4*>(dst) = make_float4(fmaf(o[a][0][c], down, zz), fmaf(o[a][1][c], down / 16.f, zz),
                                                              fmaf(o[a][0][c + 2], down, zz), fmaf(o[a][1][c + 2], down / 16.f, zz));
                *reinterpret_cast<float4*>(dst + 4) = make_float4(fmaf(o[a][2][c], down, zz), fmaf(o[a][3][c], down / 16.f, zz),
                                                                  fmaf(o[a][2][c + 2], down, zz), fmaf(o[a][3][c + 2], down / 16.f, zz));
            }
        }
    }
    __syncthreads();
    // the CTA's sums of a query, over its columns of all warps with any token, into the place of warp 0's first
    const int n_warps = min(WARPS, max(1, part_n));                 // (warps behind have none)
    const int place = row * gridDim.x + blockIdx.x;
    float* my_parts = partials + (size_t)place * gridDim.z * RC * (DH + 4);
    for (int idx = threadIdx.x; idx < n_q * (DH / 4); idx += WARPS * 32) {
        const int qi = idx / (DH / 4), c4 = idx % (DH / 4);
        float M = -INFINITY;
        for (int w = 0; w < n_warps; ++w)
#pragma unroll
            for (int c = 0; c < CP; ++c) M = fmaxf(M, w_max[w][c * RC + qi]);
        const float use = M == -INFINITY ? 0.f : M;
        float L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int w = 0; w < n_warps; ++w)
#pragma unroll
            for (int c = 0; c < CP; ++c) {
                const float f = pd_exp2(w_max[w][c * RC + qi] - use);            // (−inf gives 0; sums that are not numbers stay so)
                const float4 v = *reinterpret_cast<const float4*>(all + ((size_t)w * 8 + c * RC + qi) * DH + c4 * 4);
                L = fmaf(w_sum[w][c * RC + qi], f, L);
                acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
            }
        if (parts == 1) {
            const float inv = (L > 0.f || L != L) ? 1.f / L : 0.f;
            *reinterpret_cast<uint2*>(out + (size_t)at_row * ld_out + (size_t)(hk * R + q0 + qi) * DH + c4 * 4) =
                make_uint2(pd_pack(acc.x * inv, acc.y * inv), pd_pack(acc.z * inv, acc.w * inv));
        } else {
            float* mine = my_parts + (size_t)(part * RC + qi) * (DH + 4);
            *reinterpret_cast<float4*>(mine + c4 * 4) = acc;
            if (c4 == 0) *reinterpret_cast<float2*>(mine + DH) = make_float2(M, L);
        }
    }
    if (parts == 1) return;
    // the CTA that finds all parts there merges them, each in its turn, so the sum does not depend on who came last
    __syncthreads();
    if (threadIdx.x == 0) {
        __threadfence();                                            // (of everything that the barrier has shown this thread)
        const int before = atomicAdd(&counters[place], 1);
        s_last = before == parts - 1;
        if (s_last) counters[place] = 0;                            // left as it was found
        __threadfence();
    }
    __syncthreads();
    if (!s_last) return;
    // lanes of threads: SHARES of them take every SHARES-th part of a piece of four numbers, and meet in shared memory
    constexpr int N4 = RC * (DH / 4), SHARES = WARPS * 32 / N4 > 0 ? WARPS * 32 / N4 : 1;
    float* meet = reinterpret_cast<float*>(pd_raw);                 // [SHARES][N4][8]
    for (int idx = threadIdx.x; idx < SHARES * N4; idx += WARPS * 32) {
        const int share = idx / N4, i4 = idx % N4, qi = i4 / (DH / 4), c4 = i4 % (DH / 4);
        float M = -INFINITY, L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        if (qi < n_q) {
#pragma unroll 8
            for (int p = share; p < parts; p += SHARES) {
                const float* theirs = my_parts + (size_t)(p * RC + qi) * (DH + 4);
                const float2 ml = __ldcg(reinterpret_cast<const float2*>(theirs + DH));
                const float4 v = __ldcg(reinterpret_cast<const float4*>(theirs + c4 * 4));
                const float m_new = fmaxf(M, ml.x), use = m_new == -INFINITY ? 0.f : m_new;
                const float fa = pd_exp2(M - use), fb = pd_exp2(ml.x - use);       // (−inf gives 0)
                L = fmaf(L, fa, ml.y * fb);
                acc.x = fmaf(acc.x, fa, v.x * fb); acc.y = fmaf(acc.y, fa, v.y * fb); acc.z = fmaf(acc.z, fa, v.z * fb); acc.w = fmaf(acc.w, fa, v.w * fb);
                M = m_new;
            }
        }
        *reinterpret_cast<float4*>(meet + (size_t)idx * 8) = acc;
        *reinterpret_cast<float2*>(meet + (size_t)idx * 8 + 4) = make_float2(M, L);
    }
    __syncthreads();
    for (int i4 = threadIdx.x; i4 < n_q * (DH / 4); i4 += WARPS * 32) {
        float M = -INFINITY, L = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int x = 0; x < SHARES; ++x) M = fmaxf(M, meet[(size_t)(x * N4 + i4) * 8 + 4]);
        const float use = M == -INFINITY ? 0.f : M;
#pragma unroll
        for (int x = 0; x < SHARES; ++x) {
            const float* from = meet + (size_t)(x * N4 + i4) * 8;
            const float f = pd_exp2(from[4] - use);
            const float4 v = *reinterpret_cast<const float4*>(from);
            L = fmaf(from[5], f, L);
            acc.x = fmaf(v.x, f, acc.x); acc.y = fmaf(v.y, f, acc.y); acc.z = fmaf(v.z, f, acc.z); acc.w = fmaf(v.w, f, acc.w);
        }
        const float inv = (L > 0.f || L != L) ? 1.f / L : 0.f;
        *reinterpret_cast<uint2*>(out + (size_t)at_row * ld_out + (size_t)(hk * R + q0 + i4 / (DH / 4)) * DH + i4 % (DH / 4) * 4) =
            make_uint2(pd_pack(acc.x * inv, acc.y * inv), pd_pack(acc.z * inv, acc.w * inv));
    }
}

template <int NG, int RC, bool FEW>
int pd_launch(const void* qkv, int ld, int q_off, const void* Kq, const void* Kp, const void* Vq, const void* Vp, int n_blocks, const int* block_table,
              int max_blocks, const int* tok_slot, const int* tok_pos, const int* row_of, void* out, int ld_out, int rows, int H, int Hkv, float scale, int window, int n_split, int part_tiles,
              float* partials, int* counters, int* dev_err, cudaStream_t stream) {
    const int R = H / Hkv, q_tiles = (R + RC - 1) / RC;
    constexpr size_t smem = pd_smem(NG, FEW);
    static_assert(PD_STAGES * pd_tile_bytes(NG) >= 8 * NG * 64 * 4, "a warp's sums fit its ring");
    static_assert(smem >= (size_t)RC * NG * 16 * 32 && smem >= (size_t)pd_warps(NG, FEW) * 32 * 32, "the merge's shares fit");
    static DeviceMarks marks;
    auto kern = attn_packed_decode_kernel<NG, RC, FEW>;
    cudaError_t e = allow_shared_memory(marks, kern, smem);
    if (e != cudaSuccess) return vlrf_fail(VLRF_ERR_CUDA, "attn_packed_decode: %zu bytes of shared memory: %s", smem, cudaGetErrorString(e));
    e = launch_chained(kern, dim3(Hkv * q_tiles, rows, n_split), dim3(pd_warps(NG, FEW) * 32), smem, stream, (const __nv_bfloat16*)qkv, ld, q_off,
                       (const unsigned char*)Kq, (const unsigned char*)Kp, (const unsigned char*)Vq, (const unsigned char*)Vp, n_blocks, block_table, max_blocks,
                       tok_slot, tok_pos, row_of, (__nv_bfloat16*)out, ld_out, R, Hkv, q_tiles, scale, window, part_tiles, partials, counters, dev_err);
    if (e != cudaSuccess) return vlrf_fail(VLRF_ERR_CUDA, "attn_packed_decode: %s", cudaGetErrorString(e));
    return vlrf_check_launch("attn_packed_decode");
}

constexpr int pd_columns(int dh, int R) { return dh > 128 || R > 4 ? 8 : R > 2 ? 4 : 2; }
}  // namespace

extern "C" int vlrf_attn_packed_decode_takes(int H, int Hkv, int dh, int BT, int ld, int q_off, int ld_out) {
    return H > 0 && Hkv > 0 && H % Hkv == 0 && dh > 0 && dh % 64 == 0 && dh <= 256 && BT == PD_TOKENS && ld % 8 == 0 && q_off % 8 == 0 && ld_out % 8 == 0;
}

// Scratch of a launch with n_split > 1: float32 numbers of partials, int32 numbers of counters.
extern "C" int vlrf_attn_packed_decode_scratch(int rows, int H, int Hkv, int dh, int n_split, long long* floats, long long* ints) {
    VLRF_REQUIRE(rows >= 0 && H > 0 && Hkv > 0 && H % Hkv == 0 && dh > 0 && n_split >= 1, "attn_packed_decode: bad sizes");
    const int R = H / Hkv, RC = pd_columns(dh, R);
    const long long places = (long long)rows * Hkv * ((R + RC - 1) / RC);
    *floats = n_split > 1 ? places * n_split * RC * (dh + 4) : 0;
    *ints = n_split > 1 ? places : 0;
    return VLRF_OK;
}

extern "C" int vlrf_attn_packed_decode(const void* qkv, int ld, int q_off, const void* Kq, const void* Kp, const void* Vq, const void* Vp, int n_blocks,
                                       const int* block_table, int max_blocks, const int* tok_slot, const int* tok_pos, const int* row_of, void* out,
                                       int ld_out, int rows, int H, int Hkv, int dh, int BT, float scale, int window, int few, int n_split, int part_tiles, float* partials,
                                       int* counters, int* dev_err, cudaStream_t stream) {
    VLRF_REQUIRE(vlrf_attn_packed_decode_takes(H, Hkv, dh, BT, ld, q_off, ld_out),
                 "attn_packed_decode: %d heads over %d of %d, blocks of %d, row strides %d and %d are not taken", H, Hkv, dh, BT, ld, ld_out);
    VLRF_REQUIRE(rows >= 0 && rows <= 65535 && max_blocks > 0 && n_blocks >= 0 && window >= 0 && dev_err != nullptr, "attn_packed_decode: bad arguments");
    VLRF_REQUIRE(n_split >= 1 && n_split <= PD_MAX_SPLIT && part_tiles >= 1 && (n_split == 1 || (partials != nullptr && counters != nullptr)),
                 "attn_packed_decode: %d parts (1 to %d; more than one wants scratch)", n_split, PD_MAX_SPLIT);
    for (const void* p : {qkv, Kq, Kp, Vq, Vp, (const void*)out, (const void*)partials})
        VLRF_REQUIRE((reinterpret_cast<uintptr_t>(p) & 15) == 0, "attn_packed_decode: tensors begin on 16 bytes");
    if (rows == 0) return VLRF_OK;
    const int R = H / Hkv, RC = pd_columns(dh, R);
#define GO(NG, C) (few ? pd_launch<NG, C, true>(ARGS) : pd_launch<NG, C, false>(ARGS))
#define ARGS qkv, ld, q_off, Kq, Kp, Vq, Vp, n_blocks, block_table, max_blocks, tok_slot, tok_pos, row_of, out, ld_out, rows, H, Hkv, scale, window, n_split, part_tiles, \
             partials, counters, dev_err, stream
    if (dh == 64) return RC == 2 ? GO(1, 2) : RC == 4 ? GO(1, 4) : GO(1, 8);
    if (dh == 128) return RC == 2 ? GO(2, 2) : RC == 4 ? GO(2, 4) : GO(2, 8);
    return dh == 192 ? GO(3, 8) : GO(4, 8);
#undef GO
#undef ARGS
}
