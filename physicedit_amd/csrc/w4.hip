// Linears of a few rows with 4-bit weights and group scales (pe_gemv_w4).
//
//   y[m,n] = r[m] * sum_g s[n,g] * sum_{k in g} (c[n,k] - z[n,g]) x[m,k] + bias[n],     c, z in 0 .. 15, s bf16, g = 32, 64 or 128 inputs
//   r[m] = rsqrt(mean_k x[m,k]^2 + eps) (an RMSNorm whose weight is folded into the weight's columns) or 1
//   out = y + res,  or with the gated-MLP epilogue  out[m,f] = silu(y[m,f]) * y[m,F+f];  sums in fp32, one rounding to bf16 at the end.
//
// Every weight byte is used once, so the kernel is bound by HBM: N K / 2 bytes + 4 N K / g.  The products run on
// v_mfma_f32_16x16x32_bf16 even for one row: with the weights as the 16-row operand an instruction takes 512 weights in 16 cycles of its
// SIMD, four times what HBM delivers to a CU, and up to 16 rows of x cost what one does.
// A code becomes a bf16 by ORing it into the mantissa of 128.0: (u >> 4 i) & 0x000f000f | 0x43004300 is the pair 128 + c, so two weights cost
// two instructions (a shift and an and-or).  The offset and the zero point leave through the row sum of x over the group,
//   sum (c - z) x = sum (128 + c) x - (128 + z) sum x,
// which one more MFMA per 32 inputs (ones as the weights) gives every lane for the rows it holds; products of two bf16 are exact in
// fp32, so this costs about 2^-24 * 136 * sum |x| of a group, far below the output's bf16 rounding: of 25088 outputs at K = 18944, 42 round otherwise than
// the exact value, 28 of the plain fp32 form's.  (In the mantissa of 16.0 it costs 24 instead of 136, 15 of 25088 round otherwise, and two more instructions a
// code word and scale: gated, one row 18.3 -> 20.0 us; vocabulary 56.3 -> 58.9.)  r comes the same way: x as BOTH operands leaves sum x^2 on the diagonal.
// 143 |x| summed over a group has to stay finite, and sum x^2 where it is asked for: |x| <= 2^100, or 2^50 with the norm, keeps all of them far from the end.
//
// Layout of the codes: tiles of 16 outputs x 128 inputs, 1 KiB, [N/16][K/128][lane][step]: the lane's four words are its A fragments of the
// four 32-input steps (output lane & 15, inputs 32 step + 8 (lane >> 4) + e, element e in nibble (e >> 1) + 4 (e & 1)), one coalesced 16-byte load
// per lane and tile.  Scales and zero points are one word, [N/16][groups][16]: the scale's bf16 and -(128 + zero)
// as a bf16, exact, above it: each is one instruction away from the fp32 it is used as.  N and K are padded to 16 and 128 with scales of 0.
//
// A work-group of W waves takes R tiles of 16 outputs; its waves take turns at the 128-input chunks and join their fp32 sums in LDS in a
// fixed order: results do not depend on scheduling.  Rows from M to the next multiple of four are row M - 1 again, those behind what the LDS held:
// a row of x is a column of its own in every product, and theirs are never stored.
#include "common.h"
#include "kernels.h"

namespace pe {

struct W4Args {
    const bf16* x;
    const u32x4* codes;
    const u32x4* scale;       // words: scale bf16 | -(128 + zero) bf16 << 16
    const bf16* bias;
    const bf16* res;
    bf16* out;
    long long ldx, ldr, ldo;
    int M, N, K, KC, G;       // KC = chunks of 128 inputs, G = groups (K padded to 128)
    int pair_tiles;           // gated epilogue: tile of the up row = tile of the gate row + pair_tiles
    float eps;
};

PE_DEV bf16x8 w4_fragment(uint32_t u) {
    u32x4 f;
#pragma unroll
    for (int i = 0; i < 4; ++i) f[i] = ((u >> (4 * i)) & 0x000f000fu) | 0x43004300u;
    return __builtin_bit_cast(bf16x8, f);
}

// MT: tiles of 16 rows of x.  R: weight tiles of a work-group.  W: waves.
// GS: 32-input steps of a group (1, 2, 4).
template <int MT, int R, int W, int GS, bool NORM, bool SWIGLU>
__global__ void __launch_bounds__(W * 64) gemv_w4_kernel(W4Args a) {
    // a wave's chunk of x, 16 MT rows of 256 bytes, and later its sums
    constexpr int XB = MT * 4096, PB = R * 1024, SB = XB > PB ? XB : PB;
    __shared__ __attribute__((aligned(16))) uint8_t stage[W][SB];
    __shared__ float sq[W][MT * 16];
    constexpr int GC = 4 / GS;                 // groups of a chunk
    const int lane = lane_id(), w = wave_id(), j = lane >> 4, c = lane & 15;
    const int ntiles = (a.N + 15) >> 4;
    int tile[R];
#pragma unroll
    for (int r = 0; r < R; ++r) {
        const int t = SWIGLU ? (int)blockIdx.x * (R / 2) + (r >> 1) : (int)blockIdx.x * R + r;
        tile[r] = SWIGLU ? min(t, a.pair_tiles - 1) + (r & 1) * a.pair_tiles : min(t, ntiles - 1);
    }
    f32x4 acc[R][MT] = {};
    f32x4 gram[MT] = {};
    bf16x8 ones;
#pragma unroll
    for (int e = 0; e < 8; ++e) ones[e] = (bf16)1.0f;

    // A chunk on its way.  x goes straight into LDS, four rows of 256 bytes an instruction: 16 consecutive lanes read one row.  (As fragments, 16 lanes read
    // 16 rows and a load takes 64 steps of the address unit instead of 16: N = 3584, K = 18944, 7 rows 18.6 us against 13.9, 64 rows 74.6 against 38.0.)
    // Piece p (16 bytes) of row m goes to slot p ^ (m & 15): the fragment reads below find their 16 rows in 16 different slots.  The steps that pad K have
    // scales of 0 (their groups are padding too), their x is any part of the row.  The barriers: or the scheduler sinks the loads to their uses to save
    // registers, one round trip after another.
#define PE_W4_FETCH(CHUNK, WQ, SC)                                                                                                      \
    {                                                                                                                                   \
        _Pragma("unroll") for (int q = 0; q < MT * 4; ++q)                                                                              \
            if (4 * q < a.M) {                                                                                                          \
                const int m = 4 * q + j, k = (CHUNK) * 128 + 8 * (c ^ (m & 15));                                                        \
                glds16(a.x + (size_t)min(m, a.M - 1) * a.ldx + min(k, a.K - 8), stage[w] + q * 1024);                                   \
            }                                                                                                                           \
        __builtin_amdgcn_sched_barrier(0);                                                                                              \
        _Pragma("unroll") for (int r = 0; r < R; ++r)                                                                                   \
            WQ[r] = __builtin_nontemporal_load(a.codes + ((size_t)tile[r] * a.KC + (CHUNK)) * 64 + lane);                               \
        _Pragma("unroll") for (int r = 0; r < R; ++r)                                                                                   \
            _Pragma("unroll") for (int g = 0; g < GC; ++g) SC[r][g] = a.scale[((size_t)tile[r] * a.G + (CHUNK) * GC + g) * 4 + j];      \
        __builtin_amdgcn_sched_barrier(0);                                                                                              \
    }
    // Waves that take many chunks of few tiles ask for the next chunk as soon as this one is in registers (N = 3584, K = 18944: one row 13.5 -> 12.4 us, 24
    // rows 22.6 -> 20.2; 33 rows, N = 37888, gated: 46.9 -> 40.6).  Elsewhere the registers cost more waves than that hides (N = 152064, one row: R = 4
    // 55.5 -> 72; 60 rows, N = 12001, R, W = 2, 4: 15.3 -> 21.3).
    constexpr bool AHEAD = R == 1 || (MT == 3 && W == 4);
    u32x4 nq[R], ns[R][GC];
    if (AHEAD && w < a.KC) PE_W4_FETCH(w, nq, ns)
    for (int kc = w; kc < a.KC; kc += W) {
        u32x4 wq[R], sc[R][GC];
        bf16x8 b[MT][4];
        // The compiler's own waits between copies into LDS and reads of it are not there in every variant.  Each wait here is for everything, whatever loads
        // the compiler emits beside them, and no memory access passes it: the last chunk's reads are done before its place is filled again, and the
        // copies before they are read.  (A wait for the copies alone, by the number of younger loads, is no faster: 14.1, 13.1, 20.3 and 56.4 us against
        // 14.3, 13.2, 20.4 and 55.9 -- N, K = 3584, 18944 with 7 rows, 5001, 3424 with 33, 3584, 18944 with 24, 152064, 3584 with one; gated, one row: 18.4, 18.5.)
        if (!AHEAD) {
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
            PE_W4_FETCH(kc, wq, sc)
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int s = 0; s < 4; ++s)
#pragma unroll
            for (int mt = 0; mt < MT; ++mt) b[mt][s] = *(const bf16x8*)(stage[w] + (mt * 16 + c) * 256 + ((4 * s + j) ^ c) * 16);
        if (AHEAD) {
#pragma unroll
            for (int r = 0; r < R; ++r) {
                wq[r] = nq[r];
#pragma unroll
                for (int g = 0; g < GC; ++g) sc[r][g] = ns[r][g];
            }
            __builtin_amdgcn_sched_barrier(0);
            asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");         // the chunk is in registers, its place in LDS is free
            __builtin_amdgcn_sched_barrier(0);
            if (kc + W < a.KC) PE_W4_FETCH(kc + W, nq, ns)
        }
        if (NORM) {
#pragma unroll
            for (int s = 0; s < 4; ++s)
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) {
                    const bf16x8 f = kc * 128 + 32 * s < a.K ? b[mt][s] : bf16x8{};
                    gram[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, f, gram[mt], 0, 0, 0);
                }
        }
#pragma unroll
        for (int g = 0; g < GC; ++g) {
            f32x4 sum[R][MT] = {}, sx[MT] = {};
#pragma unroll
            for (int s = g * GS; s < (g + 1) * GS; ++s) {
#pragma unroll
                for (int mt = 0; mt < MT; ++mt) sx[mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(ones, b[mt][s], sx[mt], 0, 0, 0);
#pragma unroll
                for (int r = 0; r < R; ++r) {
                    const bf16x8 f = w4_fragment(wq[r][s]);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt) sum[r][mt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, b[mt][s], sum[r][mt], 0, 0, 0);
                }
            }
#pragma unroll
            for (int r = 0; r < R; ++r)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float scale = __uint_as_float(sc[r][g][i] << 16), off = __uint_as_float(sc[r][g][i] & 0xffff0000u);
#pragma unroll
                    for (int mt = 0; mt < MT; ++mt)
                        acc[r][mt][i] = __builtin_fmaf(scale, __builtin_fmaf(off, sx[mt][i], sum[r][mt][i]), acc[r][mt][i]);
                }
        }
    }
#undef PE_W4_FETCH

    if (NORM) {             // the diagonal: row 4 j + i == column c
#pragma unroll
        for (int mt = 0; mt < MT; ++mt)
#pragma unroll
            for (int i = 0; i < 4; ++i)
                if (4 * j + i == c) sq[w][mt * 16 + c] = gram[mt][i];
    }
#pragma unroll
    for (int mt = 0; mt < MT; ++mt) {
#pragma unroll
        for (int r = 0; r < R; ++r) *(f32x4*)(stage[w] + (r * 64 + lane) * 16) = acc[r][mt];
        __syncthreads();
        constexpr int OUT = SWIGLU ? R / 2 : R;
        for (int o = w; o < OUT; o += W) {
            const int m = mt * 16 + c;
            float rs = 1.0f;
            if (NORM) {
                float t = 0.f;
#pragma unroll
                for (int v = 0; v < W; ++v) t += sq[v][m];
                rs = rsqrtf(t / (float)a.K + a.eps);
            }
            f32x4 y[2] = {};
#pragma unroll
            for (int p = 0; p < (SWIGLU ? 2 : 1); ++p) {
#pragma unroll
                for (int v = 0; v < W; ++v) y[p] += *(const f32x4*)(stage[v] + ((SWIGLU ? 2 * o + p : o) * 64 + lane) * 16);
            }
            const int t = (int)blockIdx.x * OUT + o;
            const int n0 = t * 16 + 4 * j, cols = SWIGLU ? a.N / 2 : a.N;
            if (m < a.M && n0 < cols) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int n = n0 + i;
                    if (n >= cols) break;
                    float v = y[0][i] * rs + (a.bias ? (float)a.bias[n] : 0.f);
                    if (SWIGLU) {
                        const float u = y[1][i] * rs + (a.bias ? (float)a.bias[cols + n] : 0.f);
                        v = v * sigmoidf_(v) * u;
                    }
                    if (a.res) v += (float)a.res[(size_t)m * a.ldr + n];
                    a.out[(size_t)m * a.ldo + n] = (bf16)v;
                }
            }
        }
        __syncthreads();
    }
}

template <int MT, int R, int W, bool SWIGLU>
static void w4_launch(const W4Args& a, int gs, bool norm, hipStream_t stream) {
    const int tiles = SWIGLU ? a.pair_tiles : (a.N + 15) / 16, per = SWIGLU ? R / 2 : R;
    const dim3 grid((tiles + per - 1) / per), block(W * 64);
#define PE_W4(GS, NORM) hipLaunchKernelGGL((gemv_w4_kernel<MT, R, W, GS, NORM, SWIGLU>), grid, block, 0, stream, a)
    if (gs == 1) { if (norm) PE_W4(1, true); else PE_W4(1, false); }
    else if (gs == 2) { if (norm) PE_W4(2, true); else PE_W4(2, false); }
    else { if (norm) PE_W4(4, true); else PE_W4(4, false); }
#undef PE_W4
}

int launch_gemv_w4(const W4Problem& p, hipStream_t stream) {
    PE_REQUIRE(p.x && p.codes && p.scale && p.out, "gemv_w4: null pointer");
    PE_REQUIRE(p.group == 32 || p.group == 64 || p.group == 128, "gemv_w4: group of %d inputs (32, 64 or 128)", p.group);
    PE_REQUIRE(p.M >= 1 && p.M <= 64, "gemv_w4: M=%d rows (1 ... 64; more rows are a matrix product)", p.M);
    PE_REQUIRE(p.N >= 1 && p.K >= p.group && p.K % p.group == 0, "gemv_w4: N=%d K=%d (K must be a multiple of the group %d)", p.N, p.K, p.group);
    PE_REQUIRE(p.N <= (1 << 26) && p.K <= (1 << 22), "gemv_w4: N=%d K=%d out of range", p.N, p.K);
    PE_REQUIRE(p.ldx >= p.K && p.ldx % 8 == 0 && ((uintptr_t)p.x & 15) == 0, "gemv_w4: rows of x must be 16-byte aligned (ldx=%lld)", p.ldx);
    PE_REQUIRE(((uintptr_t)p.codes & 15) == 0 && ((uintptr_t)p.scale & 15) == 0, "gemv_w4: unaligned weight");
    const int cols = p.swiglu ? p.N / 2 : p.N;
    PE_REQUIRE(!p.swiglu || p.N % 32 == 0, "gemv_w4: the gated epilogue needs a multiple of 16 gate and up rows (N=%d)", p.N);
    PE_REQUIRE(!(p.swiglu && p.res), "gemv_w4: no residual with the gated epilogue");
    PE_REQUIRE(p.out != p.x, "gemv_w4: out may be res, not x (every work-group reads all of x)");
    PE_REQUIRE(p.ldo >= cols && (!p.res || p.ldr >= cols), "gemv_w4: row stride below the %d columns", cols);
    W4Args a;
    a.x = (const bf16*)p.x; a.codes = (const u32x4*)p.codes; a.scale = (const u32x4*)p.scale;
    a.bias = (const bf16*)p.bias; a.res = (const bf16*)p.res; a.out = (bf16*)p.out;
    a.ldx = p.ldx; a.ldr = p.ldr; a.ldo = p.ldo;
    a.M = p.M; a.N = p.N; a.K = p.K; a.KC = (p.K + 127) / 128; a.G = a.KC * (128 / p.group);
    a.pair_tiles = p.swiglu ? p.N / 32 : 0;
    a.eps = p.eps;
    const int gs = p.group / 32;
    // Weight tiles (R) and waves (W) of a work-group.  At most a tile per CU: each gets all the waves that fit (N = 3584, K = 18944, one row: R, W = 1, 16
    // 12.3 us, 1, 8 17.2, 2, 8 20.7); up to two, the same with pairs (N = 5120, K = 13824: 2, 16 12.1 us, 1, 8 14.9, 1, 16 16.1).  Some per CU: R = 1 leaves them balanced (N = 10000, K = 3584: 1, 8 7.0 us, 4, 8 8.8).  Many: a work-group's start,
    // end and reads of x are shared (N = 152064: 1, 8 79.5 us, 2, 8 65.9, 4, 8 53.2).  From two row tiles on x weighs more (20 rows, N = 5001: 1, 8 11.1 us, 2, 8 10.1;
    // 33: 19.1 and 13.1), from three on its chunks fill the LDS (60 rows, N = 12001: 2, 8 18.1 us, 2, 4 15.0, 4, 4 17.3; 64 rows, N = 152064: 199, 179, 202).
    const int tiles = (p.N + 15) / 16, mt = (p.M + 15) / 16;
    const int size = tiles <= 256 ? 0 : tiles <= (mt >= 3 ? 512 : 1024) ? 1 : 2;
    // The gated epilogue works on pairs of tiles: with many, one pair and four waves for few rows (N = 37888, one row: 2, 4 18.4 us, 4, 8 19.7; 16 rows: 22.0, 21.3).
#define PE_W4(MT, R, W) { if (p.swiglu) w4_launch<MT, (R == 1 ? 2 : R), (R == 1 ? 8 : W), true>(a, gs, p.norm, stream); else w4_launch<MT, R, W, false>(a, gs, p.norm, stream); }
    if (p.swiglu && size == 2 && p.M <= 8) w4_launch<1, 2, 4, true>(a, gs, p.norm, stream);
    else if (!p.swiglu && mt == 1 && size == 1 && tiles <= 512) w4_launch<1, 2, 16, false>(a, gs, p.norm, stream);
    else
    if (mt == 1) { if (size == 0) PE_W4(1, 1, 16) else if (size == 1) PE_W4(1, 1, 8) else PE_W4(1, 4, 8) }
    else if (mt == 2) { if (size == 0) PE_W4(2, 1, 8) else if (size == 1) PE_W4(2, 2, 8) else PE_W4(2, 4, 8) }
    else if (mt == 3) { if (size == 0) PE_W4(3, 1, 8) else if (size == 1) PE_W4(3, 2, 8) else PE_W4(3, 2, 4) }
    else { if (size == 0) PE_W4(4, 1, 8) else if (size == 1) PE_W4(4, 2, 8) else PE_W4(4, 2, 4) }
#undef PE_W4
    return check_launch("gemv_w4_kernel");
}

}  // namespace pe
