// The e4m3 key/value cache: written (rotary embedding and quantisation in one pass) and read back by the attention of one token or of a
// tree of drafted tokens.
//
// A row is one (sequence, token, kv head): D codes (OCP e4m3fn) and one fp32 scale, value = code * scale,
//   scale = max(max|x| * (1/448), 2^-126),   code = e4m3(x / scale)     (fp32 division, round to nearest even)
// A row that holds a value that is not finite gets the scale NaN and codes of zero: codes are never NaN, so a masked row can be
// multiplied by a probability of zero whatever was written there, and an unmasked one shows in the result.
//
// Layout: keys [B][H][cap][D]; values [B][H][cap/64][D][64], transposed inside blocks of 64 tokens, because the second product of the
// attention wants 16 consecutive TOKENS of one channel per lane; scales [B][H][cap].  cap is a multiple of 64.
#include "common.h"
#include "kernels.h"

namespace pe {

constexpr float E4M3_STEP = 1.0f / 448.0f, SCALE_MIN = 1.17549435e-38f;    // 2^-126

// ------------------------------------------------------------------------------------------------
// write: a lane holds 8 channels of the lower and the 8 channels half a head above, so the rotation
//   x' = x cos + rot(x) sin,  rot(x)[i] = -x[i + D/2] (i < D/2), x[i - D/2] (else)
// stays in the lane and a row is D / 16 lanes.  fp32, products rounded before the sum (no contraction), one rounding at the end.
// Bound by the bytes where many tokens are written, by the launch where one is.
// ------------------------------------------------------------------------------------------------
PE_DEV void load_half(const bf16* p, float (&x)[8]) {
    const bf16x8 t = *(const bf16x8*)p;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)t[e];
}
PE_DEV void load_half(const float* p, float (&x)[8]) {
    const f32x4 a = *(const f32x4*)p, b = *(const f32x4*)(p + 4);
#pragma unroll
    for (int e = 0; e < 4; ++e) { x[e] = a[e]; x[4 + e] = b[e]; }
}

// codes and scale of a row spread over LPR lanes
template <int LPR>
PE_DEV float quantise_row(const float (&lo)[8], const float (&hi)[8], u32x2& clo, u32x2& chi) {
    uint32_t top = 0;                 // |x| compared as integers: a NaN is above infinity, which is above every number
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        top = max(top, __float_as_uint(lo[e]) & 0x7fffffffu);
        top = max(top, __float_as_uint(hi[e]) & 0x7fffffffu);
    }
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if (top >= 0x7f800000u) {
        clo = chi = u32x2{0, 0};
        return __uint_as_float(0x7fc00000u);
    }
    const float scale = fmaxf(__uint_as_float(top) * E4M3_STEP, SCALE_MIN);
    // x / scale, correctly rounded, from one division per row: with r the rounded reciprocal, q = x r and the exact remainder e = x - q scale, q + e r rounds
    // to the quotient (Markstein 1990) as long as e does not underflow; rows so small that it could are divided
    const float r = 1.0f / scale;
    const bool tiny = scale < 0x1p-96f;
    auto over = [&](float x) __attribute__((always_inline)) {
        const float q = x * r;
        return __builtin_fmaf(__builtin_fmaf(-q, scale, x), r, q);
    };
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        if (tiny) {
            clo[h] = pack4_e4m3(lo[4 * h] / scale, lo[4 * h + 1] / scale, lo[4 * h + 2] / scale, lo[4 * h + 3] / scale);
            chi[h] = pack4_e4m3(hi[4 * h] / scale, hi[4 * h + 1] / scale, hi[4 * h + 2] / scale, hi[4 * h + 3] / scale);
        } else {
            clo[h] = pack4_e4m3(over(lo[4 * h]), over(lo[4 * h + 1]), over(lo[4 * h + 2]), over(lo[4 * h + 3]));
            chi[h] = pack4_e4m3(over(hi[4 * h]), over(hi[4 * h + 1]), over(hi[4 * h + 2]), over(hi[4 * h + 3]));
        }
    }
    return scale;
}

// how many of the T tokens of a sequence are written; start outside the cache: none
PE_DEV int append_count(int start, int T, int cap) { return start < 0 || start >= cap ? 0 : min(T, cap - start); }

// grid: x = blocks of tokens, y = groups of HG query heads, then of HG key heads, then value heads, z = sequences.  A row's lanes take the HG heads of
// their token together: the rotary tables are read once for them.  HG = 4, or 1 where few tokens are written and a row's latency counts (1 token, 28 + 4
// heads: 3.5 us against 5.3).
template <int D, int HG, typename TAB>
__global__ void __launch_bounds__(256) kv_append_kernel(KvAppend a) {
    constexpr int LPR = D / 16, ROWS = 256 / LPR;
    __shared__ __attribute__((aligned(16))) uint8_t turn[D][64 + 4];     // a block of values, transposed; rows of 17 words: no bank conflicts
    const int tid = (int)threadIdx.x, l = tid % LPR, d0 = 8 * l, b = (int)blockIdx.z;
    const int start = a.start[b], count = append_count(start, a.T, a.cap);
    int y = (int)blockIdx.y;
    if (y < a.q_groups + a.k_groups) {
        const bool is_q = y < a.q_groups;
        const int h0 = (is_q ? y : y - a.q_groups) * HG, heads = min(HG, (is_q ? a.n_q : a.H) - h0);
        const long long t0 = (long long)blockIdx.x * ROWS + tid / LPR;
        if (t0 >= a.T) return;                                    // a row's lanes leave together
        const int t = (int)t0;
        const bool there = t < count;
        const bf16* src = (is_q ? a.q + b * a.qs[0] + t * a.qs[1] + h0 * a.qs[2] : a.k + b * a.ks[0] + t * a.ks[1] + h0 * a.ks[2]) + d0;
        const long long hs = is_q ? a.qs[2] : a.ks[2];
        float lo[HG][8], hi[HG][8];
#pragma unroll
        for (int h = 0; h < HG; ++h) {
            const bf16* p = src + min(h, heads - 1) * hs;
            load_half(p, lo[h]);
            load_half(p + D / 2, hi[h]);
        }
        if (a.cos) {
            const int pos = !there ? 0 : a.positions ? a.positions[(size_t)b * a.T + t] : start + t;
            const bool known = pos >= 0 && pos < a.table_rows;     // no such row in the tables: the row becomes NaN
            const size_t at = (size_t)(known ? pos : 0) * D + d0;
            const TAB *cs = (const TAB*)a.cos + at, *sn = (const TAB*)a.sin + at;
            float cl[8], ch[8], sl[8], sh[8];
            load_half(cs, cl); load_half(cs + D / 2, ch); load_half(sn, sl); load_half(sn + D / 2, sh);
#pragma unroll
            for (int h = 0; h < HG; ++h)
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const float x = lo[h][e], z = hi[h][e];
                    lo[h][e] = known ? x * cl[e] + -z * sl[e] : __uint_as_float(0x7fc00000u);
                    hi[h][e] = known ? z * ch[e] + x * sh[e] : lo[h][e];
                }
        }
        if (is_q) {
            bf16* dst = a.q_out + (((size_t)b * a.T + t) * a.n_q + h0) * D + d0;
#pragma unroll
            for (int h = 0; h < HG; ++h) {
                if (h >= heads) break;
                bf16x8 ol, oh;
#pragma unroll
                for (int e = 0; e < 8; ++e) { ol[e] = there ? (bf16)lo[h][e] : (bf16)0.f; oh[e] = there ? (bf16)hi[h][e] : (bf16)0.f; }
                *(bf16x8*)(dst + h * D) = ol;
                *(bf16x8*)(dst + h * D + D / 2) = oh;
            }
            return;
        }
#pragma unroll
        for (int h = 0; h < HG; ++h) {
            if (h >= heads) break;
            u32x2 clo, chi;
            const float scale = quantise_row<LPR>(lo[h], hi[h], clo, chi);
            if (!there) continue;
            const size_t dst = ((size_t)b * a.H + h0 + h) * a.cap + start + t;
            *(u32x2*)(a.kc + dst * D + d0) = clo;
            *(u32x2*)(a.kc + dst * D + D / 2 + d0) = chi;
            if (l == 0) a.ksc[dst] = scale;
        }
        return;
    }
    // ---- values: one work-group per (b, head, block of 64 cache rows)
    const int h = y - a.q_groups - a.k_groups;
    const long long first0 = (long long)(start & ~63) + (long long)blockIdx.x * 64;      // cache row of the block's first token
    if (count == 0 || first0 >= start + count) return;
    const int first = (int)first0;
    const bool whole = first >= start && first + 64 <= start + count;
    const size_t plane = ((size_t)b * a.H + h) * a.cap;
    uint8_t* vdst = a.vc + (plane + first) * D;
#pragma unroll
    for (int r0 = 0; r0 < 64; r0 += ROWS) {
        const int r = r0 + tid / LPR, t = first + r - start;
        const bool mine = t >= 0 && t < count;
        float lo[8] = {}, hi[8] = {};
        if (mine) {
            const bf16* src = a.v + b * a.vs[0] + t * a.vs[1] + h * a.vs[2];
            load_half(src + d0, lo);
            load_half(src + D / 2 + d0, hi);
        }
        u32x2 clo, chi;
        const float scale = quantise_row<LPR>(lo, hi, clo, chi);
        if (!mine) continue;
        if (l == 0) a.vsc[plane + first + r] = scale;
        uint8_t* dst = whole ? &turn[d0][r] : vdst + (size_t)d0 * 64 + r;       // a block's other tokens stay as they are
        const int ld = whole ? 68 : 64;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            dst[e * ld] = (uint8_t)(clo[e >> 2] >> (8 * (e & 3)));
            dst[(D / 2 + e) * ld] = (uint8_t)(chi[e >> 2] >> (8 * (e & 3)));
        }
    }
    if (!whole) return;
    __syncthreads();
    for (int i = tid; i < D * 4; i += 256) {
        const int d = i >> 2, part = i & 3;
        const uint32_t* src = (const uint32_t*)&turn[d][16 * part];
        *(u32x4*)(vdst + (size_t)d * 64 + 16 * part) = u32x4{src[0], src[1], src[2], src[3]};
    }
}

int launch_kv_append(const KvAppend& in, hipStream_t stream) {
    KvAppend a = in;
    PE_REQUIRE(a.kc && a.vc && a.ksc && a.vsc && a.k && a.v && a.start, "kv_append: null pointer");
    PE_REQUIRE(a.D == 64 || a.D == 128, "kv_append: heads of %d (64 or 128)", a.D);
    PE_REQUIRE(a.B >= 1 && a.H >= 1 && a.T >= 1 && a.n_q >= 0 && a.cap >= 64 && a.cap % 64 == 0 && a.cap <= (1 << 30),
               "kv_append: bad shape (B=%d H=%d T=%d cap=%d)", a.B, a.H, a.T, a.cap);
    PE_REQUIRE((a.cos != nullptr) == (a.sin != nullptr) && (!a.cos || a.table_rows >= 1), "kv_append: cos and sin tables come together");
    PE_REQUIRE(a.n_q == 0 || (a.q && a.q_out && a.cos), "kv_append: queries are rotated: q, its output and the tables are needed");
    PE_REQUIRE(!a.positions || a.cos, "kv_append: positions without tables");
    const uintptr_t mis = (uintptr_t)a.kc | (uintptr_t)a.vc | (uintptr_t)a.k | (uintptr_t)a.v | (uintptr_t)a.q | (uintptr_t)a.q_out | (uintptr_t)a.cos | (uintptr_t)a.sin;
    PE_REQUIRE((mis & 15) == 0, "kv_append: pointers must be 16-byte aligned");
    for (int i = 0; i < 3; ++i)
        PE_REQUIRE(a.ks[i] % 8 == 0 && a.vs[i] % 8 == 0 && (a.n_q == 0 || a.qs[i] % 8 == 0), "kv_append: strides must be multiples of 8 elements");
    const int hg = (long long)a.B * a.T >= 256 ? 4 : 1;
    a.q_groups = (a.n_q + hg - 1) / hg;
    a.k_groups = (a.H + hg - 1) / hg;
    const long long tokens = 256 / (a.D / 16), row_blocks = (a.T + tokens - 1) / tokens;
    long long v_blocks = ((long long)a.T + 126) / 64;               // blocks of the cache that T rows from anywhere touch
    if (v_blocks > a.cap / 64) v_blocks = a.cap / 64;
    const dim3 grid((unsigned)(row_blocks > v_blocks ? row_blocks : v_blocks), a.q_groups + a.k_groups + a.H, a.B);
    PE_REQUIRE(grid.y <= 65535 && a.B <= 65535, "kv_append: too many heads or sequences");
#define PE_KV_APPEND(D, HG, TAB) hipLaunchKernelGGL((kv_append_kernel<D, HG, TAB>), grid, dim3(256), 0, stream, a)
#define PE_KV_APPEND_TAB(D, HG) if (a.table_f32) PE_KV_APPEND(D, HG, float); else PE_KV_APPEND(D, HG, bf16)
    if (a.D == 64) { if (hg == 1) { PE_KV_APPEND_TAB(64, 1); } else { PE_KV_APPEND_TAB(64, 4); } }
    else { if (hg == 1) { PE_KV_APPEND_TAB(128, 1); } else { PE_KV_APPEND_TAB(128, 4); } }
#undef PE_KV_APPEND_TAB
#undef PE_KV_APPEND
    return check_launch("kv_append_kernel");
}

// ------------------------------------------------------------------------------------------------
// read: T new tokens (1 ... 64) of a sequence against its context rows [0, start) and, where bit j of their word says so, the new row
// start + j:
//   s = (q . code_k) * scale_k * softmax_scale,   o = sum exp(s - max) scale_v code_v / sum exp(s - max),   nothing visible: o = 0
//
// Bound by the cache's bytes (2 D + 8 per row and kv head).  The query heads of a kv head and the new tokens share every byte: they are the
// columns (T * n_q / H of them, in tiles of 16) of v_mfma_f32_16x16x32_bf16, with 64 cache rows per step as the other operand.
//   S^T tile h (0 .. 3): A = codes of the keys, row r = token 16 (r >> 2) + 4 h + (r & 3) of the 64 -- so the lanes 16 j + c end up with the 16
//   CONSECUTIVE tokens 16 j ... 16 j + 15 of column c in their four results -- and B = the queries, bf16 as they came;
//   O^T += V^T P^T: A = 16 consecutive tokens of channel c, the 16 bytes that the transposed value blocks hold side by side.  P never leaves
//   the lane that computed it.
// e4m3 -> bf16 is exact (v_cvt_scalef32_pk_bf16_fp8, two codes an instruction); scale_k multiplies the fp32 score, scale_v the fp32
// probability.  The product p * scale_v goes into the matrix unit as TWO bf16, its rounding and the remainder: the matrix unit has time to spare here
// and the sum then carries 16 bits of each term instead of 8.
// Scores, maximum, sums and O are fp32.  A wave walks every fourth block of its work-group's range with a reference of its own for the exponentials; waves and
// work-groups (the cache's axis is split over `splits` of them) are joined in a fixed order.
// ------------------------------------------------------------------------------------------------
PE_DEV bf16x8 codes8(uint32_t a, uint32_t b) {
    typedef __attribute__((ext_vector_type(2))) __bf16 v2;
    const v2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false), x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
    const v2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false), x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
    return bf16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}

// maximum and sum over the four lanes 16 j + c of a column
PE_DEV float max_over_j(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(a[0]), __uint_as_float(a[1]));
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(b[0]), __uint_as_float(b[1]));
}
PE_DEV float sum_over_j(float x) {
    const auto a = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(a[0]) + __uint_as_float(a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(b[0]) + __uint_as_float(b[1]);
}

// rows of the cache that exist, and how many of the splits have a block of them (the first always takes part)
PE_DEV int kv_rows(int start, int T, int cap) { return start < 0 ? 0 : min(min(start, cap) + T, cap); }
PE_DEV int kv_used_splits(int start, int T, int cap, int splits) {
    const int blocks = (kv_rows(start, T, cap) + 63) >> 6, per = (blocks + splits - 1) / splits;
    return per == 0 ? 1 : (blocks + per - 1) / per;
}

// WR row tiles x WK shares of the cache's blocks = the waves of a work-group: with one row tile (decode: T * n_q / H <= 16 rows) all waves share its
// blocks and are joined in LDS; with more rows a wave takes 16 of them and the waves read the same blocks through the cache.
template <int D, int WR, int WK>
__global__ void __launch_bounds__(WR * WK * 64, 2) kv_attention_kernel(KvAttention a) {
    constexpr int DT = D / 16, KS = D / 32;
    constexpr bool SHARED = WR > 1;                 // the row tiles' waves read the same blocks: through LDS, two of them in it
    constexpr int BB = 64 * D, SO = WK > 1 ? WR * WK * DT * 1024 : 0, SX = SHARED ? WK * 2 * 2 * BB : 0;
    __shared__ __attribute__((aligned(16))) uint8_t lds[SO > SX ? SO : SX > 0 ? SX : 16];
    __shared__ float lds_m[WR * WK][16], lds_l[WR * WK][16];
    float (*lds_o)[DT][64][4] = (float (*)[DT][64][4])lds;       // [wave][channel tile][lane]
    const int lane = lane_id(), w = wave_id(), wr = w % WR, wk = w / WR, j = lane >> 4, c = lane & 15;
    const int split = (int)blockIdx.x, hk = (int)blockIdx.y;
    const int b = a.row_blocks == 1 ? (int)blockIdx.z : (int)blockIdx.z / a.row_blocks, rb = (int)blockIdx.z - b * a.row_blocks;
    const int G = a.n_q / a.H, rows = a.T * G;
    const int start = min(a.start[b], a.cap);
    const int n = kv_rows(start, a.T, a.cap);
    const int blocks = (n + 63) >> 6;
    const int per = (blocks + a.splits - 1) / a.splits;
    const int lo = split * per, hi = min(lo + per, blocks);
    if (split > 0 && lo >= hi) return;                                       // nothing left for this split: the join leaves it out too
    const size_t plane = ((size_t)b * a.H + hk) * a.cap;
    // lane addresses of block 0
    const uint8_t* kc = a.kc + (plane + 16 * (c >> 2) + (c & 3)) * D + 16 * j;
    const uint8_t* vc = a.vc + plane * D + c * 64 + 16 * j;
    const float *ksc = a.ksc + plane + 16 * j, *vsc = a.vsc + plane + 16 * j;

    struct Block {
        u32x4 k[4][D / 64], v[DT];
        f32x4 ks[4], vs[4];
    };
    auto load = [&](Block& t, int blk) __attribute__((always_inline)) {
        const size_t t0 = (size_t)blk * 64;
        if (!SHARED) {
#pragma unroll
            for (int h = 0; h < 4; ++h)
#pragma unroll
                for (int s = 0; s < D / 64; ++s) t.k[h][s] = *(const u32x4*)(kc + (t0 + 4 * h) * D + 64 * s);
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) t.ks[h] = *(const f32x4*)(ksc + t0 + 4 * h);
        if (!SHARED) {
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) t.v[dt] = *(const u32x4*)(vc + t0 * D + dt * 1024);
        }
#pragma unroll
        for (int h = 0; h < 4; ++h) t.vs[h] = *(const f32x4*)(vsc + t0 + 4 * h);
        __builtin_amdgcn_sched_barrier(0);      // all of a block's loads are under way before anything is waited for
    };
    // SHARED: a block's keys are 64 rows of D bytes, its values D rows of 64; the WR waves of a share copy a WR-th each, 1 KiB an instruction, in the order
    // of the addresses.  Piece p (16 bytes) of row r goes to slot p ^ turn(r): the fragments' reads, 16 rows at a time, then spread over all banks.
    constexpr int KP = D / 16;                      // pieces of a key row
    auto turn_k = [](int r) { return D == 128 ? ((r >> 4) & 3) | ((r >> 1) & 1) << 2 : (r >> 4) & 3; };
    auto turn_v = [](int r) { return (r >> 2) & 3; };
    auto copy = [&](int blk, int buf) __attribute__((always_inline)) {
        uint8_t* kd = lds + (wk * 2 + buf) * 2 * BB;
        const uint8_t *ksrc = a.kc + (plane + (size_t)blk * 64) * D, *vsrc = a.vc + (plane + (size_t)blk * 64) * D;
#pragma unroll
        for (int i = 0; i < D / 16 / WR; ++i) {
            const int q = i * WR + wr, at = q * 64 + lane;
            const int rk = at / KP, rv = at >> 2;
            glds16(ksrc + rk * D + (((at % KP) ^ turn_k(rk)) * 16), kd + q * 1024);
            glds16(vsrc + rv * 64 + (((at & 3) ^ turn_v(rv)) * 16), kd + BB + q * 1024);
        }
    };
    auto fetch = [&](Block& t, int buf) __attribute__((always_inline)) {
        const uint8_t* kd = lds + (wk * 2 + buf) * 2 * BB;
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int s = 0; s < D / 64; ++s) {
                const int r = 16 * (c >> 2) + 4 * h + (c & 3);
                t.k[h][s] = *(const u32x4*)(kd + r * D + (((4 * s + j) ^ turn_k(r)) * 16));
            }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            const int r = dt * 16 + c;
            t.v[dt] = *(const u32x4*)(kd + BB + r * 64 + ((j ^ turn_v(r)) * 16));
        }
    };

    const int row = (rb * WR + wr) * 16 + c;                                 // this lane's column
    const int r_q = min(row, rows - 1);
    const int t_q = (int)(((float)r_q + 0.5f) * __builtin_amdgcn_rcpf((float)G));        // r_q / G: exact below 2^21 rows
    const int h_q = hk * G + r_q - t_q * G;
    bf16x8 qf[KS];
    const bf16* q = a.q + b * a.qs[0] + t_q * a.qs[1] + h_q * a.qs[2] + 16 * j;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *(const bf16x8*)(q + 64 * (s >> 1) + 8 * (s & 1));
    const unsigned long long word = a.tree ? a.tree[(size_t)b * a.T + t_q] : (2ull << t_q) - 1;
    f32x4 o[DT] = {};
    float m = -INFINITY, l = 0.f;                                            // reference of the exponentials (scores times log2 e) and their sum

    auto work = [&](Block& t, int blk) __attribute__((always_inline)) {
        f32x4 s4[4] = {};                         // four independent accumulators in turn: an MFMA's result is not there for the next one
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
            for (int h = 0; h < 4; ++h)
                s4[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes8(t.k[h][s >> 1][2 * (s & 1)], t.k[h][s >> 1][2 * (s & 1) + 1]), qf[s], s4[h], 0, 0, 0);
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) s4[h][i] *= t.ks[h][i] * a.scale_log2;
        const int t0 = blk * 64;
        if (t0 + 64 > start) {                    // the last blocks: rows that are not there, new tokens that a column does not descend from
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int tok = t0 + 16 * j + i, d = tok - start;
                const bool seen = tok < n && (d < 0 || ((word >> (d & 63)) & 1));
                s4[i >> 2][i & 3] = seen ? s4[i >> 2][i & 3] : -INFINITY;
                t.vs[i >> 2][i & 3] = seen ? t.vs[i >> 2][i & 3] : 0.f;      // a scale of NaN included
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) top = fmaxf(top, s4[h][i]);
        top = max_over_j(top);
        // The reference of the exponentials is raised to 8 above the maximum where that has passed it, so most blocks find it high enough: the rescaling costs.
        // Probabilities stay at or below 1 (the largest between 2^-8 and 1 when its block is done), so |O| never passes the sum of the visible |v|.
        if (__any(top > m)) {
            const float m_new = fmaxf(m, top + 8.f);
            const float alpha = m_new == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - m_new);        // 0 from -inf
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[dt][i] *= alpha;
            m = m_new;
        }
        const float m_use = m == -INFINITY ? 0.f : m;
        u32x4 ph[2], pl[2];                       // p * scale_v as its upper 16 bits (a bf16) and the rest, rounded to bf16
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int i = 0; i < 4; i += 2) {
                const float p0 = __builtin_amdgcn_exp2f(s4[h][i] - m_use), p1 = __builtin_amdgcn_exp2f(s4[h][i + 1] - m_use);
                l += p0 + p1;
                const float w0 = p0 * t.vs[h][i], w1 = p1 * t.vs[h][i + 1];
                const uint32_t u0 = __float_as_uint(w0), u1 = __float_as_uint(w1);
                typedef __attribute__((ext_vector_type(2))) __bf16 v2;
                const v2 rest = {(bf16)(w0 - __uint_as_float(u0 & 0xffff0000u)), (bf16)(w1 - __uint_as_float(u1 & 0xffff0000u))};
                ph[h >> 1][2 * (h & 1) + (i >> 1)] = __builtin_amdgcn_perm(u1, u0, 0x07060302u);
                pl[h >> 1][2 * (h & 1) + (i >> 1)] = __builtin_bit_cast(uint32_t, rest);
            }
#pragma unroll
        for (int s = 0; s < 2; ++s) {
            bf16x8 f[DT];
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                f[dt] = codes8(t.v[dt][2 * s], t.v[dt][2 * s + 1]);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[dt], __builtin_bit_cast(bf16x8, ph[s]), o[dt], 0, 0, 0);
            }
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f[dt], __builtin_bit_cast(bf16x8, pl[s]), o[dt], 0, 0, 0);
        }
    };
    if (SHARED) {
        // every wave takes part in every step: the barrier at its top says that this block is there and that the one before is done with.  The next block
        // is asked for after this one's fragments are read (a read of LDS waits for all copies into it) and without a branch (or the wait for the scales
        // would wait for it too); past the end it is the last block again
        const int steps = (hi - lo + WK - 1) / WK;
        if (steps > 0) copy(min(lo + wk, hi - 1), 0);
        for (int i = 0; i < steps; ++i) {
            const int blk = min(lo + i * WK + wk, hi - 1);
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            Block t;
            load(t, blk);
            fetch(t, i & 1);
            __builtin_amdgcn_sched_barrier(0);
            copy(min(blk + WK, hi - 1), (i + 1) & 1);
            __builtin_amdgcn_sched_barrier(0);
            if (lo + i * WK + wk < hi) work(t, blk);
        }
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");          // the last copy is into LDS that is used again below
        __syncthreads();
    } else {
        for (int blk = lo + wk; blk < hi; blk += WK) {
            Block t;
            load(t, blk);
            work(t, blk);
        }
    }

    // ---- join the waves of a row tile; lane (j, c) finishes channels 16 dt + 4 j + i of row c, wave wk those of dt = wk, wk + WK, ...
    l = sum_over_j(l);
    float f[WK];
    if (WK > 1) {
        if (j == 0) { lds_m[w][c] = m; lds_l[w][c] = l; }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) *(f32x4*)lds_o[w][dt][lane] = o[dt];
        __syncthreads();
        m = -INFINITY;
        l = 0.f;
#pragma unroll
        for (int v = 0; v < WK; ++v) m = fmaxf(m, lds_m[v * WR + wr][c]);
#pragma unroll
        for (int v = 0; v < WK; ++v) {
            f[v] = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(lds_m[v * WR + wr][c] - m);
            l += lds_l[v * WR + wr][c] * f[v];
        }
    }
    if (row >= rows) return;
    const float inv = l == 0.f ? 0.f : 1.0f / l;       // nothing visible: zeros
    const size_t orow = ((size_t)b * a.T + t_q) * a.n_q + h_q;
#pragma unroll
    for (int dd = 0; dd < DT / WK; ++dd) {
        const int dt = dd * WK + (WK > 1 ? wk : 0);
        f32x4 y = {};
        if (WK > 1) {
#pragma unroll
            for (int v = 0; v < WK; ++v) {
                const f32x4 x = *(const f32x4*)lds_o[v * WR + wr][dt][lane];
#pragma unroll
                for (int i = 0; i < 4; ++i) y[i] = __builtin_fmaf(x[i], f[v], y[i]);
            }
        } else {
            y = o[dd];
        }
        if (a.splits == 1) {
            bf16x4 z;
#pragma unroll
            for (int i = 0; i < 4; ++i) z[i] = (bf16)(y[i] * inv);
            *(bf16x4*)(a.out + orow * D + dt * 16 + 4 * j) = z;
        } else {
            *(f32x4*)(a.part_o + (orow * a.splits + split) * D + dt * 16 + 4 * j) = y;
        }
    }
    if (a.splits > 1 && wk == 0 && j == 0) {
        a.part_ml[(orow * a.splits + split) * 2] = m;
        a.part_ml[(orow * a.splits + split) * 2 + 1] = l;
    }
}

// joins the splits of one output row (grid: rows of a sequence, sequences): 256 / (D / 4) of them at a time, four channels a lane, and these sums in order
template <int D>
__global__ void __launch_bounds__(256) kv_attention_join_kernel(const float* part_o, const float* part_ml, bf16* out, const int* start, int T, int cap,
                                                                int splits) {
    constexpr int LPR = D / 4, P = 256 / LPR;
    __shared__ f32x4 lds_y[P][LPR];
    __shared__ float lds_s[P];
    const size_t row = (size_t)blockIdx.y * gridDim.x + blockIdx.x;
    const int tid = (int)threadIdx.x, p = tid / LPR, l = tid % LPR;
    const float* ml = part_ml + row * splits * 2;
    const float* po = part_o + row * splits * D + 4 * l;
    float mx = -INFINITY;
    f32x4 y = {};
    float sum = 0.f;
    // the first eight splits of a lane are on their way before their number and the maximum over all of them are known: what no split wrote is not used
    f32x4 x[8];
    f32x2 t[8];
#pragma unroll
    for (int u = 0; u < 8; ++u) {
        const int s = min(p + u * P, splits - 1);
        x[u] = *(const f32x4*)(po + (size_t)s * D);
        t[u] = *(const f32x2*)(ml + 2 * s);
    }
    const float m0 = ml[2 * min(tid & 63, splits - 1)];
    const int used = kv_used_splits(start[blockIdx.y], T, cap, splits);
    if ((tid & 63) < used) mx = fmaxf(mx, m0);
    for (int s = (tid & 63) + 64; s < used; s += 64) mx = fmaxf(mx, ml[2 * s]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    auto add = [&](const f32x4& v, const f32x2& w) __attribute__((always_inline)) {
        const float f = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(w[0] - mx);
        sum = __builtin_fmaf(w[1], f, sum);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __builtin_fmaf(v[i], f, y[i]);
    };
#pragma unroll
    for (int u = 0; u < 8; ++u)
        if (p + u * P < used) add(x[u], t[u]);
    for (int s = p + 8 * P; s < used; s += P) add(*(const f32x4*)(po + (size_t)s * D), *(const f32x2*)(ml + 2 * s));
    // a split that saw nothing has m = -inf and weight 0 -- or, where every score is NaN, sums of NaN: they stay
    lds_y[p][l] = y;
    if (l == 0) lds_s[p] = sum;
    __syncthreads();
    if (p != 0) return;
    for (int v = 1; v < P; ++v) {
        sum += lds_s[v];
        y += lds_y[v][l];
    }
    const float inv = sum == 0.f ? 0.f : 1.0f / sum;
    bf16x4 z;
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = (bf16)(y[i] * inv);
    *(bf16x4*)(out + row * D + 4 * l) = z;
}

// How the work is cut: row tiles of a work-group, row blocks, splits of the cache's axis.  One work-group per CU is 256 of them, no more (21 rows a head,
// 12 work-groups, 15000 cache rows: 21 splits 25.6 us, 22 31.4); more splits than that only add partials to join (8 sequences' heads, 30000 rows: 32
// splits 19.9 us, 64 21.4, 117 25.4) -- except where the sequences of a batch differ in length and the longest would be left over: 24 x 8 heads,
// 0 ... 40000 rows: 2 splits 153 us, 3 115, 6 98, 11 96, and where several row tiles walk far: their steps are chains of dependent instructions, and a
// second work-group on the CU fills the gaps (33 tokens, 2 x 4 heads, 12000 rows: 8 splits 42.3 us, 16 28.6; 64 tokens, 4 heads, 15000 rows: 9 46.1, 18
// 42.6; not below four blocks a wave: 3 trees of 21, 2777 rows: 8 20.7, 14 21.9).  A split is never shorter
// than one block of 64 rows for each wave that shares the cache, and two where none do (21 rows a head, cap 1536: 128 rows 9.2 us, 256 10.8).
struct KvPlan { int wr, rb, splits; };
static KvPlan kv_plan(int B, int H, int T, int n_q, int cap) {
    KvPlan p;
    const int rows = T * (n_q / H);
    p.wr = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    p.rb = (rows + 16 * p.wr - 1) / (16 * p.wr);
    const long long wgs = (long long)B * H * p.rb, one = 256 / wgs, two = 512 / wgs, even = (2048 + wgs - 1) / wgs;
    long long s = one > 8 ? one : even < 8 ? even : 8;
    if (p.wr > 1 && two > s && cap / 64 >= 4 * (4 / p.wr) * two) s = two;
    const int most = (cap + (p.wr == 1 ? 255 : 127)) / (p.wr == 1 ? 256 : 128);
    p.splits = (int)(s < most ? s : most);
    return p;
}
size_t kv_attention_workspace_bytes(int B, int H, int T, int n_q, int D, int cap) {
    if (B < 1 || H < 1 || T < 1 || n_q < H || D < 1 || cap < 64) return 0;
    const int s = kv_plan(B, H, T, n_q, cap).splits;
    return s == 1 ? 0 : (size_t)B * T * n_q * s * (D + 2) * sizeof(float);
}

int launch_kv_attention(const KvAttention& in, void* workspace, size_t workspace_bytes, hipStream_t stream) {
    KvAttention a = in;
    PE_REQUIRE(a.kc && a.vc && a.ksc && a.vsc && a.q && a.out && a.start, "kv_attention: null pointer");
    PE_REQUIRE(a.D == 64 || a.D == 128, "kv_attention: heads of %d (64 or 128)", a.D);
    PE_REQUIRE(a.B >= 1 && a.B <= 65535 && a.H >= 1 && a.n_q >= a.H && a.n_q % a.H == 0 && a.cap >= 64 && a.cap % 64 == 0 && a.cap <= (1 << 30),
               "kv_attention: bad shape (B=%d, %d query and %d kv heads, cap=%d)", a.B, a.n_q, a.H, a.cap);
    PE_REQUIRE(a.T >= 1 && a.T <= 64, "kv_attention: T=%d new tokens (1 ... 64)", a.T);
    const uintptr_t mis = (uintptr_t)a.kc | (uintptr_t)a.vc | (uintptr_t)a.ksc | (uintptr_t)a.vsc | (uintptr_t)a.q | (uintptr_t)a.out | (uintptr_t)workspace;
    PE_REQUIRE((mis & 15) == 0 && ((uintptr_t)a.tree & 7) == 0, "kv_attention: pointers must be 16-byte aligned");
    PE_REQUIRE(a.qs[0] % 8 == 0 && a.qs[1] % 8 == 0 && a.qs[2] % 8 == 0, "kv_attention: strides must be multiples of 8 elements");
    const KvPlan plan = kv_plan(a.B, a.H, a.T, a.n_q, a.cap);
    PE_REQUIRE(a.H <= 65535 && (long long)a.B * plan.rb <= 65535 && a.T * (a.n_q / a.H) < (1 << 21), "kv_attention: too many heads or sequences");
    a.splits = plan.splits;
    a.row_blocks = plan.rb;
    const size_t need = kv_attention_workspace_bytes(a.B, a.H, a.T, a.n_q, a.D, a.cap);
    PE_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "kv_attention: workspace of %zu bytes, 16-byte aligned, needed", need);
    const size_t out_rows = (size_t)a.B * a.T * a.n_q;
    PE_REQUIRE(out_rows < (1ull << 31), "kv_attention: too many rows");
    a.part_o = (float*)workspace;
    a.part_ml = a.part_o ? a.part_o + out_rows * a.splits * a.D : nullptr;
    const dim3 grid(a.splits, a.H, a.B * plan.rb);
#define PE_KV_ATT(D, WR, WK) hipLaunchKernelGGL((kv_attention_kernel<D, WR, WK>), grid, dim3(WR * WK * 64), 0, stream, a)
    if (a.D == 64) { if (plan.wr == 1) PE_KV_ATT(64, 1, 4); else if (plan.wr == 2) PE_KV_ATT(64, 2, 2); else PE_KV_ATT(64, 4, 1); }
    else { if (plan.wr == 1) PE_KV_ATT(128, 1, 4); else if (plan.wr == 2) PE_KV_ATT(128, 2, 2); else PE_KV_ATT(128, 4, 1); }
#undef PE_KV_ATT
    if (const int rc = check_launch("kv_attention_kernel")) return rc;
    if (a.splits > 1) {
        const dim3 rows(a.T * a.n_q, a.B);
        if (a.D == 64) hipLaunchKernelGGL(kv_attention_join_kernel<64>, rows, dim3(256), 0, stream, a.part_o, a.part_ml, a.out, a.start, a.T, a.cap, a.splits);
        else hipLaunchKernelGGL(kv_attention_join_kernel<128>, rows, dim3(256), 0, stream, a.part_o, a.part_ml, a.out, a.start, a.T, a.cap, a.splits);
        return check_launch("kv_attention_join_kernel");
    }
    return PE_OK;
}

}  // namespace pe
