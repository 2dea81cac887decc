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
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        clo[h] = pack4_e4m3(lo[4 * h] / scale, lo[4 * h + 1] / scale, lo[4 * h + 2] / scale, lo[4 * h + 3] / scale);
        chi[h] = pack4_e4m3(hi[4 * h] / scale, hi[4 * h + 1] / scale, hi[4 * h + 2] / scale, hi[4 * h + 3] / scale);
    }
    return scale;
}

// first row that tokens of sequence b go to, and how many of the T tokens are written; start outside the cache: none
PE_DEV int append_count(int start, int T, int cap) { return start < 0 || start >= cap ? 0 : min(T, cap - start); }

template <int D, typename TAB>
__global__ void __launch_bounds__(256) kv_append_kernel(KvAppend a) {
    constexpr int LPR = D / 16, ROWS = 256 / LPR;
    __shared__ __attribute__((aligned(16))) uint8_t turn[D][64 + 4];     // a block of values, transposed; rows of 17 words: no bank conflicts
    const int lane = lane_id(), tid = (int)threadIdx.x;
    const int l = tid % LPR, d0 = 8 * l;
    if ((int)blockIdx.x < a.qk_blocks) {
        // ---- queries and keys: rows (b, t, head), the query heads first
        const int heads = a.n_q + a.H;
        const long long row = (long long)blockIdx.x * ROWS + tid / LPR;
        const bool in = row < (long long)a.B * a.T * heads;       // no early return: the row's lanes shuffle
        const long long rr = in ? row : 0;
        const int h = (int)(rr % heads);
        const long long bt = rr / heads;
        const int t = (int)(bt % a.T), b = (int)(bt / a.T);
        const int start = a.start[b];
        const bool is_q = h < a.n_q;
        const bf16* src = is_q ? a.q + b * a.qs[0] + t * a.qs[1] + h * a.qs[2] : a.k + b * a.ks[0] + t * a.ks[1] + (h - a.n_q) * a.ks[2];
        float lo[8], hi[8];
        load_half(src + d0, lo);
        load_half(src + D / 2 + d0, hi);
        const bool there = in && t < append_count(start, a.T, a.cap);
        if (a.cos) {
            const int pos = !there ? 0 : a.positions ? a.positions[bt] : start + t;
            const bool known = pos >= 0 && pos < a.table_rows;     // no such row in the tables: the row becomes NaN
            const size_t at = (size_t)(known ? pos : 0) * D + d0;
            const TAB *cs = (const TAB*)a.cos + at, *sn = (const TAB*)a.sin + at;
            float cl[8], ch[8], sl[8], sh[8];
            load_half(cs, cl); load_half(cs + D / 2, ch); load_half(sn, sl); load_half(sn + D / 2, sh);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const float x = lo[e], y = hi[e];
                lo[e] = known ? x * cl[e] + -y * sl[e] : __uint_as_float(0x7fc00000u);
                hi[e] = known ? y * ch[e] + x * sh[e] : lo[e];
            }
        }
        if (is_q) {
            if (!in) return;                                      // whole rows leave together: nothing below shuffles for them
            bf16x8 ol, oh;
#pragma unroll
            for (int e = 0; e < 8; ++e) { ol[e] = there ? (bf16)lo[e] : (bf16)0.f; oh[e] = there ? (bf16)hi[e] : (bf16)0.f; }
            bf16* dst = a.q_out + (bt * a.n_q + h) * D + d0;
            *(bf16x8*)dst = ol;
            *(bf16x8*)(dst + D / 2) = oh;
            return;
        }
        u32x2 clo, chi;
        const float scale = quantise_row<LPR>(lo, hi, clo, chi);
        if (!there) return;
        const size_t dst = ((size_t)b * a.H + (h - a.n_q)) * a.cap + start + t;
        *(u32x2*)(a.kc + dst * D + d0) = clo;
        *(u32x2*)(a.kc + dst * D + D / 2 + d0) = chi;
        if (l == 0) a.ksc[dst] = scale;
        return;
    }
    // ---- values: one work-group per (b, head, block of 64 cache rows)
    const int id = (int)blockIdx.x - a.qk_blocks;
    const int blk = id % a.v_blocks, h = id / a.v_blocks % a.H, b = id / a.v_blocks / a.H;
    const int start = a.start[b], count = append_count(start, a.T, a.cap);
    const int first = (start & ~63) + blk * 64;                 // cache row of the block's first token
    if (count == 0 || first >= start + count) return;
    const bool whole = first >= start && first + 64 <= start + count;
    const size_t plane = ((size_t)b * a.H + h) * a.cap;
    uint8_t* vdst = a.vc + (plane + first) * D;
    for (int r0 = 0; r0 < 64; r0 += ROWS) {
        const int r = r0 + tid / LPR, t = first + r - start;
        const bool mine = r < 64 && t >= 0 && t < count;
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
    const int rows = 256 / (a.D / 16);
    const long long qk = ((long long)a.B * a.T * (a.n_q + a.H) + rows - 1) / rows;
    a.v_blocks = (int)(((long long)a.T + 126) / 64);
    if (a.v_blocks > a.cap / 64) a.v_blocks = a.cap / 64;
    const long long grid = qk + (long long)a.B * a.H * a.v_blocks;
    PE_REQUIRE(grid < (1ll << 31), "kv_append: too many rows");
    a.qk_blocks = (int)qk;
#define PE_KV_APPEND(D, TAB) hipLaunchKernelGGL((kv_append_kernel<D, TAB>), dim3((unsigned)grid), dim3(256), 0, stream, a)
    if (a.D == 64) { if (a.table_f32) PE_KV_APPEND(64, float); else PE_KV_APPEND(64, bf16); }
    else { if (a.table_f32) PE_KV_APPEND(128, float); else PE_KV_APPEND(128, bf16); }
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
// Scores, maximum, sums and O are fp32.  A wave walks every fourth block of its work-group's range with a running maximum of its own; waves and
// work-groups (the cache's axis is split over `splits` of them) are joined in a fixed order.
// ------------------------------------------------------------------------------------------------
PE_DEV bf16x8 codes8(uint32_t a, uint32_t b) {
    typedef __attribute__((ext_vector_type(2))) __bf16 v2;
    const v2 x0 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false), x1 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true);
    const v2 x2 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false), x3 = __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true);
    return bf16x8{x0[0], x0[1], x1[0], x1[1], x2[0], x2[1], x3[0], x3[1]};
}

// WR row tiles x WK shares of the cache's blocks = the waves of a work-group: with one row tile (decode: T * n_q / H <= 16 rows) all waves share its
// blocks and are joined in LDS; with more rows a wave takes 16 of them and the waves read the same blocks through the cache.
template <int D, int WR, int WK>
__global__ void __launch_bounds__(WR * WK * 64) kv_attention_kernel(KvAttention a) {
    constexpr int DT = D / 16, KS = D / 32;
    __shared__ float lds_o[WK > 1 ? WR * WK : 1][WK > 1 ? DT : 1][64][4];
    __shared__ float lds_m[WR * WK][16], lds_l[WR * WK][16];
    const int lane = lane_id(), w = wave_id(), wr = w % WR, wk = w / WR, j = lane >> 4, c = lane & 15;
    const int split = (int)blockIdx.x, b = (int)blockIdx.z;
    const int hk = (int)blockIdx.y % a.H, rb = (int)blockIdx.y / a.H;
    const int G = a.n_q / a.H, rows = a.T * G;
    const int start = min(a.start[b], a.cap);
    const int n = start < 0 ? 0 : min(start + a.T, a.cap);                   // rows of the cache that exist
    const int blocks = (n + 63) >> 6;
    const int per = (blocks + a.splits - 1) / a.splits;
    const int lo = split * per, hi = min(lo + per, blocks);
    const size_t plane = ((size_t)b * a.H + hk) * a.cap;
    const uint8_t* kc = a.kc + plane * D;
    const uint8_t* vc = a.vc + plane * D;
    const float *ksc = a.ksc + plane, *vsc = a.vsc + plane;

    const int row = (rb * WR + wr) * 16 + c;                                 // this lane's column
    const int t_q = min(row, rows - 1) / G, h_q = hk * G + min(row, rows - 1) % G;
    bf16x8 qf[KS];
    const bf16* q = a.q + b * a.qs[0] + t_q * a.qs[1] + h_q * a.qs[2] + 16 * j;
#pragma unroll
    for (int s = 0; s < KS; ++s) qf[s] = *(const bf16x8*)(q + 64 * (s >> 1) + 8 * (s & 1));
    const unsigned long long word = a.tree ? a.tree[(size_t)b * a.T + t_q] : (2ull << t_q) - 1;
    f32x4 o[DT] = {};
    float m = -INFINITY, l = 0.f;

    for (int blk = lo + wk; blk < hi; blk += WK) {
        const int t0 = blk * 64;
        u32x4 kf[4][D / 64], vf[DT];
        f32x4 ks[4], vs[4];
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int s = 0; s < D / 64; ++s)
                kf[h][s] = *(const u32x4*)(kc + (size_t)(t0 + 16 * (c >> 2) + 4 * h + (c & 3)) * D + 64 * s + 16 * j);
#pragma unroll
        for (int h = 0; h < 4; ++h) ks[h] = *(const f32x4*)(ksc + t0 + 16 * j + 4 * h);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) vf[dt] = *(const u32x4*)(vc + (size_t)t0 * D + (size_t)(dt * 16 + c) * 64 + 16 * j);
#pragma unroll
        for (int h = 0; h < 4; ++h) vs[h] = *(const f32x4*)(vsc + t0 + 16 * j + 4 * h);
        __builtin_amdgcn_sched_barrier(0);      // all of the block's loads are under way before the first is waited for
        f32x4 s4[4] = {};
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int s = 0; s < KS; ++s)
                s4[h] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(codes8(kf[h][s >> 1][2 * (s & 1)], kf[h][s >> 1][2 * (s & 1) + 1]), qf[s], s4[h], 0, 0, 0);
        uint32_t seen = 0xffffu;                  // bit 4 h + i: this lane's token is visible to its column
        if (t0 + 64 > start) {
            seen = 0;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int t = t0 + 16 * j + i, d = t - start;
                const bool v = t < n && (d < 0 || ((word >> (d & 63)) & 1));
                seen |= (uint32_t)v << i;
            }
        }
        float top = -INFINITY;
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float s = s4[h][i] * (ks[h][i] * a.scale_log2);
                s4[h][i] = (seen >> (4 * h + i)) & 1 ? s : -INFINITY;
                top = fmaxf(top, s4[h][i]);
            }
        top = fmaxf(top, __shfl_xor(top, 16, 64));
        top = fmaxf(top, __shfl_xor(top, 32, 64));
        const float m_new = fmaxf(m, top);
        const float m_use = m_new == -INFINITY ? 0.f : m_new;
        if (__any(m_new > m)) {
            const float alpha = __builtin_amdgcn_exp2f(m - m_use);       // 0 from -inf
            l *= alpha;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt)
#pragma unroll
                for (int i = 0; i < 4; ++i) o[dt][i] *= alpha;
            m = m_new;
        }
        bf16x8 ph[2], pl[2];
#pragma unroll
        for (int h = 0; h < 4; ++h)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float p = __builtin_amdgcn_exp2f(s4[h][i] - m_use);
                l += p;
                const float pv = (seen >> (4 * h + i)) & 1 ? p * vs[h][i] : 0.f;
                const bf16 top8 = (bf16)pv;
                ph[h >> 1][4 * (h & 1) + i] = top8;
                pl[h >> 1][4 * (h & 1) + i] = (bf16)(pv - (float)top8);
            }
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int s = 0; s < 2; ++s) {
                const bf16x8 f = codes8(vf[dt][2 * s], vf[dt][2 * s + 1]);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, ph[s], o[dt], 0, 0, 0);
                o[dt] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(f, pl[s], o[dt], 0, 0, 0);
            }
    }

    // ---- join the waves of a row tile; lane (j, c) finishes channels 16 dt + 4 j + i of row c, wave wk those of dt = wk, wk + WK, ...
    l += __shfl_xor(l, 16, 64);
    l += __shfl_xor(l, 32, 64);
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
            for (int i = 0; i < 4; ++i) z[i] = l == 0.f ? (bf16)0.f : (bf16)(y[i] / l);
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

// joins the splits of one output row: 256 / (D / 4) of them at a time, four channels a lane, and these sums in order
template <int D>
__global__ void __launch_bounds__(256) kv_attention_join_kernel(const float* part_o, const float* part_ml, bf16* out, int splits) {
    constexpr int LPR = D / 4, P = 256 / LPR;
    __shared__ f32x4 lds_y[P][LPR];
    __shared__ float lds_s[P];
    const size_t row = blockIdx.x;
    const int tid = (int)threadIdx.x, p = tid / LPR, l = tid % LPR;
    const float* ml = part_ml + row * splits * 2;
    float mx = -INFINITY;
    for (int s = tid & 63; s < splits; s += 64) mx = fmaxf(mx, ml[2 * s]);
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor(mx, o, 64));
    f32x4 y = {};
    float sum = 0.f;
#pragma unroll 4
    for (int s = p; s < splits; s += P) {
        const float f = mx == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(ml[2 * s] - mx);
        const f32x4 x = *(const f32x4*)(part_o + (row * splits + s) * D + 4 * l);
        sum = __builtin_fmaf(ml[2 * s + 1], f, sum);
#pragma unroll
        for (int i = 0; i < 4; ++i) y[i] = __builtin_fmaf(x[i], f, y[i]);
    }
    // a split that saw nothing has m = -inf and weight 0 -- or, where every score is NaN, sums of NaN: they stay
    lds_y[p][l] = y;
    if (l == 0) lds_s[p] = sum;
    __syncthreads();
    if (p != 0) return;
    for (int v = 1; v < P; ++v) {
        sum += lds_s[v];
        y += lds_y[v][l];
    }
    bf16x4 z;
#pragma unroll
    for (int i = 0; i < 4; ++i) z[i] = sum == 0.f ? (bf16)0.f : (bf16)(y[i] / sum);
    *(bf16x4*)(out + row * D + 4 * l) = z;
}

// How the work is cut: row tiles and shares of the cache a work-group takes, row blocks, splits of the cache's axis.
struct KvPlan { int wr, rb, splits; };
static KvPlan kv_plan(int B, int H, int T, int n_q, int cap) {
    KvPlan p;
    const int rows = T * (n_q / H);
    p.wr = rows <= 16 ? 1 : rows <= 32 ? 2 : 4;
    p.rb = (rows + 16 * p.wr - 1) / (16 * p.wr);
    const long long wgs = (long long)B * H * p.rb;
    const long long s = wgs >= 512 ? 1 : (512 + wgs - 1) / wgs;
    const int most = (cap + 255) / 256;
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
    PE_REQUIRE((long long)a.H * plan.rb <= 65535, "kv_attention: too many heads");
    a.splits = plan.splits;
    const size_t need = kv_attention_workspace_bytes(a.B, a.H, a.T, a.n_q, a.D, a.cap);
    PE_REQUIRE(need == 0 || (workspace && workspace_bytes >= need), "kv_attention: workspace of %zu bytes, 16-byte aligned, needed", need);
    const size_t out_rows = (size_t)a.B * a.T * a.n_q;
    a.part_o = (float*)workspace;
    a.part_ml = a.part_o ? a.part_o + out_rows * a.splits * a.D : nullptr;
    const dim3 grid(a.splits, a.H * plan.rb, a.B);
#define PE_KV_ATT(D, WR, WK) hipLaunchKernelGGL((kv_attention_kernel<D, WR, WK>), grid, dim3(WR * WK * 64), 0, stream, a)
    if (a.D == 64) { if (plan.wr == 1) PE_KV_ATT(64, 1, 4); else if (plan.wr == 2) PE_KV_ATT(64, 2, 2); else PE_KV_ATT(64, 4, 1); }
    else { if (plan.wr == 1) PE_KV_ATT(128, 1, 4); else if (plan.wr == 2) PE_KV_ATT(128, 2, 2); else PE_KV_ATT(128, 4, 1); }
#undef PE_KV_ATT
    if (const int rc = check_launch("kv_attention_kernel")) return rc;
    if (a.splits > 1) {
        if (a.D == 64) hipLaunchKernelGGL(kv_attention_join_kernel<64>, dim3((unsigned)out_rows), dim3(256), 0, stream, a.part_o, a.part_ml, a.out, a.splits);
        else hipLaunchKernelGGL(kv_attention_join_kernel<128>, dim3((unsigned)out_rows), dim3(256), 0, stream, a.part_o, a.part_ml, a.out, a.splits);
        return check_launch("kv_attention_join_kernel");
    }
    return PE_OK;
}

}  // namespace pe
