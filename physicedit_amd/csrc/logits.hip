// Next-token scores: penalties for repeated tokens, biases and masks (pe_process_logits), and the greedy choice among the processed
// scores without writing them (pe_select_token).
//
// In fp32, in this order, for token v of a row (counts[v]: bit 15 = the prompt holds it, bits 0 .. 14 = how often it was generated):
//   seen (counts != 0):  l = l > 0 ? l / repetition : l * repetition
//   l -= frequency * generated;  l -= presence * (generated > 0);  l += bias[v];  bit v of the mask clear: l = -inf, whatever l was
// One pass over the row, bound by its bytes; 8 tokens per lane and step.  Rows of an odd vocabulary start at odd addresses: the loads say so
// (aligned to one element), which the hardware takes at full width.
#include "common.h"
#include "kernels.h"

namespace pe {

constexpr int LOGITS_PER_BLOCK = 256 * 8;

template <typename V, typename E>
PE_DEV V load_at(const E* p) {            // a vector load that needs no more than one element's alignment
    V v;
    __builtin_memcpy(&v, p, sizeof(V));
    return v;
}
typedef __attribute__((ext_vector_type(8))) short s16x8;
typedef __attribute__((ext_vector_type(8))) float f32x8;

template <typename T>
PE_DEV f32x8 load_logits(const T* p);
template <>
PE_DEV f32x8 load_logits<bf16>(const bf16* p) {
    const bf16x8 t = load_at<bf16x8>(p);
    f32x8 x;
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = (float)t[e];
    return x;
}
template <>
PE_DEV f32x8 load_logits<float>(const float* p) { return load_at<f32x8>(p); }

PE_DEV float process_one(float l, int count, float rep, float presence, float frequency, float bias, bool allowed) {
    const float made = (float)(count & 0x7fff);
    if (count) l = l > 0.f ? l / rep : l * rep;
    l = l - frequency * made;
    l = l - (made > 0.f ? presence : 0.f);
    l = l + bias;
    return allowed ? l : -INFINITY;
}

// the row's eight scores at v .. v + 7 (v a multiple of 8), those at and behind V left out (-inf)
template <typename T>
PE_DEV f32x8 process8(const LogitsArgs& a, size_t row, int v, float rep, float presence, float frequency) {
    const T* lg = (const T*)a.logits + row * a.ld + v;
    const short* ct = a.counts ? a.counts + row * a.ldc + v : nullptr;
    const float* bs = a.bias ? a.bias + row * a.ldb + v : nullptr;
    const uint32_t word = a.allowed ? a.allowed[row * a.ldm + (v >> 5)] : 0xffffffffu;       // used last: a shift here would wait for it alone
    f32x8 x, b = {};
    s16x8 n = {};
    if (v + 8 <= a.V) {
        x = load_logits<T>(lg);
        if (ct) n = load_at<s16x8>(ct);
        if (bs) b = load_at<f32x8>(bs);
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const bool in = v + e < a.V;
            x[e] = in ? (float)lg[e] : -INFINITY;
            n[e] = in && ct ? ct[e] : (short)0;
            b[e] = in && bs ? bs[e] : 0.f;
        }
    }
    const uint32_t bits = word >> (v & 31);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const bool ok = ((bits >> e) & 1) && v + e < a.V;
        if (a.counts) x[e] = process_one(x[e], (int)(uint16_t)n[e], rep, presence, frequency, b[e], ok);
        else { const float l = a.bias ? x[e] + b[e] : x[e]; x[e] = ok ? l : -INFINITY; }
    }
    return x;
}

PE_DEV void row_penalties(const LogitsArgs& a, size_t row, float& rep, float& presence, float& frequency) {
    // vector loads of a uniform address: a scalar load's wait is a wait for all of them, here it joins the queue of the scores
    int zero;
    asm("v_mov_b32 %0, 0" : "=v"(zero));
    const float* p = a.penalties + row * a.ldp + zero;
    rep = a.penalties ? p[0] : 1.f;
    presence = a.penalties ? p[1] : 0.f;
    frequency = a.penalties ? p[2] : 0.f;
}

template <typename T>
__global__ void __launch_bounds__(256) process_logits_kernel(LogitsArgs a) {
    const size_t row = blockIdx.y;
    float rep, presence, frequency;
    row_penalties(a, row, rep, presence, frequency);
    const int v = (int)(blockIdx.x * 256 + threadIdx.x) * 8;
    if (v >= a.V) return;
    const f32x8 x = process8<T>(a, row, v, rep, presence, frequency);
    float* out = a.out + row * (size_t)a.V + v;
    if (v + 8 <= a.V) {
        __builtin_memcpy(out, &x, sizeof(x));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (v + e < a.V) out[e] = x[e];
    }
}

// first maximum: the larger score, and among equals the lower index.  NaN is never chosen; idx = NONE where nothing is above -inf.
constexpr int NONE = 0x7fffffff;
PE_DEV void better(float& best, int& idx, float ov, int oi) {
    if (ov > best || (ov == best && oi < idx)) { best = ov; idx = oi; }
}
PE_DEV void wave_best(float& best, int& idx) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) better(best, idx, __shfl_xor(best, o, 64), __shfl_xor(idx, o, 64));
}

// bits 0 .. 14 of a count go up and stop at 32767; prompt: bit 15 is set instead
PE_DEV uint32_t counted(uint32_t n, int times, bool prompt) { return prompt ? n | 0x8000u : (n & 0x8000u) | (uint32_t)min((int)(n & 0x7fffu) + min(times, 0x7fff), 0x7fff); }

// a count that no other lane touches
PE_DEV void count_alone(short* p, int times, bool prompt) { *p = (short)counted((uint16_t)*p, times, prompt); }

// One of the two counts of a 32-bit word, both of which belong to the row.  Only its own half changes, so any order of concurrent additions gives the
// same counts.
PE_DEV void count_shared(short* p, bool prompt) {
    uint32_t* word = (uint32_t*)((uintptr_t)p & ~(uintptr_t)3);
    const int shift = ((uintptr_t)p & 2) ? 16 : 0;
    uint32_t old = *word, seen;
    do {
        seen = old;
        old = atomicCAS(word, seen, (seen & ~(0xffffu << shift)) | (counted((seen >> shift) & 0xffffu, 1, prompt) << shift));
    } while (old != seen);
}

// what becomes of a row's choice
PE_DEV void take_token(int idx, size_t row, int* token, short* counts, long long ldc, int* out_ids, int* step, int max_steps) {
    const int t = idx == NONE ? -1 : idx;
    token[row] = t;
    if (counts && t >= 0) count_alone(counts + row * ldc + t, 1, false);       // this lane writes the row's only count
    if (step) {                                   // one row only: the decode step's counter
        const int st = *step;
        if (st >= 0 && st < max_steps) out_ids[st] = t;
        *step = st + 1;
    }
}

// A row's best in one work-group (up to 8192 tokens: one launch instead of two) or a part's.  THREADS lanes of 8 tokens.
template <typename T, int THREADS, bool WHOLE>
__global__ void __launch_bounds__(THREADS) select_part_kernel(LogitsArgs a, float* part_v, int* part_i, int* token, short* counts, int* out_ids, int* step,
                                                              int max_steps) {
    __shared__ float bv[THREADS / 64];
    __shared__ int bi[THREADS / 64];
    const size_t row = blockIdx.y;
    float rep, presence, frequency;
    row_penalties(a, row, rep, presence, frequency);
    float best = -INFINITY;
    int idx = NONE;
#pragma unroll 2
    for (int v = (int)(blockIdx.x * THREADS + threadIdx.x) * 8; v < a.V; v += THREADS * 8) {
        const f32x8 x = process8<T>(a, row, v, rep, presence, frequency);
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (x[e] > best) { best = x[e]; idx = v + e; }        // ascending: the first maximum stays
        if (!WHOLE) break;
    }
    wave_best(best, idx);
    if (lane_id() == 0) { bv[wave_id()] = best; bi[wave_id()] = idx; }
    __syncthreads();
    if (threadIdx.x == 0) {
        for (int w = 1; w < THREADS / 64; ++w) better(best, idx, bv[w], bi[w]);
        if (WHOLE) {
            take_token(idx, row, token, counts, a.ldc, out_ids, step, max_steps);
        } else {
            part_v[row * gridDim.x + blockIdx.x] = best;
            part_i[row * gridDim.x + blockIdx.x] = idx;
        }
    }
}

__global__ void __launch_bounds__(64) select_join_kernel(const float* part_v, const int* part_i, int parts, int* token, short* counts,
                                                         long long ldc, int* out_ids, int* step, int max_steps) {
    const size_t row = blockIdx.x;
    float best = -INFINITY;
    int idx = NONE;
    for (int i = lane_id(); i < parts; i += 64) better(best, idx, part_v[row * parts + i], part_i[row * parts + i]);
    wave_best(best, idx);
    if (lane_id() == 0) take_token(idx, row, token, counts, ldc, out_ids, step, max_steps);
}

// A row whose counts begin or end in the middle of a 32-bit word shares that word with the row beside it or with memory that is not the caller's: the
// row's first work-group counts how often that one token comes and writes its 16 bits alone (one row of 151937, 600 tokens 3.7 us, 15000 7.6; of 151936 3.3 and 6.7).
constexpr int COUNT_THREADS = 1024;
__global__ void __launch_bounds__(COUNT_THREADS) token_counts_add_kernel(short* counts, long long ldc, int V, const int* tokens, int n, int prompt) {
    __shared__ int times[2];
    const size_t row = blockIdx.y;
    const int tid = (int)threadIdx.x;
    short* c = counts + row * ldc;
    tokens += row * n;
    const bool head = ((uintptr_t)c & 2) != 0, tail = ((uintptr_t)(c + V) & 2) != 0;       // tokens 0 and V - 1; for V = 1 at most one of them
    const long long i = (long long)blockIdx.x * COUNT_THREADS + tid;
    if (i < n) {
        const int v = tokens[i];
        if (v >= 0 && v < V && !(head && v == 0) && !(tail && v == V - 1)) count_shared(c + v, prompt != 0);
    }
    if (blockIdx.x != 0 || !(head || tail)) return;                                        // the whole work-group leaves
    if (tid < 2) times[tid] = 0;
    __syncthreads();
    int first = 0, last = 0;
#pragma unroll 4
    for (long long k = tid; k < n; k += COUNT_THREADS) {
        const int v = tokens[k];
        first += v == 0;
        last += v == V - 1;
    }
    if (first) atomicAdd(&times[0], first);
    if (last) atomicAdd(&times[1], last);
    __syncthreads();
    if (tid != 0) return;
    if (head && times[0]) count_alone(c, times[0], prompt != 0);
    if (tail && times[1]) count_alone(c + V - 1, times[1], prompt != 0);
}

static int check_logits(const LogitsArgs& a, const char* who) {
    PE_REQUIRE(a.logits, "%s: null logits", who);
    PE_REQUIRE(a.rows >= 1 && a.rows <= 65535 && a.V >= 1 && a.V <= (1 << 30), "%s: bad shape (%d rows of %d)", who, a.rows, a.V);
    PE_REQUIRE(a.ld >= a.V, "%s: row stride %lld below the vocabulary %d", who, a.ld, a.V);
    PE_REQUIRE(((uintptr_t)a.logits & (a.f32 ? 3 : 1)) == 0 && ((uintptr_t)a.counts & 1) == 0 && ((uintptr_t)a.bias & 3) == 0 && ((uintptr_t)a.allowed & 3) == 0,
               "%s: unaligned pointer", who);
    PE_REQUIRE(!a.counts || a.ldc >= a.V, "%s: row stride of counts below the vocabulary", who);
    PE_REQUIRE(!a.penalties || a.counts, "%s: penalties need the counts", who);
    PE_REQUIRE(a.ldb == 0 || a.ldb >= a.V, "%s: row stride of the bias below the vocabulary", who);
    PE_REQUIRE(a.ldm == 0 || a.ldm >= (a.V + 31) / 32, "%s: row stride of the mask below its words", who);
    return PE_OK;
}

int launch_process_logits(const LogitsArgs& a, hipStream_t stream) {
    if (const int rc = check_logits(a, "process_logits")) return rc;
    PE_REQUIRE(a.out && ((uintptr_t)a.out & 3) == 0, "process_logits: null or unaligned output");
    const dim3 grid((a.V + LOGITS_PER_BLOCK - 1) / LOGITS_PER_BLOCK, a.rows);
    if (a.f32) hipLaunchKernelGGL(process_logits_kernel<float>, grid, dim3(256), 0, stream, a);
    else hipLaunchKernelGGL(process_logits_kernel<bf16>, grid, dim3(256), 0, stream, a);
    return check_launch("process_logits_kernel");
}

// one work-group reads a short row in the time that a second launch costs (1 row, bf16 with counts: 2000 tokens 3.6 us against 5.4, 8000 5.1 and 5.8,
// 16000 7.1 and 5.9)
constexpr int SELECT_WHOLE = 8192;
size_t select_token_workspace_bytes(int rows, int V) {
    return rows < 1 || V <= SELECT_WHOLE ? 0 : (size_t)rows * ((V + LOGITS_PER_BLOCK - 1) / LOGITS_PER_BLOCK) * 8;
}

int launch_select_token(const LogitsArgs& a, int* token, short* count_into, int* out_ids, int* step, int max_steps, void* workspace,
                        size_t workspace_bytes, hipStream_t stream) {
    if (const int rc = check_logits(a, "select_token")) return rc;
    PE_REQUIRE(token, "select_token: null token");
    PE_REQUIRE(!step || (out_ids && max_steps >= 1 && a.rows == 1), "select_token: a step counter belongs to one row and its list of tokens");
    const size_t need = select_token_workspace_bytes(a.rows, a.V);
    PE_REQUIRE(need == 0 || (workspace && workspace_bytes >= need && ((uintptr_t)workspace & 3) == 0), "select_token: workspace of %zu bytes needed", need);
    const int parts = (a.V + LOGITS_PER_BLOCK - 1) / LOGITS_PER_BLOCK;
    float* pv = (float*)workspace;
    int* pi = (int*)(pv + (size_t)a.rows * parts);
#define PE_SELECT(T, THREADS, WHOLE, X)                                                                                          \
    hipLaunchKernelGGL((select_part_kernel<T, THREADS, WHOLE>), dim3(X, a.rows), dim3(THREADS), 0, stream, a, pv, pi, token, count_into, out_ids, step, max_steps)
    if (need == 0) {
        if (a.V <= LOGITS_PER_BLOCK) { if (a.f32) PE_SELECT(float, 256, true, 1); else PE_SELECT(bf16, 256, true, 1); }
        else { if (a.f32) PE_SELECT(float, 1024, true, 1); else PE_SELECT(bf16, 1024, true, 1); }
        return check_launch("select_part_kernel");
    }
    if (a.f32) PE_SELECT(float, 256, false, parts);
    else PE_SELECT(bf16, 256, false, parts);
#undef PE_SELECT
    if (const int rc = check_launch("select_part_kernel")) return rc;
    hipLaunchKernelGGL(select_join_kernel, dim3(a.rows), dim3(64), 0, stream, pv, pi, parts, token, count_into, a.ldc, out_ids, step, max_steps);
    return check_launch("select_join_kernel");
}

int launch_token_counts_add(short* counts, long long ldc, int rows, int V, const int* tokens, int n, int prompt, hipStream_t stream) {
    PE_REQUIRE(counts && tokens && ((uintptr_t)counts & 1) == 0 && ((uintptr_t)tokens & 3) == 0, "token_counts_add: null or unaligned pointer");
    PE_REQUIRE(rows >= 1 && rows <= 65535 && V >= 1 && n >= 1 && ldc >= V, "token_counts_add: bad shape (%d rows of %d, %d tokens)", rows, V, n);
    hipLaunchKernelGGL(token_counts_add_kernel, dim3((unsigned)(((long long)n + COUNT_THREADS - 1) / COUNT_THREADS), rows), dim3(COUNT_THREADS), 0, stream, counts, ldc,
                       V, tokens, n, prompt);
    return check_launch("token_counts_add_kernel");
}

}  // namespace pe
