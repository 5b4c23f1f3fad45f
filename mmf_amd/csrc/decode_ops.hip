// mmf_amd :: decoding with a paged key / value cache and several beams per request — everything around the attention
// (paged_attention.hip): the plan of a step (pages and slots from lengths), the write of new keys and values, the selection of
// the best continuations, and the block tables after it.  M4C's decoding loop (mmf/models/m4c.py:284-304) is greedy and re-runs the
// whole transformer per step; mmf/utils/text.py's BeamSearch keeps its beams on the host.
#include "common.h"
#include "mmf_amd.h"
#include "paged_common.h"

namespace {

// inclusive sum over the workgroup (up to 16 waves); `total` gets the sum of all.  lds: 16 values
template <typename T> DEVI T wave_upto(T v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T t = __shfl_up(v, o, 64);
        if (lane >= o) v += t;
    }
    return v;
}
template <typename T> DEVI T block_scan(T v, int64_t* lds, T& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, waves = blockDim.x >> 6;
    const T s = wave_upto(v, lane);
    __syncthreads();
    if (lane == 63) lds[wave] = s;
    __syncthreads();
    T x = lane < waves ? (T)lds[lane] : 0;
    const T own = __shfl(x, wave, 64);
#pragma unroll
    for (int o = 1; o < 16; o <<= 1) {
        const T t = __shfl_up(x, o, 64);
        if (lane >= o) x += t;
    }
    total = __shfl(x, 15, 64);
    return s + __shfl(x, wave, 64) - own;
}

// ------------------------------------------------------------------------------------------------
// the plan of a step.  Whole numbers only; a few bytes per request and 12 per new token: latency is all there is to it.  One workgroup takes back the pages of
// finished groups and scans the groups (a thread each: what a group needs, what those before it took); the rows' tokens and blocks are filled in by the
// same launch where they are few, and by a second one over the whole chip where not.  32 groups of 5 beams with a token each: 4.3 us;
// 512 requests, 51 of them released, with 136 thousand new tokens: 13.6 us (four dependent trips to memory, two for the released pages, and three scans) and 4.3 for the rows.
// ------------------------------------------------------------------------------------------------
struct PlanGroup {      // what the scan leaves for the rows of a group
    int base;           // pages taken by the groups before it
    int forks;          // bit w: beam w takes a page for the block it shares so far
    int kv;             // tokens in the cache before this step
    int granted;        // new tokens; -1 - n: none of the n asked for
};

constexpr int PLAN_THREADS = 1024;       // (256 where that is a thread per group)
constexpr int PLAN_MANY = 128;           // tokens from which a row is walked by the whole workgroup

DEVI int blocks_of(int tokens, int shift) { return (int)(((int64_t)tokens + (1 << shift) - 1) >> shift); }

// Pages of released groups, back on the stack in the order of their rows and blocks; returns the new top.  As many rows at a time as there are threads: those to
// release are listed, in any order; 16 lanes count the pages of a listed row, the counts are scanned over the rows, and 16 lanes push them from there.
struct Release { int blocks[PLAN_THREADS], place[PLAN_THREADS], list[PLAN_THREADS], listed; };
DEVI int plan_release(const mmf_paged_plan_desc& d, int shift, int top, Release& x, int64_t* lds) {
    const int tid = threadIdx.x, l16 = tid & 15, team = tid >> 4, teams = blockDim.x >> 4, R = d.groups * d.beams;
#pragma unroll 1
    for (int r0 = 0; r0 < R; r0 += blockDim.x) {
        const int g = min(r0 + tid, R - 1) / d.beams, q = d.q_lens[g], kv = d.kv_lens[g];
        if (tid == 0) x.listed = 0;
        __syncthreads();
        x.place[tid] = 0;
        if (r0 + tid < R && q < 0) {
            x.blocks[tid] = min(blocks_of(max(kv, 0), shift), d.blocks);
            x.list[atomicAdd(&x.listed, 1)] = tid;
        }
        __syncthreads();
        const int listed = x.listed;
#pragma unroll 1
        for (int k = team; k < listed; k += teams) {
            const int r = x.list[k], blocks = x.blocks[r];
            const int* owned = d.owned + (size_t)(r0 + r) * d.blocks;
            int n = 0;
#pragma unroll 8
            for (int j = l16; j < blocks; j += 16) n += owned[j] >= 0;
#pragma unroll
            for (int o = 8; o > 0; o >>= 1) n += __shfl_xor(n, o, 64);
            if (l16 == 0) x.place[r] = n;
        }
        __syncthreads();
        const int n = x.place[tid];
        int total;
        const int upto = block_scan(n, lds, total);
        x.place[tid] = top + upto - n;
        __syncthreads();
#pragma unroll 1
        for (int k = team; k < listed; k += teams) {
            const int r = x.list[k], blocks = x.blocks[r];
            const int* owned = d.owned + (size_t)(r0 + r) * d.blocks;
            int at = x.place[r];
            for (int j0 = 0; j0 < blocks; j0 += 64) {
                int p[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) p[e] = j0 + 16 * e + l16 < blocks ? owned[j0 + 16 * e + l16] : -1;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t m = (uint32_t)(__ballot(p[e] >= 0) >> (tid & 48)) & 0xffff;
                    const int to = at + __popc(m & ((1u << l16) - 1));
                    if (p[e] >= 0) {
                        if (to < d.free_capacity) d.free_pages[to] = p[e];
                        else flag_page_error();                  // more pages came back than the pool has: one was given back twice
                    }
                    at += __popc(m);
                }
            }
        }
        top = min(top + total, d.free_capacity);
        __syncthreads();
    }
    return top;
}

// the tokens and blocks of one row, by `nthr` threads
DEVI void plan_row(const mmf_paged_plan_desc& d, int shift, const PlanGroup& g, int r, int w, int start, int top, int tid, int nthr) {
    const bool gets = !d.shared || w == 0;                        // has tokens and pages of its own
    if (g.granted > 0) {
        const int have = blocks_of(g.kv, shift), want = blocks_of(g.kv + g.granted, shift), below = (1 << shift) - 1;
        const bool fork = (g.forks >> w) & 1;
        const int lo = fork ? g.kv >> shift : have;
        int rank = g.base;                                        // the row's first page, counted from the top of the stack
        if (!d.shared) rank += w * (want - have) + __popc(g.forks & ((1u << w) - 1u));
        const int* from = d.free_pages + (top - 1 - rank + lo);   // from[-j]: the page of block j >= lo
        int* table = d.tables + (size_t)r * d.blocks;
        int* owned = d.owned + (size_t)r * d.blocks;
        const int part = have > 0 ? table[have - 1] : -1;         // the block that is not full yet, unless the row gets a page for it
        if (gets)
            for (int i = tid; i < g.granted; i += nthr) {
                const int pos = g.kv + i, j = pos >> shift;
                const int page = j >= lo ? from[-j] : part;
                if (page < 0) flag_page_error();                  // (the token has no slot; a page beyond the pool is the write's to see)
                d.slots[start + i] = page < 0 ? -1 : ((int64_t)page << shift) + (pos & below);
                d.positions[start + i] = pos;
            }
        for (int j = lo + tid; j < want; j += nthr) {
            const int page = from[-j];
            if (fork && j == lo) {
                int* c = d.copies + 3 * (size_t)r;
                c[0] = part; c[1] = page; c[2] = g.kv & below;
                if (part < 0) flag_page_error();                  // (nothing to copy from)
            }
            table[j] = page;
            owned[j] = gets ? page : -1;                          // a shared block belongs to the group's first row
        }
    } else if (gets) {                                            // the tokens of a request that has to wait
        const int n = min(-1 - g.granted, d.rows - start);
        for (int i = tid; i < n; i += nthr) { d.slots[start + i] = -1; d.positions[start + i] = -1; }
    }
}

// rows_too: a row by one thread, by eight where some have more than four tokens, by all where it has many; else the second launch takes workgroups for each
__global__ __launch_bounds__(PLAN_THREADS) void plan_kernel(mmf_paged_plan_desc d, int shift, int rows_too) {
    __shared__ int64_t lds[PLAN_THREADS / 64];
    __shared__ int taken, refused, flags;                         // flags: 1 a group is released, 2 a row has many tokens
    __shared__ Release release;
    const int tid = threadIdx.x, threads = blockDim.x, W = d.beams, per = d.shared ? 1 : W;
    PlanGroup* ws = reinterpret_cast<PlanGroup*>(d.ws);
    int* tail = reinterpret_cast<int*>(ws + d.groups);             // [0]: the top the pages are taken from
    if (tid == 0) { taken = 0; refused = 0; flags = 0; }
    const int g_first = min(tid, d.groups - 1), q_first = d.q_lens[g_first], kv_first = d.kv_lens[g_first];
    for (int i = tid; i < 3 * d.groups * W; i += threads) d.copies[i] = -1;
    const int told = d.free_top[0];
    int top = min(max(told, 0), d.free_capacity);
    if (tid == 0 && top != told) flag_page_error();
    __syncthreads();
    int most = max(q_first, 0), least = min(q_first, 0);
    for (int g = tid + threads; g < d.groups; g += threads) {
        const int q = d.q_lens[g];
        most = max(most, q);
        least = min(least, q);
    }
    const int f = (least < 0) | (most > 4) << 1 | (most > PLAN_MANY) << 2;
    if (f) atomicOr(&flags, f);
    __syncthreads();
    if (flags & 1) top = plan_release(d, shift, top, release, lds);
    const int per_row = flags & 2 ? 8 : 1;
    int carry_need = 0, total;
    int64_t carry_rows = 0, total64;
#pragma unroll 1
    for (int g0 = 0; g0 < d.groups; g0 += threads) {
        const int g = g0 + tid;
        const bool in = g < d.groups;
        const int q = !in ? 0 : g0 ? d.q_lens[g] : q_first, kv = !in ? 0 : max(g0 ? d.kv_lens[g] : kv_first, 0), n = max(q, 0);
        const int64_t rows = (int64_t)per * n, start = carry_rows + block_scan(rows, lds, total64) - rows;
        carry_rows += total64;
        const bool fits = (int64_t)kv + n <= (int64_t)d.blocks << shift && start + rows <= d.rows;
        int need = 0, forks = 0;
        if (n > 0 && fits) {
            if (!d.shared && (kv & ((1 << shift) - 1))) {
                const int* owned = d.owned + (size_t)g * W * d.blocks + (kv >> shift);
#pragma unroll 4
                for (int w = 1; w < W; ++w) forks |= (owned[(size_t)w * d.blocks] < 0) << w;
            }
            need = per * (blocks_of(kv + n, shift) - blocks_of(kv, shift)) + __popc(forks);
        }
        const int upto = carry_need + block_scan(need, lds, total);
        carry_need += total;
        const bool served = in && q >= 0 && fits && (need == 0 || upto <= top);
        if (in) {
            d.granted[g] = served ? n : 0;
            d.kv_out[g] = q < 0 ? 0 : kv + (served ? n : 0);
            ws[g] = PlanGroup{upto - need, served ? forks : 0, kv, served ? n : -1 - n};
            for (int w = 0; w < per; ++w) d.q_start[(size_t)g * per + w] = (int)min(start + (int64_t)w * n, (int64_t)d.rows);
            if (served && need) atomicMax(&taken, upto);          // (all that is asked for before a group that gets pages is served too)
            if (q >= 0 && !served) atomicAdd(&refused, 1);
        }
    }
    for (int64_t i = carry_rows + tid; i < d.rows; i += threads) { d.slots[i] = -1; d.positions[i] = -1; }
    __syncthreads();
    if (tid == 0) {
        d.top_out[0] = top - taken;
        d.refused[0] = refused;
        tail[0] = top;
    }
    if (!rows_too) return;
    if (tid == 0) release.listed = 0;
    __syncthreads();
#pragma unroll 1
    for (int r = tid / per_row; r < d.groups * W; r += threads / per_row) {
        const int g = r / W;
        const PlanGroup x = ws[g];
        if ((flags & 4) && x.granted > PLAN_MANY) {
            if (tid % per_row == 0) release.list[atomicAdd(&release.listed, 1)] = r;
        } else plan_row(d, shift, x, r, r - g * W, d.shared ? d.q_start[g] : d.q_start[r], top, tid % per_row, per_row);
    }
    if (!(flags & 4)) return;
    __syncthreads();
#pragma unroll 1
    for (int k = 0; k < release.listed; ++k) {
        const int r = release.list[k], g = r / W;
        plan_row(d, shift, ws[g], r, r - g * W, d.shared ? d.q_start[g] : d.q_start[r], top, tid, threads);
    }
}
__global__ __launch_bounds__(256) void plan_rows_kernel(mmf_paged_plan_desc d, int shift) {
    const PlanGroup* ws = reinterpret_cast<const PlanGroup*>(d.ws);
    const int r = blockIdx.x, g = r / d.beams;
    plan_row(d, shift, ws[g], r, r - g * d.beams, d.shared ? d.q_start[g] : d.q_start[r], reinterpret_cast<const int*>(ws + d.groups)[0],
             blockIdx.y * 256 + threadIdx.x, gridDim.y * 256);
}

// ------------------------------------------------------------------------------------------------
// new keys and values into their slots.  Every byte moves once each way, and memory bounds it: 16384 rows of 8 heads of 128 in bf16, 27 us for 121 MB; 160 rows of 12 heads
// of 64: 2.8 us, an empty launch.  A thread moves one VT: 16 bytes, or one element where a row does not start on 16 bytes (134 MB that caches hold: 22 us by 16 bytes,
// 122 by elements).
// ------------------------------------------------------------------------------------------------
template <typename VT>
__global__ __launch_bounds__(256) void paged_write_kernel(mmf_paged_write_desc d, int esize, int per_token) {
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int t = (int)(i / per_token);
    if (t >= d.tokens) return;
    int c = (int)(i - (int64_t)t * per_token);
    const int64_t slot = d.slots[t];
    if (slot < 0) return;
    if (slot >= (int64_t)d.pages * d.page_size) {
        if (c == 0) flag_page_error();
        return;
    }
    const bool is_v = c >= per_token / 2;
    if (is_v) c -= per_token / 2;
    const int per_head = d.head_dim * esize / (int)sizeof(VT), h = c / per_head, e = (c - h * per_head) * (int)sizeof(VT);
    const int64_t page = slot / d.page_size, pos = slot - page * d.page_size;
    const char* src = (const char*)(is_v ? d.v : d.k) + ((is_v ? (int64_t)t * d.v_row + (int64_t)h * d.v_head : (int64_t)t * d.k_row + (int64_t)h * d.k_head) * esize + e);
    char* dst = (char*)(is_v ? d.v_cache : d.k_cache) + ((page * d.page_stride + h * d.head_stride + pos * d.pos_stride) * esize + e);
    *reinterpret_cast<VT*>(dst) = *reinterpret_cast<const VT*>(src);
}

// ------------------------------------------------------------------------------------------------
// the best continuations of a group.  Candidate (w, v) of an unfinished beam: score[w] + logit[w][v] - lse[w]; of a finished one: the
// end token at score[w].  The W largest, the lowest flat index w * V + v first among equals.  Values of different beams meet in 64 bits:
// in 32 the sum would round candidates together that are apart.
//
// Within a row the order is the logits' own, so a first kernel takes every row in segments, a workgroup each with the segment in its registers, and leaves the segment's
// maximum, its sum of exponentials and its W largest; a second one merges the segments and beams of a group.  Both pick W out of N in the same way: of the maxima of
// 64 groups of threads the W-th largest is a bar that at least W values reach, and few more do; those are ranked by counting.
//
// 128 rows of 128000 logits in bf16, 8 beams: 15 us for the rows (33 MB; vector instructions, 23 a logit of which the exponential and its correction are 7, issue in 40 % of
// its cycles, and start when most loads have landed) and 10 for the merge; 160 rows of 5050 in fp32, 5 beams: 6.3 and 7.5 us.  The merge is a chain of trips to memory and to
// LDS by a workgroup per group: what does not wait for the sums (lists, segments, the history's first columns) is read first.
// ------------------------------------------------------------------------------------------------
constexpr double NEG_INF = -__builtin_huge_val();
constexpr int CHUNKS = 4, LIST = 1024, KEEP = LIST / 256;                            // 16-byte pieces of a segment per thread
template <typename T> constexpr int seg_max = 256 * CHUNKS * 16 / (int)sizeof(T);

struct Picked { float v; int i; };                                // i: index in the row, -1: none
struct Segment { double sum; float top; int pad; };               // sum of exp(x - top)
DEVI bool better(double av, int64_t ai, double bv, int64_t bi) { return av > bv || (av == bv && ai < bi); }

// The W-th largest of the maxima of 64 groups of four threads; `top` gets the largest.  Every wave ranks all 64 among 16 of them
struct Bar { float4 best[16]; int rank[4][64]; float top[4]; };
DEVI float bar_of(float mine, int W, Bar& b, float& top) {
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    mine = fmaxf(mine, __shfl_xor(mine, 1, 64));
    mine = fmaxf(mine, __shfl_xor(mine, 2, 64));
    float* best = reinterpret_cast<float*>(b.best);
    if ((tid & 3) == 0) best[tid >> 2] = mine;
    __syncthreads();
    const float x = best[lane];
    const int from = lane - 16 * wave;
    int rank = 0;
    float most = -INFINITY;
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        const float4 y = b.best[4 * wave + j];
        most = fmaxf(most, fmaxf(fmaxf(y.x, y.y), fmaxf(y.z, y.w)));
        rank += (y.x > x || (y.x == x && 4 * j < from)) + (y.y > x || (y.y == x && 4 * j + 1 < from)) + (y.z > x || (y.z == x && 4 * j + 2 < from)) +
                (y.w > x || (y.w == x && 4 * j + 3 < from));
    }
    b.rank[wave][lane] = rank;
    if (lane == 0) b.top[wave] = most;
    __syncthreads();
    rank = b.rank[0][lane] + b.rank[1][lane] + b.rank[2][lane] + b.rank[3][lane];
    top = fmaxf(fmaxf(b.top[0], b.top[1]), fmaxf(b.top[2], b.top[3]));
    return __shfl(x, __ffsll((unsigned long long)__ballot(rank == W - 1)) - 1, 64);
}

// exp(x) for x <= 0, the rounding of x log2 e carried along: relative 2^-23 at any x
DEVI float exp_down(float x) {
    x = fmaxf(x, -200.f);                                         // (a masked value: its power is 0 all the same)
    const float a = x * 1.44269504088896340736f, r = fmaf(x, 1.9259629911266174e-8f, fmaf(x, 1.44269504088896340736f, -a));
    return __builtin_amdgcn_exp2f(a) * fmaf(r, 0.693147180559945309f, 1.f);
}
// log(x) of a normal x > 0 in 64 bits: x = m 2^e with m in [sqrt 1/2, sqrt 2), log m = 2 atanh(s), s = (m - 1) / (m + 1), |s| < 0.172: the series ends below 1e-13
DEVI double log_of(double x) {
    int e = __builtin_amdgcn_frexp_exp(x);
    double m = __builtin_amdgcn_frexp_mant(x);
    if (m < 0.70710678118654752) { m *= 2.0; e -= 1; }
    const double s = (m - 1.0) / (m + 1.0), q = s * s;
    double p = 1.0 / 15.0;
#pragma unroll
    for (int k = 13; k >= 1; k -= 2) p = p * q + 1.0 / k;
    return 2.0 * s * p + e * 0.69314718055994530942;
}

// 16 bytes of a row; WIDE: rows start on 4 bytes, else on an element.  Behind the end: -inf.  (NaN loses every comparison and maximum below, as -inf does.)
template <typename T, bool WIDE> struct Piece {
    static constexpr int VEC = 16 / (int)sizeof(T);
    typedef uint32_t u32x4a __attribute__((ext_vector_type(4), aligned(4)));
    T x[VEC];
    DEVI void load(const T* row, int at, int n) {
        if (WIDE && at + VEC <= n) {
            const u32x4a w = *reinterpret_cast<const u32x4a*>(row + at);
            __builtin_memcpy(x, &w, 16);
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) x[e] = at + e < n ? row[at + e] : (T)-INFINITY;
        }
    }
};

template <typename T, bool WIDE>
__global__ __launch_bounds__(256, WIDE ? 8 : 4) void beam_rows_kernel(mmf_beam_select_desc d, int segments, int length) {
    typedef Piece<T, WIDE> P;
    constexpr int VEC = P::VEC;
    __shared__ Bar maxima;
    __shared__ float cand_v[LIST];
    __shared__ int cand_i[LIST], count;
    __shared__ double sums[4];
    const int row = blockIdx.y, seg = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, W = d.beams;
    const float score = d.scores[row];
    if (d.finished[row] || !(score > -INFINITY)) return;          // (the second kernel does not look at these rows either)
    const int64_t first = (int64_t)seg * length;
    const int n = (int)min((int64_t)length, d.vocab - first);
    const T* x = (const T*)d.logits + (int64_t)row * d.ld + first;
    if (tid == 0) count = 0;
    P p[CHUNKS];
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
        if (c == 0 || 256 * VEC * c < n) p[c].load(x, (256 * c + tid) * VEC, n);
    float mine = -INFINITY;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
        if (c == 0 || 256 * VEC * c < n)
#pragma unroll
            for (int e = 0; e < VEC; ++e) mine = fmaxf(mine, (float)p[c].x[e]);
    float top;
    const float bar = bar_of(mine, W, maxima, top), base = top > -INFINITY && top < INFINITY ? top : 0.f;
    double s = 0.0;
#pragma unroll
    for (int c = 0; c < CHUNKS; ++c)
        if (c == 0 || 256 * VEC * c < n) {
#pragma unroll
            for (int e = 0; e < VEC; e += 4)
                s += (double)((exp_down((float)p[c].x[e] - base) + exp_down((float)p[c].x[e + 1] - base)) +
                              (exp_down((float)p[c].x[e + 2] - base) + exp_down((float)p[c].x[e + 3] - base)));
        }
    if (mine >= bar && mine > -INFINITY) {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c)
            if (c == 0 || 256 * VEC * c < n)
#pragma unroll
                for (int e = 0; e < VEC; ++e) {
                    const float y = (float)p[c].x[e];
                    if (y >= bar && y > -INFINITY) {
                        const int to = atomicAdd(&count, 1);
                        if (to < LIST) { cand_v[to] = y; cand_i[to] = (256 * c + tid) * VEC + e; }
                    }
                }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if (lane == 0) sums[wave] = s;
    __syncthreads();
    Picked* out = (Picked*)d.ws + ((int64_t)row * segments + seg) * W;
    Segment* seg_out = (Segment*)((Picked*)d.ws + (((int64_t)d.groups * W * segments * W + 1) & ~1ll)) + (int64_t)row * segments + seg;
    if (tid == 0) *seg_out = Segment{sums[0] + sums[1] + sums[2] + sums[3], top, 0};
    const int found = count;
    if (found <= LIST) {
        for (int i = tid; i < found; i += 256) {
            const float a = cand_v[i];
            const int ai = cand_i[i];
            int rank = 0;
            for (int j = 0; j < found; ++j) {
                const float bv = cand_v[j];
                rank += bv > a || (bv == a && cand_i[j] < ai);
            }
            if (rank < W) out[rank] = Picked{a, (int)first + ai};
        }
        if (tid >= found && tid < W) out[tid] = Picked{-INFINITY, -1};
        return;
    }
    float last = INFINITY;                                        // a plateau of equal values wider than the list: one round per value picked
    int last_i = -1;
#pragma unroll 1
    for (int k = 0; k < W; ++k) {
        float bv = -INFINITY;
        int bi = 0x7fffffff;
#pragma unroll 1
        for (int i = tid; i < n; i += 256) {
            const float y = (float)x[i];
            if (y > -INFINITY && (y < last || (y == last && i > last_i)) && (y > bv || (y == bv && i < bi))) { bv = y; bi = i; }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const float ov = __shfl_xor(bv, o, 64);
            const int oi = __shfl_xor(bi, o, 64);
            if (ov > bv || (ov == bv && oi < bi)) { bv = ov; bi = oi; }
        }
        __syncthreads();
        if (lane == 0) { cand_v[wave] = bv; cand_i[wave] = bi; }
        __syncthreads();
        for (int u = 0; u < 4; ++u)
            if (cand_v[u] > bv || (cand_v[u] == bv && cand_i[u] < bi)) { bv = cand_v[u]; bi = cand_i[u]; }
        last = bv;
        last_i = bi;
        if (tid == 0) out[k] = bi == 0x7fffffff ? Picked{-INFINITY, -1} : Picked{bv, (int)first + bi};
    }
}

// step_at: the column of the new tokens where the host does not know it (a captured call that is replayed), else null
__global__ __launch_bounds__(256) void beam_merge_kernel(mmf_beam_select_desc d, int segments, const int32_t* step_at) {
    __shared__ double cand_v[LIST], score[MMF_BEAMS_MAX], lse[MMF_BEAMS_MAX], best_v[MMF_BEAMS_MAX], red_v[4];
    __shared__ int64_t cand_i[LIST], best_i[MMF_BEAMS_MAX], red_i[4];
    __shared__ int done[MMF_BEAMS_MAX], parent[MMF_BEAMS_MAX], count;
    __shared__ Bar maxima;
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, W = d.beams;
    const int64_t V = d.vocab;
    const Picked* picked = (const Picked*)d.ws + (int64_t)g * W * segments * W;
    const Segment* segs = (const Segment*)((const Picked*)d.ws + (((int64_t)d.groups * W * segments * W + 1) & ~1ll)) + (int64_t)g * W * segments;
    if (tid < W) {                                                // (scores and finished may be updated in place)
        const float s = d.scores[g * W + tid];
        score[tid] = s == s ? (double)s : NEG_INF;
        done[tid] = d.finished[g * W + tid] != 0;
        best_v[tid] = NEG_INF;
        best_i[tid] = -1;
    }
    if (tid == 0) count = 0;
    const int64_t step = step_at ? *step_at : d.step;             // (read with the first loads; needed last)
    const int per = segments * W, cols = (int)min((int64_t)(LIST / W), d.length);
    const float one = 1.f / per, per_col = 1.f / cols;            // k / per for k < 2^20 (a vocabulary of 2^22): half a unit is more than the rounding
    auto beam_of = [&](int k) { return (int)(((float)k + 0.5f) * one); };
    const int64_t at = (int64_t)g * W * d.length;
    Picked early[KEEP];                                           // what does not wait for the sums
    int64_t past[KEEP];
#pragma unroll
    for (int e = 0; e < KEEP; ++e) {
        const int k = tid + 256 * e;
        early[e] = Picked{-INFINITY, -1};
        past[e] = 0;
        if (k < W * per) early[e] = picked[k];
        if (d.history && k < W * cols) {
            const int w = (int)(((float)k + 0.5f) * per_col);
            past[e] = d.history[at + w * d.length + k - w * cols];
        }
    }
    const int l16 = tid & 15;
    Segment first = {0.0, -INFINITY, 0};
    if (tid >> 4 < W && l16 < segments) first = segs[(tid >> 4) * segments + l16];
    __syncthreads();
    for (int w0 = 0; w0 < W; w0 += 16) {                          // lse, by 16 lanes each: NaN marks a row without candidates
        const int w = w0 + (tid >> 4);
        const bool live = w < W && !done[w] && score[w] > NEG_INF;
        if (w0) first = live && l16 < segments ? segs[w * segments + l16] : Segment{0.0, -INFINITY, 0};
        float m = live ? first.top : -INFINITY;
        for (int s = live ? l16 + 16 : segments; s < segments; s += 16) m = fmaxf(m, segs[w * segments + s].top);
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o, 64));
        double sum = live && first.top > -INFINITY ? first.sum * (double)exp_down(first.top - m) : 0.0;
        for (int s = live ? l16 + 16 : segments; s < segments; s += 16) {
            const Segment x = segs[w * segments + s];
            if (x.top > -INFINITY) sum += x.sum * (double)exp_down(x.top - m);
        }
#pragma unroll
        for (int o = 8; o > 0; o >>= 1) sum += __shfl_xor(sum, o, 64);
        if (l16 == 0 && w < W) lse[w] = live && m > -INFINITY && m < INFINITY ? (double)m + log_of(sum) : __builtin_nan("");
    }
    __syncthreads();
    // candidate k of beam w's lists; a finished beam's only one stands first in its lists
    auto cand = [&](int k, const Picked& p, int64_t& i) {
        const int w = beam_of(k);
        double v = NEG_INF;
        i = w * V;
        if (done[w]) {
            if (k == w * per) { v = score[w]; i += d.eos; }
        } else if (lse[w] == lse[w] && p.i >= 0) { v = score[w] + ((double)p.v - lse[w]); i += p.i; }
        return v;
    };
    float mine = -INFINITY;                                       // (rounding to 32 bits keeps the order)
    int64_t at_i[KEEP];
    double at_v[KEEP];
#pragma unroll
    for (int e = 0; e < KEEP; ++e) {
        at_v[e] = tid + 256 * e < W * per ? cand(tid + 256 * e, early[e], at_i[e]) : NEG_INF;
        mine = fmaxf(mine, (float)at_v[e]);
    }
#pragma unroll 4
    for (int k = tid + 256 * KEEP; k < W * per; k += 256) {
        int64_t i;
        mine = fmaxf(mine, (float)cand(k, picked[k], i));
    }
    float top;
    const float bar = bar_of(mine, W, maxima, top);
    auto keep = [&](double v, int64_t i) {
        if (v > NEG_INF && (float)v >= bar) {
            const int to = atomicAdd(&count, 1);
            if (to < LIST) { cand_v[to] = v; cand_i[to] = i; }
        }
    };
    if (mine >= bar && mine > -INFINITY) {
#pragma unroll
        for (int e = 0; e < KEEP; ++e) keep(at_v[e], at_i[e]);
#pragma unroll 1
        for (int k = tid + 256 * KEEP; k < W * per; k += 256) {
            int64_t i;
            const double v = cand(k, picked[k], i);
            keep(v, i);
        }
    }
    __syncthreads();
    const int found = count;
    if (found <= LIST) {
        for (int a = tid; a < found; a += 256) {
            const double v = cand_v[a];
            const int64_t i = cand_i[a];
            int rank = 0;
            for (int b = 0; b < found; ++b) rank += better(cand_v[b], cand_i[b], v, i);
            if (rank < W) { best_v[rank] = v; best_i[rank] = i; }
        }
    } else {
        double last = -NEG_INF;
        int64_t last_i = -1;
#pragma unroll 1
        for (int r = 0; r < W; ++r) {
            double bv = NEG_INF;
            int64_t bi = INT64_MAX;
#pragma unroll 1
            for (int k = tid; k < W * per; k += 256) {
                int64_t i;
                const double v = cand(k, picked[k], i);
                if (v > NEG_INF && better(last, last_i, v, i) && better(v, i, bv, bi)) { bv = v; bi = i; }
            }
#pragma unroll 1
            for (int o = 32; o > 0; o >>= 1) {
                const double ov = __shfl_xor(bv, o, 64);
                const int64_t oi = __shfl_xor((long long)bi, o, 64);
                if (better(ov, oi, bv, bi)) { bv = ov; bi = oi; }
            }
            __syncthreads();
            if (lane == 0) { red_v[wave] = bv; red_i[wave] = bi; }
            __syncthreads();
            for (int u = 0; u < 4; ++u)
                if (better(red_v[u], red_i[u], bv, bi)) { bv = red_v[u]; bi = red_i[u]; }
            last = bv;
            last_i = bi;
            if (tid == 0 && bi != INT64_MAX) { best_v[r] = bv; best_i[r] = bi; }
        }
    }
    __syncthreads();
    if (tid == 0 && best_i[W - 1] < 0) {                          // fewer live candidates than beams: the others are equal, the lowest indices go first
        int have = 0;
        while (best_i[have] >= 0) ++have;
        int64_t i = 0;
        for (int r = have; r < W; ++i) {
            bool used = false;
            for (int b = 0; b < have; ++b) used |= best_i[b] == i;
            if (!used) best_i[r++] = i;
        }
    }
    __syncthreads();
    if (tid < W) {
        const int64_t i = best_i[tid];
        int p = 0;
        while ((p + 1) * V <= i) ++p;
        const int64_t token = i - p * V;
        parent[tid] = p;
        best_i[tid] = token;
        d.scores_out[g * W + tid] = (float)best_v[tid];
        d.parents[g * W + tid] = p;
        d.tokens[g * W + tid] = token;
        d.finished_out[g * W + tid] = done[p] || token == d.eos;
    }
    __syncthreads();
    if (!d.history) return;
    if (tid == 0 && (step < 0 || step >= d.length)) flag_page_error();       // (no column is the step's: the parents' rows come back as they are)
    // through LDS, many columns at a time: in place as well
    for (int64_t t0 = 0; t0 < d.length; t0 += cols) {
#pragma unroll
        for (int e = 0; e < KEEP; ++e) {                              // these columns, and the next ones on their way
            const int k = tid + 256 * e, w = (int)(((float)k + 0.5f) * per_col);
            const int64_t t = t0 + cols + k - w * cols;
            if (k < W * cols) {
                cand_i[k] = past[e];
                if (t < d.length) past[e] = d.history[at + w * d.length + t];
            }
        }
        __syncthreads();
#pragma unroll
        for (int e = 0; e < KEEP; ++e) {
            const int k = tid + 256 * e, w = (int)(((float)k + 0.5f) * per_col);
            const int64_t t = t0 + k - w * cols;
            if (k < W * cols && t < d.length) d.history_out[at + w * d.length + t] = t == step ? best_i[w] : cand_i[parent[w] * cols + k - w * cols];
        }
        __syncthreads();
    }
}

// Segments of a row: as long as a workgroup holds, and shorter where few rows would leave compute units idle (four workgroups for each; with two or eight the two sizes
// above take the same within 2 %), down to a piece per thread
int beam_segments(int rows, int64_t vocab, bool f32, int* length) {
    const int64_t least = (vocab + (f32 ? seg_max<float> : seg_max<bf16>) - 1) / (f32 ? seg_max<float> : seg_max<bf16>), fill = (1024 + rows - 1) / rows;
    const int64_t most = vocab / (f32 ? 1024 : 2048);
    int64_t n = fill < most ? fill : most;
    if (n < least) n = least;
    const int64_t len = ((vocab + n - 1) / n + 7) / 8 * 8;
    *length = (int)len;
    return (int)((vocab + len - 1) / len);
}

// ------------------------------------------------------------------------------------------------
// block tables after a selection.  A block that is full is only read from here on: the children share it.  The block that goes on being
// written has to be each beam's own: the first child of a beam keeps its page, the other children take the pages of the beams that have
// no child, of which there are exactly as many, and get its tokens copied.  A page that is copied from is never copied to.
// The tables are a workgroup per group; the copies a launch over rows and planes that leaves at once where there is nothing to copy.  32 groups of 5 beams, 8 planes of
// 12 heads of 64, half a page of 16 to copy: 8.7 us for 12.5 MB, two launches and their trips to memory; 8 groups of 8 beams, 32 planes of 8 heads of 128, 68 MB: 21 us.
// ------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void reorder_tables_kernel(mmf_paged_reorder_desc d) {
    __shared__ int pages[LIST], copied[MMF_BEAMS_MAX];
    __shared__ int parent[MMF_BEAMS_MAX], source[MMF_BEAMS_MAX];  // source[w]: the beam whose last page beam w goes on writing
    const int g = blockIdx.x, tid = threadIdx.x, W = d.beams;
    if (tid < W) {
        int64_t p = d.parents[(size_t)g * W + tid];
        if (p < 0 || p >= W) { flag_page_error(); p = tid; }
        parent[tid] = (int)p;
    }
    __syncthreads();
    if (tid == 0) {
        uint32_t kept = 0;
        for (int w = 0; w < W; ++w) kept |= 1u << parent[w];
        uint32_t idle = ~kept, seen = 0;
        for (int w = 0; w < W; ++w) {
            if (!((seen >> parent[w]) & 1)) { source[w] = parent[w]; seen |= 1u << parent[w]; }
            else { source[w] = __ffs(idle) - 1; idle &= idle - 1; }
        }
    }
    __syncthreads();
    const int told = d.kv_lens[g], kv = max(told, 0), rest = kv & (d.page_size - 1), part = rest ? kv / d.page_size : -1, cols = LIST / W;
    const int* from = d.tables + (size_t)g * W * d.blocks;
    int* to = d.tables_out + (size_t)g * W * d.blocks;
    for (int j0 = 0; j0 < d.blocks; j0 += cols) {                 // through LDS, many columns at a time: in place as well
        for (int k = tid; k < W * cols; k += 256) {
            const int w = k / cols, j = j0 + k - w * cols;
            if (j < d.blocks) pages[k] = from[(size_t)(j == part ? source[w] : parent[w]) * d.blocks + j];
        }
        if (part >= j0 && part < j0 + cols && part < d.blocks && tid < W) copied[tid] = source[tid] != parent[tid] ? from[(size_t)parent[tid] * d.blocks + part] : -1;
        __syncthreads();
        for (int k = tid; k < W * cols; k += 256) {
            const int w = k / cols, j = j0 + k - w * cols;
            if (j < d.blocks) to[(size_t)w * d.blocks + j] = pages[k];
        }
        if (part >= j0 && part < j0 + cols && part < d.blocks && tid < W) {
            int* c = d.copies + 3 * ((size_t)g * W + tid);
            const bool copy = source[tid] != parent[tid];
            c[0] = copied[tid];
            c[1] = copy ? pages[tid * cols + part - j0] : -1;
            c[2] = copy ? rest : -1;
            if (copy && (c[0] < 0 || c[1] < 0)) flag_page_error();               // (left out; a page beyond the pool is the copy's to see)
        }
        __syncthreads();
    }
    if (tid == 0 && (told < 0 || kv > (int64_t)d.blocks * d.page_size)) flag_page_error();       // (a length that the table has no blocks for: full blocks only)
    if ((part < 0 || part >= d.blocks) && tid < 3 * W) d.copies[3 * (size_t)g * W + tid] = -1;
}

// the first copies[r][2] tokens of page copies[r][0] to page copies[r][1], in every plane (keys and values of every layer).  VT: 16 bytes, or an element where rows
// do not start on 16 (64 pages of 8 heads of 17 tokens in 32 planes: 20 us with 128 columns, 32 with 125)
template <typename VT>
__global__ __launch_bounds__(256) void copy_pages_kernel(mmf_paged_copy_desc d, int esize) {
    const int r = blockIdx.x;
    const int src = d.copies[3 * (size_t)r], dst = d.copies[3 * (size_t)r + 1], tokens = min(d.copies[3 * (size_t)r + 2], d.page_size);
    if (src == dst || src < 0 || dst < 0 || tokens <= 0) return;
    if (src >= d.pages || dst >= d.pages) {
        if (threadIdx.x == 0 && blockIdx.y == 0) flag_page_error();
        return;
    }
    char* base = (char*)d.cache + blockIdx.y * d.plane_stride * esize;
    char* to = base + dst * d.page_stride * esize;
    const char* from = base + src * d.page_stride * esize;
    const int per_pos = d.head_dim * esize / (int)sizeof(VT), n = tokens * per_pos, lane = threadIdx.x & 63;
    const bool dense = d.pos_stride == d.head_dim;
    for (int h = threadIdx.x >> 6; h < d.kv_heads; h += 4)        // a wave per head
#pragma unroll 4
        for (int i = lane; i < n; i += 64) {
            const int pos = dense ? 0 : i / per_pos;
            const int64_t off = (h * d.head_stride + pos * d.pos_stride) * esize + (int64_t)(i - pos * per_pos) * (int)sizeof(VT);
            *reinterpret_cast<VT*>(to + off) = *reinterpret_cast<const VT*>(from + off);
        }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

extern "C" {

int mmf_decode_take_error(void) { return take_page_error(); }

int64_t mmf_paged_plan_ws_bytes(int groups, int beams) {
    return groups > 0 && beams > 0 ? (int64_t)groups * (int64_t)sizeof(PlanGroup) + 16 : 0;
}

int mmf_paged_plan(const mmf_paged_plan_desc* d, void* stream) {
    MMF_CHECK_ARG(d && d->q_lens && d->kv_lens && d->tables && d->owned && d->free_pages && d->free_top, "paged_plan: null operand");
    MMF_CHECK_ARG(d->q_start && d->granted && d->kv_out && d->slots && d->positions && d->copies && d->top_out && d->refused && d->ws, "paged_plan: null output");
    MMF_CHECK_ARG(d->groups > 0 && d->blocks > 0 && d->rows > 0 && d->free_capacity > 0, "paged_plan: bad shape");
    MMF_CHECK_ARG(d->beams >= 1 && d->beams <= MMF_BEAMS_MAX && d->groups <= 0x0fffffff / d->beams, "paged_plan: 1 .. 32 beams");
    MMF_CHECK_ARG(d->page_size >= 1 && d->page_size <= MMF_PAGE_MAX && (d->page_size & (d->page_size - 1)) == 0, "paged_plan: page_size is a power of two up to 1024");
    MMF_CHECK_ARG((int64_t)d->blocks * d->page_size <= 0x40000000 && d->rows <= 0x40000000, "paged_plan: more than 2^30 tokens");
    // One workgroup walks up to a thousand tokens, or a few for each of as many rows as it has threads; more is work for the whole chip and a second launch.  32 groups of 5
    // beams, a token each: 4.3 us in one launch, 6.0 in two; 512 prompts of up to 2048 tokens: 306 us in one, 17.4 in two.
    const int64_t rows = (int64_t)d->groups * d->beams;
    const int64_t walked = (int64_t)d->rows * (d->shared ? d->beams : 1);      // (every row of a shared group fills its table; rows of many tokens: fewer than a thread each)
    const bool one = walked <= 1024 || (walked <= 4 * rows && rows <= 4 * PLAN_THREADS);
    const int shift = __builtin_ctz(d->page_size);
    page_kernels_used();
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(rows <= 256 ? 256 : PLAN_THREADS), 0, (hipStream_t)stream, *d, shift, (int)one);
    MMF_CHECK_LAUNCH();
    if (!one) {                                                   // a workgroup per row, and a few where rows have many tokens on average: some have many times that
        const int64_t wide = d->rows / rows / 64;
        const unsigned y = (unsigned)(wide < 1 ? 1 : wide > 8 ? 8 : wide);
        hipLaunchKernelGGL(plan_rows_kernel, dim3((unsigned)rows, y), dim3(256), 0, (hipStream_t)stream, *d, shift);
        MMF_CHECK_LAUNCH();
    }
    return 0;
}

int mmf_paged_write(const mmf_paged_write_desc* d, void* stream) {
    MMF_CHECK_ARG(d && d->k && d->v && d->k_cache && d->v_cache && d->slots, "paged_write: null operand");
    MMF_CHECK_ARG(d->tokens >= 0 && d->pages > 0 && d->kv_heads > 0 && d->head_dim > 0, "paged_write: bad shape");
    MMF_CHECK_ARG(d->page_size >= 1 && d->page_size <= MMF_PAGE_MAX, "paged_write: bad page_size");
    if (d->tokens == 0) return 0;
    const int es = d->is_f32 ? 4 : 2, unit = 16 / es;
    const bool wide = aligned16(d->k) && aligned16(d->v) && aligned16(d->k_cache) && aligned16(d->v_cache) && d->head_dim % unit == 0 && d->k_row % unit == 0 &&
                      d->k_head % unit == 0 && d->v_row % unit == 0 && d->v_head % unit == 0 && d->page_stride % unit == 0 && d->head_stride % unit == 0 &&
                      d->pos_stride % unit == 0;
    const int64_t per_token = 2ll * d->kv_heads * d->head_dim / (wide ? unit : 1), blocks = (d->tokens * per_token + 255) / 256;
    MMF_CHECK_ARG(per_token <= 0x3fffffff && blocks <= 0x7fffffff, "paged_write: too many elements for one call");
    const dim3 grid((unsigned)blocks);
    page_kernels_used();
    if (wide) hipLaunchKernelGGL(paged_write_kernel<uint4>, grid, dim3(256), 0, (hipStream_t)stream, *d, es, (int)per_token);
    else if (es == 4) hipLaunchKernelGGL(paged_write_kernel<uint32_t>, grid, dim3(256), 0, (hipStream_t)stream, *d, es, (int)per_token);
    else hipLaunchKernelGGL(paged_write_kernel<uint16_t>, grid, dim3(256), 0, (hipStream_t)stream, *d, es, (int)per_token);
    MMF_CHECK_LAUNCH();
    return 0;
}

int64_t mmf_beam_select_ws_bytes(int groups, int beams, int64_t vocab, int is_f32) {
    if (groups < 1 || beams < 1 || vocab < 1) return 0;
    int length;
    const int64_t rows = (int64_t)groups * beams, n = beam_segments((int)rows, vocab, is_f32 != 0, &length);
    return ((rows * n * beams + 1) & ~1ll) * (int64_t)sizeof(Picked) + rows * n * (int64_t)sizeof(Segment);
}

static int beam_select(const mmf_beam_select_desc* d, const int32_t* step_at, void* stream) {
    MMF_CHECK_ARG(d && d->logits && d->scores && d->finished && d->scores_out && d->parents && d->tokens && d->finished_out && d->ws, "beam_select: null operand");
    MMF_CHECK_ARG(d->groups > 0 && d->beams >= 1 && d->beams <= MMF_BEAMS_MAX && d->vocab > 0 && d->ld >= d->vocab, "beam_select: bad shape");
    MMF_CHECK_ARG(d->vocab <= 1 << 22 && (int64_t)d->groups * d->beams <= 65535, "beam_select: 2^22 tokens and 65535 rows at most");
    MMF_CHECK_ARG(d->eos >= 0 && d->eos < d->vocab, "beam_select: the end token is not in the vocabulary");
    MMF_CHECK_ARG(!d->history || (d->history_out && d->length > 0 && (step_at || (d->step >= 0 && d->step < d->length))), "beam_select: step is not a column of the history");
    int length;
    const int segments = beam_segments(d->groups * d->beams, d->vocab, d->is_f32 != 0, &length);
    const dim3 grid(segments, d->groups * d->beams);
    const bool wide = ((uintptr_t)d->logits & 3) == 0 && (d->ld & 1) == 0;
    page_kernels_used();
    if (d->is_f32) hipLaunchKernelGGL((beam_rows_kernel<float, true>), grid, dim3(256), 0, (hipStream_t)stream, *d, segments, length);
    else if (wide) hipLaunchKernelGGL((beam_rows_kernel<bf16, true>), grid, dim3(256), 0, (hipStream_t)stream, *d, segments, length);
    else hipLaunchKernelGGL((beam_rows_kernel<bf16, false>), grid, dim3(256), 0, (hipStream_t)stream, *d, segments, length);
    MMF_CHECK_LAUNCH();
    hipLaunchKernelGGL(beam_merge_kernel, dim3(d->groups), dim3(256), 0, (hipStream_t)stream, *d, segments, step_at);
    MMF_CHECK_LAUNCH();
    return 0;
}

int mmf_beam_select(const mmf_beam_select_desc* d, void* stream) { return beam_select(d, nullptr, stream); }

int mmf_beam_select_at(const mmf_beam_select_desc* d, const int32_t* step, void* stream) {
    MMF_CHECK_ARG(step, "beam_select: null operand");
    return beam_select(d, step, stream);
}

int mmf_paged_reorder(const mmf_paged_reorder_desc* d, void* stream) {
    MMF_CHECK_ARG(d && d->parents && d->kv_lens && d->tables && d->tables_out && d->copies, "paged_reorder: null operand");
    MMF_CHECK_ARG(d->groups > 0 && d->beams >= 1 && d->beams <= MMF_BEAMS_MAX && d->blocks > 0, "paged_reorder: bad shape");
    MMF_CHECK_ARG(d->page_size >= 1 && d->page_size <= MMF_PAGE_MAX && (d->page_size & (d->page_size - 1)) == 0, "paged_reorder: page_size is a power of two up to 1024");
    page_kernels_used();
    hipLaunchKernelGGL(reorder_tables_kernel, dim3(d->groups), dim3(256), 0, (hipStream_t)stream, *d);
    MMF_CHECK_LAUNCH();
    return 0;
}

int mmf_paged_copy(const mmf_paged_copy_desc* d, void* stream) {
    MMF_CHECK_ARG(d && d->copies && d->cache, "paged_copy: null operand");
    MMF_CHECK_ARG(d->rows > 0 && d->planes > 0 && d->planes <= 65535 && d->pages > 0 && d->kv_heads > 0 && d->head_dim > 0, "paged_copy: bad shape");
    MMF_CHECK_ARG(d->page_size >= 1 && d->page_size <= MMF_PAGE_MAX && (int64_t)d->kv_heads * d->page_size * d->head_dim <= 0x3fffffff, "paged_copy: bad page");
    const int es = d->is_f32 ? 4 : 2, unit = 16 / es;
    const bool wide = aligned16(d->cache) && d->head_dim % unit == 0 && d->plane_stride % unit == 0 && d->page_stride % unit == 0 && d->head_stride % unit == 0 &&
                      d->pos_stride % unit == 0;
    const dim3 grid(d->rows, d->planes);
    page_kernels_used();
    if (wide) hipLaunchKernelGGL(copy_pages_kernel<uint4>, grid, dim3(256), 0, (hipStream_t)stream, *d, es);
    else if (es == 4) hipLaunchKernelGGL(copy_pages_kernel<uint32_t>, grid, dim3(256), 0, (hipStream_t)stream, *d, es);
    else hipLaunchKernelGGL(copy_pages_kernel<uint16_t>, grid, dim3(256), 0, (hipStream_t)stream, *d, es);
    MMF_CHECK_LAUNCH();
    return 0;
}

}  // extern "C"
