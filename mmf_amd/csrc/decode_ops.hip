// mmf_amd :: decoding with a paged key / value cache and several beams per request — everything around the attention
// (paged_attention.hip): the plan of a step (pages and slots from lengths), the write of new keys and values, the selection of
// the best continuations, and the block tables after it.  M4C's decoding loop (mmf/models/m4c.py:284-304) is greedy and re-runs the
// whole transformer per step; mmf/utils/text.py's BeamSearch keeps its beams on the host.
#include "common.h"
#include "mmf_amd.h"
#include "paged_common.h"

namespace {

constexpr int PLAN_THREADS = 1024;

// inclusive sum over the workgroup's PLAN_THREADS threads; `total` gets the sum of all
template <typename T> DEVI T block_scan(T v, int64_t* lds, T& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    T s = v;
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const T t = __shfl_up(s, o, 64);
        if (lane >= o) s += t;
    }
    __syncthreads();
    if (lane == 63) lds[wave] = s;
    __syncthreads();
    T before = 0;
    total = 0;
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / 64; ++w) {
        const T x = (T)lds[w];
        if (w < wave) before += x;
        total += x;
    }
    return s + before;
}

// ------------------------------------------------------------------------------------------------
// the plan of a step.  Whole numbers only; a few bytes per request and 12 per new token: latency is all there is to it.
// ------------------------------------------------------------------------------------------------
struct PlanGroup {      // what the scan leaves for the rows of a group
    int base;           // pages taken by the groups before it
    int forks;          // bit w: beam w takes a page for the block it shares so far
    int kv;             // tokens in the cache before this step
    int granted;        // new tokens, -1: none (released, refused)
};

DEVI int blocks_of(int tokens, int page_size) { return (int)(((int64_t)tokens + page_size - 1) / page_size); }

// pages of released groups, back on the stack in the order of their rows and blocks; returns the new top
DEVI int plan_release(const mmf_paged_plan_desc& d, int64_t* lds) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int R = d.groups * d.beams;
    int top = d.free_top[0];
    top = min(max(top, 0), d.free_capacity);
    if (threadIdx.x == 0 && top != d.free_top[0]) flag_page_error();
    for (int r0 = 0; r0 < R; r0 += PLAN_THREADS / 64) {          // one wave per row: count, place, push
        const int r = r0 + wave;
        int n = 0, blocks = 0;
        if (r < R && d.q_lens[r / d.beams] < 0) {
            blocks = min(blocks_of(max(d.kv_lens[r / d.beams], 0), d.page_size), d.blocks);
            for (int j0 = 0; j0 < blocks; j0 += 64) n += __popcll(__ballot(j0 + lane < blocks && d.owned[(size_t)r * d.blocks + j0 + lane] >= 0));
        }
        __syncthreads();
        if (lane == 0) lds[wave] = n;
        __syncthreads();
        int at = top, total = 0;
#pragma unroll
        for (int w = 0; w < PLAN_THREADS / 64; ++w) {
            const int x = (int)lds[w];
            if (w < wave) at += x;
            total += x;
        }
        for (int j0 = 0; j0 < blocks && n > 0; j0 += 64) {
            const int p = j0 + lane < blocks ? d.owned[(size_t)r * d.blocks + j0 + lane] : -1;
            const uint64_t m = __ballot(p >= 0);
            const int to = at + __popcll(m & ((1ull << lane) - 1));
            if (p >= 0) {
                if (to < d.free_capacity) d.free_pages[to] = p;
                else flag_page_error();                          // more pages came back than the pool has: a page was given back twice
            }
            at += __popcll(m);
        }
        top = min(top + total, d.free_capacity);
    }
    return top;
}

// the tokens and blocks of one row, by `nthr` threads
DEVI void plan_row(const mmf_paged_plan_desc& d, const PlanGroup& g, int r, int start, int top, int tid, int nthr) {
    const int w = r % d.beams, ps = d.page_size;
    const bool first = w == 0;
    if (g.granted > 0) {
        const int have = blocks_of(g.kv, ps), want = blocks_of(g.kv + g.granted, ps);
        const bool fork = (g.forks >> w) & 1;
        const int lo = fork ? g.kv / ps : have;
        int rank = g.base;                                        // the row's first page, counted from the top of the stack
        if (!d.shared) rank += w * (want - have) + __popc(g.forks & ((1u << w) - 1u));
        int* table = d.tables + (size_t)r * d.blocks;
        int* owned = d.owned + (size_t)r * d.blocks;
        for (int j = lo + tid; j < want; j += nthr) {
            const int page = d.free_pages[top - 1 - (rank + j - lo)];
            if (fork && j == lo) { d.copies[3 * r] = table[j]; d.copies[3 * r + 1] = page; d.copies[3 * r + 2] = g.kv % ps; }
            table[j] = page;
            owned[j] = (!d.shared || first) ? page : -1;          // a shared block belongs to the group's first row
        }
        if (!d.shared || first) {
            for (int i = tid; i < g.granted; i += nthr) {
                const int pos = g.kv + i, j = pos / ps;
                const int page = j >= lo ? d.free_pages[top - 1 - (rank + j - lo)] : table[j];
                d.slots[start + i] = page < 0 ? -1 : (int64_t)page * ps + (pos - j * ps);
                d.positions[start + i] = pos;
            }
        }
    } else if (!d.shared || first) {                              // the tokens of a request that has to wait
        const int n = min(-1 - g.granted, d.rows - start);
        for (int i = tid; i < n; i += nthr) { d.slots[start + i] = -1; d.positions[start + i] = -1; }
    }
}

__global__ __launch_bounds__(PLAN_THREADS) void plan_kernel(mmf_paged_plan_desc d) {
    __shared__ int64_t lds[PLAN_THREADS / 64];
    const int tid = threadIdx.x, W = d.beams, ps = d.page_size, per = d.shared ? 1 : W;
    PlanGroup* ws = reinterpret_cast<PlanGroup*>(d.ws);
    const int top = plan_release(d, lds);
    int carry_need = 0, carry_refused = 0, carry_taken = 0, total;
    int64_t carry_rows = 0, total_rows;
    for (int g0 = 0; g0 < d.groups; g0 += PLAN_THREADS) {
        const int g = g0 + tid;
        const bool in = g < d.groups;
        const int q = in ? d.q_lens[g] : 0, kv = in ? max(d.kv_lens[g], 0) : 0, n = max(q, 0);
        const int64_t rows = (int64_t)per * n, start64 = carry_rows + block_scan(rows, lds, total_rows) - rows;
        carry_rows += total_rows;
        const bool fits = (int64_t)kv + n <= (int64_t)d.blocks * ps && start64 + rows <= d.rows;
        int need = 0, forks = 0;
        if (in && n > 0 && fits) {
            const int fresh = blocks_of(kv + n, ps) - blocks_of(kv, ps);
            if (!d.shared && kv % ps != 0)
                for (int w = 1; w < W; ++w)
                    if (d.owned[((size_t)g * W + w) * d.blocks + kv / ps] < 0) forks |= 1 << w;
            need = per * fresh + __popc(forks);
        }
        const int upto = carry_need + block_scan(need, lds, total);
        carry_need += total;
        const bool served = in && q >= 0 && fits && (need == 0 || upto <= top);
        if (in) {
            d.granted[g] = served ? n : 0;
            d.kv_out[g] = q < 0 ? 0 : kv + (served ? n : 0);
            ws[g] = PlanGroup{upto - need, served ? forks : 0, kv, served ? n : -1 - n};
            for (int w = 0; w < per; ++w) d.q_start[(size_t)g * per + w] = (int)min(start64 + (int64_t)w * n, (int64_t)d.rows);
        }
        block_scan(served ? need : 0, lds, total);
        carry_taken += total;
        block_scan((int)(in && q >= 0 && !served), lds, total);
        carry_refused += total;
    }
    if (tid == 0) {
        d.top_out[0] = top - carry_taken;
        d.refused[0] = carry_refused;
    }
    for (int i = tid; i < 3 * d.groups * W; i += PLAN_THREADS) d.copies[i] = -1;
    for (int64_t i = carry_rows + tid; i < d.rows; i += PLAN_THREADS) { d.slots[i] = -1; d.positions[i] = -1; }
    __syncthreads();
    const int lane = tid & 63;
    for (int r = tid >> 6; r < d.groups * W; r += PLAN_THREADS / 64) {
        const int g = r / W;
        plan_row(d, ws[g], r, d.shared ? d.q_start[g] : d.q_start[r], top, lane, 64);
    }
}

// ------------------------------------------------------------------------------------------------
// new keys and values into their slots.  Every byte moves once each way; a thread moves one VT (16 bytes, or one element
// where a row does not start on 16 bytes).
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
// ------------------------------------------------------------------------------------------------
constexpr double NEG_INF = -__builtin_huge_val();

struct Cand { double v; int64_t i; };
DEVI bool better(double av, int64_t ai, double bv, int64_t bi) { return av > bv || (av == bv && ai < bi); }

template <typename T> DEVI float logit(const T* x, int64_t v) {
    const float f = (float)x[v];
    return f == f ? f : -INFINITY;
}

template <typename T>
__global__ __launch_bounds__(256) void beam_select_kernel(mmf_beam_select_desc d) {
    __shared__ double red_v[4], lse[MMF_BEAMS_MAX], score[MMF_BEAMS_MAX];
    __shared__ int64_t red_i[4], token[MMF_BEAMS_MAX];
    __shared__ int parent[MMF_BEAMS_MAX], done[MMF_BEAMS_MAX];
    const int g = blockIdx.x, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, W = d.beams;
    const int64_t V = d.vocab;
    if (tid < W) {                                                // (scores and finished may be updated in place)
        score[tid] = (double)d.scores[g * W + tid];
        done[tid] = d.finished[g * W + tid] != 0;
    }
    for (int w = 0; w < W; ++w) {
        const T* x = (const T*)d.logits + ((size_t)g * W + w) * d.ld;
        float m = -INFINITY;
        for (int64_t v = tid; v < V; v += 256) m = fmaxf(m, logit(x, v));
        m = wave_max(m);
        __syncthreads();
        if (lane == 0) red_v[wave] = m;
        __syncthreads();
        m = (float)fmax(fmax(red_v[0], red_v[1]), fmax(red_v[2], red_v[3]));
        double s = 0.0;
        if (m > -INFINITY)
            for (int64_t v = tid; v < V; v += 256) s += (double)expf(logit(x, v) - m);
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
        __syncthreads();
        if (lane == 0) red_v[wave] = s;
        __syncthreads();
        if (tid == 0) lse[w] = (double)m + log(red_v[0] + red_v[1] + red_v[2] + red_v[3]);
    }
    __syncthreads();
    double last_v = -NEG_INF;
    int64_t last_i = -1;
    for (int k = 0; k < W; ++k) {                                 // the best candidate behind the last one chosen
        double bv = NEG_INF;
        int64_t bi = INT64_MAX;
        for (int w = 0; w < W; ++w) {
            const T* x = (const T*)d.logits + ((size_t)g * W + w) * d.ld;
            for (int64_t v = tid; v < V; v += 256) {
                double c = done[w] ? (v == d.eos ? score[w] : NEG_INF) : score[w] + ((double)logit(x, v) - lse[w]);
                if (!(c == c)) c = NEG_INF;
                const int64_t i = w * V + v;
                if (better(last_v, last_i, c, i) && better(c, i, bv, bi)) { bv = c; bi = i; }
            }
        }
#pragma unroll
        for (int o = 32; o > 0; o >>= 1) {
            const double ov = __shfl_xor(bv, o, 64);
            const int64_t oi = __shfl_xor((long long)bi, o, 64);
            if (better(ov, oi, bv, bi)) { bv = ov; bi = oi; }
        }
        __syncthreads();
        if (lane == 0) { red_v[wave] = bv; red_i[wave] = bi; }
        __syncthreads();
        for (int u = 0; u < 4; ++u)
            if (u == 0 || better(red_v[u], red_i[u], bv, bi)) { bv = red_v[u]; bi = red_i[u]; }
        last_v = bv;
        last_i = bi;
        if (tid == 0) {
            const int p = (int)(bi / V);
            parent[k] = p;
            token[k] = bi - (int64_t)p * V;
            d.scores_out[g * W + k] = (float)bv;
            d.parents[g * W + k] = p;
            d.tokens[g * W + k] = token[k];
        }
    }
    __syncthreads();
    if (tid < W) d.finished_out[g * W + tid] = done[parent[tid]] || token[tid] == d.eos;
    if (d.history)
        for (int64_t t = tid; t < d.length; t += 256) {           // a column at a time: in place as well
            int64_t h[MMF_BEAMS_MAX];
            for (int w = 0; w < W; ++w) h[w] = t == d.step ? token[w] : d.history[((size_t)g * W + parent[w]) * d.length + t];
            for (int w = 0; w < W; ++w) d.history_out[((size_t)g * W + w) * d.length + t] = h[w];
        }
}

// ------------------------------------------------------------------------------------------------
// block tables after a selection.  A block that is full is only read from here on: the children share it.  The block that goes on being
// written has to be each beam's own: the first child of a beam keeps its page, the other children take the pages of the beams that have
// no child, of which there are exactly as many, and get its tokens copied.  A page that is copied from is never copied to.
// ------------------------------------------------------------------------------------------------
__global__ __launch_bounds__(256) void reorder_tables_kernel(mmf_paged_reorder_desc d) {
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
    const int kv = max(d.kv_lens[g], 0), part = kv % d.page_size ? kv / d.page_size : -1;
    for (int j = tid; j < d.blocks; j += 256) {                   // a column at a time: in place as well
        int t[MMF_BEAMS_MAX];
        for (int w = 0; w < W; ++w) t[w] = d.tables[((size_t)g * W + w) * d.blocks + j];
        for (int w = 0; w < W; ++w) d.tables_out[((size_t)g * W + w) * d.blocks + j] = t[j == part ? source[w] : parent[w]];
        if (j == part)
            for (int w = 0; w < W; ++w) {
                const bool copy = source[w] != parent[w];
                int* c = d.copies + 3 * ((size_t)g * W + w);
                c[0] = copy ? t[parent[w]] : -1;
                c[1] = copy ? t[source[w]] : -1;
                c[2] = copy ? kv % d.page_size : -1;
            }
    }
    if ((part < 0 || part >= d.blocks) && tid < 3 * W) d.copies[3 * (size_t)g * W + tid] = -1;
}

// the first copies[r][2] tokens of page copies[r][0] to page copies[r][1], in every plane (keys and values of every layer)
template <typename VT>
__global__ __launch_bounds__(256) void copy_pages_kernel(mmf_paged_copy_desc d, int esize) {
    const int r = blockIdx.x;
    const int src = d.copies[3 * (size_t)r], dst = d.copies[3 * (size_t)r + 1], tokens = min(d.copies[3 * (size_t)r + 2], d.page_size);
    if (src == dst || src < 0 || dst < 0 || tokens <= 0) return;
    if (src >= d.pages || dst >= d.pages) {
        if (threadIdx.x == 0 && blockIdx.y == 0) flag_page_error();
        return;
    }
    const int per_pos = d.head_dim * esize / (int)sizeof(VT), n = d.kv_heads * tokens * per_pos;
    char* base = (char*)d.cache + blockIdx.y * d.plane_stride * esize;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int h = i / (tokens * per_pos), k = i - h * tokens * per_pos, pos = k / per_pos, e = (k - pos * per_pos) * (int)sizeof(VT);
        const int64_t off = (h * d.head_stride + pos * d.pos_stride) * esize + e;
        *reinterpret_cast<VT*>(base + dst * d.page_stride * esize + off) = *reinterpret_cast<const VT*>(base + src * d.page_stride * esize + off);
    }
}

bool aligned16(const void* p) { return (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

}  // namespace

extern "C" {

int mmf_decode_take_error(void) {
    int v = 0;
    if (hipMemcpyFromSymbol(&v, HIP_SYMBOL(g_page_error), sizeof(int)) != hipSuccess) { mmf_amd_set_error("take_index_error: copy failed"); return -1; }
    if (v) { const int z = 0; (void)hipMemcpyToSymbol(HIP_SYMBOL(g_page_error), &z, sizeof(int)); }
    return v;
}

int64_t mmf_paged_plan_ws_bytes(int groups) { return (int64_t)(groups > 0 ? groups : 0) * (int64_t)sizeof(PlanGroup) + 16; }

int mmf_paged_plan(const mmf_paged_plan_desc* d, void* stream) {
    MMF_CHECK_ARG(d && d->q_lens && d->kv_lens && d->tables && d->owned && d->free_pages && d->free_top, "paged_plan: null operand");
    MMF_CHECK_ARG(d->q_start && d->granted && d->kv_out && d->slots && d->positions && d->copies && d->top_out && d->refused && d->ws, "paged_plan: null output");
    MMF_CHECK_ARG(d->groups > 0 && d->blocks > 0 && d->rows > 0 && d->free_capacity > 0, "paged_plan: bad shape");
    MMF_CHECK_ARG(d->beams >= 1 && d->beams <= MMF_BEAMS_MAX && d->groups <= 0x3fffffff / d->beams, "paged_plan: 1 .. 32 beams");
    MMF_CHECK_ARG(d->page_size >= 1 && d->page_size <= MMF_PAGE_MAX && (d->page_size & (d->page_size - 1)) == 0, "paged_plan: page_size is a power of two up to 1024");
    MMF_CHECK_ARG((int64_t)d->blocks * d->page_size <= 0x3fffffff && d->rows <= 0x3fffffff, "paged_plan: more than 2^30 tokens");
    hipLaunchKernelGGL(plan_kernel, dim3(1), dim3(PLAN_THREADS), 0, (hipStream_t)stream, *d);
    MMF_CHECK_LAUNCH();
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
    if (wide) hipLaunchKernelGGL(paged_write_kernel<uint4>, grid, dim3(256), 0, (hipStream_t)stream, *d, es, (int)per_token);
    else if (es == 4) hipLaunchKernelGGL(paged_write_kernel<uint32_t>, grid, dim3(256), 0, (hipStream_t)stream, *d, es, (int)per_token);
    else hipLaunchKernelGGL(paged_write_kernel<uint16_t>, grid, dim3(256), 0, (hipStream_t)stream, *d, es, (int)per_token);
    MMF_CHECK_LAUNCH();
    return 0;
}

int64_t mmf_beam_select_ws_bytes(int groups, int beams, int64_t vocab) { (void)groups; (void)beams; (void)vocab; return 0; }

int mmf_beam_select(const mmf_beam_select_desc* d, void* stream) {
    MMF_CHECK_ARG(d && d->logits && d->scores && d->finished && d->scores_out && d->parents && d->tokens && d->finished_out, "beam_select: null operand");
    MMF_CHECK_ARG(d->groups > 0 && d->beams >= 1 && d->beams <= MMF_BEAMS_MAX && d->vocab > 0 && d->ld >= d->vocab, "beam_select: bad shape");
    MMF_CHECK_ARG(d->eos >= 0 && d->eos < d->vocab, "beam_select: the end token is not in the vocabulary");
    MMF_CHECK_ARG(!d->history || (d->history_out && d->length > 0 && d->step >= 0 && d->step < d->length), "beam_select: step is not a column of the history");
    if (d->is_f32) hipLaunchKernelGGL(beam_select_kernel<float>, dim3(d->groups), dim3(256), 0, (hipStream_t)stream, *d);
    else hipLaunchKernelGGL(beam_select_kernel<bf16>, dim3(d->groups), dim3(256), 0, (hipStream_t)stream, *d);
    MMF_CHECK_LAUNCH();
    return 0;
}

int mmf_paged_reorder(const mmf_paged_reorder_desc* d, void* stream) {
    MMF_CHECK_ARG(d && d->parents && d->kv_lens && d->tables && d->tables_out && d->copies, "paged_reorder: null operand");
    MMF_CHECK_ARG(d->groups > 0 && d->beams >= 1 && d->beams <= MMF_BEAMS_MAX && d->blocks > 0, "paged_reorder: bad shape");
    MMF_CHECK_ARG(d->page_size >= 1 && d->page_size <= MMF_PAGE_MAX, "paged_reorder: bad page_size");
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
    if (wide) hipLaunchKernelGGL(copy_pages_kernel<uint4>, grid, dim3(256), 0, (hipStream_t)stream, *d, es);
    else if (es == 4) hipLaunchKernelGGL(copy_pages_kernel<uint32_t>, grid, dim3(256), 0, (hipStream_t)stream, *d, es);
    else hipLaunchKernelGGL(copy_pages_kernel<uint16_t>, grid, dim3(256), 0, (hipStream_t)stream, *d, es);
    MMF_CHECK_LAUNCH();
    return 0;
}

}  // extern "C"
