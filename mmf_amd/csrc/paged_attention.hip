// mmf_amd :: attention of new tokens over the pages of their request (mmf_paged_attention).
//   out[i] = sum_j softmax_j(scale * q[i] . k[j]) v[j]
// One pass over the keys with the running maximum m and sum l of the softmax: a block of scores s moves them to
//   m' = max(m, max s),  l' = l exp(m - m') + sum exp(s - m'),  o' = o exp(m - m') + exp(s - m') v,   out = o / l at the end.
#include "common.h"
#include "mmf_amd.h"
#include "paged_common.h"

namespace {

// One wave per (new token, query head): a lane takes one of 64 keys for the scores, and D / 64 columns of the sum.
template <typename T, int D>
__global__ __launch_bounds__(256) void paged_attn_wave_kernel(mmf_paged_attn_desc d) {
    constexpr int C = D / 64;
    const int lane = threadIdx.x & 63;
    const int64_t unit = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int h = (int)(unit % d.heads);
    const int64_t ri = unit / d.heads;
    const int r = (int)(ri / d.max_q), i = (int)(ri - (int64_t)r * d.max_q);
    if (r >= d.requests) return;
    const int kv = min(max(d.kv_lens[r / d.beams], 0), d.blocks * d.page_size), n = d.q_lens[r / d.beams];
    if (i == 0 && lane == 0 && (n > d.max_q || kv != d.kv_lens[r / d.beams])) flag_page_error();
    if (i >= n) return;
    const int64_t row = (int64_t)d.q_start[r] + i;
    if (row < 0 || row >= d.tokens) { flag_page_error(); return; }
    const T* q = (const T*)d.q + row * d.q_row + h * d.q_head;
    const int hk = h / (d.heads / d.kv_heads);
    const int end = d.causal ? min(kv, kv - n + i + 1) : kv;
    const int32_t* table = d.tables + r * d.table_row;
    float m = -INFINITY, l = 0.f, o[C];
#pragma unroll
    for (int c = 0; c < C; ++c) o[c] = 0.f;
    for (int j0 = 0; j0 < end; j0 += 64) {
        const int j = j0 + lane;
        int page = j < end ? table[j / d.page_size] : -1;
        if (j < end && (page < 0 || page >= d.pages)) { flag_page_error(); page = -1; }
        const int64_t off = (int64_t)page * d.page_stride + hk * d.head_stride + (int64_t)(j % d.page_size) * d.pos_stride;
        float s = -INFINITY;
        if (page >= 0) {
            const T* k = (const T*)d.k_cache + off;
            s = 0.f;
            for (int e = 0; e < D; ++e) s += (float)q[e] * (float)k[e];
            s *= d.scale;
        }
        const float m1 = fmaxf(m, wave_max(s)), mm = m1 == -INFINITY ? 0.f : m1;
        const float a = __expf(m - mm), p = __expf(s - mm);
        l = l * a + wave_sum(p);
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] *= a;
        for (int k = 0; k < 64 && j0 + k < end; ++k) {
            const float pk = __shfl(p, k, 64);
            const int64_t ok = __shfl((long long)off, k, 64);
            if (__shfl(page, k, 64) < 0) continue;
            const T* v = (const T*)d.v_cache + ok;
#pragma unroll
            for (int c = 0; c < C; ++c) o[c] += pk * (float)v[c * 64 + lane];
        }
        m = m1;
    }
    T* out = (T*)d.out + row * d.out_row + h * d.out_head;
#pragma unroll
    for (int c = 0; c < C; ++c) out[c * 64 + lane] = (T)(l > 0.f ? o[c] / l : 0.f);
}

}  // namespace

extern "C" {

int mmf_paged_attention_take_error(void) {
    int v = 0;
    if (hipMemcpyFromSymbol(&v, HIP_SYMBOL(g_page_error), sizeof(int)) != hipSuccess) { mmf_amd_set_error("take_index_error: copy failed"); return -1; }
    if (v) { const int z = 0; (void)hipMemcpyToSymbol(HIP_SYMBOL(g_page_error), &z, sizeof(int)); }
    return v;
}

int64_t mmf_paged_attention_ws_bytes(const mmf_paged_attn_desc* d) { (void)d; return 0; }

int mmf_paged_attention(const mmf_paged_attn_desc* d, void* stream) {
    MMF_CHECK_ARG(d && d->q && d->k_cache && d->v_cache && d->tables && d->kv_lens && d->q_start && d->q_lens && d->out, "paged_attention: null operand");
    MMF_CHECK_ARG(d->head_dim == 64 || d->head_dim == 128, "paged_attention: head_dim is 64 or 128");
    MMF_CHECK_ARG(d->heads > 0 && d->kv_heads > 0 && d->heads % d->kv_heads == 0, "paged_attention: heads is a multiple of kv_heads");
    MMF_CHECK_ARG(d->requests > 0 && d->beams >= 1 && d->beams <= MMF_BEAMS_MAX && d->blocks > 0 && d->pages > 0 && d->tokens >= 0, "paged_attention: bad shape");
    MMF_CHECK_ARG(d->page_size >= 1 && d->page_size <= MMF_PAGE_MAX && (d->page_size & (d->page_size - 1)) == 0, "paged_attention: page_size is a power of two up to 1024");
    MMF_CHECK_ARG((int64_t)d->blocks * d->page_size <= 0x3fffffff, "paged_attention: more than 2^30 keys");
    MMF_CHECK_ARG(d->max_q >= 1, "paged_attention: max_q is at least 1");
    if (d->tokens == 0) return 0;
    const int64_t units = (int64_t)d->requests * d->max_q * d->heads, blocks = (units + 3) / 4;
    MMF_CHECK_ARG(blocks <= 0x7fffffff, "paged_attention: too many rows for one call");
    const dim3 grid((unsigned)blocks);
    if (d->is_f32 && d->head_dim == 64) hipLaunchKernelGGL((paged_attn_wave_kernel<float, 64>), grid, dim3(256), 0, (hipStream_t)stream, *d);
    else if (d->is_f32) hipLaunchKernelGGL((paged_attn_wave_kernel<float, 128>), grid, dim3(256), 0, (hipStream_t)stream, *d);
    else if (d->head_dim == 64) hipLaunchKernelGGL((paged_attn_wave_kernel<bf16, 64>), grid, dim3(256), 0, (hipStream_t)stream, *d);
    else hipLaunchKernelGGL((paged_attn_wave_kernel<bf16, 128>), grid, dim3(256), 0, (hipStream_t)stream, *d);
    MMF_CHECK_LAUNCH();
    return 0;
}

}  // extern "C"
