// mmf_amd :: attention of new tokens over the pages of their request (mmf_paged_attention).
//   out[i] = sum_j softmax_j(scale * q[i] . k[j]) v[j]
// One pass over the keys with the running maximum m and sum l of the softmax: a tile of scores s moves them to
//   m' = max(m, max s),  l' = l exp(m - m') + sum exp(s - m'),  o' = o exp(m - m') + exp(s - m') v,   out = o / l at the end.
//
// The rows of a product are (new token, query head) pairs that read one key head, 32 to a wave: with q the column of S^T = K Q^T a lane holds one row's
// scores (16 keys of every 32; lane ^ 32 the others), so maximum and sum need one exchange, and the probabilities are in the register order that the second
// product O^T = V^T P^T takes (v_mfma_f32_32x32x16_bf16, or v_mfma_f32_32x32x2_f32 for the fp32 pool, whose operands are one row element per lane).
//
//   chunks (more than 32 rows per request and key head): a workgroup takes 128 rows (fp32: 64), its waves share the staged K and V tiles;
//   steps  (at most 32 rows):                           a workgroup takes all beams of a group that fit 32 rows, its four waves take different tiles.
//
// Keys are split over workgroups in runs of equal length for all requests, chosen on the device from the actual lengths (Plan below); runs are joined by a
// second kernel, launched only where a request can be split at all.
//
// What bounds it, and what it measured (MI355X; a copy of 1 GiB reaches 5.18 TB/s, a bf16 product of 8192^3 1262 TFLOP/s, an fp32 one of 4096^3 139):
//   long caches   8 requests of 16384 .. 65536 keys, 32 heads on 8, head_dim 128, one token: 191 us, 5.3 TB/s of pages.  Memory.
//   steps         32 groups of 5 beams, 120 .. 181 keys of which the prompt's pages are shared, 12 heads of 64: 11.9 us for 21.5 MB.  The chain lengths, table,
//                 first tile, four tiles, meeting of the waves; with every beam reading the shared pages itself 25.3 us.  The fp32 pool: 27.3 us for 43 MB.
//   fp32 tokens   8 requests of 2048 .. 8192 keys, 32 heads on 8, one token: 110.8 us at head_dim 128 (2.3 TB/s), 51.5 at 64 (2.5).  A tile's load waits for the score
//                 products of the one before, and a product takes 32 rows where 4 are the request's.
//   chunks        270 GFLOP over caches, 32 heads on 8, head_dim 128: 333 us, 808 TFLOP/s (340 on another card), 15 of it to join runs.  Products (512 cycles per 32
//                 keys of a wave) and vector instructions (545) of the two waves that a SIMD holds: the matrix units are busy in 37 % of the cycles, vector instructions
//                 issue in 44 %.  Of 340 us, copies without exponentials took 320, without staging 293, without barriers too 280.  At head_dim 64 (135 GFLOP) 194 us,
//                 694 TFLOP/s; 32 prompts of 70 .. 170 tokens, 12 heads of 64, not causal: 15.2 us.
//   fp32 prompts  the same 32 prompts: 35.6 us.  The products of the longest prompts (3.5 us per 32 keys for two waves on a SIMD) behind 10 us
//                 of lengths, plan, queries, first tile and output.
#include "common.h"
#include "mmf_amd.h"
#include "paged_common.h"
#include <atomic>

namespace {

typedef __attribute__((address_space(3))) void* lds_vp;
typedef const __attribute__((address_space(1))) void* glb_vp;
static __device__ uint4 g_zero16;

constexpr int STEP_ROWS = 32;
// Rows of a chunk's workgroup, a wave per 32.  fp32 is bound by its products and not by what it stages: fewer waves without rows at the end of a prompt count for more
// (32 prompts of 70 .. 170 tokens, 12 heads of 64: 36.9 us with 128 rows, 35.6 with 64; bf16 reads every tile twice as often with 64).
template <typename T> constexpr int chunk_rows = sizeof(T) == 2 ? 128 : 64;
constexpr int UNITS_MAX = 960;         // requests (chunks) or groups of beams (steps) per launch
constexpr int PREFIX_MAX = 4 * (UNITS_MAX + 1) * 4;

struct Args {
    mmf_paged_attn_desc d;
    int page_shift, group;             // group: query heads per key head
    int units, nb, per_group;          // nb: beams a unit takes together (steps), per_group: units per group of beams
    int target, run_min;               // workgroups to aim at when keys are split; shortest run
    int parts;                         // partial results that the workspace has room for
    int split;                         // whether keys may be split at all
    float c;                           // |scale| log2 e (1 when scale is 0)
    uint32_t q_and, q_xor;             // the scale's sign on the queries' bits: their sign bits turned over (scale < 0), all bits cleared (scale 0)
};

// ---- LDS image of rows of RB bytes, 16-byte chunks XOR-swizzled so that 16 rows at one chunk, and 4 rows x 4 chunks, meet no bank twice ----
template <int RB> DEVI int swz(int row) { return RB == 128 ? (row >> 1) & 7 : ((row & 3) << 2) | ((row >> 2) & 3); }
template <int RB> DEVI int at(int row, int chunk) { return row * RB + ((chunk ^ swz<RB>(row)) << 4); }

// Keys key0 .. + ROWS into K and V images by LDS-DMA; keys >= end, and keys on pages outside the pool, come as zeros.  `page` holds, in lane l, the page of
// key0 + (l % ROWS).  NW waves share the tile, ROWS / NW rows in a row each.  Chunks, where these lie in one page (a tile starts on a page, or ROWS divide the page and
// the tile's start): the wave reads them through a buffer descriptor that ends behind the last of them, and all that a lane adds to it is its place among them, the same
// for every tile.  Otherwise every lane has an address of its own; in steps too, whose few tiles wait for the first bytes and not for the instructions before them (32
// groups of 5 beams: 11.9 us, and 12.5 by descriptors; 270 GFLOP of chunks: 350 us, and 340 by descriptors).
template <typename T, int D, int ROWS, int NW> struct Stager {
    static constexpr int RB = D * (int)sizeof(T), CPR = RB / 16, RPI = 64 / CPR, OWN = ROWS / NW, N = OWN / RPI;
    uint32_t offset[N];                // of a row's 16 bytes, in its page or among the wave's rows
    uint64_t head;                     // page 0 of the head
    int64_t to_v;
    uint32_t page_bytes, pos_bytes;
    DEVI static bool one_page(const Args& a) { return NW > 1 && a.d.page_size >= OWN; }
    DEVI Stager(const Args& a, int64_t head_off, int wave, int lane) {
        page_bytes = (uint32_t)(a.d.page_stride * (int)sizeof(T));
        pos_bytes = (uint32_t)(a.d.pos_stride * (int)sizeof(T));
        to_v = (const char*)a.d.v_cache - (const char*)a.d.k_cache;
        head = (uint64_t)a.d.k_cache + (uint64_t)head_off * sizeof(T);
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int mine = i * RPI + lane / CPR, row = wave * OWN + mine;
            offset[i] = (one_page(a) ? mine : row & (a.d.page_size - 1)) * pos_bytes + ((lane % CPR) ^ swz<RB>(row)) * 16;
        }
    }
    DEVI void operator()(const Args& a, int key0, int end, int page, unsigned char* k_img, unsigned char* v_img, int wave, int lane) const {
        const bool in = key0 + (lane & (ROWS - 1)) < end, ok = in && (unsigned)page < (unsigned)a.d.pages;
        if (in != ok) flag_page_error();
        if (one_page(a)) {
            const int key = __builtin_amdgcn_readfirstlane(key0) + wave * OWN, left = __builtin_amdgcn_readfirstlane(end) - key, p = __builtin_amdgcn_readlane(page, wave * OWN);
            const int bytes = left > 0 && (unsigned)p < (unsigned)a.d.pages ? (min(left, OWN) - 1) * (int)pos_bytes + RB : 0;
            const uint64_t k = head + (uint64_t)(uint32_t)p * page_bytes + (uint32_t)(key & (a.d.page_size - 1)) * pos_bytes;
            const auto rk = __builtin_amdgcn_make_buffer_rsrc((void*)k, 0, bytes, 0x00020000), rv = __builtin_amdgcn_make_buffer_rsrc((void*)(k + to_v), 0, bytes, 0x00020000);
#pragma unroll
            for (int i = 0; i < N; ++i) {
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rk, (lds_vp)(k_img + (wave * OWN + i * RPI) * RB), 16, offset[i], 0, 0, 0);
                __builtin_amdgcn_raw_ptr_buffer_load_lds(rv, (lds_vp)(v_img + (wave * OWN + i * RPI) * RB), 16, offset[i], 0, 0, 0);
            }
            return;
        }
        const int use = ok ? page : -1;
        const uint64_t tile = head + (uint32_t)(key0 & (a.d.page_size - 1)) * pos_bytes, zero = (uint64_t)&g_zero16;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const int row = wave * OWN + i * RPI, p = __shfl(use, row + lane / CPR, 64);
            const uint64_t k = (uint64_t)(uint32_t)p * page_bytes + tile + offset[i];
            const uint64_t kk = p >= 0 ? k : zero, vv = p >= 0 ? k + to_v : zero;
            __builtin_amdgcn_global_load_lds((glb_vp)kk, (lds_vp)(k_img + row * RB), 16, 0, 0);
            __builtin_amdgcn_global_load_lds((glb_vp)vv, (lds_vp)(v_img + row * RB), 16, 0, 0);
        }
    }
};
// The page of key key0 + l % ROWS, for lane l (behind the end: any).  No branch: the value is first looked at a tile later, and may not be waited for before.
template <int ROWS> DEVI int page_of(const Args& a, const int32_t* table, int key0, int end, int lane) {
    return table[max(min(key0 + (lane & (ROWS - 1)), end - 1), 0) >> a.page_shift];
}

// ---- the rows of a wave: their queries, and the operands of a tile of 32 keys as the two products take them ----
// A tile's operands are all read before the first product that needs them: keys, then the score products; values, which land while the softmax is worked out, then
// the products that add them up.  Left to itself the compiler reads each operand right before its product, and waits for LDS 32 times a tile.
//
// A key that a row does not see adds 0 * v to it, which is 0 unless v is an infinity or no number.  Where the rows of a tile see different keys its values are looked
// through for those; zeros take their place, and once all tiles are added up they are added to the rows that see them, from the cache (add_odd).
DEVI int key_of(int r, int lane) { return 8 * (r >> 2) + 4 * (lane >> 5) + (r & 3); }        // the key of a lane's score r

template <typename T, int D> struct Operands;
template <typename T, int D> struct Rows;

template <int D> struct Operands<bf16, D> {
    bf16x8 k[D / 16], v[2][D / 32];
    DEVI void read_k(const unsigned char* img, int lane) {
#pragma unroll
        for (int u = 0; u < D / 16; ++u) k[u] = *reinterpret_cast<const bf16x8*>(img + at<2 * D>(lane & 31, 2 * u + (lane >> 5)));
    }
    // V^T by ds_read_b64_tr_b16 (16 lanes read 4 rows x 16 columns, lane i gets column i): step u takes keys 16 u .. + 16 in the order that a lane holds their scores.
    DEVI void read_v(const unsigned char* img, int lane) {
        typedef s16x4 __attribute__((address_space(3))) * lds_p;
        typedef short s16x8 __attribute__((ext_vector_type(8)));
        const int g = lane >> 4, i = lane & 15;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int t = 0; t < D / 32; ++t) {
                const int row = 16 * u + 4 * (g >> 1) + (i >> 2), col = 32 * t + 16 * (g & 1) + (i & 3) * 4;
                const s16x4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(img + at<2 * D>(row, col >> 3) + (col & 7) * 2));
                const s16x4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(img + at<2 * D>(row + 8, col >> 3) + (col & 7) * 2));
                const s16x8 x = {lo[0], lo[1], lo[2], lo[3], hi[0], hi[1], hi[2], hi[3]};
                v[u][t] = __builtin_bit_cast(bf16x8, x);
            }
    }
    DEVI bool odd() const {
        typedef uint16_t u16x2 __attribute__((ext_vector_type(2)));
        u16x2 most = 0;
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int t = 0; t < D / 32; ++t)
#pragma unroll
                for (int e = 0; e < 4; ++e) most = __builtin_elementwise_max(most, __builtin_bit_cast(u16x2, __builtin_bit_cast(u32x4, v[u][t])[e] & 0x7fff7fffu));
        return __ballot(most[0] >= 0x7f80 || most[1] >= 0x7f80) != 0;
    }
    DEVI void clear_odd() {
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int t = 0; t < D / 32; ++t) {
                u32x4 w = __builtin_bit_cast(u32x4, v[u][t]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if ((w[e] & 0x7f800000u) == 0x7f800000u) w[e] &= 0x0000ffffu;
                    if ((w[e] & 0x7f80u) == 0x7f80u) w[e] &= 0xffff0000u;
                }
                v[u][t] = __builtin_bit_cast(bf16x8, w);
                __builtin_amdgcn_sched_barrier(0);
            }
    }
};
template <int D> struct Rows<bf16, D> {
    bf16x8 q[D / 16];
    DEVI void load(const bf16* p, bool ok, const Args& a, int lane) {
#pragma unroll
        for (int s = 0; s < D / 16; ++s) {
            u32x4 x = {};
            if (ok) x = *reinterpret_cast<const u32x4*>(p + 16 * s + 8 * (lane >> 5));
            q[s] = __builtin_bit_cast(bf16x8, (x & a.q_and) ^ (a.q_xor | a.q_xor >> 16));
        }
    }
    DEVI void scores(const Operands<bf16, D>& x, f32x16& s) const {
#pragma unroll
        for (int u = 0; u < D / 16; ++u) s = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.k[u], q[u], s, 0, 0, 0);
    }
    // sums += V^T p.  p is rounded to bf16: relative 2^-8 of each, the pool's own precision.
    DEVI static void add(f32x16 (&o)[D / 32], const f32x16& p, const Operands<bf16, D>& x) {
        bf16x8 pb[2];
#pragma unroll
        for (int r = 0; r < 16; ++r) pb[r >> 3][r & 7] = (bf16)p[r];
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
            for (int t = 0; t < D / 32; ++t) o[t] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(x.v[u][t], pb[u], o[t], 0, 0, 0);
    }
};

// fp32: a step of v_mfma_f32_32x32x2_f32 takes one element per lane, lanes 0 - 31 of reduction slot 0 and lanes 32 - 63 of slot 1
template <int D> struct Operands<float, D> {
    f32x4 k[D / 8];                                                // element (t, e) of half h: column 8 t + 4 h + e
    float v[16][D / 32];                                           // step r: key_of(r), as a lane holds the scores
    DEVI void read_k(const unsigned char* img, int lane) {
#pragma unroll
        for (int t = 0; t < D / 8; ++t) k[t] = *reinterpret_cast<const f32x4*>(img + at<4 * D>(lane & 31, 2 * t + (lane >> 5)));
    }
    DEVI void read_v(const unsigned char* img, int lane) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int t = 0; t < D / 32; ++t) {
                const int col = 32 * t + (lane & 31);
                v[r][t] = *reinterpret_cast<const float*>(img + at<4 * D>(key_of(r, lane), col >> 2) + (col & 3) * 4);
            }
    }
    DEVI bool odd() const {
        float most = 0.f;
        bool none = false;
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int t = 0; t < D / 32; ++t) {
                none |= v[r][t] != v[r][t];
                most = fmaxf(most, fabsf(v[r][t]));
            }
        return __ballot(none || most == INFINITY) != 0;
    }
    DEVI void clear_odd() {
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int t = 0; t < D / 32; ++t) v[r][t] = fabsf(v[r][t]) < INFINITY ? v[r][t] : 0.f;
    }
};
template <int D> struct Rows<float, D> {
    f32x4 q[D / 8];
    DEVI void load(const float* p, bool ok, const Args& a, int lane) {
#pragma unroll
        for (int t = 0; t < D / 8; ++t) {
            u32x4 x = {};
            if (ok) x = *reinterpret_cast<const u32x4*>(p + 8 * t + 4 * (lane >> 5));
            q[t] = __builtin_bit_cast(f32x4, (x & a.q_and) ^ a.q_xor);
        }
    }
    DEVI void scores(const Operands<float, D>& x, f32x16& s) const {
#pragma unroll
        for (int t = 0; t < D / 8; ++t)
#pragma unroll
            for (int e = 0; e < 4; ++e) s = __builtin_amdgcn_mfma_f32_32x32x2f32(x.k[t][e], q[t][e], s, 0, 0, 0);
    }
    DEVI static void add(f32x16 (&o)[D / 32], const f32x16& p, const Operands<float, D>& x) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
#pragma unroll
            for (int t = 0; t < D / 32; ++t) o[t] = __builtin_amdgcn_mfma_f32_32x32x2f32(x.v[r][t], p[r], o[t], 0, 0, 0);
    }
};

// the values of one key that are infinite or no number, to the rows that see it
template <typename T, int D> DEVI void add_odd(const Args& a, f32x16 (&o)[D / 32], const int32_t* table, int h, int key, bool sees, int lane) {
    typedef T T4 __attribute__((ext_vector_type(4)));
    const int page = table[key >> a.page_shift];
    if ((unsigned)page >= (unsigned)a.d.pages) return;
    const T* v = (const T*)a.d.v_cache + page * a.d.page_stride + h * a.d.head_stride + (key & (a.d.page_size - 1)) * a.d.pos_stride + 4 * (lane >> 5);
#pragma unroll
    for (int t = 0; t < D / 32; ++t)
#pragma unroll
        for (int r = 0; r < 16; r += 4) {
            const T4 x = *reinterpret_cast<const T4*>(v + 32 * t + 2 * r);
#pragma unroll
            for (int e = 0; e < 4; ++e) o[t][r + e] += sees && !(fabsf((float)x[e]) < INFINITY) ? (float)x[e] : 0.f;
        }
}

// a value and that of lane ^ 32: v_permlane32_swap_b32 leaves the lower half's in one register and the upper half's in the other (the second copy is kept
// apart from the first: of two equal operands the compiler returns the first result for both)
DEVI void halves(float x, float& lower, float& upper) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    uint32_t v = u;
    asm("" : "+v"(v));
    const auto r = __builtin_amdgcn_permlane32_swap(u, v, false, false);
    lower = __builtin_bit_cast(float, (uint32_t)r[0]);
    upper = __builtin_bit_cast(float, (uint32_t)r[1]);
}
DEVI float max_halves(float x) { float a, b; halves(x, a, b); return fmaxf(a, b); }
DEVI float add_halves(float x) { float a, b; halves(x, a, b); return a + b; }
DEVI int wave_min(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v = min(v, __shfl_xor(v, o, 64));
    return __builtin_amdgcn_readfirstlane(v);
}

// One tile of 32 keys, key0 its first, for the rows of a wave; lim: keys this lane's row sees.  m (in units of log2) may lag up to 8 behind the largest score:
// a probability is then at most 2^8, and the sums need no rescaling on most tiles.
// `ahead` is called once the tile's operands are read: loads into LDS that are under way when the transposed values are read would be waited for first.
template <typename T, int D, typename F>
DEVI void tile_step(const Rows<T, D>& rows, const unsigned char* k, const unsigned char* v, int key0, int lim, bool masked, float c, float& m, float& l, f32x16 (&o)[D / 32],
                    int lane, bool& odd, F ahead) {
    f32x16 s = {};
    Operands<T, D> x;
    x.read_k(k, lane);
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);                                           // a wave at its products goes before one at its softmax
    rows.scores(x, s);
    __builtin_amdgcn_s_setprio(0);
    __builtin_amdgcn_sched_barrier(0);
    x.read_v(v, lane);
    __builtin_amdgcn_sched_barrier(0);
    ahead();
    __builtin_amdgcn_sched_barrier(0);
    float top = -INFINITY;
    if (masked) {
#pragma unroll
        for (int r = 0; r < 16; ++r)
            if (key0 + key_of(r, lane) >= lim) s[r] = -INFINITY;
        if (x.odd()) { x.clear_odd(); odd = true; }
    }
#pragma unroll
    for (int r = 0; r < 16; ++r) top = fmaxf(top, s[r]);
    top = max_halves(top) * c;
    if (__ballot(top > m + 8.f) != 0) {
        const float next = fmaxf(m, top), keep = next == -INFINITY ? 1.f : __builtin_amdgcn_exp2f(m - next);
        m = next;
        l *= keep;
#pragma unroll
        for (int t = 0; t < D / 32; ++t)
#pragma unroll
            for (int r = 0; r < 16; ++r) o[t][r] *= keep;
    }
    const float mm = m == -INFINITY ? 0.f : m;
    float sum = 0.f;
#pragma unroll
    for (int r = 0; r < 16; ++r) {
        s[r] = __builtin_amdgcn_exp2f(fmaf(s[r], c, -mm));
        sum += s[r];
    }
    l += sum;
    __builtin_amdgcn_s_setprio(1);
    Rows<T, D>::add(o, s, x);
    __builtin_amdgcn_s_setprio(0);
}

// ------------------------------------------------------------------------------------------------
// who computes what.  Unit u (a request; or nb beams of a group) has tiles(u) row tiles and keys(u) keys; keys are cut into runs of `run` keys so that about
// `target` workgroups have work, and a unit with one run writes its result itself.
// ------------------------------------------------------------------------------------------------
struct Unit { int req, nb, n, n_all, kv; };    // first request, beams, new tokens (up to max_q), all new tokens, keys
DEVI Unit unit_of(const Args& a, int u) {
    Unit x;
    const int g = u / a.per_group, w0 = (u - g * a.per_group) * a.nb;
    x.req = g * a.d.beams + w0;
    x.nb = min(a.nb, a.d.beams - w0);
    if (a.nb == 1) { x.req = u; x.nb = 1; }
    const int len = x.req / a.d.beams;
    x.n_all = max(a.d.q_lens[len], 0);
    x.n = min(x.n_all, a.d.max_q);
    x.kv = min(max(a.d.kv_lens[len], 0), a.d.blocks * a.d.page_size);
    return x;
}

struct Plan {
    bool split;
    int run, items, parts, joins;
    int* order;      // [units] the units, longest first (up to 64 of them: else as they come)
    int* item0;      // [units + 1] first item of each unit, in that order
    int* part0;      // first partial result (units with several runs)
    int* join0;      // first (tile, head) to join
};
template <int TILE> DEVI int tiles_of(const Args& a, const Unit& x) { return (x.nb * x.n * a.group + TILE - 1) / TILE; }

DEVI int64_t wave_add(int64_t v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor((long long)v, o, 64);
    return v;
}
DEVI int wave_upto(int v, int lane) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
        const int t = __shfl_up(v, o, 64);
        if (lane >= o) v += t;
    }
    return v;
}

DEVI int wave_sum_int(int v) {
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
    return v;
}

// Whether there is anything to split: tables may have room for long requests (a.split) that are not there.  32 requests of 150 keys, 12 heads of 64, in tables for 4096:
// 9.6 us with this look at the lengths, 17.7 without it, 7.8 in tables for 512.
DEVI bool any_long(const Args& a) {
    if (!a.split) return false;
    int most = 0;
#pragma unroll 4
    for (int i = threadIdx.x & 63; i < a.d.requests / a.d.beams; i += 64) most = max(most, a.d.kv_lens[i]);
    return __ballot(most > a.run_min) != 0;
}

// `lds`: 4 (units + 1) ints; every wave ends with the same plan (the first one writes it).  Where nothing is split there is no run to choose, and steps have nothing to
// plan: item = (unit, head).
template <int TILE> DEVI Plan make_plan(const Args& a, bool split_any, int* lds) {
    const int lane = threadIdx.x & 63;
    Plan p;
    p.run = 0x3fffffff;
    p.split = split_any;
    if (!split_any && TILE == STEP_ROWS) {
        p.items = a.units * a.d.kv_heads;
        return p;
    }
    p.item0 = lds;
    p.part0 = lds + a.units + 1;
    p.join0 = lds + 2 * (a.units + 1);
    p.order = lds + 3 * (a.units + 1);
    const Unit first = unit_of(a, min(lane, a.units - 1));                    // (64 units at most, as a rule: looked up once)
    int64_t work = 0;
    for (int u = split_any ? lane : a.units; u < a.units; u += 64) {
        const Unit x = u < 64 ? first : unit_of(a, u);
        work += (int64_t)tiles_of<TILE>(a, x) * x.kv;
    }
    work = wave_add(work) * a.d.kv_heads;
    int64_t want = (work + a.target - 1) / a.target;
    // Steps: each request's last run is a short one; lengthen the runs until the workgroups that are resident together hold all of them.
    // Either: lengthen them until the partial results have room.
#pragma unroll 1
    for (int round = 0; split_any; ++round) {
        p.run = round < 12 ? (int)((max((int64_t)a.run_min, min(want, (int64_t)0x1fffffff)) + 63) / 64 * 64) : 0x3fffffff;
        int n = 0, split = 0;
        for (int u = lane; u < a.units; u += 64) {
            const Unit x = u < 64 ? first : unit_of(a, u);
            const int runs = max(1, (int)(((int64_t)x.kv + p.run - 1) / p.run)), k = tiles_of<TILE>(a, x) * a.d.kv_heads * runs;
            n += k;
            if (runs > 1) split += k;
        }
        n = wave_sum_int(n);
        split = wave_sum_int(split);
        if (split <= a.parts && (TILE != STEP_ROWS || split == 0 || n <= a.target || round >= 4)) break;
        want = (int64_t)p.run + (int64_t)p.run * max(n - a.target, a.target / 8) / a.target;
    }
    // longest first: workgroups that come free late then get short work (makespan over 6 requests of 1711 .. 16771 keys: 1.07 of the mean, 1.4 in any order)
    if (a.units <= 64) {
        const int mine = lane < a.units ? first.kv : -1;
        int rank = 0;
#pragma unroll 4
        for (int v = 0; v < a.units; ++v) {
            const int kv = __builtin_amdgcn_readlane(mine, v);
            rank += kv > mine || (kv == mine && v < lane);
        }
        if (lane < a.units) p.order[rank] = lane;
    } else {
        for (int u = lane; u < a.units; u += 64) p.order[u] = u;
    }
    __syncthreads();
    int items = 0, parts = 0, joins = 0;
    for (int u0 = 0; u0 < a.units; u0 += 64) {
        const int u = u0 + lane;
        int i = 0, q = 0, j = 0;
        if (u < a.units) {
            const Unit x = unit_of(a, p.order[u]);
            const int t = tiles_of<TILE>(a, x) * a.d.kv_heads, runs = max(1, (int)(((int64_t)x.kv + p.run - 1) / p.run));
            i = t * runs;
            if (runs > 1) { q = i; j = t; }
        }
        const int iu = wave_upto(i, lane), qu = wave_upto(q, lane), ju = wave_upto(j, lane);
        if (u < a.units && threadIdx.x < 64) { p.item0[u] = items + iu - i; p.part0[u] = parts + qu - q; p.join0[u] = joins + ju - j; }
        items += __shfl(iu, 63, 64);
        parts += __shfl(qu, 63, 64);
        joins += __shfl(ju, 63, 64);
    }
    p.items = items;
    p.parts = parts;
    p.joins = joins;
    if (threadIdx.x == 0) { p.item0[a.units] = items; p.part0[a.units] = parts; p.join0[a.units] = joins; }
    __syncthreads();
    return p;
}
DEVI int find(const int* first, int units, int i) {          // the last unit whose first is <= i and that is not empty
    int lo = 0, hi = units;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (first[mid] <= i) lo = mid;
        else hi = mid;
    }
    return lo;
}

// place in the order, run, tile and head of an item
struct Item { int u, run, tile, head; Unit x; };
template <int TILE> DEVI Item item_of(const Args& a, const Plan& plan, int item) {
    Item it;
    if (plan.split || TILE != STEP_ROWS) {
        it.u = find(plan.item0, a.units, item);
        it.x = unit_of(a, plan.order[it.u]);
        int rest = item - plan.item0[it.u];
        it.head = rest % a.d.kv_heads;
        rest /= a.d.kv_heads;
        const int tiles = tiles_of<TILE>(a, it.x);
        it.run = rest / tiles;
        it.tile = tiles - 1 - (rest - it.run * tiles);                        // the last tokens, which see most, first (4096 tokens of one prompt: 220 -> 194 us)
    } else {
        it.u = item / a.d.kv_heads;
        it.head = item - it.u * a.d.kv_heads;
        it.tile = it.run = 0;
        it.x = unit_of(a, it.u);
    }
    // the same for the whole workgroup: in scalar registers from here on
    int* f[] = {&it.u, &it.run, &it.tile, &it.head, &it.x.req, &it.x.nb, &it.x.n, &it.x.n_all, &it.x.kv};
#pragma unroll
    for (int k = 0; k < 9; ++k) *f[k] = __builtin_amdgcn_readfirstlane(*f[k]);
    if (it.tile == 0 && it.run == 0 && it.head == 0 && threadIdx.x == 0 && (it.x.n_all > a.d.max_q || it.x.kv != a.d.kv_lens[it.x.req / a.d.beams])) flag_page_error();
    return it;
}

// a row of a unit: beam, token, query head within the group -> its token row, or -1 where it has none
struct Row { int64_t token; int head, beam, i; };
DEVI Row row_of(const Args& a, const Unit& x, int row) {
    Row r;
    const int t = row / a.group;
    r.head = row - t * a.group;
    r.beam = x.nb == 1 ? 0 : t / x.n;
    r.i = t - r.beam * x.n;
    r.token = -1;
    if (row < x.nb * x.n * a.group) {
        r.token = (int64_t)a.d.q_start[x.req + r.beam] + r.i;
        if (r.token < 0 || r.token >= a.d.tokens) { flag_page_error(); r.token = -1; }
    }
    return r;
}
DEVI int sees(const Args& a, const Unit& x, int i) { return a.d.causal ? max(0, min(x.kv, x.kv - x.n_all + i + 1)) : x.kv; }

template <typename T, int D> DEVI T* out_row(const Args& a, const Row& r, int h) {
    return (T*)a.d.out + r.token * a.d.out_row + (int64_t)(h * a.group + r.head) * a.d.out_head;
}
// partial results: [part][TILE][D] sums, then [part][TILE][2] maximum (log2) and sum
template <int D, int TILE> DEVI float* part_o(const Args& a, int part) { return (float*)a.d.ws + (int64_t)part * TILE * D; }
template <int D, int TILE> DEVI float* part_ml(const Args& a, int part) { return (float*)a.d.ws + (int64_t)a.parts * TILE * D + (int64_t)part * TILE * 2; }

DEVI void store4(bf16* p, float a, float b, float c, float d) { *reinterpret_cast<bf16x4*>(p) = pack4(a, b, c, d); }
DEVI void store4(float* p, float a, float b, float c, float d) { *reinterpret_cast<f32x4*>(p) = f32x4{a, b, c, d}; }

// ------------------------------------------------------------------------------------------------
// chunks
// ------------------------------------------------------------------------------------------------
template <typename T> constexpr int chunk_subtiles = sizeof(T) == 2 ? 2 : 1;      // 64 keys a tile in bf16, 32 in fp32: 32 or 16 KB of K and V at head_dim 64 or 128 either way
template <typename T, int D> constexpr int chunk_lds = 2 * 2 * 32 * chunk_subtiles<T> * D * (int)sizeof(T);

template <typename T, int D>
__global__ __launch_bounds__(2 * chunk_rows<T>, D * (int)sizeof(T) >= 512 ? 1 : 2) void paged_attn_chunk_kernel(Args a) {
    extern __shared__ unsigned char lds[];
    constexpr int CHUNK_ROWS = chunk_rows<T>, NW = CHUNK_ROWS / 32, NS = chunk_subtiles<T>, KT = 32 * NS, RB = D * (int)sizeof(T), IMG = KT * RB;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Plan plan = make_plan<CHUNK_ROWS>(a, any_long(a), reinterpret_cast<int*>(lds + 4 * IMG));
    for (int item = blockIdx.x; item < plan.items; item += gridDim.x) {
        const Item it = item_of<CHUNK_ROWS>(a, plan, item);
        const Unit& x = it.x;
        const int u = it.u, h = it.head, run = it.run, row0 = it.tile * CHUNK_ROWS;
        const bool whole = plan.run >= x.kv;
        const int last = min(x.n * a.group, row0 + CHUNK_ROWS) - 1;
        const int end = min(sees(a, x, last / a.group), (run + 1) * plan.run);
        const int start = run * plan.run;
        const Row row = row_of(a, x, row0 + 32 * wave + (lane & 31));
        const int lim = row.token >= 0 ? sees(a, x, row.i) : 0x7fffffff;      // (rows without a token compute on zeros: nothing of them is written)
        Rows<T, D> rows;
        rows.load((const T*)a.d.q + row.token * a.d.q_row + (int64_t)(h * a.group + row.head) * a.d.q_head, row.token >= 0, a, lane);
        const int free_to = wave_min(lim), see_to = -wave_min(row.token >= 0 ? -lim : 0);       // keys that every row of the wave sees, that any does
        const bool idle = row0 + 32 * wave >= x.n * a.group;                     // a wave without rows only helps to stage
        float m = -INFINITY, l = 0.f;
        bool odd = false;
        f32x16 o[D / 32] = {};
        const int32_t* table = a.d.tables + x.req * a.d.table_row;
        const int64_t head_off = h * a.d.head_stride;
        const int steps = end > start ? (end - start + KT - 1) / KT : 0;
        const Stager<T, D, KT, NW> stage(a, head_off, wave, lane);
        int page = page_of<KT>(a, table, start, end, lane);
        __syncthreads();                                                         // the item before has read its last tile
        if (steps > 0) stage(a, start, end, page, lds, lds + IMG, wave, lane);
        page = page_of<KT>(a, table, start + KT, end, lane);
        for (int j = 0; j < steps; ++j) {
            const int key0 = start + j * KT;
            unsigned char* img = lds + (j & 1) * 2 * IMG;
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            __syncthreads();
            auto ahead = [&] {
                if (j + 1 < steps) {
                    unsigned char* next = lds + ((j + 1) & 1) * 2 * IMG;
                    stage(a, key0 + KT, end, page, next, next + IMG, wave, lane);
                    page = page_of<KT>(a, table, key0 + 2 * KT, end, lane);
                }
            };
            const int subs = idle ? 0 : (min(min(see_to, end) - key0, KT) + 31) >> 5;
            if (subs <= 0) { ahead(); continue; }
            { const int n = 0; tile_step<T, D>(rows, img + n * 32 * RB, img + IMG + n * 32 * RB, key0 + 32 * n, min(lim, end), key0 + 32 * n + 32 > min(free_to, end), a.c, m, l, o, lane, odd, ahead); }
            if (subs == 2) { const int n = 1; tile_step<T, D>(rows, img + n * 32 * RB, img + IMG + n * 32 * RB, key0 + 32 * n, min(lim, end), key0 + 32 * n + 32 > min(free_to, end), a.c, m, l, o, lane, odd, [] {}); }
        }
        l = add_halves(l);
        if (odd) {                                                               // from the first tile that not every row sees
            const int mixed = max(min(free_to, end) - start, 0) / 32 * 32 + start;
#pragma unroll 1
            for (int key = mixed; key < min(see_to, end); ++key) add_odd<T, D>(a, o, table, h, key, key < lim, lane);
        }
        if (whole) {
            if (row.token >= 0) {
                T* out = out_row<T, D>(a, row, h);
                const float inv = l != 0.f ? 1.f / l : 0.f;
#pragma unroll
                for (int t = 0; t < D / 32; ++t)
#pragma unroll
                    for (int r = 0; r < 16; r += 4)
                        store4(out + 32 * t + 2 * r + 4 * (lane >> 5), o[t][r] * inv, o[t][r + 1] * inv, o[t][r + 2] * inv, o[t][r + 3] * inv);
            }
        } else {
            const int part = plan.part0[u] + (item - plan.item0[u]);
            const int at_row = 32 * wave + (lane & 31);
            float* po = part_o<D, CHUNK_ROWS>(a, part) + at_row * D;
#pragma unroll
            for (int t = 0; t < D / 32; ++t)
#pragma unroll
                for (int r = 0; r < 16; r += 4) store4(po + 32 * t + 2 * r + 4 * (lane >> 5), o[t][r], o[t][r + 1], o[t][r + 2], o[t][r + 3]);
            if (lane < 32) {
                float* ml = part_ml<D, CHUNK_ROWS>(a, part) + 2 * at_row;
                ml[0] = m;
                ml[1] = l;
            }
        }
    }
}

// ------------------------------------------------------------------------------------------------
// steps
// ------------------------------------------------------------------------------------------------
template <typename T, int D> constexpr int step_lds = 4 * 2 * 32 * D * (int)sizeof(T);       // a tile of 32 keys per wave

template <typename T, int D>
__global__ __launch_bounds__(256, D * (int)sizeof(T) >= 512 ? 1 : 2) void paged_attn_step_kernel(Args a) {
    extern __shared__ unsigned char lds[];
    constexpr int RB = D * (int)sizeof(T), IMG = 32 * RB;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    unsigned char* mine = lds + wave * 2 * IMG;
    int* shared_to = reinterpret_cast<int*>(lds + 8 * IMG);
    const Plan plan = make_plan<STEP_ROWS>(a, any_long(a), shared_to + 4);
    for (int item = blockIdx.x; item < plan.items; item += gridDim.x) {
        const Item it = item_of<STEP_ROWS>(a, plan, item);
        const Unit& x = it.x;
        const int u = it.u, h = it.head, run = it.run;
        if (x.n == 0) continue;
        const int start = run * plan.run, end = min(x.kv, start + plan.run);
        const bool whole = plan.run >= x.kv;
        const int n_rows = x.nb * x.n * a.group;
        const Row row = row_of(a, x, lane & 31);
        const int lim = row.token >= 0 ? sees(a, x, row.i) : 0x7fffffff;
        Rows<T, D> rows;
        rows.load((const T*)a.d.q + row.token * a.d.q_row + (int64_t)(h * a.group + row.head) * a.d.q_head, row.token >= 0, a, lane);
        const int free_to = wave_min(lim);
        const int32_t* table = a.d.tables + x.req * a.d.table_row;
        const int64_t head_off = h * a.d.head_stride;
        // pages that are the same for every beam are read once for all of them: up to the first block that differs
        __syncthreads();                                                         // the item before has read shared_to and the tiles
        int shared_end = max(end, start);
        if (x.nb > 1 && end > start) {
            int differs = 0x7fffffff;
            const int b1 = (end - 1) >> a.page_shift;
            for (int b = (start >> a.page_shift) + threadIdx.x; b <= b1; b += 256) {
                const int p = table[b];
                bool same = true;
#pragma unroll 4
                for (int w = 1; w < x.nb; ++w) same &= table[w * a.d.table_row + b] == p;
                if (!same) differs = min(differs, b);
            }
#pragma unroll
            for (int o = 32; o > 0; o >>= 1) differs = min(differs, __shfl_xor(differs, o, 64));
            if (lane == 0) shared_to[wave] = differs;
            __syncthreads();
            differs = min(min(shared_to[0], shared_to[1]), min(shared_to[2], shared_to[3]));
            differs = __builtin_amdgcn_readfirstlane(differs);
            if (differs <= b1) shared_end = max(start, differs << a.page_shift);
        }
        // jobs: the shared tiles, then each beam's own
        const int shared_tiles = (shared_end - start + 31) / 32, jobs = shared_tiles + (max(end - shared_end, 0) + 31) / 32 * x.nb;
        struct Job { int key0, end, beam; };
        auto job = [&](int j) {
            const int k = j - shared_tiles;
            return k < 0 ? Job{start + 32 * j, shared_end, -1} : Job{shared_end + 32 * (k / x.nb), j < jobs ? end : 0, k % x.nb};
        };
        auto pages = [&](const Job& b) { return page_of<32>(a, table + max(b.beam, 0) * a.d.table_row, b.key0, b.end, lane); };
        float m = -INFINITY, l = 0.f;
        bool odd = false;
        f32x16 o[D / 32] = {};
        Job now = job(wave), next = job(wave + 4);
        int page = pages(now), page_next = pages(next);
        const Stager<T, D, 32, 1> stage(a, head_off, 0, lane);
        if (wave < jobs) stage(a, now.key0, now.end, page, mine, mine + IMG, 0, lane);
        for (int j = wave; j < jobs; j += 4) {
            asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
            const Job after = job(j + 8);
            // once the tile's operands are in registers, the next tile lands in its place
            auto ahead = [&] {
                asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
                if (j + 4 < jobs) stage(a, next.key0, next.end, page_next, mine, mine + IMG, 0, lane);
                page_next = pages(after);
            };
            const int see = min(lim, now.end);
            const bool take = now.beam < 0 || row.beam == now.beam;              // a tile of one beam: the other beams' rows see none of it
            tile_step<T, D>(rows, mine, mine + IMG, now.key0, take ? see : 0, now.beam >= 0 || now.key0 + 32 > min(free_to, now.end), a.c, m, l, o, lane, odd, ahead);
            now = next; next = after;
        }
        l = add_halves(l);
        if (odd) {
#pragma unroll 1
            for (int j = wave; j < jobs; j += 4) {
                const Job b = job(j);
                if (b.beam < 0 && b.key0 + 32 <= min(free_to, b.end)) continue;
#pragma unroll 1
                for (int key = b.key0; key < min(b.key0 + 32, b.end); ++key)
                    add_odd<T, D>(a, o, table + max(b.beam, 0) * a.d.table_row, h, key, key < lim && (b.beam < 0 || row.beam == b.beam), lane);
            }
        }
        // the four waves' sums meet: [wave][row][D] fp32 in the tiles' place, [wave][row][2] behind
        __syncthreads();
        constexpr int LD = D + 4;                                                // (rows of D floats alone would put every row's column on one bank)
        float* so = reinterpret_cast<float*>(lds);
        float* sml = so + 4 * 8 * LD;
        for (int r0 = 0; r0 < n_rows; r0 += 8) {                                 // 8 rows at a time: 4 x 8 x (D + 4) floats fit any form's tiles
            const int at_row = (lane & 31) - r0;
            if (at_row >= 0 && at_row < 8) {
#pragma unroll
                for (int t = 0; t < D / 32; ++t)
#pragma unroll
                    for (int r = 0; r < 16; r += 4)
                        *reinterpret_cast<f32x4*>(so + (wave * 8 + at_row) * LD + 32 * t + 2 * r + 4 * (lane >> 5)) = f32x4{o[t][r], o[t][r + 1], o[t][r + 2], o[t][r + 3]};
                if (lane < 32) { sml[(wave * 8 + at_row) * 2] = m; sml[(wave * 8 + at_row) * 2 + 1] = l; }
            }
            __syncthreads();
            for (int i = threadIdx.x; i < 8 * (D / 4); i += 256) {
                const int rr = i / (D / 4), e = (i - rr * (D / 4)) * 4;
                if (r0 + rr >= n_rows) continue;
                float top = -INFINITY;
#pragma unroll
                for (int w = 0; w < 4; ++w) top = fmaxf(top, sml[(w * 8 + rr) * 2]);
                const float mm = top == -INFINITY ? 0.f : top;
                f32x4 sum = {};
                float den = 0.f;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float f = __builtin_amdgcn_exp2f(sml[(w * 8 + rr) * 2] - mm);
                    den += f * sml[(w * 8 + rr) * 2 + 1];
                    sum += f * *reinterpret_cast<const f32x4*>(so + (w * 8 + rr) * LD + e);
                }
                if (whole) {
                    const Row to = row_of(a, x, r0 + rr);
                    const float inv = den != 0.f ? 1.f / den : 0.f;
                    if (to.token >= 0) store4(out_row<T, D>(a, to, h) + e, sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv);
                } else {
                    const int part = plan.part0[u] + (item - plan.item0[u]);
                    *reinterpret_cast<f32x4*>(part_o<D, STEP_ROWS>(a, part) + (r0 + rr) * D + e) = sum;
                    if (e == 0) { float* ml = part_ml<D, STEP_ROWS>(a, part) + 2 * (r0 + rr); ml[0] = top; ml[1] = den; }
                }
            }
            __syncthreads();
        }
    }
}

// ------------------------------------------------------------------------------------------------
// the runs of a split request, joined in their order
// ------------------------------------------------------------------------------------------------
template <typename T, int D, int TILE>
__global__ __launch_bounds__(256) void paged_attn_join_kernel(Args a) {
    extern __shared__ unsigned char lds[];
    if (!any_long(a)) return;
    const Plan plan = make_plan<TILE>(a, true, reinterpret_cast<int*>(lds));
    constexpr int PER = D / 4, ROWS = 256 / PER;                                 // threads per row, rows at a time
    constexpr int SLICES = TILE / ROWS;
    for (int i = blockIdx.x; i < plan.joins * SLICES; i += gridDim.x) {
        const int j = i / SLICES, slice = i - j * SLICES;
        const int u = find(plan.join0, a.units, j);
        const Unit x = unit_of(a, plan.order[u]);
        const int h = (j - plan.join0[u]) % a.d.kv_heads, tile = (j - plan.join0[u]) / a.d.kv_heads, tiles = tiles_of<TILE>(a, x);
        const int runs = (x.kv + plan.run - 1) / plan.run;
        const int at_row = slice * ROWS + threadIdx.x / PER, e = (threadIdx.x % PER) * 4;
        const Row row = row_of(a, x, tile * TILE + at_row);
        if (row.token < 0) continue;
        float top = -INFINITY, den = 0.f;
        f32x4 sum = {};
        constexpr int AT_ONCE = 8;
        for (int r0 = 0; r0 < runs; r0 += AT_ONCE) {                             // loads of eight runs in flight
            float mr[AT_ONCE], lr[AT_ONCE];
            f32x4 v[AT_ONCE];
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                const int part = plan.part0[u] + (min(r0 + k, runs - 1) * tiles + tiles - 1 - tile) * a.d.kv_heads + h;
                const float* ml = part_ml<D, TILE>(a, part) + 2 * at_row;
                mr[k] = ml[0];
                lr[k] = ml[1];
                v[k] = *reinterpret_cast<const f32x4*>(part_o<D, TILE>(a, part) + at_row * D + e);
            }
#pragma unroll
            for (int k = 0; k < AT_ONCE; ++k) {
                if (r0 + k >= runs) continue;
                const float next = fmaxf(top, mr[k]), mm = next == -INFINITY ? 0.f : next;
                const float fa = __builtin_amdgcn_exp2f(top - mm), fb = __builtin_amdgcn_exp2f(mr[k] - mm);
                den = den * fa + lr[k] * fb;
                sum = sum * fa + v[k] * fb;
                top = next;
            }
        }
        const float inv = den != 0.f ? 1.f / den : 0.f;
        store4(out_row<T, D>(a, row, h) + e, sum[0] * inv, sum[1] * inv, sum[2] * inv, sum[3] * inv);
    }
}

// Which kernel, and how keys are split.  Up to 32 rows per key head go through the step kernel, whose waves take different keys; more have rows enough for a wave each.
// Workgroups to aim at when keys are split: 512 steps (two on every compute unit; long caches: 191 us, with 256 190, with 1024 199), 768 chunks of 128 rows (with 512
// 340 us as well, with 1024 347: longest first, the short last runs fill the gaps).  Shortest run 512 keys: one request of 500 keys takes 8.2 us in one piece and 14.9 split
// by 256, 4 requests of 1000 keys 19.9 and 17.7; 2 chunks of 64 tokens over 4000 keys take 37.4 us, 43.8 with runs of 1024 and 45.5 with runs of 256.
struct Shape { bool chunk, split; int nb, target, run_min, parts; int64_t ws; };
Shape shape_of(const mmf_paged_attn_desc* d) {
    Shape s;
    const int64_t rows = (int64_t)d->max_q * (d->heads / d->kv_heads);
    s.chunk = rows > STEP_ROWS;
    s.nb = s.chunk ? 1 : (int)(STEP_ROWS / rows < d->beams ? STEP_ROWS / rows : d->beams);
    const int tile = !s.chunk ? STEP_ROWS : d->is_f32 ? chunk_rows<float> : chunk_rows<bf16>;
    s.target = s.chunk ? 768 * 128 / tile : 512;
    s.run_min = 512;
    s.parts = s.chunk ? 2 * s.target : 1024;
    s.split = (int64_t)d->blocks * d->page_size > s.run_min;
    s.ws = s.split ? (int64_t)s.parts * tile * (d->head_dim + 2) * 4 : 0;
    return s;
}

// more than 64 KB of LDS are asked for once per kernel and device
template <typename K> int allow_lds(K* kernel, int bytes, std::atomic<uint64_t>& done) {
    int dev = 0;
    if (hipGetDevice(&dev) != hipSuccess) return 1;
    const uint64_t bit = 1ull << (dev & 63);
    if (done.load(std::memory_order_relaxed) & bit) return 0;
    if (hipFuncSetAttribute(reinterpret_cast<const void*>(kernel), hipFuncAttributeMaxDynamicSharedMemorySize, bytes) != hipSuccess) return 1;
    done.fetch_or(bit, std::memory_order_relaxed);
    return 0;
}

template <typename T, int D> int launch(const mmf_paged_attn_desc* d, const Shape& s, hipStream_t stream) {
    constexpr int CHUNK_ROWS = chunk_rows<T>;
    Args a;
    a.d = *d;
    a.page_shift = __builtin_ctz(d->page_size);
    a.group = d->heads / d->kv_heads;
    a.nb = s.nb;
    a.per_group = (d->beams + s.nb - 1) / s.nb;
    a.target = s.target;
    a.parts = s.parts;
    a.run_min = s.run_min;
    a.split = s.split;
    const int64_t tiles = s.chunk ? ((int64_t)d->max_q * a.group + CHUNK_ROWS - 1) / CHUNK_ROWS : 1;
    a.c = d->scale != 0.f ? fabsf(d->scale) * 1.44269504088896340736f : 1.f;
    a.q_and = d->scale != 0.f ? 0xffffffffu : 0u;
    a.q_xor = d->scale < 0.f ? 0x80000000u : 0u;
    const int step = UNITS_MAX / a.per_group * d->beams;         // requests per launch: whole groups
    for (int r0 = 0; r0 < d->requests; r0 += step) {
        const int n = d->requests - r0 < step ? d->requests - r0 : step;
        a.d.requests = n;
        a.d.tables = d->tables + r0 * d->table_row;
        a.d.kv_lens = d->kv_lens + r0 / d->beams;
        a.d.q_lens = d->q_lens + r0 / d->beams;
        a.d.q_start = d->q_start + r0;
        a.units = s.nb == 1 ? n : n / d->beams * a.per_group;
        const int prefix = 4 * (a.units + 1) * 4;
        const int64_t most = tiles * a.units * d->kv_heads;
        MMF_CHECK_ARG(most <= 0x3fffffff, "paged_attention: too many rows for one call");
        const int cap = s.chunk ? 2048 * 128 / CHUNK_ROWS : 512, grid = s.split || most > cap ? cap : (int)most;
        if (s.chunk) {
            const int lds = chunk_lds<T, D> + prefix;
            static std::atomic<uint64_t> done{0};
            MMF_CHECK_ARG(!allow_lds(paged_attn_chunk_kernel<T, D>, chunk_lds<T, D> + PREFIX_MAX, done), "paged_attention: LDS");
            hipLaunchKernelGGL((paged_attn_chunk_kernel<T, D>), dim3(grid), dim3(2 * CHUNK_ROWS), lds, stream, a);
        } else {
            const int lds = step_lds<T, D> + 16 + prefix;
            static std::atomic<uint64_t> done{0};
            MMF_CHECK_ARG(!allow_lds(paged_attn_step_kernel<T, D>, step_lds<T, D> + 16 + PREFIX_MAX, done), "paged_attention: LDS");
            hipLaunchKernelGGL((paged_attn_step_kernel<T, D>), dim3(grid), dim3(256), lds, stream, a);
        }
        MMF_CHECK_LAUNCH();
        if (s.split) {
            if (s.chunk) hipLaunchKernelGGL((paged_attn_join_kernel<T, D, CHUNK_ROWS>), dim3(1024), dim3(256), prefix, stream, a);
            else hipLaunchKernelGGL((paged_attn_join_kernel<T, D, STEP_ROWS>), dim3(512), dim3(256), prefix, stream, a);
            MMF_CHECK_LAUNCH();
        }
    }
    return 0;
}

}  // namespace

extern "C" {

int mmf_paged_attention_take_error(void) { return take_page_error(); }

int64_t mmf_paged_attention_ws_bytes(const mmf_paged_attn_desc* d) {
    if (!d || d->kv_heads <= 0 || d->heads < d->kv_heads || d->max_q < 1 || d->beams < 1) return 0;
    return shape_of(d).ws;
}

int mmf_paged_attention(const mmf_paged_attn_desc* d, void* stream) {
    MMF_CHECK_ARG(d && d->q && d->k_cache && d->v_cache && d->tables && d->kv_lens && d->q_start && d->q_lens && d->out, "paged_attention: null operand");
    MMF_CHECK_ARG(d->head_dim == 64 || d->head_dim == 128, "paged_attention: head_dim is 64 or 128");
    MMF_CHECK_ARG(d->heads > 0 && d->kv_heads > 0 && d->heads % d->kv_heads == 0, "paged_attention: heads is a multiple of kv_heads");
    MMF_CHECK_ARG(d->requests > 0 && d->beams >= 1 && d->beams <= MMF_BEAMS_MAX && d->blocks > 0 && d->pages > 0 && d->tokens >= 0, "paged_attention: bad shape");
    MMF_CHECK_ARG(d->requests % d->beams == 0, "paged_attention: requests come in groups of beams");
    MMF_CHECK_ARG(d->page_size >= 1 && d->page_size <= MMF_PAGE_MAX && (d->page_size & (d->page_size - 1)) == 0, "paged_attention: page_size is a power of two up to 1024");
    MMF_CHECK_ARG((int64_t)d->blocks * d->page_size <= 0x3fffffff, "paged_attention: more than 2^30 keys");
    MMF_CHECK_ARG(d->max_q >= 1 && (int64_t)d->max_q * d->heads <= 0x3fffffff, "paged_attention: max_q is at least 1, and max_q * heads under 2^30");
    const int unit = d->is_f32 ? 4 : 8;
    MMF_CHECK_ARG(((uintptr_t)d->q & 15) == 0 && ((uintptr_t)d->k_cache & 15) == 0 && ((uintptr_t)d->v_cache & 15) == 0 && ((uintptr_t)d->out & 15) == 0 &&
                      d->q_row % unit == 0 && d->q_head % unit == 0 && d->page_stride % unit == 0 && d->head_stride % unit == 0 && d->pos_stride % unit == 0 &&
                      d->out_row % unit == 0 && d->out_head % unit == 0, "paged_attention: rows start on 16 bytes");
    const int64_t size = d->is_f32 ? 4 : 2;
    MMF_CHECK_ARG(d->page_stride >= 0 && d->page_stride * size <= 0xffffffffll && d->pos_stride >= 0 && d->pos_stride * d->page_size * size <= 0x7fffffff && d->head_stride >= 0,
                  "paged_attention: a page within 2 GiB, pages within 4 GiB of each other");
    if (d->tokens == 0) return 0;
    const Shape s = shape_of(d);
    page_kernels_used();
    MMF_CHECK_ARG(s.ws == 0 || (d->ws && ((uintptr_t)d->ws & 15) == 0), "paged_attention: null workspace");
    if (d->is_f32) return d->head_dim == 64 ? launch<float, 64>(d, s, (hipStream_t)stream) : launch<float, 128>(d, s, (hipStream_t)stream);
    return d->head_dim == 64 ? launch<bf16, 64>(d, s, (hipStream_t)stream) : launch<bf16, 128>(d, s, (hipStream_t)stream);
}

}  // extern "C"
