// The paged 8-bit cache (paged.h): block tables and slot maps from request lengths, and the append of new keys and values.
#include "paged.h"

// ---- block tables and slot maps ---------------------------------------------------------------------------------------------------
// For every row b, in order (all sums exclusive prefix sums over the rows):
//   take  = clamp(new, 0, min(max_new, rows - start)), start = sum(take)  (row_stride > 0: start = b * row_stride)
//   want  = max(0, ceil(min(past + take, max_len) / block) - held), got = clamp(avail - sum(want), 0, want)
//   table[held + i] = ring[(head + sum(want) + i) mod blocks], i < got
//   new < 0: the row has ended; its blocks go to the ring's end in order, its table entries become -1
// Then every token row's slot = table[pos / block] * block + pos % block.  Latency is all that matters (a step of 256 rows moves
// 7 KB): one workgroup does both halves where the work is small, otherwise the scan runs in one workgroup and the filling in
// many -- a second launch instead of a grid-wide wait.
struct SlotRow { int start, take, past, kept, held, base, back, gone; };      // 32 bytes a row, in the caller's scratch

struct SlotArgs {
    const int32_t* past; const int32_t* fresh; int32_t* held; int32_t* table; int32_t* ring; int32_t* counters;
    int n, width, block, blocks, max_len, max_new, rows, row_stride;
    int32_t* starts; int32_t* slots; int32_t* positions; SlotRow* desc;
};

#define SLOT_THREADS 1024
#define SLOT_WAVES (SLOT_THREADS / 64)

// exclusive prefix sum over the workgroup, and the total; `lds`: SLOT_WAVES + 1 entries of its own
__device__ __forceinline__ int64_t slot_scan(int64_t v, int64_t* lds, int64_t& total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t inc = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t o = __shfl_up(inc, off, 64);
        if (lane >= off) inc += o;
    }
    if (lane == 63) lds[wave] = inc;
    __syncthreads();
    if (threadIdx.x == 0) {
        int64_t run = 0;
        for (int w = 0; w < SLOT_WAVES; ++w) { const int64_t s = lds[w]; lds[w] = run; run += s; }
        lds[SLOT_WAVES] = run;
    }
    __syncthreads();
    const int64_t r = inc - v + lds[wave];
    total = lds[SLOT_WAVES];
    __syncthreads();
    return r;
}

__device__ __forceinline__ void slot_scan_rows(const SlotArgs& a)
{
    __shared__ int64_t lds[SLOT_WAVES + 1];
    const int head = (int) ((uint32_t) a.counters[0] % (uint32_t) a.blocks);
    const int avail = min(max(a.counters[1], 0), a.blocks);
    int64_t rows_before = 0, want_before = 0, back_before = 0;
    for (int b0 = 0; b0 < a.n; b0 += SLOT_THREADS) {
        const int b = b0 + threadIdx.x;
        const bool in = b < a.n;
        const int fresh = in ? a.fresh[b] : 0;
        const int held = in ? min(max(a.held[b], 0), a.width) : 0;
        const int past = in ? max(a.past[b], 0) : 0;
        int take = min(max(fresh, 0), a.max_new), start = 0;
        int64_t total;
        if (a.row_stride > 0) {
            const int64_t s = (int64_t) b * a.row_stride;
            start = (int) min(s, (int64_t) a.rows);
            take = min(min(take, a.row_stride), a.rows - start);
        } else {
            const int64_t s = rows_before + slot_scan(take, lds, total);
            rows_before += total;
            start = (int) min(s, (int64_t) a.rows);
            take = min(take, a.rows - start);
        }
        const bool gone = fresh < 0;
        const int end = (int) min((int64_t) past + take, (int64_t) a.max_len);
        const int want = in && !gone ? max(0, (end + a.block - 1) / a.block - held) : 0;
        const int64_t base = want_before + slot_scan(want, lds, total);
        want_before += total;
        const int back = gone ? held : 0;
        const int64_t back_base = back_before + slot_scan(back, lds, total);
        back_before += total;
        if (in) {
            const int got = (int) min(max((int64_t) avail - base, (int64_t) 0), (int64_t) want);
            SlotRow r;
            r.start = start; r.take = take; r.past = past; r.held = held;
            r.kept = gone ? 0 : held + got;
            r.base = (int) ((head + base) % a.blocks);
            r.back = (int) ((head + avail + back_base) % a.blocks);
            r.gone = gone;
            a.desc[b] = r;
            a.starts[b] = start;
            a.held[b] = r.kept;
        }
    }
    __syncthreads();                                          // every thread has read the counters
    if (threadIdx.x == 0) {
        const int got = (int) min(want_before, (int64_t) avail);
        a.counters[0] = (head + got) % a.blocks;
        a.counters[1] = (int) min((int64_t) avail - got + back_before, (int64_t) a.blocks);
        a.counters[2] = (int) min(want_before - got, (int64_t) 0x7fffffff);
        a.counters[3] = 0;
        a.starts[a.n] = (int) min(a.row_stride > 0 ? (int64_t) a.n * a.row_stride : rows_before, (int64_t) a.rows);
    }
}

__device__ __forceinline__ int slot_ring(const SlotArgs& a, int at) { return a.ring[at >= a.blocks ? at - a.blocks : at]; }

// the table and the ring of rows first, first + step, ... (a wave each)
__device__ __forceinline__ void slot_fill_rows(const SlotArgs& a, int first, int step)
{
    const int lane = threadIdx.x & 63;
    for (int b = first; b < a.n; b += step) {
        const SlotRow r = a.desc[b];
        int32_t* row = a.table + (size_t) b * a.width;
        if (r.gone) {
            for (int i = lane; i < r.held; i += 64) {
                const int at = (int) (((int64_t) r.back + i) % a.blocks);
                a.ring[at] = row[i];
                row[i] = -1;
            }
        } else {
            for (int i = r.held + lane; i < r.kept; i += 64) row[i] = slot_ring(a, r.base + i - r.held);
        }
    }
}

// the slots and positions of token rows first, first + step, ...
__device__ __forceinline__ void slot_fill_tokens(const SlotArgs& a, int first, int step)
{
    for (int t = first; t < a.rows; t += step) {
        int lo = 0, hi = a.n;                                 // the last row that starts at or before t (rows of no token share a start: the last one)
        if (a.row_stride > 0) lo = min(t / a.row_stride, a.n - 1);
        else while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (a.desc[mid].start <= t) lo = mid; else hi = mid; }
        const SlotRow r = a.desc[lo];
        const int i = t - r.start;
        int slot = -1, pos = 0;
        if (i < r.take) {
            pos = (int) min((int64_t) r.past + i, (int64_t) 0x7fffffff);
            const int k = pos / a.block;
            if (pos < a.max_len && k < r.kept) {
                // (entries that this call adds are still being written by other waves: they are read where they come from)
                const int id = k < r.held ? a.table[(size_t) lo * a.width + k] : slot_ring(a, r.base + k - r.held);
                if (id >= 0 && id < a.blocks) slot = id * a.block + pos % a.block;
            }
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
    }
}

__global__ __launch_bounds__(SLOT_THREADS) void paged_slots_small_kernel(SlotArgs a)
{
    slot_scan_rows(a);
    __syncthreads();                                          // desc, of this workgroup alone
    slot_fill_tokens(a, threadIdx.x, SLOT_THREADS);
    slot_fill_rows(a, threadIdx.x >> 6, SLOT_WAVES);
}

__global__ __launch_bounds__(SLOT_THREADS) void paged_slots_scan_kernel(SlotArgs a) { slot_scan_rows(a); }

__global__ __launch_bounds__(256) void paged_slots_fill_kernel(SlotArgs a, int token_groups)
{
    if ((int) blockIdx.x < token_groups) slot_fill_tokens(a, blockIdx.x * 256 + threadIdx.x, token_groups * 256);
    else slot_fill_rows(a, (blockIdx.x - token_groups) * 4 + (threadIdx.x >> 6), (gridDim.x - token_groups) * 4);
}

extern "C" int exl_paged_slots(const int32_t* past_lens, const int32_t* new_lens, int32_t* held, int32_t* block_table, int32_t* ring,
                               int32_t* counters, int n_rows, int table_width, int block_size, int num_blocks, int max_len, int max_new, int rows,
                               int row_stride, int32_t* starts, int32_t* slots, int32_t* positions, int32_t* scratch, void* stream)
{
    EXL_REQUIRE(past_lens && new_lens && held && block_table && ring && counters && starts && slots && positions && scratch, EXL_E_INVALID,
                "paged_slots: null pointer");
    EXL_REQUIRE(n_rows > 0 && table_width > 0 && num_blocks > 0 && rows >= 0 && max_new >= 0 && row_stride >= 0 && max_len >= 0, EXL_E_INVALID,
                "paged_slots: bad shape");
    EXL_TRY(paged_check_block("paged_slots", block_size, num_blocks));
    EXL_REQUIRE((int64_t) max_len <= (int64_t) table_width * block_size, EXL_E_INVALID, "paged_slots: max_len (%d) exceeds the block table (%d blocks of %d)",
                max_len, table_width, block_size);
    SlotArgs a = {past_lens, new_lens, held, block_table, ring, counters, n_rows, table_width, block_size, num_blocks, max_len, max_new, rows,
                  row_stride, starts, slots, positions, (SlotRow*) scratch};
    hipStream_t s = (hipStream_t) stream;
    if (rows <= 4096 && n_rows <= 1024) {
        hipLaunchKernelGGL(paged_slots_small_kernel, dim3(1), dim3(SLOT_THREADS), 0, s, a);
    } else {
        hipLaunchKernelGGL(paged_slots_scan_kernel, dim3(1), dim3(SLOT_THREADS), 0, s, a);
        EXL_LAUNCH_CHECK();
        const int tg = (int) ((rows + 255L) / 256 < 2048 ? (rows + 255L) / 256 : 2048), rg = (n_rows + 3) / 4 < 2048 ? (n_rows + 3) / 4 : 2048;
        hipLaunchKernelGGL(paged_slots_fill_kernel, dim3(tg + rg), dim3(256), 0, s, a, tg);
    }
    EXL_LAUNCH_CHECK();
    return 0;
}

int paged_check_block(const char* what, int block_size, int num_blocks)
{
    EXL_REQUIRE(block_size == 16 || block_size == 32 || block_size == 64 || block_size == 128, EXL_E_UNSUPPORTED,
                "%s: block_size (%d) must be 16, 32, 64 or 128", what, block_size);
    EXL_REQUIRE((int64_t) num_blocks * block_size <= 0x7fffffff, EXL_E_UNSUPPORTED, "%s: %d blocks of %d tokens exceed 2^31 slots", what, num_blocks,
                block_size);
    return 0;
}

// ---- append -----------------------------------------------------------------------------------------------------------------------
// A RUN is the longest stretch of token rows whose slots are consecutive inside one page.  Per run and kv head, keys and values each:
//   amax = max |x| (x clamped to +-top * 2^hi, NaN left out), e = the least exponent with amax <= top * 2^e; a run that does not start
//   its page keeps the page's earlier tokens: e = max(e, the page's), their codes move by 2^(e_old - e);  code = round(x / 2^e)
// Keys are rotated first when sin / cos are given: lo * cos - hi * sin in 64 bits and rounded to odd in 32, so that the code is one
// rounding of the exact rotation.  Short runs (single tokens, a few drafted ones) take a wave each; from APPEND_LONG tokens on, and
// head_dim % 16 == 0, the whole workgroup takes the run: every number is read once and stays in registers between the maximum and the
// rounding, and the values' codes are transposed in LDS.
struct AppendArgs {
    const f16* k; const f16* v; const int32_t* slots; const int32_t* positions; const f16* sin; const f16* cos;
    uint8_t* kp; uint8_t* vp; float* ks; float* vs;
    int rows, kv_heads, hd, hd16, block, blocks, chunk, angle_rows;
    long k_stride, v_stride;
};

#define APPEND_LONG 8

// a * b - c * d (sign = -1) or a * b + c * d of fp16 numbers: exact products, the sum in 64 bits, rounded to odd (a later rounding to
// fewer bits then is the exact value's)
__device__ __forceinline__ float rot_odd(f16 a, f16 b, f16 c, f16 d, float sign)
{
    const float p = (float) a * (float) b, q = (float) c * (float) d * sign;
    const double s = (double) p + (double) q;
    float r = (float) s;
    if ((double) r != s && s == s) {
        uint32_t u = __float_as_uint(r);
        if (fabs((double) r) > fabs(s)) u -= 1;                // towards zero
        r = __uint_as_float(u | 1);
    }
    return r;
}

// x of four columns d .. d + 3 of a key or value row; zeros behind head_dim
template <bool ROPE> __device__ __forceinline__ void append_load(const f16* row, const f16* sin, const f16* cos, int d, int hd, float (&x)[4])
{
#pragma unroll
    for (int i = 0; i < 4; ++i) x[i] = 0.f;
    if (d >= hd) return;
    const f16x4 v = *(const f16x4_a4*) (row + d);
    if (!ROPE) {
#pragma unroll
        for (int i = 0; i < 4; ++i) x[i] = (float) v[i];
        return;
    }
    const int half = hd >> 1;                                 // (half is even, d a multiple of four: a group of four may lie across the middle)
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const int c = d + i;
        const f16 o = row[c < half ? c + half : c - half];
        x[i] = rot_odd(v[i], cos[c], o, sin[c], c < half ? -1.f : 1.f);
    }
}

template <int CODE, bool ROPE, bool IS_KEY>
__device__ __forceinline__ void append_run(const AppendArgs& a, int h, int t, int n, int page, int off)
{
    const int lane = threadIdx.x & 63;
    const f16* x0 = IS_KEY ? a.k + (size_t) t * a.k_stride + (size_t) h * a.hd : a.v + (size_t) t * a.v_stride + (size_t) h * a.hd;
    const long stride = IS_KEY ? a.k_stride : a.v_stride;
    uint8_t* codes = (IS_KEY ? a.kp : a.vp) + ((size_t) page * a.kv_heads + h) * a.block * a.hd16;
    float* scale = (IS_KEY ? a.ks : a.vs) + (size_t) page * a.kv_heads + h;
    const int per = a.hd16 >> 2, words = n * per;
    const float cap = PagedRange<CODE>::top * paged_pow2(PagedRange<CODE>::hi);
    auto fetch = [&](int w, float (&x)[4], int& i, int& d) {
        i = w / per;
        d = (w - i * per) * 4;
        const int pos = ROPE ? min(max(a.positions[t + i], 0), a.angle_rows - 1) : 0;
        append_load<ROPE && IS_KEY>(x0 + (size_t) i * stride, a.sin + (size_t) pos * a.hd, a.cos + (size_t) pos * a.hd, d, a.hd, x);
    };
    float amax = 0.f;
    for (int w = lane; w < words; w += 64) {
        float x[4]; int i, d;
        fetch(w, x, i, d);
#pragma unroll
        for (int j = 0; j < 4; ++j) amax = fmaxf(amax, fabsf(x[j]));           // (fmaxf leaves a NaN out)
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor(amax, o, 64));
    int e = paged_exp_for<CODE>(fminf(amax, cap));
    if (off > 0) {
        const int old = paged_scale_exp<CODE>(*scale);
        if (e <= old) e = old;
        else {                                                  // the earlier tokens' codes under the new scale
            const float f = paged_pow2(old - e);
            const int old_words = IS_KEY ? off * per : a.hd16 * (a.block >> 2);
            for (int w = lane; w < old_words; w += 64) {
                uint32_t* p = (uint32_t*) codes + w;
                const int first = IS_KEY ? 0 : (w % (a.block >> 2)) * 4;       // values: tokens first .. first + 3 of one column
                if (!IS_KEY && first >= off) continue;
                const uint32_t was = *p;
                float x[4];
                paged_decode4<CODE>(was, x);
                const uint32_t now = paged_encode4<CODE>(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
                const int left = IS_KEY ? 4 : off - first;
                const uint32_t mask = left >= 4 ? 0xffffffffu : (1u << (8 * left)) - 1;
                *p = (now & mask) | (was & ~mask);
            }
        }
    }
    if (lane == 0) *scale = paged_pow2(e);
    const float inv = paged_pow2(-e);
    for (int w = lane; w < words; w += 64) {
        float x[4]; int i, d;
        fetch(w, x, i, d);
        const uint32_t c = paged_encode4<CODE>(x[0] * inv, x[1] * inv, x[2] * inv, x[3] * inv);
        if (IS_KEY) *(uint32_t*) (codes + (size_t) (off + i) * a.hd16 + d) = c;
        else {
#pragma unroll
            for (int j = 0; j < 4; ++j) codes[(size_t) (d + j) * a.block + off + i] = (uint8_t) (c >> (8 * j));
        }
    }
}

// The exponent of a page that a run of largest magnitude `amax` at offset `off` joins; `old`: the exponent before (== the new one: nothing moves)
template <int CODE> __device__ __forceinline__ int append_exp(float amax, int off, const float* scale, int& old)
{
    const float cap = PagedRange<CODE>::top * paged_pow2(PagedRange<CODE>::hi);
    const int e = paged_exp_for<CODE>(fminf(amax, cap));
    old = off > 0 ? paged_scale_exp<CODE>(*scale) : e;
    return max(e, old);
}

// A run of n tokens by the whole workgroup (256 threads).  `per` = head_dim / 16 threads share a token, each with 16 of its numbers: columns
// 8 j .. 8 j + 7 of both halves of a key (what a rotation pairs), columns 16 j .. 16 j + 15 of a value.  P: passes over the tokens.
template <int CODE, bool ROPE, int P>
__device__ __forceinline__ void append_run_wide(const AppendArgs& a, int h, int t, int n, int page, int off, uint8_t* lds, float* red)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = a.hd >> 4, step = 256 / per, half = a.hd >> 1;
    const int j = tid % per, i0 = tid / per;
    const bool on = i0 < step;                                    // (256 is no multiple of head_dim / 16: 80, 96, ...)
    float k[P][16];
    f16x8 v[P][2];
    float kmax = 0.f, vmax = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int i = i0 + p * step;
        if (!on || i >= n) continue;
        const f16* kr = a.k + (size_t) (t + i) * a.k_stride + (size_t) h * a.hd + 8 * j;
        const f16* vr = a.v + (size_t) (t + i) * a.v_stride + (size_t) h * a.hd + 16 * j;
        const f16x8 lo = *(const f16x8_a8*) kr, hi = *(const f16x8_a8*) (kr + half);
        v[p][0] = *(const f16x8_a8*) vr;
        v[p][1] = *(const f16x8_a8*) (vr + 8);
        if (ROPE) {
            const size_t at = (size_t) min(max(a.positions[t + i], 0), a.angle_rows - 1) * a.hd + 8 * j;
            const f16x8 sl = *(const f16x8_a8*) (a.sin + at), sh = *(const f16x8_a8*) (a.sin + at + half);
            const f16x8 cl = *(const f16x8_a8*) (a.cos + at), ch = *(const f16x8_a8*) (a.cos + at + half);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                k[p][e] = rot_odd(lo[e], cl[e], hi[e], sl[e], -1.f);
                k[p][8 + e] = rot_odd(hi[e], ch[e], lo[e], sh[e], 1.f);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) { k[p][e] = (float) lo[e]; k[p][8 + e] = (float) hi[e]; }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            kmax = fmaxf(kmax, fabsf(k[p][e]));
            vmax = fmaxf(vmax, fabsf((float) v[p][e >> 3][e & 7]));
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { kmax = fmaxf(kmax, __shfl_xor(kmax, o, 64)); vmax = fmaxf(vmax, __shfl_xor(vmax, o, 64)); }
    __syncthreads();                                              // (the last run's LDS is free)
    if (lane == 0) { red[wave] = kmax; red[4 + wave] = vmax; }
    __syncthreads();
    kmax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    vmax = fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7]));
    const size_t ph = (size_t) page * a.kv_heads + h, at = ph * a.block * a.hd16;
    uint8_t* kc = a.kp + at;
    uint8_t* vc = a.vp + at;
    int kold, vold;
    const int ke = append_exp<CODE>(kmax, off, a.ks + ph, kold), ve = append_exp<CODE>(vmax, off, a.vs + ph, vold);
    __syncthreads();                                              // every thread has read the scales
    if (tid == 0) { a.ks[ph] = paged_pow2(ke); a.vs[ph] = paged_pow2(ve); }
    if (ke != kold) {                                             // the earlier tokens' codes under the new scale
        const float f = paged_pow2(kold - ke);
        for (int w = tid; w < off * (a.hd16 >> 2); w += 256) {
            float x[4];
            paged_decode4<CODE>(((const uint32_t*) kc)[w], x);
            ((uint32_t*) kc)[w] = paged_encode4<CODE>(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
        }
    }
    if (ve != vold) {
        const float f = paged_pow2(vold - ve);
        const int words = a.block >> 2;
        for (int w = tid; w < a.hd16 * words; w += 256) {
            const int first = (w % words) * 4;
            if (first >= off) continue;
            float x[4];
            paged_decode4<CODE>(((const uint32_t*) vc)[w], x);
            const uint32_t now = paged_encode4<CODE>(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
            if (first + 4 <= off) ((uint32_t*) vc)[w] = now;
            else for (int b = 0; b < off - first; ++b) vc[4 * w + b] = (uint8_t) (now >> (8 * b));       // (the word's other bytes belong to the new tokens)
        }
    }
    const float kinv = paged_pow2(-ke), vinv = paged_pow2(-ve);
    const int row = a.block + 4;                                  // bytes of a value column in LDS: the columns of a wave's threads lie in different banks
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int i = i0 + p * step;
        if (!on || i >= n) continue;
        uint32_t c[4];
#pragma unroll
        for (int w = 0; w < 4; ++w) c[w] = paged_encode4<CODE>(k[p][4 * w] * kinv, k[p][4 * w + 1] * kinv, k[p][4 * w + 2] * kinv, k[p][4 * w + 3] * kinv);
        uint8_t* kr = kc + (size_t) (off + i) * a.hd16 + 8 * j;
        *(uint2*) kr = make_uint2(c[0], c[1]);
        *(uint2*) (kr + half) = make_uint2(c[2], c[3]);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            const f16x8 x = v[p][w >> 1];
            const int e = (w & 1) * 4;
            const uint32_t u = paged_encode4<CODE>((float) x[e] * vinv, (float) x[e + 1] * vinv, (float) x[e + 2] * vinv, (float) x[e + 3] * vinv);
#pragma unroll
            for (int b = 0; b < 4; ++b) lds[(16 * j + 4 * w + b) * row + off + i] = (uint8_t) (u >> (8 * b));
        }
    }
    __syncthreads();
    const int pieces = a.block >> 4;                              // 16 tokens of a column at a time
    for (int w = tid; w < a.hd * pieces; w += 256) {
        const int d = w / pieces, first = (w % pieces) * 16;
        const uint8_t* src = lds + d * row + first;
        uint8_t* dst = vc + (size_t) d * a.block + first;
        if (first >= off && first + 16 <= off + n) {
            const uint32_t* x = (const uint32_t*) src;
            *(uint4*) dst = make_uint4(x[0], x[1], x[2], x[3]);
        } else {
            for (int b = max(first, off); b < min(first + 16, off + n); ++b) dst[b - first] = src[b - first];
        }
    }
}

// One workgroup = `chunk` token rows of one head: it does the runs that begin there.  P = 0: a wave for every run.
template <int CODE, bool ROPE, int P> __global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float red[8];
    __shared__ int longs[16][4];                                  // the long runs: token row, tokens, page, offset
    __shared__ int count;
    const int h = blockIdx.y, lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int t0 = blockIdx.x * a.chunk, t1 = min(t0 + a.chunk, a.rows);
    if (P) {
        if (threadIdx.x == 0) count = 0;
        __syncthreads();
    }
    for (int t = t0 + wave; t < t1; t += 4) {
        const int slot = a.slots[t];
        if (slot < 0 || slot / a.block >= a.blocks) continue;
        const int page = slot / a.block, off = slot % a.block;
        if (t > 0 && off > 0 && a.slots[t - 1] == slot - 1) continue;          // not the first of its run
        int n = 1;                                              // lanes look at the following rows
        for (int base = 1; base < a.block - off; base += 64) {
            const int i = base + lane;
            const bool on = i < a.block - off && t + i < a.rows && a.slots[t + i] == slot + i;
            const uint64_t m = __ballot(!on);
            n = base + (m ? __ffsll((unsigned long long) m) - 1 : 64);
            if (m) break;
        }
        n = min(n, a.block - off);
        if (P && n >= APPEND_LONG) {
            if (lane == 0) { const int x = atomicAdd(&count, 1); longs[x][0] = t; longs[x][1] = n; longs[x][2] = page; longs[x][3] = off; }
            continue;
        }
        append_run<CODE, ROPE, true>(a, h, t, n, page, off);
        append_run<CODE, ROPE, false>(a, h, t, n, page, off);
    }
    if (P) {
        __syncthreads();
        for (int x = 0; x < count; ++x)                           // (runs of different pages: their order does not matter)
            append_run_wide<CODE, ROPE, P ? P : 1>(a, h, longs[x][0], longs[x][1], longs[x][2], longs[x][3], lds, red);
    }
}

extern "C" int exl_paged_append(const void* key_states, const void* value_states, long key_stride, long value_stride, const int32_t* slots, int rows,
                                void* key_pages, void* value_pages, float* key_scales, float* value_scales, int code, int num_blocks, int num_kv_heads,
                                int block_size, int head_dim, const int32_t* positions, const void* sin, const void* cos, int angle_rows, void* stream)
{
    EXL_REQUIRE(key_states && value_states && slots && key_pages && value_pages && key_scales && value_scales, EXL_E_INVALID, "paged_append: null pointer");
    EXL_REQUIRE(rows >= 0 && num_blocks > 0 && num_kv_heads > 0 && num_kv_heads <= 65535, EXL_E_INVALID, "paged_append: bad shape");
    EXL_TRY(paged_check_block("paged_append", block_size, num_blocks));
    EXL_TRY(paged_check_head("paged_append", code, head_dim));
    EXL_REQUIRE((sin == nullptr) == (cos == nullptr) && (!sin || (positions && angle_rows > 0)), EXL_E_INVALID,
                "paged_append: a rotation needs sin, cos and positions");
    EXL_REQUIRE(key_stride >= (long) num_kv_heads * head_dim && value_stride >= (long) num_kv_heads * head_dim && key_stride % 4 == 0 &&
                value_stride % 4 == 0 && ((uintptr_t) key_states | (uintptr_t) value_states) % 8 == 0, EXL_E_INVALID,
                "paged_append: key / value rows must be 8-byte aligned and at least kv_heads * head_dim apart");
    EXL_REQUIRE(((uintptr_t) key_pages | (uintptr_t) value_pages) % 16 == 0, EXL_E_INVALID, "paged_append: pages must be 16-byte aligned");
    if (rows == 0) return 0;
    AppendArgs a = {(const f16*) key_states, (const f16*) value_states, slots, positions, (const f16*) sin, (const f16*) cos,
                    (uint8_t*) key_pages, (uint8_t*) value_pages, key_scales, value_scales, rows, num_kv_heads, head_dim, (head_dim + 15) / 16 * 16,
                    block_size, num_blocks, 4, angle_rows, key_stride, value_stride};
    const int passes = head_dim % 16 ? 0 : (block_size * (head_dim / 16) + 255) / 256;       // (256 / (head_dim / 16) tokens a pass, or a few less)
    a.chunk = (long) rows * num_kv_heads <= 16384 ? 4 : 16;       // few rows: a run for every wave at once
    const dim3 grid((unsigned) ((rows + a.chunk - 1L) / a.chunk), (unsigned) num_kv_heads);
    const size_t lds = passes ? (size_t) head_dim * (block_size + 4) : 0;
    hipStream_t s = (hipStream_t) stream;
    const int p = !passes ? 0 : passes * (256 / (head_dim / 16)) >= block_size ? passes : passes + 1;
#define APPEND(C, R, P) hipLaunchKernelGGL((paged_append_kernel<C, R, P>), grid, dim3(256), lds, s, a)
#define APPEND_P(C, R) do { if (p == 0) APPEND(C, R, 0); else if (p == 1) APPEND(C, R, 1); else if (p == 2) APPEND(C, R, 2); else if (p <= 4) APPEND(C, R, 4); \
                            else APPEND(C, R, 8); } while (0)
    if (code == EXL_PAGE_FP8) { if (sin) APPEND_P(EXL_PAGE_FP8, true); else APPEND_P(EXL_PAGE_FP8, false); }
    else                      { if (sin) APPEND_P(EXL_PAGE_INT8, true); else APPEND_P(EXL_PAGE_INT8, false); }
#undef APPEND_P
#undef APPEND
    EXL_LAUNCH_CHECK();
    return 0;
}

int paged_check_head(const char* what, int code, int head_dim)
{
    EXL_REQUIRE(code == EXL_PAGE_FP8 || code == EXL_PAGE_INT8, EXL_E_INVALID, "%s: unknown page code %d", what, code);
    EXL_REQUIRE(head_dim > 0 && head_dim <= 256 && head_dim % 4 == 0, EXL_E_UNSUPPORTED, "%s: head_dim (%d) must be a multiple of 4, at most 256", what,
                head_dim);
    return 0;
}
