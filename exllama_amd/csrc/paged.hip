// The paged 8-bit cache (paged.h): block tables and slot maps from request lengths, and the append of new keys and values.
#include "paged.h"
#include <type_traits>

// ---- block tables and slot maps ---------------------------------------------------------------------------------------------------
// For every row b, in order (all sums exclusive prefix sums over the rows):
//   take  = clamp(new, 0, min(max_new, rows - start)), start = sum(take)  (row_stride > 0: start = b * row_stride)
//   want  = max(0, ceil(min(past + take, max_len) / block) - held), got = clamp(avail - sum(want), 0, want)
//   table[held + i] = ring[(head + sum(want) + i) mod blocks], i < got
//   new < 0: the row has ended; its blocks go to the ring's end in order, its table entries become -1
//   past > held * block, and new or held > 0: earlier tokens found no block.  want = 0, what the row lacks counts as missing: a block handed out now would
//   begin with what another row left in it, in place of those tokens
// Then every token row's slot = table[pos / block] * block + pos % block.  Latency is all that matters (a step of 256 rows moves
// 7 KB): one workgroup does both halves where the work is small, otherwise the scan runs in one workgroup and the filling in
// many -- a second launch instead of a grid-wide wait.  Measured, us, one workgroup / scan + filling and
// another launch: one row 3.0 / 2.8 + 1.6, 64 rows of 64 tokens 3.9 / 3.4 + 3.1, 256 rows 7.2 / 3.5 + 2.5, 512 rows (the limit) 9.2 / 5.2 + 3.5;
// 2048 prompts of 300 k tokens 8.1 + 5.5 (2.4 MB of slots and positions).
struct SlotRow { int start, take, past, kept, held, base, back, gone; };      // 32 bytes a row

struct SlotArgs {
    const int32_t* past; const int32_t* fresh; int32_t* held; int32_t* table; int32_t* ring; int32_t* counters;
    int n, width, lbs, blocks, max_len, max_new, rows, row_stride;               // lbs: log2 of the block size
    int32_t* starts; int32_t* slots; int32_t* positions;
};

#define SLOT_THREADS 1024
#define SLOT_WAVES (SLOT_THREADS / 64)
#define SLOT_SMALL_ROWS 512                                       // rows and token rows up to which one workgroup does it all
#define SLOT_SMALL_TOKENS 4096

// exclusive prefix sum over the workgroup, and the total; `lds`: SLOT_WAVES entries.  Up to 64 rows only the first wave has numbers: no barrier.
__device__ __forceinline__ int64_t slot_scan(int64_t v, int64_t* lds, bool one_wave, int64_t& total)
{
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int64_t inc = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int64_t o = __shfl_up(inc, off, 64);
        if (lane >= off) inc += o;
    }
    total = __shfl(inc, 63, 64);
    if (one_wave) return inc - v;
    __syncthreads();                                              // (the last sums have been read)
    if (lane == 63) lds[wave] = inc;
    __syncthreads();
    int64_t before = lds[lane & (SLOT_WAVES - 1)];                // every wave scans the waves' sums for itself
#pragma unroll
    for (int off = 1; off < SLOT_WAVES; off <<= 1) {
        const int64_t o = __shfl_up(before, off, SLOT_WAVES);
        if ((lane & (SLOT_WAVES - 1)) >= off) before += o;
    }
    total = __shfl(before, SLOT_WAVES - 1, 64);
    const int64_t mine = __shfl(before, wave ? wave - 1 : 0, 64);
    return inc - v + (wave ? mine : 0);
}

// R consecutive rows for a thread
template <int R> __device__ __forceinline__ void slot_scan_rows(const SlotArgs& a, SlotRow* desc)
{
    __shared__ int64_t lds[SLOT_WAVES];
    __shared__ unsigned long long lacking;                        // blocks that rows without their earlier tokens' lack
    const bool one_wave = a.n <= 64 * R;
    if (one_wave && threadIdx.x >= 64) return;
    if (threadIdx.x == 0) lacking = 0;                            // (a scan's barrier, or in one wave this fence, stands between this and the first sum)
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int head = (int) ((uint32_t) a.counters[0] % (uint32_t) a.blocks);
    const int avail = min(max(a.counters[1], 0), a.blocks);
    int64_t rows_before = 0, want_before = 0, back_before = 0;
    for (int b0 = 0; b0 < a.n; b0 += SLOT_THREADS * R) {
        const int first = b0 + threadIdx.x * R;
        int fresh[R], held[R], past[R], take[R], start[R], want[R], back[R], lost[R];
        int64_t mine = 0, total;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            const bool in = first + i < a.n;
            fresh[i] = in ? a.fresh[first + i] : 0;
            held[i] = in ? a.held[first + i] : 0;
            past[i] = in ? a.past[first + i] : 0;
        }
#pragma unroll
        for (int i = 0; i < R; ++i) {
            held[i] = min(max(held[i], 0), a.width);
            past[i] = max(past[i], 0);
            take[i] = min(max(fresh[i], 0), a.max_new);
            mine += take[i];
        }
        int64_t at = 0;
        if (a.row_stride <= 0) {
            at = rows_before + slot_scan(mine, lds, one_wave, total);
            rows_before += total;
        }
        mine = 0;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (a.row_stride > 0) {
                at = (int64_t) (first + i) * a.row_stride;
                take[i] = min(take[i], a.row_stride);
            }
            start[i] = (int) min(at, (int64_t) a.rows);
            at += take[i];
            take[i] = min(take[i], a.rows - start[i]);
            const int end = (int) min((int64_t) past[i] + take[i], (int64_t) a.max_len);
            const int need = (int) (((int64_t) end + (1 << a.lbs) - 1) >> a.lbs);
            want[i] = first + i < a.n && fresh[i] >= 0 ? max(0, need - held[i]) : 0;
            lost[i] = (fresh[i] > 0 || held[i] > 0) && (past[i] - 1) >> a.lbs >= held[i] ? want[i] : 0;
            want[i] -= lost[i];
            back[i] = fresh[i] < 0 ? held[i] : 0;
            mine += (int64_t) want[i] << 32 | back[i];
        }
        const int64_t both = slot_scan(mine, lds, one_wave, total);      // (both sums are less than the table's entries: 2^31)
        int64_t base = want_before + (both >> 32), back_base = back_before + (both & 0xffffffff);
        want_before += total >> 32;
        back_before += total & 0xffffffff;
#pragma unroll
        for (int i = 0; i < R; ++i) {
            if (first + i >= a.n) break;
            if (lost[i]) atomicAdd(&lacking, (unsigned long long) lost[i]);
            const int got = (int) min(max((int64_t) avail - base, (int64_t) 0), (int64_t) want[i]);
            SlotRow r;
            r.start = start[i]; r.take = take[i]; r.past = past[i]; r.held = held[i];
            r.gone = fresh[i] < 0;
            r.kept = r.gone ? 0 : held[i] + got;
            r.base = got ? (int) (head + base < a.blocks ? head + base : head + base - a.blocks) : 0;      // (got: base < avail <= blocks)
            r.back = r.gone ? (int) ((head + avail + back_base) % a.blocks) : 0;
            desc[first + i] = r;
            a.starts[first + i] = start[i];
            a.held[first + i] = r.kept;
            base += want[i];
            back_base += back[i];
        }
    }
    if (!one_wave) __syncthreads();                               // every thread has read the counters, and added what its rows lack
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    if (threadIdx.x == 0) {
        const int got = (int) min(want_before, (int64_t) avail);
        a.counters[0] = (head + got) % a.blocks;
        a.counters[1] = (int) min((int64_t) avail - got + back_before, (int64_t) a.blocks);
        a.counters[2] = (int) min(want_before - got + (int64_t) lacking, (int64_t) 0x7fffffff);
        a.counters[3] = 0;
        a.starts[a.n] = (int) min(a.row_stride > 0 ? (int64_t) a.n * a.row_stride : rows_before, (int64_t) a.rows);
    }
}

__device__ __forceinline__ int slot_ring(const SlotArgs& a, int at) { return a.ring[at >= a.blocks ? at - a.blocks : at]; }

// the table and the ring of rows first, first + step, ... (a wave each)
__device__ __forceinline__ void slot_fill_rows(const SlotArgs& a, const SlotRow* desc, int first, int step)
{
    const int lane = threadIdx.x & 63;
    for (int b = first; b < a.n; b += step) {
        const SlotRow r = desc[b];
        int32_t* row = a.table + (size_t) b * a.width;
        if (r.gone) {
            for (int i = lane; i < r.held; i += 64) {
                const int at = (int) (((uint32_t) r.back + (uint32_t) i) % (uint32_t) a.blocks);
                a.ring[at] = row[i];
                row[i] = -1;
            }
        } else {
            for (int i = r.held + lane; i < r.kept; i += 64) row[i] = slot_ring(a, r.base + i - r.held);
        }
    }
}

// the slots and positions of token rows first, first + step, ...
__device__ __forceinline__ void slot_fill_tokens(const SlotArgs& a, const SlotRow* desc, int first, int step)
{
    for (int t = first; t < a.rows; t += step) {
        int lo = 0, hi = a.n;                                 // the last row that starts at or before t (rows of no token share a start: the last one)
        if (a.row_stride > 0) lo = min(t / a.row_stride, a.n - 1);
        else while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (desc[mid].start <= t) lo = mid; else hi = mid; }
        const SlotRow r = desc[lo];
        const int i = t - r.start;
        int slot = -1, pos = 0;
        if (i < r.take) {
            pos = (int) min((int64_t) r.past + i, (int64_t) 0x7fffffff);
            const int k = pos >> a.lbs;
            if (pos < a.max_len && k < r.kept) {
                // (entries that this call adds are still being written by other waves: they are read where they come from)
                const int id = k < r.held ? a.table[(size_t) lo * a.width + k] : slot_ring(a, r.base + k - r.held);
                if (id >= 0 && id < a.blocks) slot = (id << a.lbs) + (pos & ((1 << a.lbs) - 1));
            }
        }
        a.slots[t] = slot;
        a.positions[t] = pos;
    }
}

__global__ __launch_bounds__(SLOT_THREADS) void paged_slots_small_kernel(SlotArgs a)
{
    __shared__ SlotRow desc[SLOT_SMALL_ROWS];
    slot_scan_rows<1>(a, desc);
    __syncthreads();
    slot_fill_tokens(a, desc, threadIdx.x, SLOT_THREADS);
    slot_fill_rows(a, desc, threadIdx.x >> 6, SLOT_WAVES);
}

__global__ __launch_bounds__(SLOT_THREADS) void paged_slots_scan_kernel(SlotArgs a, SlotRow* desc) { slot_scan_rows<4>(a, desc); }

__global__ __launch_bounds__(256) void paged_slots_fill_kernel(SlotArgs a, const SlotRow* desc, int token_groups)
{
    if ((int) blockIdx.x < token_groups) slot_fill_tokens(a, desc, blockIdx.x * 256 + threadIdx.x, token_groups * 256);
    else slot_fill_rows(a, desc, (blockIdx.x - token_groups) * 4 + (threadIdx.x >> 6), (gridDim.x - token_groups) * 4);
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
    EXL_REQUIRE((int64_t) n_rows * table_width < 0x7fffffff, EXL_E_UNSUPPORTED, "paged_slots: the block table exceeds 2^31 entries");
    SlotArgs a = {past_lens, new_lens, held, block_table, ring, counters, n_rows, table_width, 31 - __builtin_clz((unsigned) block_size), num_blocks, max_len,
                  max_new, rows, row_stride, starts, slots, positions};
    hipStream_t s = (hipStream_t) stream;
    if (rows <= SLOT_SMALL_TOKENS && n_rows <= SLOT_SMALL_ROWS) {
        hipLaunchKernelGGL(paged_slots_small_kernel, dim3(1), dim3(SLOT_THREADS), 0, s, a);
    } else {
        hipLaunchKernelGGL(paged_slots_scan_kernel, dim3(1), dim3(SLOT_THREADS), 0, s, a, (SlotRow*) scratch);
        EXL_LAUNCH_CHECK();
        const int tg = (int) ((rows + 255L) / 256 < 2048 ? (rows + 255L) / 256 : 2048), rg = (n_rows + 3) / 4 < 2048 ? (n_rows + 3) / 4 : 2048;
        hipLaunchKernelGGL(paged_slots_fill_kernel, dim3(tg + rg), dim3(256), 0, s, a, (const SlotRow*) scratch, tg);
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
// Keys are rotated first when sin / cos are given; the code is one rounding of the exact rotation.  Short runs (single tokens, a few drafted
// ones) take a wave each; from APPEND_LONG tokens on, and head_dim % 16 == 0, the whole workgroup takes the run: every number is read once and
// stays in registers between the maximum and the rounding, and the values' codes are transposed in LDS.  (APPEND_LONG 4 / 8 / 32: 300 runs of 6
// tokens x 8 heads 19 / 16 / 16 us, 128 of 16 13 / 15 / 22, 30 k ragged tokens 42 / 42 / 53.)
// Bound by HBM for long runs (30 k ragged int8 tokens x 8 heads, 188 MB: 39 us = 4.8 TB/s; a prompt of 2048 x 32 heads with rotation, 51 MB: 18.8 us =
// 2.7 TB/s, one round of workgroups), by latency for few (64 tokens x 8 heads: 5.6 us), by the values' columns for many single tokens (1024 x 32
// heads 93 us: a token's value touches every line of its 8 KB page, which attention reads in whole lines for it).
struct AppendArgs {
    const f16* k; const f16* v; const int32_t* slots; const int32_t* positions; const f16* sin; const f16* cos;
    uint8_t* kp; uint8_t* vp; float* ks; float* vs;
    int rows, kv_heads, hd, hd16, lbs, blocks, chunk, angle_rows;  // lbs: log2 of the block size
    int k_stride, v_stride;
    uint32_t by_words, by_16, by_4;                               // dividing thread numbers by hd16 / 4, hd / 16 and hd / 4: n * by >> 32
};

// n / d for n < 2^16, d <= 64 (by = 2^32 / d rounded up, 0 for d = 1); a division by a number in a register is twenty instructions
__device__ __forceinline__ int over(int n, uint32_t by) { return by ? (int) __umulhi((uint32_t) n, by) : n; }

#define APPEND_LONG 8

// a * b + sign * c * d of fp16 numbers as a 32-bit number that rounds to a code (7 bits at most) and compares with a scale's border as the
// exact one does.  One fma of an exact product rounds once; a second rounding can only go wrong where the first ended on a border, that
// is with 15 zeros below: there the sum is rounded to odd instead (its error is exact by Knuth's two-sum; an inexact even sum moves one
// step towards the exact one).  Rounding every sum to odd made 16 instructions a number instead of 5.
__device__ __forceinline__ float rot_code(f16 a, f16 b, f16 c, f16 d, float sign)
{
#pragma clang fp contract(off)
    const float q = (float) c * (float) d * sign;
    float s = __builtin_fmaf((float) a, (float) b, q);
    if (__any((__float_as_uint(s) & 0x7fff) == 0)) {
        const float p = (float) a * (float) b;
        const float bb = s - p;
        const float err = (p - (s - bb)) + (q - bb);
        const uint32_t u = __float_as_uint(s);
        if (!(u & 1) && (err < 0.f || err > 0.f)) s = __uint_as_float((err < 0.f) == (s < 0.f) ? u + 1 : u - 1);
    }
    return s;
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
        x[i] = rot_code(v[i], cos[c], o, sin[c], c < half ? -1.f : 1.f);
    }
}

// The exponent of a page that numbers of largest magnitude `amax` join at offset `off`; `old`: the exponent before (== the new one: nothing moves)
template <int CODE> __device__ __forceinline__ int append_exp(float amax, int off, float scale, int& old)
{
    const float cap = PagedRange<CODE>::top * paged_pow2(PagedRange<CODE>::hi);
    const int e = paged_exp_for<CODE>(fminf(amax, cap));
    old = off > 0 ? paged_scale_exp<CODE>(scale) : e;
    return max(e, old);
}

// The codes of a page's first `off` tokens under a scale that is 1 / f of what it was, by `threads` threads
template <int CODE> __device__ __forceinline__ void append_move_keys(uint8_t* codes, int off, int hd16, float f, int thread, int threads)
{
    for (int w = thread; w < off * (hd16 >> 2); w += threads) {
        float x[4];
        paged_decode4<CODE>(((const uint32_t*) codes)[w], x);
        ((uint32_t*) codes)[w] = paged_encode4<CODE, false>(x[0], x[1], x[2], x[3], f);
    }
}
template <int CODE> __device__ __forceinline__ void append_move_values(uint8_t* codes, int off, int hd16, int lbs, float f, int thread, int threads)
{
    for (int w = thread; w < hd16 << (lbs - 2); w += threads) {
        const int first = (w & ((1 << (lbs - 2)) - 1)) * 4;
        if (first >= off) continue;
        float x[4];
        paged_decode4<CODE>(((const uint32_t*) codes)[w], x);
        const uint32_t now = paged_encode4<CODE, false>(x[0], x[1], x[2], x[3], f);
        if (first + 4 <= off) ((uint32_t*) codes)[w] = now;
        else for (int b = 0; b < off - first; ++b) codes[4 * w + b] = (uint8_t) (now >> (8 * b));          // (the word's other bytes belong to the new tokens)
    }
}

// A short run by one wave: a lane has four columns of a token, of the key and of the value at once (one round of loads and one of shuffles).
template <int CODE, bool ROPE> __device__ __forceinline__ void append_run(const AppendArgs& a, int h, int t, int n, int page, int off)
{
    const int lane = threadIdx.x & 63;
    const f16* k0 = a.k + (size_t) t * a.k_stride + (size_t) h * a.hd;
    const f16* v0 = a.v + (size_t) t * a.v_stride + (size_t) h * a.hd;
    const size_t ph = (size_t) page * a.kv_heads + h, at = ph * a.hd16 << a.lbs;
    uint8_t* kc = a.kp + at;
    uint8_t* vc = a.vp + at;
    const float kscale = a.ks[ph], vscale = a.vs[ph];
    const int per = a.hd16 >> 2, words = n * per;
    const float cap = PagedRange<CODE>::top * paged_pow2(PagedRange<CODE>::hi);
    auto fetch = [&](int w, float (&k)[4], float (&v)[4], int& i, int& d) {
        i = over(w, a.by_words);
        d = (w - i * per) * 4;
        const int pos = ROPE ? min(max(a.positions[t + i], 0), a.angle_rows - 1) : 0;
        append_load<false>(v0 + (size_t) i * a.v_stride, nullptr, nullptr, d, a.hd, v);
        append_load<ROPE>(k0 + (size_t) i * a.k_stride, a.sin + (size_t) pos * a.hd, a.cos + (size_t) pos * a.hd, d, a.hd, k);
    };
    float k[4], v[4], kmax = 0.f, vmax = 0.f;
    int i, d;
    for (int w = lane; w < words; w += 64) {
        fetch(w, k, v, i, d);
#pragma unroll
        for (int j = 0; j < 4; ++j) { kmax = fmaxf(kmax, fabsf(k[j])); vmax = fmaxf(vmax, fabsf(v[j])); }       // (fmaxf leaves a NaN out)
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { kmax = fmaxf(kmax, __shfl_xor(kmax, o, 64)); vmax = fmaxf(vmax, __shfl_xor(vmax, o, 64)); }
    int kold, vold;
    const int ke = append_exp<CODE>(kmax, off, kscale, kold), ve = append_exp<CODE>(vmax, off, vscale, vold);
    if (ke != kold) append_move_keys<CODE>(kc, off, a.hd16, paged_pow2(kold - ke), lane, 64);
    if (ve != vold) append_move_values<CODE>(vc, off, a.hd16, a.lbs, paged_pow2(vold - ve), lane, 64);
    if (lane == 0) { a.ks[ph] = paged_pow2(ke); a.vs[ph] = paged_pow2(ve); }
    const float kinv = paged_pow2(-ke), vinv = paged_pow2(-ve);
    const bool big = kmax > cap || vmax > cap;
    for (int w = lane; w < words; w += 64) {
        if (words > 64) fetch(w, k, v, i, d);
        const uint32_t x = big ? paged_encode4<CODE, true>(k[0], k[1], k[2], k[3], kinv) : paged_encode4<CODE, false>(k[0], k[1], k[2], k[3], kinv);
        const uint32_t y = big ? paged_encode4<CODE, true>(v[0], v[1], v[2], v[3], vinv) : paged_encode4<CODE, false>(v[0], v[1], v[2], v[3], vinv);
        *(uint32_t*) (kc + (off + i) * a.hd16 + d) = x;
#pragma unroll
        for (int j = 0; j < 4; ++j) vc[((d + j) << a.lbs) + off + i] = (uint8_t) (y >> (8 * j));
    }
}

// A run of n tokens by the whole workgroup (256 threads).  Keys: head_dim / 16 threads share a token, each with columns 8 j .. 8 j + 7 of both
// halves (what a rotation pairs).  Values: a thread has four columns of four tokens that make up one word of each column in the page,
// so that they are transposed by the encoding itself.  P: passes of 256 threads over the page, keys and values alike.
template <int CODE, bool ROPE, int P>
__device__ __forceinline__ void append_run_wide(const AppendArgs& a, int h, int t, int n, int page, int off, uint8_t* lds, float* red)
{
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int per = a.hd >> 4, half = a.hd >> 1, cols = a.hd >> 2, step = over(256, a.by_16);
    const int i0 = over(tid, a.by_16), j = tid - i0 * per;        // (256 need not be a multiple of head_dim / 16: the last threads then repeat)
    const int w0 = off >> 2, words = ((off + n - 1) >> 2) - w0 + 1;
    const f16* k0 = a.k + (size_t) t * a.k_stride + (size_t) h * a.hd + 8 * j;
    const f16* v0 = a.v + (size_t) t * a.v_stride + (size_t) h * a.hd;
    const size_t ph = (size_t) page * a.kv_heads + h, at = ph * a.hd16 << a.lbs;
    uint8_t* kc = a.kp + at;
    uint8_t* vc = a.vp + at;
    const float kscale = a.ks[ph], vscale = a.vs[ph];
    // all loads go out before anything is computed; threads behind the run's end repeat its last token, which changes no maximum
    f16x8 lo[P], hi[P];
    f16x4 v[P][4];
    int pos[P];
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int i = min(i0 + p * step, n - 1);
        lo[p] = *(const f16x8_a8*) (k0 + i * a.k_stride);
        hi[p] = *(const f16x8_a8*) (k0 + i * a.k_stride + half);
        if (ROPE) pos[p] = a.positions[t + i];
    }
#pragma unroll
    for (int p = 0; p < P; ++p) {
        const int x = tid + 256 * p, w = over(x, a.by_4), d = 4 * (x - w * cols), i = 4 * (w0 + min(w, words - 1)) - off;
#pragma unroll
        for (int b = 0; b < 4; ++b) v[p][b] = *(const f16x4_a4*) (v0 + min(max(i + b, 0), n - 1) * a.v_stride + d);
    }
    float k[P][16], kmax = 0.f, vmax = 0.f;
#pragma unroll
    for (int p = 0; p < P; ++p) {
        if (ROPE) {
            const size_t to = (size_t) min(max(pos[p], 0), a.angle_rows - 1) * a.hd + 8 * j;
            const f16x8 sl = *(const f16x8_a2*) (a.sin + to), sh = *(const f16x8_a2*) (a.sin + to + half);
            const f16x8 cl = *(const f16x8_a2*) (a.cos + to), ch = *(const f16x8_a2*) (a.cos + to + half);
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                k[p][e] = rot_code(lo[p][e], cl[e], hi[p][e], sl[e], -1.f);
                k[p][8 + e] = rot_code(hi[p][e], ch[e], lo[p][e], sh[e], 1.f);
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) { k[p][e] = (float) lo[p][e]; k[p][8 + e] = (float) hi[p][e]; }
        }
#pragma unroll
        for (int e = 0; e < 16; ++e) {
            kmax = fmaxf(kmax, fabsf(k[p][e]));
            vmax = fmaxf(vmax, fabsf((float) v[p][e >> 2][e & 3]));
        }
    }
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) { kmax = fmaxf(kmax, __shfl_xor(kmax, o, 64)); vmax = fmaxf(vmax, __shfl_xor(vmax, o, 64)); }
    __syncthreads();                                              // (the last run's LDS is free; every thread has read the scales)
    if (lane == 0) { red[wave] = kmax; red[4 + wave] = vmax; }
    __syncthreads();
    kmax = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
    vmax = fmaxf(fmaxf(red[4], red[5]), fmaxf(red[6], red[7]));
    int kold, vold;
    const int ke = append_exp<CODE>(kmax, off, kscale, kold), ve = append_exp<CODE>(vmax, off, vscale, vold);
    if (ke != kold) append_move_keys<CODE>(kc, off, a.hd16, paged_pow2(kold - ke), tid, 256);
    if (ve != vold) append_move_values<CODE>(vc, off, a.hd16, a.lbs, paged_pow2(vold - ve), tid, 256);
    if (tid == 0) { a.ks[ph] = paged_pow2(ke); a.vs[ph] = paged_pow2(ve); }
    const float kinv = paged_pow2(-ke), vinv = paged_pow2(-ve), cap = PagedRange<CODE>::top * paged_pow2(PagedRange<CODE>::hi);
    const int row = (1 << a.lbs) + 4;                             // bytes of a value column in LDS: the columns of a wave's threads lie in different banks
    auto encode = [&](auto saturate) {
        constexpr bool S = decltype(saturate)::value;
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int i = i0 + p * step;
            uint32_t c[4];
#pragma unroll
            for (int w = 0; w < 4; ++w) c[w] = paged_encode4<CODE, S>(k[p][4 * w], k[p][4 * w + 1], k[p][4 * w + 2], k[p][4 * w + 3], kinv);
            uint8_t* kr = kc + (off + i) * a.hd16 + 8 * j;
            if (i0 < step && i < n) {
                *(uint2*) kr = make_uint2(c[0], c[1]);
                *(uint2*) (kr + half) = make_uint2(c[2], c[3]);
            }
        }
#pragma unroll
        for (int p = 0; p < P; ++p) {
            const int x = tid + 256 * p, w = over(x, a.by_4);
            uint8_t* dst = lds + 4 * (x - w * cols) * row + 4 * (w0 + w);
            if (w < words)
#pragma unroll
                for (int e = 0; e < 4; ++e)
                    *(uint32_t*) (dst + e * row) = paged_encode4<CODE, S>((float) v[p][0][e], (float) v[p][1][e], (float) v[p][2][e], (float) v[p][3][e], vinv);
        }
    };
    if (kmax > cap || vmax > cap) encode(std::true_type()); else encode(std::false_type());
    __syncthreads();
    for (int w = tid; w < a.hd << (a.lbs - 4); w += 256) {         // 16 tokens of a column at a time
        const int d = w >> (a.lbs - 4), first = (w & ((1 << (a.lbs - 4)) - 1)) * 16;
        const uint8_t* src = lds + d * row + first;
        uint8_t* dst = vc + (d << a.lbs) + first;
        if (first >= off && first + 16 <= off + n) {
            const uint32_t* x = (const uint32_t*) src;
            *(uint4*) dst = make_uint4(x[0], x[1], x[2], x[3]);
        } else {
            for (int b = max(first, off); b < min(first + 16, off + n); ++b) dst[b - first] = src[b - first];
        }
    }
}

// One workgroup = `chunk` (at most 63) token rows of one head: it does the runs that begin there.  The chunk's slots and the page that may follow
// (at most 63 + 127 of them, and the one before) are read in one round of loads, by one wave for all four (they have to agree on the runs whatever happens to the
// slots meanwhile); a bit for each row says whether it continues the row before it.
// P = 0, head_dim no multiple of 16: a wave for every run, its codes stored byte by byte, however long: a prompt of 2048 x 32 heads of 100 takes
// 127 us, of 112 19.5 (single tokens, 64 x 32 heads: 7.6 and 8.2).
template <int CODE, bool ROPE, int P> __global__ __launch_bounds__(256) void paged_append_kernel(AppendArgs a)
{
    extern __shared__ __attribute__((aligned(16))) uint8_t lds[];
    __shared__ float red[8];
    __shared__ int slots[192];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    // heads next to each other in launch order: what runs at one time reads whole token rows
    const int h = blockIdx.x % a.kv_heads, t0 = (int) (blockIdx.x / a.kv_heads) * a.chunk, count = min(a.chunk, a.rows - t0);
    int slot[3];                                                  // of token rows t0 - 1 + lane + 64 i
    uint64_t on[4];                                               // bit: the row continues the one before it
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        const int64_t t = (int64_t) t0 - 1 + lane + 64 * i;
        if (wave == 0) slots[lane + 64 * i] = t >= 0 && t < a.rows ? a.slots[t] : -1;
    }
    __syncthreads();
#pragma unroll
    for (int i = 0; i < 3; ++i) slot[i] = slots[lane + 64 * i];
#pragma unroll
    for (int i = 0; i < 3; ++i) {
        int before = __shfl_up(slot[i], 1, 64);
        if (i) { const int last = __shfl(slot[i ? i - 1 : 0], 63, 64); if (lane == 0) before = last; }
        else if (lane == 0) before = -2;
        on[i] = __ballot(slot[i] > 0 && (slot[i] & ((1 << a.lbs) - 1)) != 0 && slot[i] == before + 1);
    }
    on[3] = 0;
    const int page_here = slot[0] >> a.lbs;
    const uint64_t starts = __ballot(slot[0] >= 0 && page_here < a.blocks) & ~on[0];
    for (int x = 0, nth = 0; x < count; ++x) {
        if (!(starts >> (x + 1) & 1)) continue;
        const int s = __shfl(slot[0], x + 1, 64), page = s >> a.lbs, off = s & ((1 << a.lbs) - 1);
        int n = 1, at = x + 2;                                    // the ones that follow
        while (at < 192) {
            const uint64_t rest = ~(on[at >> 6] >> (at & 63));    // (zeros come in from above: the word ends the stretch at the latest)
            const int ones = rest ? __ffsll((unsigned long long) rest) - 1 : 64, room = 64 - (at & 63);
            n += min(ones, room);
            at += min(ones, room);
            if (ones < room) break;
        }
        n = min(n, (1 << a.lbs) - off);
        if (P && n >= APPEND_LONG) {
            append_run_wide<CODE, ROPE, P ? P : 1>(a, h, t0 + x, n, page, off, lds, red);
        } else if ((nth++ & 3) == wave) {
            append_run<CODE, ROPE>(a, h, t0 + x, n, page, off);
        }
    }
}

extern "C" int exl_paged_append(const void* key_states, const void* value_states, long key_stride, long value_stride, const int32_t* slots, int rows,
                                void* key_pages, void* value_pages, float* key_scales, float* value_scales, int code, int num_blocks, int num_kv_heads,
                                int block_size, int head_dim, const int32_t* positions, const void* sin, const void* cos, int angle_rows, void* stream)
{
    EXL_REQUIRE(((key_states && value_states && slots) || rows == 0) && key_pages && value_pages && key_scales && value_scales, EXL_E_INVALID,
                "paged_append: null pointer");                    // (empty tensors have no address)
    EXL_REQUIRE(rows >= 0 && num_blocks > 0 && num_kv_heads > 0 && num_kv_heads <= 65535, EXL_E_INVALID, "paged_append: bad shape");
    EXL_TRY(paged_check_block("paged_append", block_size, num_blocks));
    EXL_TRY(paged_check_head("paged_append", code, head_dim));
    EXL_REQUIRE((sin == nullptr) == (cos == nullptr) && (!sin || ((positions || rows == 0) && angle_rows > 0)), EXL_E_INVALID,
                "paged_append: a rotation needs sin, cos and positions");
    EXL_REQUIRE(key_stride >= (long) num_kv_heads * head_dim && value_stride >= (long) num_kv_heads * head_dim && key_stride % 4 == 0 &&
                value_stride % 4 == 0 && ((uintptr_t) key_states | (uintptr_t) value_states) % 8 == 0, EXL_E_INVALID,
                "paged_append: key / value rows must be 8-byte aligned and at least kv_heads * head_dim apart");
    EXL_REQUIRE(((uintptr_t) key_pages | (uintptr_t) value_pages) % 16 == 0, EXL_E_INVALID, "paged_append: pages must be 16-byte aligned");
    if (rows == 0) return 0;
    EXL_REQUIRE(key_stride <= 1 << 22 && value_stride <= 1 << 22, EXL_E_UNSUPPORTED, "paged_append: key / value rows more than 2^22 elements apart");
    auto by = [](int d) { return (uint32_t) ((0x100000000ull + d - 1) / d); };
    const int hd16 = (head_dim + 15) / 16 * 16;
    AppendArgs a = {(const f16*) key_states, (const f16*) value_states, slots, positions, (const f16*) sin, (const f16*) cos,
                    (uint8_t*) key_pages, (uint8_t*) value_pages, key_scales, value_scales, rows, num_kv_heads, head_dim, hd16,
                    31 - __builtin_clz((unsigned) block_size), num_blocks, 4, angle_rows, (int) key_stride, (int) value_stride, by(hd16 / 4),
                    head_dim % 16 ? 0u : by(head_dim / 16), by(head_dim / 4)};
    // passes of the wide form over a page: block tokens x head_dim / 16 threads (256 / (head_dim / 16) whole tokens at a time)
    const int step = head_dim % 16 ? 0 : 256 / (head_dim / 16), p = step ? (block_size + step - 1) / step : 0;
    // Token rows of a workgroup.  Few: the runs of single tokens go to many waves; many: fewer workgroups that find no run's beginning (they
    // cost as much of the machine's registers as the others while they wait for their slots).  Measured, us, chunks of 4 / 16 / 32 / 63, head_dim 128:
    //   256 single tokens x 8 heads 8.2 / 14.8 / 24 / 44      512 x 32: 35 / 33 / 40 / 54       256 runs of 8 x 32: 45 / 42 / 41 / 62
    //   one prompt of 512 x 8 heads 10.1 / 7.7 / 8.1 / 7.8    2048 x 8: 17 / 12 / 9.6 / 9.4     2048 x 32: 37 / 21 / 19 / 16
    //   8192 x 8 in pages of 128 (four passes: twice the registers) 84 / 56 / 48 / 29           30 k ragged tokens x 8: 156 / 63 / 42 / 39
    const int64_t work = (int64_t) rows * num_kv_heads;
    a.chunk = work <= 12000 ? 4 : work <= 24000 ? 16 : work <= 131072 && p < 4 ? 32 : 63;
    const int64_t groups = ((int64_t) rows + a.chunk - 1) / a.chunk * num_kv_heads;
    EXL_REQUIRE(groups <= 0x7fffffff, EXL_E_UNSUPPORTED, "paged_append: too many rows for %d kv heads", num_kv_heads);
    const dim3 grid((unsigned) groups);
    const size_t lds = p ? (size_t) head_dim * (block_size + 4) : 0;
    hipStream_t s = (hipStream_t) stream;
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
