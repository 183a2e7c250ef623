// Attention over the paged 8-bit cache (paged.h).
//   o[t, h] = sum_j p_j V[j] / sum_j p_j,   p_j = exp(s_j - max s),   s_j = scale * rope(q[t, h]) . K[j],   j <= past + i, j < past + new
// Two forms, told apart by what the host knows, the most queries that a row has for one kv head (max_new * heads / kv_heads): up to 32 (head_dim over
// 128: 16) the cache's bytes bound the work, above it the products do.  Measured (us, few / many; 32 queries a row, head_dim 128): 16 rows of 4000 keys
// 51 / 68, one of 16000 30 / 40, 96 ragged ones 49 / 66, 8 of 300 19 / 17.
// Rounding: codes * scale are fp16 numbers exactly (448 * 2^7, 127 * 2^9); weights are rounded to fp16 for the product with the values, the
// denominator adds them as they are: 2^-11 of a weight, for one below 2^-21 of the largest (there fp16 is subnormal) 2^-32 of the largest;
// sums, maxima and the softmax's denominator are 32 bits; a rotated query is an fp16 number and its
// rest, also fp16 (2^-22) -- but for head_dim over 128 in the form for many queries; the result is rounded to fp16 once.
#include "paged.h"
#include <type_traits>

struct PagedAttn {
    const f16* q; const int32_t* starts; const int32_t* past; const int32_t* fresh; const int32_t* table;
    const uint8_t* kp; const uint8_t* vp; const float* ks; const float* vs; const f16* sin; const f16* cos; f16* out;
    int n, rows, max_new, width, blocks, block, heads, kv_heads, hd, hd16, angle_rows;
    long q_stride;
    float scale;
};

// A row of the batch as the kernels see it, whatever the device memory says: start + fresh <= rows, keys inside the table.
struct PaRow { int start, fresh, past, keys; };
__device__ __forceinline__ PaRow pa_row(const PagedAttn& a, int b)
{
    PaRow r;
    r.start = min(max(a.starts[b], 0), a.rows);
    r.fresh = min(min(max(a.fresh[b], 0), a.max_new), a.rows - r.start);
    r.past = max(a.past[b], 0);
    r.keys = r.fresh ? (int) min((int64_t) r.past + r.fresh, (int64_t) a.width * a.block) : 0;
    return r;
}

// ---- rows of few queries: the cache's bytes are all that counts ------------------------------------------------------------------------
// The tiles of 64 keys of all rows lie in one line, row behind row (each with PA_BEGIN places before it, for what beginning a row costs), and
// every wave takes an equal stretch of it for one kv head: whatever the rows' lengths, all waves end together, none waits for another, and the
// next row's first tile is on its way while the last one's last is worked on.
// A wave does all queries of its row that read the kv head (up to 16 * NT: tokens * heads of the group, GQA reads the cache once).  A row
// that lies in one stretch is written; the others leave one partial result for each stretch, joined in order by a second kernel -- the cut
// depends on the lengths alone, so results do not depend on scheduling.
// Bound by HBM: 8 rows of 65536 keys x 8 kv heads x 128 (1.07 GB) 199 us = 5.4 TB/s, 96 rows of 0 .. 16384 (434 MB) 93 us = 4.7 TB/s; one row of 2048 keys
// x 32 heads (16.8 MB) is latency: 9 us, and 4 us for the joining kernel.
// PA_BEGIN, measured 0 / 2 / 4: 96 ragged rows 134 / 104 / 105 us, five rows of four tokens 22 / 17 / 16, 96 equal rows 99 / 99 / 103.
// Both products are MFMAs on fp16 numbers converted from the codes in registers; nothing goes through LDS:
//   S^T = K Q^T   (16x16x32): A = keys.  MFMA row m of product t4 is key 16 * (m >> 2) + 4 * t4 + (m & 3) of the tile, so that a lane (query
//                 column c = lane & 15, group g = lane >> 4) gets the 16 scores of keys 16 g .. 16 g + 15, in order, over the four products;
//   O^T = V^T P^T : A = value columns, 16 bytes = keys 16 g .. 16 g + 15 of one column, as the page holds them; B = the lane's own 16 weights.
#define PA_WAVES 4
#define PA_KEYS 64
#define PA_BEGIN 2
#define PA_MOST 15.f                                              // the largest weight: 2^15
#define PA_BIAS 7.f                                               // the largest weight of a tile that moves the reference: 2^7

// A page's scale as the conversions take it.  int8: 2^e is the exponent field of the fp16 numbers that a code's byte becomes the mantissa of:
// (1024 + u) * 2^e with u = code + 128, minus 1152 * 2^e -- up to e = 5; beyond (`big`, for every lane as soon as one has it) a product follows.
struct PaScale { float f; uint32_t top; f16x2 sub, mul; };
template <int CODE> __device__ __forceinline__ PaScale pa_scale(float s)
{
    PaScale r = {};
    const int e = paged_scale_exp<CODE>(s);
    r.f = paged_pow2(e);
    if (CODE == EXL_PAGE_INT8) {
        const uint32_t field = (uint32_t) (min(e, 5) + 25) << 2;
        r.top = field * 0x01010101u;
        r.sub = __builtin_bit_cast(f16x2, (field << 8 | 0x80) * 0x00010001u);
        r.mul = (f16x2) ((f16) paged_pow2(max(e - 5, 0)));
    }
    return r;
}
template <int CODE> __device__ __forceinline__ bool pa_big(const PaScale& s) { return CODE == EXL_PAGE_INT8 && __any((float) s.mul[0] != 1.f); }

template <int CODE, bool BIG> __device__ __forceinline__ f16x8 pa_numbers(uint32_t lo, uint32_t hi, const PaScale& scale)     // 8 codes * scale, exact
{
    union { uint32_t u[4]; f16x2 h[4]; f16x8 v; } x;
    if (CODE == EXL_PAGE_FP8) {
        x.h[0] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int) lo, scale.f, false);
        x.h[1] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int) lo, scale.f, true);
        x.h[2] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int) hi, scale.f, false);
        x.h[3] = __builtin_amdgcn_cvt_scalef32_pk_f16_fp8((int) hi, scale.f, true);
    } else {
        const uint32_t a = lo ^ 0x80808080u, b = hi ^ 0x80808080u;
        x.u[0] = __builtin_amdgcn_perm(scale.top, a, 0x04010400u);
        x.u[1] = __builtin_amdgcn_perm(scale.top, a, 0x04030402u);
        x.u[2] = __builtin_amdgcn_perm(scale.top, b, 0x04010400u);
        x.u[3] = __builtin_amdgcn_perm(scale.top, b, 0x04030402u);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            x.h[i] = x.h[i] - scale.sub;
            if (BIG) x.h[i] = x.h[i] * scale.mul;
        }
    }
    return x.v;
}

// A value that is NaN and that only some of a tile's queries see (a token of this call, in e4m3 pages): a weight of 0 does not hide it from the
// others.  In tiles on the border such codes become 0 in the product with the weights, and the sums that they belong to become NaN: few queries: by
// two more products, of bf16's largest number at every NaN with the same number at every key that a query sees, which is infinity, and
// with its negative (sums set by a comparison each would be copied out of the matrix cores' registers and back); many queries: behind the last tile.
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ uint32_t pa_nan4(uint32_t codes) { return (((codes & 0x7f7f7f7fu) + 0x01010101u) & 0x80808080u) >> 7; }       // 1 in each byte that is NaN
__device__ __forceinline__ uint32_t pa_bits4(uint32_t ones) { return ones * 0x10204080u >> 28; }                                        // four bytes of 0 or 1 as four bits
__device__ __forceinline__ bf16x8 pa_holes(uint32_t lo, uint32_t hi)                                      // of eight bytes of 0 or 1
{
    union { uint32_t u[4]; bf16x8 v; } x;
    lo *= 0x7f; hi *= 0x7f;
    x.u[0] = __builtin_amdgcn_perm(0, lo, 0x01010000u); x.u[1] = __builtin_amdgcn_perm(0, lo, 0x03030202u);
    x.u[2] = __builtin_amdgcn_perm(0, hi, 0x01010000u); x.u[3] = __builtin_amdgcn_perm(0, hi, 0x03030202u);
    return x.v;
}
__device__ __forceinline__ bf16x8 pa_seen(int n, bool negative)                                           // the first n of eight
{
    union { uint32_t u[4]; bf16x8 v; } x;
    const uint32_t most = negative ? 0xff7fff7fu : 0x7f7f7f7fu;
#pragma unroll
    for (int i = 0; i < 4; ++i) x.u[i] = n >= 2 * i + 2 ? most : n == 2 * i + 1 ? most & 0xffff : 0u;
    return x.v;
}

// Query elements d .. d + 7 of one token and head (zeros behind head_dim), rotated at `pos` when there are tables.  A rotated query is no fp16
// number, and up to sqrt(2) times as large as the largest: it is taken by halves (exact, the scores are doubled: pa_c1); hi is the nearest fp16
// number, lo what it leaves (0 without a rotation).
struct PaQuery { f16x8 hi, lo; };
__device__ __forceinline__ PaQuery pa_query(const PagedAttn& a, const f16* q, int64_t pos, int d)
{
    PaQuery r = {};
    if (d >= a.hd) return r;
    const int half = a.hd >> 1;
    const f16* sin = nullptr; const f16* cos = nullptr;
    if (a.sin) {
        const size_t at = (size_t) (pos < a.angle_rows ? pos : a.angle_rows - 1) * a.hd;
        sin = a.sin + at; cos = a.cos + at;
    }
    auto put = [&](int i, float x) { x *= 0.5f; r.hi[i] = (f16) x; r.lo[i] = (f16) (x - (float) r.hi[i]); };
    if (a.hd % 16 == 0) {
        r.hi = *(const f16x8_a8*) (q + d);
        if (sin) {
            const f16x8 x = r.hi, o = *(const f16x8_a8*) (q + (d < half ? d + half : d - half)), s = *(const f16x8_a2*) (sin + d), c = *(const f16x8_a2*) (cos + d);
            const float sign = d < half ? -1.f : 1.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) put(i, fmaf((float) x[i], (float) c[i], sign * (float) o[i] * (float) s[i]));
        }
        return r;
    }
#pragma unroll
    for (int u = 0; u < 8; u += 4) {                             // head_dim a multiple of 4: in fours, whose other halves lie in fours too, but for the four in the middle
        const int e = d + u;
        if (e >= a.hd) break;
        const f16x4 x = *(const f16x4_a4*) (q + e);
        f16x4 o = {}, si = {}, co = {};
        if (sin) {
            si = *(const f16x4_a2*) (sin + e);
            co = *(const f16x4_a2*) (cos + e);
            if (e + 4 <= half || e >= half) o = *(const f16x4_a4*) (q + (e < half ? e + half : e - half));
            else for (int i = 0; i < 4; ++i) o[i] = q[e + i < half ? e + i + half : e + i - half];
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (sin) put(u + i, fmaf((float) x[i], (float) co[i], (e + i < half ? -(float) o[i] : (float) o[i]) * (float) si[i]));
            else r.hi[u + i] = x[i];
        }
    }
    return r;
}

// What a product of query and key is multiplied by: scores in powers of two
__device__ __forceinline__ float pa_c1(const PagedAttn& a) { return a.scale * (a.sin ? 2 * 1.44269504f : 1.44269504f); }

// How the work is cut: few queries: `target` waves for a kv head, no stretch of less than `min_piece` tiles; many queries: pm_find below
struct PaCut { int target, min_piece; };

// A row by scalar loads (b is the same in every lane)
__device__ __forceinline__ PaRow pa_row_of_wave(const PagedAttn& a, int b)
{
    typedef const __attribute__((address_space(4))) int32_t* scalar;
    PaRow r;
    r.start = min(max(((scalar) a.starts)[b], 0), a.rows);
    r.fresh = min(min(max(((scalar) a.fresh)[b], 0), a.max_new), a.rows - r.start);
    r.past = max(((scalar) a.past)[b], 0);
    r.keys = r.fresh ? (int) min((int64_t) r.past + r.fresh, (int64_t) a.width * a.block) : 0;
    return r;
}

// Stretch `w` of the line: `count` places from place `from` of row `row` on, the first of them number `at` of the line; `share`: places of a stretch.
// (The host has made sure that the line has less than 2^30 places.)
struct PaStretch { int row, from, count, share, at; };
__device__ __forceinline__ PaStretch pa_stretch(const PagedAttn& a, const PaCut& cut, int w)
{
    constexpr int KEPT = 4;                                        // rows of the batch whose places stay in registers: 64 * KEPT
    const int lane = threadIdx.x & 63;
    auto places = [&](int b) { const int keys = b < a.n ? pa_row(a, b).keys : 0; return keys ? (keys + PA_KEYS - 1) / PA_KEYS + PA_BEGIN : 0; };
    int kept[KEPT], total = 0;
#pragma unroll
    for (int i = 0; i < KEPT; ++i) {
        kept[i] = 0;
        if (64 * i < a.n) kept[i] = places(lane + 64 * i);
        total += kept[i];
    }
    for (int b = lane + 64 * KEPT; b < a.n; b += 64) total += places(b);
    if (a.n > 1) {
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) total += __shfl_xor(total, off, 64);
    }
    total = __builtin_amdgcn_readfirstlane(total);
    PaStretch st = {-1, 0, 0, 0, 0};
    st.share = max((total + cut.target - 1) / cut.target, cut.min_piece);
    if ((int64_t) w * st.share >= total) return st;
    st.at = w * st.share;
    st.count = min(st.share, total - st.at);
    if (a.n == 1) { st.row = 0; st.from = st.at; return st; }
    int before = 0;
    auto look = [&](int b0, int t) {                               // 64 rows; true: found
        int inc = t;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) { const int o = __shfl_up(inc, off, 64); if (lane >= off) inc += o; }
        const int from = before + inc - t;
        const uint64_t hit = __ballot(st.at >= from && st.at < from + t);
        before += __builtin_amdgcn_readlane(inc, 63);
        if (!hit) return false;
        const int l = __ffsll((unsigned long long) hit) - 1;
        st.row = b0 + l;
        st.from = __builtin_amdgcn_readlane(st.at - from, l);
        return true;
    };
#pragma unroll
    for (int i = 0; i < KEPT; ++i) if (64 * i < a.n && look(64 * i, kept[i])) return st;
    for (int b0 = 64 * KEPT; b0 < a.n; b0 += 64) if (look(b0, places(b0 + lane))) return st;
    return st;
}

// A partial result: [queries][DP + 4] floats (o, then m and l); a stretch has room for two: of the row that it continues, and of the one that goes on
__host__ __device__ constexpr size_t pa_part_floats(int dp, int nt) { return (size_t) 16 * nt * (dp + 4); }

// Registers (DP = 128, NT = 1): 64 for a tile's bytes, twice (the next tile is on its way while one is worked on), 32 of O, 32 of Q (241 in all):
// two waves per SIMD.  Twice the queries take one wave per SIMD, and so do wider heads, without the second set of bytes.
template <int CODE, int DP, int NT>
__global__ __launch_bounds__(PA_WAVES * 64, DP * NT <= 128 ? 2 : 1) void paged_attn_few_kernel(PagedAttn a, PaCut cut, float* __restrict__ parts,
                                                                                            int2* __restrict__ firsts)
{
    constexpr int KS = DP / 64, DT = DP / 16;
    constexpr bool AHEAD = DP <= 128;
    const int lane = threadIdx.x & 63, c = lane & 15, g = lane >> 4;
    const int worker = __builtin_amdgcn_readfirstlane(blockIdx.x * PA_WAVES + (threadIdx.x >> 6)), kvh = worker % a.kv_heads, w = worker / a.kv_heads;
    const PaStretch to = pa_stretch(a, cut, w);
    if (to.row < 0) return;
    const int group = a.heads / a.kv_heads, lbs = 31 - __clz(a.block);
    const int by_group = __builtin_amdgcn_readfirstlane((65535 + group) / group);                 // n / group = n * by_group >> 16 (n, group <= 32)
    const size_t kpage = (size_t) a.block * a.hd16;              // bytes of one page of one head, keys or values
    // (columns behind head_dim: key rows read column 0 again, value pages their last 16 columns; the queries there are zeros, the results unused)
    struct Stage { uint4 k[4][KS]; uint4 v[DT]; float ks, vs; bool there; };      // (scales as they are: looking at one here would wait for every load before it)
    auto fetch = [&](int tile, const int32_t* table, Stage& st) {
        const int ik = (tile * PA_KEYS + 16 * (c >> 2)) >> lbs, iv = (tile * PA_KEYS + 16 * g) >> lbs;      // the pages of this lane's key rows and of its group's values
        struct { int k, v; } id = {ik < a.width ? table[ik] : -1, iv < a.width ? table[iv] : -1};
        const bool kok = id.k >= 0 && id.k < a.blocks, vok = id.v >= 0 && id.v < a.blocks;
        const size_t kb = (size_t) (kok ? id.k : 0) * a.kv_heads + kvh, vb = (size_t) (vok ? id.v : 0) * a.kv_heads + kvh;
        const int key = tile * PA_KEYS + 16 * (c >> 2) + (c & 3);
        const uint8_t* kp = a.kp + kb * kpage + (size_t) (key & (a.block - 1)) * a.hd16;
#pragma unroll
        for (int t4 = 0; t4 < 4; ++t4)
#pragma unroll
            for (int s = 0; s < KS; ++s) st.k[t4][s] = *(const uint4*) (kp + 4 * t4 * a.hd16 + (64 * s + 16 * g < a.hd16 ? 64 * s + 16 * g : 0));
        const uint8_t* vp = a.vp + vb * kpage + c * a.block + ((tile * PA_KEYS + 16 * g) & (a.block - 1));
#pragma unroll
        for (int t = 0; t < DT; ++t) st.v[t] = *(const uint4*) (vp + min(16 * t, a.hd16 - 16) * a.block);
        st.ks = a.ks[vb];
        st.vs = a.vs[vb];
        st.there = vok;
    };

    const float c1 = pa_c1(a);
    const PaScale one = pa_scale<CODE>(1.f);
    f16x8 qf[NT][KS][2], ql[NT][KS][2];                          // the query and what fp16 leaves of it: the matrix cores have time for both
    int limit[NT];                                               // the last key this lane's query sees
    f32x4 o[NT][DT];
    float m[NT], l[NT];
    PaRow row;
    auto lane_here = [] {                                         // the lane once more, opaque: what follows from it takes no registers in the loop over the tiles
        int zero = 0;
        asm volatile("" : "+v"(zero));
        return (int) __builtin_amdgcn_mbcnt_hi(~0u, __builtin_amdgcn_mbcnt_lo(~0u, zero));
    };
    auto begin = [&](int b) {                                     // the queries of row b
        row = pa_row_of_wave(a, b);
        const int queries = row.fresh * group;
        const int here = lane_here(), cc = here & 15, gg = here >> 4;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            const int r = nt * 16 + cc, i = r * by_group >> 16;
            const bool in = r < queries;
            limit[nt] = in ? (int) min((int64_t) row.past + i, (int64_t) row.keys - 1) : -1;
            const f16* q = a.q + (size_t) (row.start + (in ? i : 0)) * a.q_stride + (size_t) (kvh * group + (in ? r - i * group : 0)) * a.hd;
#pragma unroll
            for (int s = 0; s < KS; ++s)
#pragma unroll
                for (int half = 0; half < 2; ++half) {
                    PaQuery x = pa_query(a, q, (int64_t) row.past + i, 64 * s + 16 * gg + 8 * half);
                    if (!in) x = {};
                    qf[nt][s][half] = x.hi;
                    ql[nt][s][half] = x.lo;
                }
            m[nt] = -INFINITY; l[nt] = 0.f;
#pragma unroll
            for (int t = 0; t < DT; ++t) o[nt][t] = (f32x4) {0.f, 0.f, 0.f, 0.f};
        }
    };

    auto work = [&](int tile, Stage& st) {
        const int key0 = tile * PA_KEYS + 16 * g;
        const bool border = tile * PA_KEYS + PA_KEYS - 1 > row.past || __any(!st.there);
        if (border) {                                            // weights of 0 do not hide what may stand in bytes that hold no value: NaN
            const int n = st.there ? min(max(row.keys - key0, 0), 16) : 0;
            uint32_t mask[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) mask[i] = n >= 4 * i + 4 ? 0xffffffffu : n <= 4 * i ? 0u : (1u << (8 * (n - 4 * i))) - 1;
#pragma unroll
            for (int t = 0; t < DT; ++t) { st.v[t].x &= mask[0]; st.v[t].y &= mask[1]; st.v[t].z &= mask[2]; st.v[t].w &= mask[3]; }
        }
        f32x4 s[NT][4];
#pragma unroll
        for (int nt = 0; nt < NT; ++nt)
#pragma unroll
            for (int t4 = 0; t4 < 4; ++t4) s[nt][t4] = (f32x4) {0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t4 = 0; t4 < 4; ++t4)
#pragma unroll
            for (int u = 0; u < KS; ++u) {
                const f16x8 k0 = pa_numbers<CODE, false>(st.k[t4][u].x, st.k[t4][u].y, one), k1 = pa_numbers<CODE, false>(st.k[t4][u].z, st.k[t4][u].w, one);
#pragma unroll
                for (int nt = 0; nt < NT; ++nt) {
                    s[nt][t4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, qf[nt][u][0], s[nt][t4], 0, 0, 0);
                    s[nt][t4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, qf[nt][u][1], s[nt][t4], 0, 0, 0);
                    s[nt][t4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k0, ql[nt][u][0], s[nt][t4], 0, 0, 0);
                    s[nt][t4] = __builtin_amdgcn_mfma_f32_16x16x32_f16(k1, ql[nt][u][1], s[nt][t4], 0, 0, 0);
                }
            }
        f16x8 p[NT][2];
        const float sc = paged_pow2(paged_scale_exp<CODE>(st.ks)) * c1;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float x[16], mx = -INFINITY;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                x[i] = s[nt][i >> 2][i & 3] * sc;
                asm("" : "+v"(x[i]));                             // (rounded here, for the maximum and for the weight alike)
                if (border && (!st.there || key0 + i > limit[nt])) x[i] = -INFINITY;
                mx = fmaxf(mx, x[i]);
            }
            mx = fmaxf(mx, __shfl_xor(mx, 16, 64));
            mx = fmaxf(mx, __shfl_xor(mx, 32, 64));
            // the weights are relative to a reference, which moves only when one would pass 2^15, so that the tile's largest becomes 2^7: fp16 holds them up
            // to 2^16, and with all of its digits down to 2^-14, that is 2^-21 of the largest or less
            // (one pass at most: mx - m is then 8 or less, whatever mx - 7 was rounded to; a loop for wide heads, whose sums lie in the matrix cores' own
            // registers: what it copies out and back stays in it)
            for (bool moves = __any(mx - m[nt] > PA_MOST); moves; moves = DP > 128 && __any(mx - m[nt] > PA_MOST)) {
                const float mn = fmaxf(m[nt], mx - PA_BIAS);
                const float keep = m[nt] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m[nt] - mn);
                l[nt] *= keep;
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int j = 0; j < 4; ++j) o[nt][t][j] *= keep;
                m[nt] = mn;
            }
            const float ref = m[nt] == -INFINITY ? 0.f : m[nt];
            float sum = 0.f;                                     // (of the tile: small weights one by one beside a large sum would lose their ends, all to one side)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float e = __builtin_amdgcn_exp2f(x[i] - ref);
                sum += e;
                p[nt][i >> 3][i & 7] = (f16) e;
            }
            l[nt] += sum;
        }
        const PaScale vs = pa_scale<CODE>(st.vs);
        if (CODE == EXL_PAGE_FP8 && border && row.fresh > 1) {
            uint32_t nan = 0;
#pragma unroll
            for (int t = 0; t < DT; ++t) nan |= pa_nan4(st.v[t].x) | pa_nan4(st.v[t].y) | pa_nan4(st.v[t].z) | pa_nan4(st.v[t].w);
            if (__any(nan)) {
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    uint4& v = st.v[t];
                    asm volatile("" : "+v"(v.x), "+v"(v.y), "+v"(v.z), "+v"(v.w));       // (computed again, not kept from above)
                    const uint4 n = make_uint4(pa_nan4(v.x), pa_nan4(v.y), pa_nan4(v.z), pa_nan4(v.w));
                    v.x &= ~(n.x * 255); v.y &= ~(n.y * 255); v.z &= ~(n.z * 255); v.w &= ~(n.w * 255);
                    const bf16x8 n0 = pa_holes(n.x, n.y), n1 = pa_holes(n.z, n.w);
#pragma unroll
                    for (int nt = 0; nt < NT; ++nt)
#pragma unroll
                        for (int sign = 0; sign < 2; ++sign) {
                            int seen = st.there ? limit[nt] + 1 - key0 : 0;
                            asm volatile("" : "+v"(seen));
                            o[nt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(n0, pa_seen(seen, sign), o[nt][t], 0, 0, 0);
                            o[nt][t] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(n1, pa_seen(seen - 8, sign), o[nt][t], 0, 0, 0);
                        }
                    __builtin_amdgcn_sched_barrier(0);        // (one after the other: all at once they take too many registers)
                }
            }
        }
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            const f16x8 v0 = pa_numbers<CODE, true>(st.v[t].x, st.v[t].y, vs), v1 = pa_numbers<CODE, true>(st.v[t].z, st.v[t].w, vs);
#pragma unroll
            for (int nt = 0; nt < NT; ++nt) {
                o[nt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v0, p[nt][0], o[nt][t], 0, 0, 0);
                o[nt][t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(v1, p[nt][1], o[nt][t], 0, 0, 0);
            }
        }
    };

    // a row's (or a stretch's) end: the sums of the four groups, and out.  `part`: where a partial result goes, or null
    auto end = [&](float* part) {
        const int here = lane_here(), cc = here & 15, gg = here >> 4;
#pragma unroll
        for (int nt = 0; nt < NT; ++nt) {
            float sum = l[nt];
            sum += __shfl_xor(sum, 16, 64);
            sum += __shfl_xor(sum, 32, 64);
            const int r = nt * 16 + cc, i = r * by_group >> 16;
            if (r >= row.fresh * group) continue;
            if (part) {
                float* p = part + (size_t) r * (DP + 4);
#pragma unroll
                for (int t = 0; t < DT; ++t) *(f32x4*) (p + 16 * t + 4 * gg) = o[nt][t];
                if (gg == 0) { p[DP] = m[nt]; p[DP + 1] = sum; }
            } else {
                f16* out = a.out + (size_t) (row.start + i) * a.heads * a.hd + (size_t) (kvh * group + r - i * group) * a.hd;
                const float inv = sum == 0.f ? 0.f : 1.f / sum;
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    f16x4 x;
#pragma unroll
                    for (int e = 0; e < 4; ++e) x[e] = (f16) (o[nt][t][e] * inv);
                    if (16 * t + 4 * gg < a.hd) *(f16x4*) (out + 16 * t + 4 * gg) = x;      // (head_dim is a multiple of four)
                }
            }
        }
    };

    int b = to.row, from = to.from, left = to.count;              // the row, the first place of it that is this stretch's, places that are left
    int at = to.at - to.from;                                     // the row's first place in the line
    if (from + left <= PA_BEGIN) return;                          // (no tile)
    Stage st;
    fetch(max(from - PA_BEGIN, 0), a.table + (size_t) b * a.width, st);
    for (;;) {                                                    // the rows of the stretch
        begin(b);
        const int tiles = (row.keys + PA_KEYS - 1) / PA_KEYS, first = max(from - PA_BEGIN, 0), last = min(from + left - PA_BEGIN, tiles) - 1;
        left -= tiles + PA_BEGIN - from;
        int nb = b;                                               // the next row that has any keys, if it has a tile in this stretch
        // (b + 1 < n always holds where places are left -- but for lengths that changed under the call)
        if (left > PA_BEGIN && b + 1 < a.n) do ++nb; while (nb < a.n - 1 && pa_row_of_wave(a, nb).keys == 0);
        for (int tile = first; ; ++tile) {
            const bool more = tile < last || nb != b;
            const int32_t* table = a.table + (size_t) (tile < last ? b : nb) * a.width;
            const int ntile = tile < last ? tile + 1 : 0;
            Stage nx;
            if (AHEAD && more) fetch(ntile, table, nx);
            work(tile, st);
            if (AHEAD) st = nx;
            else if (more) fetch(ntile, table, st);
            if (tile >= last) break;
        }
        const bool whole = first == 0 && last == tiles - 1;
        float* part = parts + (((size_t) w * a.kv_heads + kvh) * 2 + (first == 0)) * pa_part_floats(DP, NT);
        end(whole ? nullptr : part);
        int share = to.share;
        asm volatile("" : "+s"(share));                           // (the division is not prepared before the loop)
        if (first == 0 && kvh == 0 && lane == 0)                  // for the joining kernel: where the row's parts begin, and how many there are
            firsts[b] = make_int2(w, (at + PA_BEGIN + tiles - 1) / share - w + 1);
        if (nb == b) return;
        at += tiles + PA_BEGIN;
        b = nb;
        from = 0;
    }
}

// The parts of a row joined: `each` (1, 2, 4, ...) queries of one row and kv head for a workgroup, dp / 4 lanes for a query; the lanes that are
// left take every so many-th part each, with a maximum of their own, and meet in LDS -- in an order that depends on the lengths alone.
// 4 us for a few rows (a launch and three rounds of loads), 9 us for 96 ragged rows x 64 heads (12 MB of parts).
__global__ __launch_bounds__(256) void paged_attn_join_kernel(PagedAttn a, const float* __restrict__ parts, const int2* __restrict__ firsts, int dp, int nt, int each, int target)
{
    __shared__ f32x4 slice_o[256];
    __shared__ float slice_m[256], slice_l[256];
    const int b = blockIdx.x, kvh = blockIdx.z, group = a.heads / a.kv_heads, tid = threadIdx.x;
    const PaRow row = pa_row(a, b);
    if (row.keys == 0 || (int) blockIdx.y * each >= row.fresh * group) return;
    const int2 first = firsts[b];                                 // (the row had a first part: it was written)
    if (first.y < 2 || first.x < 0 || first.y > target - first.x) return;      // (beyond the stretches: lengths that changed under the call)
    const int lanes = dp >> 2, slices = 256 / (lanes * each), d = (tid % lanes) * 4, q = tid / lanes % each, sl = tid / (lanes * each);
    const int r = blockIdx.y * each + q;
    const size_t size = pa_part_floats(dp, nt), step = 2 * a.kv_heads * size;
    const float* p0 = parts + (((size_t) first.x * a.kv_heads + kvh) * 2) * size + (size_t) r * (dp + 4);      // part 0 lies behind it, in the second place
    float m = -INFINITY, sum = 0.f;
    f32x4 o = {0.f, 0.f, 0.f, 0.f};
    if (r < row.fresh * group) {
        constexpr int U = 4;                                      // parts in flight
        for (int k0 = sl; k0 < first.y; k0 += U * slices) {
            float pm[U], pl[U];
            f32x4 po[U];
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const int k = min(k0 + u * slices, first.y - 1);
                const float* p = p0 + (k ? k * step : size);
                pm[u] = k0 + u * slices < first.y ? p[dp] : -INFINITY;
                pl[u] = p[dp + 1];
                po[u] = *(const f32x4*) (p + d);
            }
            float top = m;
#pragma unroll
            for (int u = 0; u < U; ++u) top = fmaxf(top, pm[u]);
            const float keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
            sum *= keep;
            o *= keep;
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (k0 + u * slices >= first.y) break;
                const float f = pm[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(pm[u] - top);
                sum += f * pl[u];
                o += f * po[u];
            }
            m = top;
        }
    }
    slice_o[tid] = o;
    slice_m[tid] = m;
    slice_l[tid] = sum;
    __syncthreads();
    if (sl || r >= row.fresh * group || d >= a.hd) return;
    float top = m;
    for (int u = 1; u < slices; ++u) top = fmaxf(top, slice_m[tid + u * lanes * each]);
    const float keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
    sum *= keep;
    o *= keep;
    for (int u = 1; u < slices; ++u) {
        const int x = tid + u * lanes * each;
        const float f = slice_m[x] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(slice_m[x] - top);
        sum += f * slice_l[x];
        o += f * slice_o[x];
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    f16x4 x;
#pragma unroll
    for (int e = 0; e < 4; ++e) x[e] = (f16) (o[e] * inv);
    *(f16x4*) (a.out + (size_t) (row.start + r / group) * a.heads * a.hd + (size_t) (kvh * group + r % group) * a.hd + d) = x;
}

// ---- rows of many queries: prompts and pieces of prompts --------------------------------------------------------------------------------
// One workgroup (4 waves) takes 128 queries (token * group + head of the group, so that GQA shares the cache's tiles) and walks tiles of 64 keys.
// The codes are converted ONCE per workgroup on their way into LDS, as fp16 in the MFMA's operand order (two buffers, one barrier a tile); each
// wave has 32 queries:
//   S^T = K Q^T (32x32x16): row m of the product is key 16 * ((m >> 2) & 1) + 4 * (m >> 3) + (m & 3) of a half tile, so that a lane (query
//   column c = lane & 31, group g = lane >> 5) gets keys 16 g .. 16 g + 15 in order;   O^T = V^T P^T: the lane's own weights are the operand.
// LDS pieces of 16 bytes are laid out by XOR so that neither the writes (one key, all columns) nor the reads (linear) meet in a bank.
// Bound by the sum of MFMA and VALU time (conversion, exp2, masks), which two workgroups a compute unit do not hide behind each other (pieces of a 70B
// prompt: 48 % and 54 % of the cycles).
// LOW, head_dim up to 128: the rest of a rotated query is multiplied too -- half as many MFMAs again: a prompt of 2048 x 32 heads (34 GFLOP causal)
// takes 86 us instead of 76, pieces of a 70B prompt (410 GFLOP) 634 instead of 523 (in turn on one GPU); without it the result is 3.8e-4 of its norm
// off, with it 2.65e-4 (2.05e-4 are its own rounding).  Wider heads have no registers for it (spilled: 127 -> 213 us).
#define PM_ROWS 128

// s * c1, rounded, and how far it lies above ref
__device__ __forceinline__ float pa_above(float s, float c1, float ref)
{
#pragma clang fp contract(off)
    const float x = s * c1;
    return x - ref;
}

// A tile of queries and a piece of its keys (all tiles of a row are cut in the same number of `pieces`)
struct PmItem { int row, tile, piece, pieces; };
struct PmFound { PmItem item; PaRow row; };                       // (the row as one thread read it: all waves walk the same tiles whatever happens to the lengths meanwhile)

// Item `w` of the launch; row < 0: none.  The cost of a row is tiles of queries * tiles of keys; with `piece` = a `target`-th of all rows' cost
// (or min_piece), rows of 1.5 times as many keys or more are cut into pieces of about that size -- 4 / 3 * target items at most, and these come
// first: an item's number is its place among the partial results.  Tiles of a row come with the last (the longest) first; where every item of the launch is resident at once, the
// second half comes shortest first: the two workgroups of a compute unit, half a launch apart, then have equal work together.
// lds: 96 bytes, free again afterwards.
__device__ __forceinline__ PmFound pm_find(const PagedAttn& a, const PaCut& cut, int w, void* lds)
{
    int64_t* sums = (int64_t*) lds;
    PmFound& found = *(PmFound*) (sums + 2 * PA_WAVES);
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, step = PA_WAVES * 64;
    struct Size { int q, keys; };
    auto size = [&](int b) -> Size {
        const PaRow r = pa_row(a, b);
        const int64_t queries = (int64_t) r.fresh * (a.heads / a.kv_heads);
        return {(int) ((queries + PM_ROWS - 1) / PM_ROWS), (r.keys + PA_KEYS - 1) / PA_KEYS};
    };
    auto total = [&](int64_t v, int at) -> int64_t {               // over the workgroup
#pragma unroll
        for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, 64);
        if (lane == 0) sums[at * PA_WAVES + wave] = v;
        __syncthreads();
        return sums[at * PA_WAVES] + sums[at * PA_WAVES + 1] + sums[at * PA_WAVES + 2] + sums[at * PA_WAVES + 3];
    };
    const Size mine = tid < a.n ? size(tid) : Size{0, 0};           // (of the first 256 rows, kept)
    int64_t cost = 0;
    for (int b = tid; b < a.n; b += step) { const Size z = b == tid ? mine : size(b); cost += (int64_t) z.q * z.keys; }
    if (tid == 0) found.item.row = -1;
    cost = total(cost, 0);
    const int64_t even = (cost + cut.target - 1) / cut.target;
    const int piece = (int) min(max(even, (int64_t) cut.min_piece), (int64_t) 1 << 30);
    auto pieces = [&](const Size& z) { return max((int) (((int64_t) z.keys + piece / 2) / piece), 1); };
    int64_t cuts = 0;
    for (int b = tid; b < a.n; b += step) { const Size z = b == tid ? mine : size(b); const int np = pieces(z); if (np > 1) cuts += (int64_t) z.q * np; }
    cuts = total(cuts, 1);
    const bool first = w < cuts;                                  // among the rows that are cut, or behind them
    int64_t before = first ? 0 : cuts, count = 0;
    for (int b0 = 0; b0 < a.n; b0 += step) {
        const int b = b0 + tid;
        const Size z = b >= a.n ? Size{0, 0} : b0 == 0 ? mine : size(b);
        const int np = pieces(z);
        const int64_t here = (np > 1) == first ? (int64_t) z.q * np : 0;
        int64_t inc = here;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) { const int64_t o = __shfl_up(inc, off, 64); if (lane >= off) inc += o; }
        __syncthreads();
        if (lane == 63) sums[wave] = inc;
        __syncthreads();
        int64_t base = before + inc - here;
        for (int u = 0; u < wave; ++u) base += sums[u];
        if (w >= base && w < base + here) {
            const int k = (int) (w - base), t = k / np, half = (z.q + 1) / 2;
            const bool fold = !first && cost <= 2 * (int64_t) cut.target * z.keys;     // (as many tiles as fit at once, or fewer: a compute unit holds two)
            found.item = {b, fold && t >= half ? t - half : z.q - 1 - t, k % np, np};
            found.row = pa_row(a, b);
        }
        before += sums[0] + sums[1] + sums[2] + sums[3];
        if (before > w) break;
    }
    __syncthreads();
    const PmFound it = found;
    __syncthreads();                                              // `lds` is the caller's again
    return it;
}

// WIDE: pages of 64 or 128 tokens, a tile lies in one: its page is looked up once, in scalar registers (pieces of a 70B prompt 651 -> 617 us).
template <int CODE, int DP, bool WIDE, bool LOW>
__global__ __launch_bounds__(PA_WAVES * 64, DP <= 128 ? 2 : 1) void paged_attn_many_kernel(PagedAttn a, PaCut cut, float* __restrict__ parts,
                                                                                        PmItem* __restrict__ items, int part_items)
{
    constexpr int KB = DP / 16, DT = DP / 32, PIECES = PA_KEYS * KB / 256;       // 16-byte pieces of codes per thread: keys, and as many of values
    extern __shared__ __attribute__((aligned(16))) unsigned char lds[];          // [2][keys: 2 * KB * 1024 bytes, values: 4 * DT * 1024 bytes], [2][DP] maps, 2 ints, [DT][256] bits
    constexpr int K_BYTES = 2 * KB * 1024, BUF = 2 * K_BYTES;
    uint64_t* nan_map = (uint64_t*) (lds + 2 * BUF);              // by buffer, of a tile on the border: the tokens whose value is NaN, a word for each column
    int* nan_tile = (int*) (nan_map + 2 * DP);                    // by buffer: the last tile on the border that held one
    // kv heads next to each other in launch order: consecutive workgroups go to different XCDs, so that those of one head (the same keys and
    // values) share an XCD's L2 where kv_heads is a multiple of 8, and every XCD gets tiles of all lengths
    const int kvh = blockIdx.x % a.kv_heads, w = blockIdx.x / a.kv_heads;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6), c = lane & 31, g = lane >> 5;
    uint16_t* hole = (uint16_t*) (nan_tile + 2) + tid;            // [DT][256]: a bit for each of this lane's sums that is NaN
    if (tid < 2) nan_tile[tid] = -1;                              // (pm_find has barriers)
    if (CODE == EXL_PAGE_FP8) for (int t = 0; t < DT; ++t) hole[t * 256] = 0;
    const PmFound found = pm_find(a, cut, w, lds);
    const PmItem it = {__builtin_amdgcn_readfirstlane(found.item.row), __builtin_amdgcn_readfirstlane(found.item.tile), __builtin_amdgcn_readfirstlane(found.item.piece),
                       __builtin_amdgcn_readfirstlane(found.item.pieces)};
    if (kvh == 0 && tid == 0 && w < part_items) items[w] = it;                   // for the joining kernel
    if (it.row < 0) return;
    const PaRow row = {__builtin_amdgcn_readfirstlane(found.row.start), __builtin_amdgcn_readfirstlane(found.row.fresh), __builtin_amdgcn_readfirstlane(found.row.past),
                       __builtin_amdgcn_readfirstlane(found.row.keys)};
    const int group = a.heads / a.kv_heads, lbs = 31 - __clz(a.block);
    const int64_t queries = (int64_t) row.fresh * group, q0 = (int64_t) it.tile * PM_ROWS;
    const int last_token = (int) ((min(q0 + PM_ROWS, queries) - 1) / group);
    const int all_tiles = (int) ((min((int64_t) row.past + last_token + 1, (int64_t) row.keys) + PA_KEYS - 1) / PA_KEYS);
    const int t_first = (int) ((int64_t) all_tiles * it.piece / it.pieces);
    const int t_last = (int) ((int64_t) all_tiles * (it.piece + 1) / it.pieces);

    // this lane's query
    const int64_t r = q0 + wave * 32 + c;
    const bool in = r < queries;
    const int token = in ? (int) (r / group) : 0, head = kvh * group + (in ? (int) (r % group) : 0);
    const int limit = in ? (int) min((int64_t) row.past + token, (int64_t) row.keys - 1) : -1;
    // the last key that all queries of this wave see.  (A tile behind what any of them sees is worked on like the others, all masked: a short cut around
    // it made the compiler keep the accumulators in two places and copy them in every tile.)
    const int64_t wave_q0 = q0 + wave * 32;
    const int wave_free = wave_q0 < queries ? (int) min((int64_t) row.past + (int) (wave_q0 / group), (int64_t) row.keys - 1) : -1;
    f16x8 qf[KB], ql[KB];                                         // the query and what fp16 leaves of it after a rotation
    {
        const f16* q = a.q + (size_t) (row.start + token) * a.q_stride + (size_t) head * a.hd;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
            PaQuery x = pa_query(a, q, (int64_t) row.past + token, 16 * kb + 8 * g);
            if (!in) x = {};
            qf[kb] = x.hi;
            ql[kb] = x.lo;
        }
    }

    const int32_t* table = a.table + (size_t) it.row * a.width;
    const size_t page_bytes = (size_t) a.block * a.hd16;
    // staging roles: keys: piece i of this thread is column chunk k_ch of key k_key + (256 / KB) * i; values: 16 keys v_kc of column v_d + 64 * i
    const int k_ch = tid % KB, k_key = tid / KB, v_kc = tid & 3, v_d = tid >> 2;
    constexpr int K_STEP = 256 / KB;
    struct Ids { int k[WIDE ? 1 : PIECES]; int v; };
    struct Stage { uint4 k[PIECES], v[PIECES]; float ks[WIDE ? 1 : PIECES], vs; int n; uint32_t there; };   // n: valid keys of the value pieces; there: a bit for each 16 keys
    auto look = [&](int tile) -> Ids {
        Ids id;
        if (WIDE) {
            const int p = (tile * PA_KEYS) >> lbs;
            id.k[0] = id.v = p < a.width ? ((const __attribute__((address_space(4))) int32_t*) table)[p] : -1;     // a scalar load
        } else {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int p = (tile * PA_KEYS + k_key + K_STEP * i) >> lbs;
                id.k[WIDE ? 0 : i] = p < a.width ? table[p] : -1;
            }
            const int p = (tile * PA_KEYS + 16 * v_kc) >> lbs;
            id.v = p < a.width ? table[p] : -1;
        }
        return id;
    };
    // offsets of this thread's pieces inside a page, for WIDE: from the tile's first key on
    const int k_at = k_key * a.hd16 + (16 * k_ch < a.hd16 ? 16 * k_ch : 0);
    int v_at[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) v_at[i] = ((v_d + 64 * i < a.hd16 ? v_d + 64 * i : 0) << lbs) + (WIDE ? 16 * v_kc : 0);
    auto fetch = [&](int tile, const Ids& id, Stage& st) {
        const bool ok = id.v >= 0 && id.v < a.blocks;
        const size_t vb = (size_t) (ok ? id.v : 0) * a.kv_heads + kvh;
        const int key = tile * PA_KEYS + 16 * v_kc;
        if (WIDE) {
            const int first = (tile * PA_KEYS) & (a.block - 1);
            const uint8_t* kp = a.kp + vb * page_bytes + first * a.hd16;
            const uint8_t* vp = a.vp + vb * page_bytes + first;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                st.k[i] = *(const uint4*) (kp + (uint32_t) (k_at + K_STEP * i * a.hd16));
                st.v[i] = *(const uint4*) (vp + (uint32_t) v_at[i]);
            }
            st.ks[0] = a.ks[vb];
        } else {
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const int at = tile * PA_KEYS + k_key + K_STEP * i, kid = id.k[WIDE ? 0 : i];
                const size_t kb = (size_t) (kid >= 0 && kid < a.blocks ? kid : 0) * a.kv_heads + kvh;
                st.k[i] = *(const uint4*) (a.kp + kb * page_bytes + (size_t) ((at & (a.block - 1)) * a.hd16 + (16 * k_ch < a.hd16 ? 16 * k_ch : 0)));
                st.ks[WIDE ? 0 : i] = a.ks[kb];
            }
            const uint8_t* vp = a.vp + vb * page_bytes + (key & (a.block - 1));
#pragma unroll
            for (int i = 0; i < PIECES; ++i) st.v[i] = *(const uint4*) (vp + v_at[i]);
        }
        st.vs = a.vs[vb];                                         // (as it is: looking at it here would wait for every load before it)
        st.n = ok ? min(max(row.keys - key, 0), 16) : 0;
        st.there = WIDE ? (ok ? 15u : 0u) : (uint32_t) __ballot(ok) & 15;
    };
    // where this thread's pieces go in a buffer
    int k_to[PIECES], v_to[PIECES];
#pragma unroll
    for (int i = 0; i < PIECES; ++i) {
        const int key = k_key + K_STEP * i, kt = key >> 5, m = 8 * ((key >> 2) & 3) + 4 * ((key >> 4) & 1) + (key & 3), d = v_d + 64 * i;
        k_to[i] = (kt * KB + k_ch) * 1024 + ((m ^ (k_ch & 7)) << 4);
        v_to[i] = K_BYTES + ((v_kc >> 1) * 2 * DT + (d >> 5)) * 1024 + ((((v_kc & 1) * 32 + (d & 31)) ^ (v_kc << 1)) << 4);
    }
    const int free_keys = (int) min((int64_t) row.past + (int) (q0 / group), (int64_t) row.keys - 1);       // the last key that all queries of the workgroup see
    auto store = [&](int tile, Stage& st) {
        unsigned char* buf = lds + ((tile - t_first) & 1) * BUF;
        const bool border = tile * PA_KEYS + PA_KEYS - 1 > free_keys;
        if (border || __any(st.n < 16)) {                         // bytes that hold no value may be anything, NaN too: a weight of 0 does not hide it
            uint32_t mask[4], nan = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) mask[i] = st.n >= 4 * i + 4 ? 0xffffffffu : st.n <= 4 * i ? 0u : (1u << (8 * (st.n - 4 * i))) - 1;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                uint4& v = st.v[i];
                v.x &= mask[0]; v.y &= mask[1]; v.z &= mask[2]; v.w &= mask[3];
                if (CODE == EXL_PAGE_FP8 && border) {
                    const uint4 n = make_uint4(pa_nan4(v.x), pa_nan4(v.y), pa_nan4(v.z), pa_nan4(v.w));
                    v.x &= ~(n.x * 255); v.y &= ~(n.y * 255); v.z &= ~(n.z * 255); v.w &= ~(n.w * 255);
                    const uint32_t bits = pa_bits4(n.x) | pa_bits4(n.y) << 4 | pa_bits4(n.z) << 8 | pa_bits4(n.w) << 12;
                    ((uint16_t*) (nan_map + ((tile - t_first) & 1) * DP + v_d + 64 * i))[v_kc] = (uint16_t) bits;
                    nan |= bits;
                }
            }
            if (nan) nan_tile[(tile - t_first) & 1] = tile;
        }
        const PaScale vscale = pa_scale<CODE>(st.vs);
        PaScale kscale[WIDE ? 1 : PIECES];
        bool big = pa_big<CODE>(vscale);
#pragma unroll
        for (int i = 0; i < (WIDE ? 1 : PIECES); ++i) { kscale[i] = pa_scale<CODE>(st.ks[i]); big = big || pa_big<CODE>(kscale[i]); }
        auto convert = [&](auto big) {
            constexpr bool BIG = decltype(big)::value;
#pragma unroll
            for (int i = 0; i < PIECES; ++i) {
                const PaScale& ks = kscale[WIDE ? 0 : i];
                *(f16x8*) (buf + k_to[i]) = pa_numbers<CODE, BIG>(st.k[i].x, st.k[i].y, ks);
                *(f16x8*) (buf + k_to[i] + 512) = pa_numbers<CODE, BIG>(st.k[i].z, st.k[i].w, ks);       // (columns 8 .. 15 of the chunk: lanes 32 .. 63)
                *(f16x8*) (buf + v_to[i]) = pa_numbers<CODE, BIG>(st.v[i].x, st.v[i].y, vscale);
                *(f16x8*) (buf + v_to[i] + DT * 1024) = pa_numbers<CODE, BIG>(st.v[i].z, st.v[i].w, vscale);
            }
        };
        if (big) convert(std::true_type()); else convert(std::false_type());
    };

    f32x16 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int j = 0; j < 16; ++j) o[t][j] = 0.f;
    float m = -INFINITY, l = 0.f;
    const float c1 = pa_c1(a);

    Stage st;
    Ids id;
    uint32_t there = 15;
    if (__builtin_expect(t_first < t_last, 1)) {
        fetch(t_first, look(t_first), st);
        there = st.there;
        store(t_first, st);
        if (t_first + 1 < t_last) fetch(t_first + 1, look(t_first + 1), st);
        if (t_first + 2 < t_last) id = look(t_first + 2);
    }
    if (__builtin_expect(t_first < t_last, 1)) for (int tile = t_first; ; ) {
        unsigned char* buf = lds + ((tile - t_first) & 1) * BUF;
        const uint32_t now = there;
        __syncthreads();                                          // this tile is in `buf`, and every wave is through with the other one
        if (tile + 1 < t_last) {
            there = st.there;
            store(tile + 1, st);
            if (tile + 2 < t_last) {
                fetch(tile + 2, id, st);
                if (tile + 3 < t_last) id = look(tile + 3);
            }
        }
        const bool border = tile * PA_KEYS + PA_KEYS - 1 > wave_free || now != 15;
        f32x16 s[2];
#pragma unroll
        for (int kt = 0; kt < 2; ++kt) {
#pragma unroll
            for (int j = 0; j < 16; ++j) s[kt][j] = 0.f;
#pragma unroll
            for (int kb = 0; kb < KB; ++kb) {
                const f16x8 k = *(const f16x8*) (buf + (kt * KB + kb) * 1024 + ((lane ^ (kb & 7)) << 4));
                s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, qf[kb], s[kt], 0, 0, 0);
                if (LOW) s[kt] = __builtin_amdgcn_mfma_f32_32x32x16_f16(k, ql[kb], s[kt], 0, 0, 0);
            }
            if (LOW) __builtin_amdgcn_sched_barrier(0);           // (fewer pieces of keys in flight: the query's second half takes their registers)
        }
        float mx = -INFINITY;
        if (__builtin_amdgcn_readfirstlane(border)) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                const int left = now >> (2 * kt + g) & 1 ? limit - (tile * PA_KEYS + 32 * kt + 16 * g) : -1;      // the last visible of these 16 keys
#pragma unroll
                for (int j = 0; j < 16; ++j) if (j > left) s[kt][j] = -INFINITY;
            }
        }
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int j = 0; j < 16; ++j) mx = fmaxf(mx, s[kt][j]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * c1;
        asm("" : "+v"(mx));                                       // (rounded here: contracted into the difference below, a pass might not be the last)
        // the reference moves as in the other form
        // (one pass at most: mx - m is then 8 or less, whatever mx - 7 was rounded to; a loop for wide heads, whose sums lie in the matrix cores' own
        // registers: what it copies out and back stays in it)
        for (bool moves = __any(mx - m > PA_MOST); moves; moves = DP > 128 && __any(mx - m > PA_MOST)) {
            const float mn = fmaxf(m, mx - PA_BIAS);
            const float keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - mn);
            l *= keep;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int j = 0; j < 16; ++j) o[t][j] *= keep;
            m = mn;
        }
        float ref = m == -INFINITY ? 0.f : m;
        // Scores so large that one fma and a product with a difference disagree by more than 2^-2: rounded as mx was.  (Wide heads always: a branch here
        // made the compiler copy sums in every tile.)
        if (DP <= 128 && __any(fabsf(ref) > 0x1p22f)) {
            const float back = 1.f / c1;
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int j = 0; j < 16; ++j) s[kt][j] = pa_above(s[kt][j], c1, ref) * back;
            ref = 0.f;
        }
        f16x8 p[2][2];
        float sum = 0.f;                                          // (of the tile, as in the other form)
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int j = 0; j < 16; ++j) {
                const float e = __builtin_amdgcn_exp2f(DP > 128 ? pa_above(s[kt][j], c1, ref) : fmaf(s[kt][j], c1, -ref));
                sum += e;
                p[kt][j >> 3][j & 7] = (f16) e;
            }
        l += sum;
#pragma unroll
        for (int kt = 0; kt < 2; ++kt)
#pragma unroll
            for (int h = 0; h < 2; ++h)
#pragma unroll
                for (int t = 0; t < DT; ++t) {
                    const f16x8 v = *(const f16x8*) (buf + K_BYTES + ((kt * 2 + h) * DT + t) * 1024 + ((lane ^ (4 * kt + 2 * g)) << 4));
                    o[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v, p[kt][h], o[t], 0, 0, 0);
                }
        if (CODE == EXL_PAGE_FP8 && tile * PA_KEYS + PA_KEYS - 1 > free_keys && __builtin_amdgcn_readfirstlane(nan_tile[(tile - t_first) & 1]) == tile) {
            uint64_t seen = 0;                                    // the keys of the tile that this lane's query sees
#pragma unroll
            for (int u = 0; u < 4; ++u) {
                const int n = now >> u & 1 ? min(max(limit - (tile * PA_KEYS + 16 * u) + 1, 0), 16) : 0;
                seen |= (uint64_t) ((1u << n) - 1) << (16 * u);
            }
            const uint64_t* map = nan_map + ((tile - t_first) & 1) * DP + 4 * g;
#pragma unroll
            for (int t = 0; t < DT; ++t) {
                uint32_t bits = 0;
#pragma unroll
                for (int j = 0; j < 16; ++j) bits = bits << 1 | ((map[32 * t + 8 * (j >> 2) + (j & 3)] & seen) ? 1u : 0u);
                hole[t * 256] |= (uint16_t) bits;
                __builtin_amdgcn_sched_barrier(0);
            }
        }
        if (++tile >= t_last) break;
    }

    // ---- out: row j of a product is column 32 t + 8 * (j >> 2) + 4 g + (j & 3)
    l += __shfl_xor(l, 32, 64);
    if (!in) return;
    if (CODE == EXL_PAGE_FP8) {
#pragma unroll
        for (int t = 0; t < DT; ++t) {
            const uint32_t bits = hole[t * 256];
            if (bits)
#pragma unroll
                for (int j = 0; j < 16; ++j) if (bits >> (15 - j) & 1) o[t][j] = NAN;
        }
    }
    if (it.pieces == 1) {
        f16* out = a.out + (size_t) (row.start + token) * a.heads * a.hd + (size_t) head * a.hd;
        const float inv = l == 0.f ? 0.f : 1.f / l;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int d = 32 * t + 8 * j + 4 * g;
                if (d >= a.hd) continue;                              // (head_dim is a multiple of four)
                f16x4 x;
#pragma unroll
                for (int e = 0; e < 4; ++e) x[e] = (f16) (o[t][4 * j + e] * inv);
                *(f16x4*) (out + d) = x;
            }
    } else {
        float* part = parts + (((size_t) w * a.kv_heads + kvh) * PM_ROWS + wave * 32 + c) * (DP + 4);
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int j = 0; j < 4; ++j) *(f32x4*) (part + 32 * t + 8 * j + 4 * g) = (f32x4) {o[t][4 * j], o[t][4 * j + 1], o[t][4 * j + 2], o[t][4 * j + 3]};
        if (g == 0) { part[DP] = m; part[DP + 1] = l; }
    }
}

// The pieces of a query tile joined, in order: 16 lanes for a query, 16 queries of an item for a workgroup (most of which find nothing to do:
// 4.5 us where no row is cut).  Four parts in flight: one at a time 100 queries x 32 heads took 21 us for six parts each.
template <int DP> __global__ __launch_bounds__(256) void paged_attn_join_many_kernel(PagedAttn a, const float* __restrict__ parts, const PmItem* __restrict__ items)
{
    constexpr int V = DP / 64, U = DP <= 128 ? 4 : 2;             // groups of four columns of a lane; pieces in flight
    const int w = blockIdx.x, kvh = blockIdx.y, lane = threadIdx.x & 15;
    const PmItem it = items[w];
    if (it.row < 0 || it.piece != 0 || it.pieces < 2) return;
    const PaRow row = pa_row(a, it.row);
    const int group = a.heads / a.kv_heads, q = blockIdx.z * 16 + (threadIdx.x >> 4);
    const size_t step = (size_t) a.kv_heads * PM_ROWS * (DP + 4);
    const int64_t r = (int64_t) it.tile * PM_ROWS + q;
    if (r >= (int64_t) row.fresh * group) return;
    const float* p0 = parts + (((size_t) w * a.kv_heads + kvh) * PM_ROWS + q) * (DP + 4);
    float m = -INFINITY, sum = 0.f;
    f32x4 o[V] = {};
    for (int k0 = 0; k0 < it.pieces; k0 += U) {
        float pm[U], pl[U];
        f32x4 po[U][V];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const float* p = p0 + min(k0 + u, it.pieces - 1) * step;
            pm[u] = k0 + u < it.pieces ? p[DP] : -INFINITY;
            pl[u] = p[DP + 1];
#pragma unroll
            for (int j = 0; j < V; ++j) po[u][j] = *(const f32x4*) (p + 64 * j + 4 * lane);
        }
        float top = m;
#pragma unroll
        for (int u = 0; u < U; ++u) top = fmaxf(top, pm[u]);
        const float keep = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - top);
        sum *= keep;
#pragma unroll
        for (int j = 0; j < V; ++j) o[j] *= keep;
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (k0 + u >= it.pieces) break;
            const float f = pm[u] == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(pm[u] - top);
            sum += f * pl[u];
#pragma unroll
            for (int j = 0; j < V; ++j) o[j] += f * po[u][j];
        }
        m = top;
    }
    const float inv = sum == 0.f ? 0.f : 1.f / sum;
    f16* out = a.out + (size_t) (row.start + (int) (r / group)) * a.heads * a.hd + (size_t) (kvh * group + (int) (r % group)) * a.hd;
#pragma unroll
    for (int j = 0; j < V; ++j) {
        const int d = 64 * j + 4 * lane;
        f16x4 x;
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = (f16) (o[j][e] * inv);
        if (d < a.hd) *(f16x4*) (out + d) = x;                    // (head_dim is a multiple of four)
    }
}

// How a call is cut, from what the host knows: most queries of a row (max_new * group) up to 16 * NT: the kernel for few queries, else the other
struct PaPlan { int dp, nt, group, items, parts, rows_y; bool many, split; PaCut cut; size_t item_bytes, part_bytes; };
static size_t pa_round(size_t n) { return (n + 255) / 256 * 256; }

static PaPlan pa_plan(int n, int rows, int max_new, int heads, int kv_heads, int hd, int width, int block)
{
    PaPlan p;
    p.dp = hd <= 64 ? 64 : hd <= 128 ? 128 : 256;
    p.group = heads / kv_heads;
    const int64_t queries = (int64_t) (max_new < rows ? max_new : rows) * p.group, longest = (int64_t) width * block;
    p.many = queries > (p.dp == 256 ? 16 : 32);
    p.nt = queries <= 16 ? 1 : 2;
    p.rows_y = (int) queries;
    if (!p.many) {
        // All waves that the machine holds at once.  Half / all / twice as many: 96 ragged rows 108 / 104 / 110 us, 32 queries a row 69 / 53 / 65.
        // Stretches of at least one tile: 1 / 2 / 4: one row of 2048 keys 12.8 / 14.8 / 18.9 us
        const int waves = 1024 * (p.dp * p.nt <= 128 ? 2 : 1);
        p.cut = {kv_heads >= waves ? 1 : waves / kv_heads, 1};
        p.split = true;
        p.items = p.parts = p.cut.target;
        p.item_bytes = pa_round((size_t) n * sizeof(int2));
        p.part_bytes = pa_round((size_t) p.parts * kv_heads * 2 * pa_part_floats(p.dp, p.nt) * sizeof(float));
    } else {
        const int64_t fresh = (int64_t) n * max_new < rows ? (int64_t) n * max_new : rows, tiles = (fresh * p.group + PM_ROWS - 1) / PM_ROWS + n;
        // A workgroup for every compute unit, pieces of 8 tiles or more.  128 / 256 / 512 workgroups: 100 tokens x 32 heads after 3000 43 / 41 / 49 us,
        // x 64 heads with 8 kv heads 58 / 45 / 48.  Pieces of at least 4 / 8 / 16 tiles: 40 / 41 / 48 and 45 / 45 / 48
        p.cut = {kv_heads >= 256 ? 1 : 256 / kv_heads, 8};
        p.split = longest > p.cut.min_piece * PA_KEYS;
        p.parts = p.split ? 2 * p.cut.target : 0;
        p.items = (int) (tiles + p.parts < 0x7fffffff ? tiles + p.parts : 0x7fffffff);
        p.item_bytes = pa_round((size_t) p.parts * sizeof(PmItem));
        p.part_bytes = pa_round((size_t) p.parts * kv_heads * PM_ROWS * (p.dp + 4) * sizeof(float));
    }
    return p;
}

template <int CODE> static int pa_launch(const PagedAttn& a, const PaPlan& p, void* workspace, hipStream_t s)
{
    float* parts = (float*) ((char*) workspace + p.item_bytes);
    EXL_REQUIRE((int64_t) p.items * a.kv_heads <= 0x7fffffff, EXL_E_UNSUPPORTED, "paged_attention: too many rows for %d kv heads", a.kv_heads);
    const unsigned items = (unsigned) p.items * (unsigned) a.kv_heads;
    const dim3 grid(p.many ? items : (items + PA_WAVES - 1) / PA_WAVES);
    if (!p.many) {
        int2* firsts = (int2*) workspace;
#define PA_FEW(DP, NT) hipLaunchKernelGGL((paged_attn_few_kernel<CODE, DP, NT>), grid, dim3(PA_WAVES * 64), 0, s, a, p.cut, parts, firsts)
        if (p.dp == 64)       { if (p.nt == 1) PA_FEW(64, 1); else PA_FEW(64, 2); }
        else if (p.dp == 128) { if (p.nt == 1) PA_FEW(128, 1); else PA_FEW(128, 2); }
        else                  PA_FEW(256, 1);
#undef PA_FEW
        EXL_LAUNCH_CHECK();
        int each = 1;                                             // queries of a joining workgroup: as many as leave work for the whole machine
        while (2 * each <= 1024 / p.dp && each < p.rows_y && (int64_t) a.n * a.kv_heads * ((p.rows_y + 2 * each - 1) / (2 * each)) >= 512) each *= 2;
        hipLaunchKernelGGL(paged_attn_join_kernel, dim3((unsigned) a.n, (unsigned) ((p.rows_y + each - 1) / each), (unsigned) a.kv_heads), dim3(256), 0, s, a, parts, firsts,
                           p.dp, p.nt, each, p.cut.target);
        EXL_LAUNCH_CHECK();
        return 0;
    }
    PmItem* list = (PmItem*) workspace;
#define PA_MANY_R(DP, WIDE, ROPE) do { static bool done[EXL_MAX_DEVICES] = {};                                                               \
    EXL_TRY(exl_lds_opt_in((const void*) paged_attn_many_kernel<CODE, DP, WIDE, ROPE>, done));                                                \
    hipLaunchKernelGGL((paged_attn_many_kernel<CODE, DP, WIDE, ROPE>), grid, dim3(PA_WAVES * 64), 2 * PA_KEYS * DP * 4 + 2 * DP * 8 + 8 + DP / 32 * 512, s, a, p.cut, parts, list, p.parts); } while (0)
#define PA_MANY(DP, WIDE) do { if (DP <= 128 && a.sin) PA_MANY_R(DP, WIDE, (DP <= 128)); else PA_MANY_R(DP, WIDE, false); } while (0)
    if (a.block >= PA_KEYS) { if (p.dp == 64) PA_MANY(64, true); else if (p.dp == 128) PA_MANY(128, true); else PA_MANY(256, true); }
    else                    { if (p.dp == 64) PA_MANY(64, false); else if (p.dp == 128) PA_MANY(128, false); else PA_MANY(256, false); }
#undef PA_MANY
#undef PA_MANY_R
    EXL_LAUNCH_CHECK();
    if (p.split) {
        const dim3 jgrid((unsigned) p.parts, (unsigned) a.kv_heads, PM_ROWS / 16);
        if (p.dp == 64)       hipLaunchKernelGGL((paged_attn_join_many_kernel<64>), jgrid, dim3(256), 0, s, a, parts, list);
        else if (p.dp == 128) hipLaunchKernelGGL((paged_attn_join_many_kernel<128>), jgrid, dim3(256), 0, s, a, parts, list);
        else                  hipLaunchKernelGGL((paged_attn_join_many_kernel<256>), jgrid, dim3(256), 0, s, a, parts, list);
        EXL_LAUNCH_CHECK();
    }
    return 0;
}

extern "C" size_t exl_paged_attention_workspace(int n_rows, int rows, int max_new, int num_heads, int num_kv_heads, int head_dim, int table_width,
                                                int block_size)
{
    if (n_rows <= 0 || rows <= 0 || max_new <= 0 || num_heads <= 0 || num_kv_heads <= 0 || num_heads % num_kv_heads || head_dim <= 0 || table_width <= 0 ||
        block_size <= 0) return 0;
    const PaPlan p = pa_plan(n_rows, rows, max_new, num_heads, num_kv_heads, head_dim, table_width, block_size);
    return p.item_bytes + p.part_bytes;
}

extern "C" int exl_paged_attention(const void* q, long q_stride, const int32_t* starts, const int32_t* past_lens, const int32_t* new_lens, int n_rows,
                                   int rows, int max_new, const int32_t* block_table, int table_width, const void* key_pages, const void* value_pages,
                                   const float* key_scales, const float* value_scales, int code, int num_blocks, int block_size, int num_heads,
                                   int num_kv_heads, int head_dim, float scale, const void* sin, const void* cos, int angle_rows, void* out,
                                   void* workspace, size_t workspace_bytes, void* stream)
{
    const bool none = rows == 0 || max_new == 0;                  // (nothing to do: empty tensors have no address)
    EXL_REQUIRE(((q && out) || none) && starts && past_lens && new_lens && block_table && key_pages && value_pages && key_scales && value_scales, EXL_E_INVALID,
                "paged_attention: null pointer");
    EXL_REQUIRE(n_rows > 0 && rows >= 0 && max_new >= 0 && table_width > 0 && num_blocks > 0 && num_heads > 0 && num_kv_heads > 0 &&
                num_heads <= 65535, EXL_E_INVALID, "paged_attention: bad shape");
    EXL_REQUIRE(num_heads % num_kv_heads == 0, EXL_E_INVALID, "paged_attention: heads (%d) %% kv_heads (%d) != 0", num_heads, num_kv_heads);
    EXL_TRY(paged_check_block("paged_attention", block_size, num_blocks));
    EXL_TRY(paged_check_head("paged_attention", code, head_dim));
    EXL_REQUIRE((sin == nullptr) == (cos == nullptr) && (!sin || angle_rows > 0), EXL_E_INVALID, "paged_attention: a rotation needs sin and cos");
    EXL_REQUIRE(q_stride >= (long) num_heads * head_dim && q_stride % 4 == 0 && ((uintptr_t) q | (uintptr_t) out) % 8 == 0, EXL_E_INVALID,
                "paged_attention: q rows must be 8-byte aligned and at least heads * head_dim apart");
    EXL_REQUIRE(((uintptr_t) key_pages | (uintptr_t) value_pages) % 16 == 0, EXL_E_INVALID, "paged_attention: pages must be 16-byte aligned");
    EXL_REQUIRE((int64_t) table_width * block_size <= 0x7fffffff - PA_KEYS, EXL_E_UNSUPPORTED,      // (lengths are rounded up to tiles in 32 bits)
                "paged_attention: the block table exceeds 2^31 - %d tokens", PA_KEYS + 1);
    EXL_REQUIRE((int64_t) n_rows * ((int64_t) table_width * block_size / PA_KEYS + PA_BEGIN + 1) < 1 << 30, EXL_E_UNSUPPORTED,
                "paged_attention: %d rows of %d blocks are too many", n_rows, table_width);
    if (none) return 0;
    EXL_REQUIRE((uintptr_t) out >= (uintptr_t) q + 2 * ((size_t) (rows - 1) * q_stride + (size_t) num_heads * head_dim) ||
                (uintptr_t) q >= (uintptr_t) out + 2 * (size_t) rows * num_heads * head_dim, EXL_E_INVALID, "paged_attention: out overlaps q");
    PagedAttn a = {(const f16*) q, starts, past_lens, new_lens, block_table, (const uint8_t*) key_pages, (const uint8_t*) value_pages, key_scales,
                   value_scales, (const f16*) sin, (const f16*) cos, (f16*) out, n_rows, rows, max_new, table_width, num_blocks, block_size, num_heads,
                   num_kv_heads, head_dim, (head_dim + 15) / 16 * 16, angle_rows, q_stride, scale > 0.f ? scale : 1.f / sqrtf((float) head_dim)};
    hipStream_t s = (hipStream_t) stream;
    const PaPlan p = pa_plan(n_rows, rows, max_new, num_heads, num_kv_heads, head_dim, table_width, block_size);
    EXL_REQUIRE(p.item_bytes + p.part_bytes == 0 || (workspace && (uintptr_t) workspace % 16 == 0 && workspace_bytes >= p.item_bytes + p.part_bytes), EXL_E_TOO_SMALL,
                "paged_attention: the workspace is too small (%zu < %zu bytes) or not 16-byte aligned", workspace_bytes, p.item_bytes + p.part_bytes);
    return code == EXL_PAGE_FP8 ? pa_launch<EXL_PAGE_FP8>(a, p, workspace, s) : pa_launch<EXL_PAGE_INT8>(a, p, workspace, s);
}
