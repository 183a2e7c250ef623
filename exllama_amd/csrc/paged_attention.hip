// Attention over the paged 8-bit cache (paged.h).
//   o[t, h] = sum_j p_j V[j] / sum_j p_j,   p_j = exp(s_j - max s),   s_j = scale * rope(q[t, h]) . K[j],   j <= past + i, j < past + new
#include "paged.h"

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

#define PA_TILE 256

// One workgroup = one query row of one head: a thread per key of a tile of 256 for the scores, then a thread per column for the sum.
template <int CODE> __global__ __launch_bounds__(PA_TILE) void paged_attn_row_kernel(PagedAttn a)
{
    __shared__ float qs[256], sc[PA_TILE], red[8];
    const int t = blockIdx.x, h = blockIdx.y, tid = threadIdx.x;
    int lo = 0, hi = a.n;
    while (hi - lo > 1) { const int mid = (lo + hi) >> 1; if (a.starts[mid] <= t) lo = mid; else hi = mid; }
    const PaRow row = pa_row(a, lo);
    const int i = t - row.start, past = row.past;
    if (i < 0 || i >= row.fresh) return;
    const int keys = (int) min((int64_t) past + i + 1, (int64_t) row.keys);
    const int kvh = h / (a.heads / a.kv_heads);
    const f16* q = a.q + (size_t) t * a.q_stride + (size_t) h * a.hd;
    if (tid < a.hd) {
        float x = (float) q[tid];
        if (a.sin) {
            const int pos = (int) min((int64_t) past + i, (int64_t) a.angle_rows - 1), half = a.hd >> 1;
            const float s = (float) a.sin[(size_t) pos * a.hd + tid], c = (float) a.cos[(size_t) pos * a.hd + tid];
            x = x * c + (tid < half ? -(float) q[tid + half] : (float) q[tid - half]) * s;
        }
        qs[tid] = x;
    }
    __syncthreads();
    float m = -INFINITY, l = 0.f, o = 0.f;
    for (int j0 = 0; j0 < keys; j0 += PA_TILE) {
        const int j = j0 + tid;
        float s = -INFINITY;
        if (j < keys) {
            const int id = a.table[(size_t) lo * a.width + j / a.block];
            if (id >= 0 && id < a.blocks) {
                const size_t base = (size_t) id * a.kv_heads + kvh;
                const uint32_t* k = (const uint32_t*) (a.kp + (base * a.block + j % a.block) * a.hd16);
                s = 0.f;
                for (int d = 0; d < a.hd; d += 4) {
                    float x[4];
                    paged_decode4<CODE>(k[d >> 2], x);
                    s += x[0] * qs[d] + x[1] * qs[d + 1] + x[2] * qs[d + 2] + x[3] * qs[d + 3];
                }
                s *= a.ks[base] * a.scale;
            }
        }
        float mx = s;
        for (int off = 32; off > 0; off >>= 1) mx = fmaxf(mx, __shfl_xor(mx, off, 64));
        if ((tid & 63) == 0) red[tid >> 6] = mx;
        __syncthreads();
        mx = fmaxf(fmaxf(red[0], red[1]), fmaxf(red[2], red[3]));
        const float mn = fmaxf(m, mx), ref = mn == -INFINITY ? 0.f : mn;
        const float p = s == -INFINITY ? 0.f : __expf(s - ref), keep = m == -INFINITY ? 0.f : __expf(m - ref);
        float sum = p;
        for (int off = 32; off > 0; off >>= 1) sum += __shfl_xor(sum, off, 64);
        if ((tid & 63) == 0) red[4 + (tid >> 6)] = sum;
        sc[tid] = p;
        __syncthreads();
        l = l * keep + red[4] + red[5] + red[6] + red[7];
        m = mn;
        o *= keep;
        if (tid < a.hd) {
            for (int u = 0; u < PA_TILE && j0 + u < keys; ++u) {
                const float w = sc[u];
                if (w == 0.f) continue;
                const int id = a.table[(size_t) lo * a.width + (j0 + u) / a.block];
                if (id < 0 || id >= a.blocks) continue;
                const size_t base = (size_t) id * a.kv_heads + kvh;
                const uint8_t* v = a.vp + (base * a.hd16 + tid) * a.block + (j0 + u) % a.block;
                float x[4];
                paged_decode4<CODE>(*v, x);
                o += w * x[0] * a.vs[base];
            }
        }
        __syncthreads();
    }
    if (tid < a.hd) a.out[(size_t) t * a.heads * a.hd + (size_t) h * a.hd + tid] = (f16) (l > 0.f || l != l ? o / l : 0.f);
}

extern "C" size_t exl_paged_attention_workspace(int n_rows, int rows, int max_new, int num_heads, int num_kv_heads, int head_dim, int table_width,
                                                int block_size)
{
    return 0;
}

extern "C" int exl_paged_attention(const void* q, long q_stride, const int32_t* starts, const int32_t* past_lens, const int32_t* new_lens, int n_rows,
                                   int rows, int max_new, const int32_t* block_table, int table_width, const void* key_pages, const void* value_pages,
                                   const float* key_scales, const float* value_scales, int code, int num_blocks, int block_size, int num_heads,
                                   int num_kv_heads, int head_dim, float scale, const void* sin, const void* cos, int angle_rows, void* out,
                                   void* workspace, size_t workspace_bytes, void* stream)
{
    EXL_REQUIRE(q && starts && past_lens && new_lens && block_table && key_pages && value_pages && key_scales && value_scales && out, EXL_E_INVALID,
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
    EXL_REQUIRE((int64_t) table_width * block_size <= 0x7fffffff, EXL_E_UNSUPPORTED, "paged_attention: the block table exceeds 2^31 tokens");
    if (rows == 0 || max_new == 0) return 0;
    PagedAttn a = {(const f16*) q, starts, past_lens, new_lens, block_table, (const uint8_t*) key_pages, (const uint8_t*) value_pages, key_scales,
                   value_scales, (const f16*) sin, (const f16*) cos, (f16*) out, n_rows, rows, max_new, table_width, num_blocks, block_size, num_heads,
                   num_kv_heads, head_dim, (head_dim + 15) / 16 * 16, angle_rows, q_stride, scale > 0.f ? scale : 1.f / sqrtf((float) head_dim)};
    hipStream_t s = (hipStream_t) stream;
    if (code == EXL_PAGE_FP8) hipLaunchKernelGGL((paged_attn_row_kernel<EXL_PAGE_FP8>), dim3(rows, num_heads), dim3(PA_TILE), 0, s, a);
    else                   hipLaunchKernelGGL((paged_attn_row_kernel<EXL_PAGE_INT8>), dim3(rows, num_heads), dim3(PA_TILE), 0, s, a);
    EXL_LAUNCH_CHECK();
    return 0;
}
