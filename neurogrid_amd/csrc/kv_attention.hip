// kv_attention.hip - attention over the 8-bit key/value cache (kv_cache.h; its
// layout: kv_cache.hpp).
//
// With a page's scales k_s, v_s, codes k, v and x_j = c k_s (q . k_j):
//   out = sum_j exp(x_j - m) v_s v_j / sum_j exp(x_j - m),  m a running maximum
// of the visible x_j, sums in 32 bits. One pass over the cache.
#include "kv_cache.hpp"

namespace ng {
namespace {

struct AttnArgs {
    const int* cu;
    const int* lens;
    const int* table;
    int max_pages, total, hq, group;
    float scale;  // softmax_scale log2(e)
    int window, sinks;
};

// One wave per query row and head, a token per lane.
template <typename T, int D>
__global__ __launch_bounds__(64) void kv_attention_row_kernel(uint16_t* out, const uint16_t* q, KvView kv, AttnArgs a) {
    constexpr int C = D / 64;
    __shared__ float s_q[D], s_p[64];
    __shared__ int s_page[64];
    const int b = blockIdx.y, hh = blockIdx.z, h = hh / a.group, lane = threadIdx.x;
    const KvRows rows = kv_rows(a.cu, b, a.total);
    const int ps = 1 << kv.ps_log2;
    const int len = min(max(a.lens[b], 0), a.max_pages << kv.ps_log2);
    const int lost = max(a.lens[b], 0) - len;  // tokens past the table are not there
    for (int i = blockIdx.x; i < rows.count; i += gridDim.x) {
        const int p = len + lost - rows.count + i;
        const size_t ro = (static_cast<size_t>(rows.first + i) * a.hq + hh) * D;
        for (int d = lane; d < D; d += 64) s_q[d] = to_f32<T>(q[ro + d]);
        __syncthreads();
        float m = -__builtin_inff(), l = 0.0f, acc[C];
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] = 0.0f;
        const int end = min(p, len - 1);
        for (int j0 = 0; j0 <= end; j0 += 64) {
            const int j = j0 + lane;
            bool seen = j <= end && (a.window == 0 || j > p - a.window || j < a.sinks);
            const int page = seen ? a.table[static_cast<size_t>(b) * a.max_pages + (j >> kv.ps_log2)] : -1;
            seen = page >= 0 && page < kv.num_pages;
            float x = -__builtin_inff(), vs = 0.0f;
            const int slot = j & (ps - 1);
            if (seen) {
                const size_t ph = static_cast<size_t>(page) * kv.hkv + h;
                const uint8_t* kc = kv.kc + ph * (static_cast<size_t>(ps) * D) + (slot >> 4) * 16 * D + (slot & 15) * 16;
                float s = 0.0f;
                for (int d = 0; d < D; ++d)
                    s += s_q[d] * static_cast<float>(static_cast<int8_t>(kc[(d >> 6) * 1024 + ((d >> 4) & 3) * 256 + (d & 15)]));
                x = s * (kv.ks[ph] * a.scale);
                vs = kv.vs[ph];
            }
            const float mn = fmaxf(m, wave_max_f32(x));
            const float ms = mn == -__builtin_inff() ? 0.0f : mn;
            const float e = seen ? __builtin_amdgcn_exp2f(x - ms) : 0.0f, f = __builtin_amdgcn_exp2f(m - ms);
            l = l * f + wave_sum_f32(e);
            m = mn;
            s_p[lane] = e * vs;
            s_page[lane] = seen ? page : -1;
            __syncthreads();
#pragma unroll
            for (int c = 0; c < C; ++c) acc[c] *= f;
            for (int t = 0; t < 64 && j0 + t <= end; ++t) {
                if (s_page[t] < 0) continue;
                const int sl = (j0 + t) & (ps - 1), tt = sl & 15;
                const uint8_t* vc = kv.vc + (static_cast<size_t>(s_page[t]) * kv.hkv + h) * (static_cast<size_t>(ps) * D) +
                                    (sl >> 4) * 16 * D;
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    const int kg = lane >> 4, i4 = (lane >> 2) & 3, r = lane & 3;
                    acc[c] += s_p[t] * static_cast<float>(static_cast<int8_t>(
                                           vc[c * 1024 + (kg * 16 + (tt >> 2) * 4 + r) * 16 + i4 * 4 + (tt & 3)]));
                }
            }
            __syncthreads();
        }
        const float inv = l == 0.0f ? 0.0f : 1.0f / l;
#pragma unroll
        for (int c = 0; c < C; ++c) out[ro + 64 * c + lane] = from_f32<T>(acc[c] * inv);
    }
}

template <typename T, int D>
int launch_attention(const dim3& grid, void* out, const void* q, const KvView& kv, const AttnArgs& a) {
    kv_attention_row_kernel<T, D><<<grid, dim3(64), 0, stream()>>>(static_cast<uint16_t*>(out),
                                                                  static_cast<const uint16_t*>(q), kv, a);
    return 0;
}

template <typename T>
int kv_attention(const char* name, void* out, const void* q, const ng_kv_int8_cache* cache, const void* cu,
                 const void* lens, const void* table, int batch, int max_pages, int total, int max_q, int max_kv,
                 int hq, float scale, int window, int sinks, void* workspace, size_t workspace_bytes) {
    if (kv_check_cache(name, cache) != 0) return -1;
    NG_REQUIRE(out && q, "%s: null pointer", name);
    if (kv_check_batch(name, cache, cu, lens, table, batch, max_pages, total, max_q) != 0) return -1;
    NG_REQUIRE(max_kv > 0, "%s: invalid max_kv_len %d", name, max_kv);
    NG_REQUIRE(hq > 0 && hq % cache->num_kv_heads == 0 && hq <= 32767,
               "%s: %d query heads on %d key/value heads", name, hq, cache->num_kv_heads);
    NG_REQUIRE(__builtin_isfinite(scale) && scale >= 0.0f, "%s: softmax_scale must be finite and >= 0", name);
    NG_REQUIRE(window >= 0 && sinks >= 0, "%s: window and sinks must be >= 0", name);
    NG_REQUIRE(aligned16(out) && aligned16(q) && aligned16(workspace), "%s: pointers must be 16-byte aligned", name);
    const AttnArgs a{static_cast<const int*>(cu), static_cast<const int*>(lens), static_cast<const int*>(table),
                     max_pages, total, hq, hq / cache->num_kv_heads, scale * 1.4426950408889634f,
                     min(window, 1 << 30), sinks};
    const dim3 grid(min(max_q, 65535), batch, hq);
    const KvView kv = kv_view(*cache);
    switch (cache->head_dim) {
        case 64: launch_attention<T, 64>(grid, out, q, kv, a); break;
        case 128: launch_attention<T, 128>(grid, out, q, kv, a); break;
        case 192: launch_attention<T, 192>(grid, out, q, kv, a); break;
        default: launch_attention<T, 256>(grid, out, q, kv, a); break;
    }
    NG_CHECK_LAUNCH(name);
    return 0;
}

}  // namespace
}  // namespace ng

using namespace ng;

extern "C" size_t ng_kv_int8_attention_workspace(const ng_kv_int8_cache* cache, int num_q_heads, int batch,
                                                 int max_q_len, int max_kv_len) {
    return 0;
}

extern "C" int ng_kv_int8_attention(void* out, const void* q, const ng_kv_int8_cache* cache, const void* cu_q,
                                    const void* kv_lens, const void* page_table, int batch, int max_pages, int total_q,
                                    int max_q_len, int max_kv_len, int num_q_heads, float softmax_scale, int window,
                                    int sinks, void* workspace, size_t workspace_bytes) {
    return kv_attention<f16>("ng_kv_int8_attention", out, q, cache, cu_q, kv_lens, page_table, batch, max_pages,
                             total_q, max_q_len, max_kv_len, num_q_heads, softmax_scale, window, sinks, workspace,
                             workspace_bytes);
}

extern "C" int ng_bf16_kv_int8_attention(void* out, const void* q, const ng_kv_int8_cache* cache, const void* cu_q,
                                         const void* kv_lens, const void* page_table, int batch, int max_pages,
                                         int total_q, int max_q_len, int max_kv_len, int num_q_heads,
                                         float softmax_scale, int window, int sinks, void* workspace,
                                         size_t workspace_bytes) {
    return kv_attention<bf16>("ng_bf16_kv_int8_attention", out, q, cache, cu_q, kv_lens, page_table, batch, max_pages,
                              total_q, max_q_len, max_kv_len, num_q_heads, softmax_scale, window, sinks, workspace,
                              workspace_bytes);
}
