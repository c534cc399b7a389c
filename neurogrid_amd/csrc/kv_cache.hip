// kv_cache.hip - writing, reading back and copying the pages of the 8-bit
// key/value cache (kv_cache.h; its layout: kv_cache.hpp).
//
// Append. A page and head is one block of quantisation, so one workgroup holds
// all of a page's new tokens of a head in registers: a wave per 16 tokens, its
// 64 lanes 4 per token with 16 elements of each 64-element chunk, which are the
// K pieces of the layout; V's are the same codes with each quad's 4 x 4 bytes
// transposed (DPP). The page's largest magnitude is a DPP maximum per wave and
// one exchange through LDS. Codes of tokens that were there before are loaded
// with the new rows, so that a scale that grows costs no further trip.
// A lane's two pieces of a row lie side by side and are two accesses: with
// default-policy loads and stores the second meets the first's line in L2, with
// non-temporal ones it did not. 4096 + 2920 + 1967 tokens of 8 heads, D = 128:
// append 11.7 us (13.0 non-temporal; 38 MB), read 11.6 us (19.7).
// Bound: a token of a step is launch latency (4.1 us), prompts are HBM.
#include "kv_cache.hpp"

namespace ng {
namespace {

// Largest finite magnitude of a vector's 8 elements, as its bit pattern.
template <typename T>
__device__ __forceinline__ uint32_t absmax_finite8(const u32x4 v, uint32_t m) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint32_t b = lane16(v, e) & 0x7fffu;
        if (b < kInfBits<T> && b > m) m = b;
    }
    return m;
}

// A block's largest magnitude m as its codes are formed with it: 127 x / m is the
// quotient of X = x (127 2^-e) and M = m 2^-e, 1 <= M < 2 (less for m below 2^-120).
// x and m have at most 11 significant bits, so X is exact, and the quotient is a
// half-integer or at least 2^-20 of itself away from one: RN(X / M) rounds to the
// code that the real quotient has. It takes no division: with inv = RN(1 / M), z =
// RN(X inv) is within a few ulp, the residual X - z M is exact, and one
// correction step gives the correctly rounded quotient (Markstein).
struct Block {
    float scale;  // 127 2^-e
    float m, inv; // M, RN(1 / M)
    int e;
};
__device__ __forceinline__ Block block_of(float m) {
    Block b;
    b.e = max(static_cast<int>(__builtin_bit_cast(uint32_t, m) >> 23), 7) - 127;
    b.scale = __builtin_ldexpf(127.0f, -b.e);
    b.m = __builtin_ldexpf(m, -b.e);
    b.inv = 1.0f / b.m;
    return b;
}
__device__ __forceinline__ uint32_t code_bits(float x, const Block& b) {
    const float z = x * b.inv;
    return __builtin_bit_cast(uint32_t, fp32_barrier(__builtin_fmaf(__builtin_fmaf(z, -b.m, x), b.inv, z)) + kRoundMagic);
}
__device__ __forceinline__ uint32_t low_bytes(uint32_t b0, uint32_t b1, uint32_t b2, uint32_t b3) {
    const uint32_t lo = __builtin_amdgcn_perm(b1, b0, 0x0c0c0400u), hi = __builtin_amdgcn_perm(b3, b2, 0x0c0c0400u);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}

// Codes of the 8 elements of a vector. Where some are not finite, by the IEEE
// quotient: infinities saturate, NaN gives 127.
template <typename T>
__device__ __forceinline__ u32x2 kv_codes8(const u32x4 v, const Block& b, bool finite) {
    u32x2 out = {0, 0};
    if (finite) {
#pragma unroll
        for (int d = 0; d < 2; ++d)
            out[d] = low_bytes(code_bits(el_mul<T, 0>(v[2 * d], b.scale), b), code_bits(el_mul<T, 1>(v[2 * d], b.scale), b),
                               code_bits(el_mul<T, 0>(v[2 * d + 1], b.scale), b),
                               code_bits(el_mul<T, 1>(v[2 * d + 1], b.scale), b));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int c = qclamp_ref(__builtin_rintf(to_f32<T>(lane16(v, e)) * b.scale / b.m));
            out[e >> 2] |= (static_cast<uint32_t>(c) & 0xffu) << ((e & 3) * 8);
        }
    }
    return out;
}

// rint(code old / m) of four codes, old = the block's magnitude before times
// 2^-e (the product is exact, so the code is again the real quotient's).
__device__ __forceinline__ uint32_t rescale4(uint32_t w, float old, const Block& b) {
    uint32_t c[4];
#pragma unroll
    for (int e = 0; e < 4; ++e) c[e] = code_bits(fp32_barrier(static_cast<float>(static_cast<int8_t>(w >> (8 * e))) * old), b);
    return low_bytes(c[0], c[1], c[2], c[3]);
}

// Grid: pages of a sequence (strided over), batch, 2 heads (K, V).
template <typename T, int D>
__global__ __launch_bounds__(512) void kv_append_kernel(KvView kv, const uint16_t* __restrict__ k,
                                                        const uint16_t* __restrict__ v, const int* __restrict__ cu,
                                                        const int* __restrict__ ctx_lens,
                                                        const int* __restrict__ table, int max_pages, int total,
                                                        int* dropped) {
    constexpr int C = D / 64;
    __shared__ uint32_t s_max[8];
    const int b = blockIdx.y, h = blockIdx.z >> 1;
    const bool is_v = blockIdx.z & 1;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int waves = blockDim.x / kWave;
    const int ps = 1 << kv.ps_log2, cap = max_pages << kv.ps_log2;
    const KvRows rows = kv_rows(cu, b, total);
    const int ctx = min(max(load_uniform(ctx_lens + b), 0), cap);
    const int n = min(rows.count, cap - ctx);
    const bool counts = dropped != nullptr && blockIdx.z == 0 && threadIdx.x == 0;
    if (counts && blockIdx.x == 0 && rows.count > n) atomicAdd(dropped, rows.count - n);
    if (n == 0) return;
    const uint16_t* x = (is_v ? v : k) + static_cast<size_t>(rows.first) * kv.hkv * D + static_cast<size_t>(h) * D;
    uint8_t* codes = is_v ? kv.vc : kv.kc;
    float* scales = is_v ? kv.vs : kv.ks;
    const size_t head_bytes = static_cast<size_t>(ps) * D;
    const int kg = lane >> 4, t = lane & 15;
    const uint32_t sel = quad_selector(lane);
    const int last = (ctx + n - 1) >> kv.ps_log2;
    for (int pg = (ctx >> kv.ps_log2) + blockIdx.x; pg <= last; pg += gridDim.x) {
        const int t0 = pg << kv.ps_log2;
        const int lo = max(ctx - t0, 0), hi = min(ctx + n - t0, ps);  // slots lo .. hi - 1 are new
        // The new rows are requested before the page is known.
        const int slot = wave * kSub + t;
        const bool is_new = slot >= lo && slot < hi;
        const u32x4 zero = {0, 0, 0, 0};
        u32x4 in[C][2], old[C];
        const uint16_t* row = x + static_cast<ptrdiff_t>(t0 + slot - ctx) * kv.hkv * D + 16 * kg;
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 2; ++j) in[c][j] = is_new ? ld16(row + 64 * c + 8 * j) : zero;
        const int page = load_uniform(table + static_cast<size_t>(b) * max_pages + pg);
        if (page < 0 || page >= kv.num_pages) {
            if (counts) atomicAdd(dropped, hi - lo);
            continue;
        }
        const size_t ph = static_cast<size_t>(page) * kv.hkv + h;
        uint8_t* mine = codes + ph * head_bytes + static_cast<size_t>(wave) * kSub * D + lane * 16;
        const bool has_old = wave * kSub < lo;  // of the wave's 16 tokens
#pragma unroll
        for (int c = 0; c < C; ++c) old[c] = has_old ? ld16(mine + 1024 * c) ^ kKvBias : zero;
        const float before = lo > 0 ? scales[ph] : 0.0f;
        uint32_t m = 0;
#pragma unroll
        for (int c = 0; c < C; ++c) m = absmax_bits8(in[c][1], absmax_bits8(in[c][0], m));
        m = wave_max_u32_dpp(m);
        const bool finite = m < kInfBits<T>;
        if (!finite) {
            m = 0;
#pragma unroll
            for (int c = 0; c < C; ++c) m = absmax_finite8<T>(in[c][1], absmax_finite8<T>(in[c][0], m));
            m = wave_max_u32_dpp(m);
        }
        if (waves > 1) {
            __syncthreads();  // the last page's maxima are read
            if (lane == 0) s_max[wave] = m;
            __syncthreads();
            for (int w = 0; w < waves; ++w) m = umax32(m, s_max[w]);
        }
        const float now = fmaxf(before, to_f32<T>(static_cast<uint16_t>(m)));
        // Every wave of the block read the old magnitude before the barrier
        // above, or is this wave.
        if (threadIdx.x == 0) scales[ph] = now;
        const bool grown = now > before;
        if (wave * kSub + kSub <= lo && !grown) continue;  // old codes only, as they were
        const Block blk = block_of(now);
        const float old_m = __builtin_ldexpf(before, -blk.e);
        // Which bytes of a dword are old tokens': all or none for K, by token for V.
        const int quad_old = min(max(lo - (wave * kSub + (t & ~3)), 0), 4);
        const uint32_t keep = is_v ? (quad_old == 4 ? ~0u : (1u << (8 * quad_old)) - 1u) : (slot < lo ? ~0u : 0u);
#pragma unroll
        for (int c = 0; c < C; ++c) {
            u32x4 q = zero;
            if (now > 0.0f) {
                const u32x2 a = kv_codes8<T>(in[c][0], blk, finite), d = kv_codes8<T>(in[c][1], blk, finite);
                q = u32x4{a[0], a[1], d[0], d[1]};
            }
            if (is_v) {
#pragma unroll
                for (int i = 0; i < 4; ++i) q[i] = quad_transpose(q[i], sel);
            }
            if (has_old) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const uint32_t o = grown ? rescale4(old[c][i], old_m, blk) : old[c][i];
                    q[i] = (o & keep) | (q[i] & ~keep);
                }
            }
            st16(mine + 1024 * c, q ^ kKvBias);
        }
    }
}

// Two codes' values as 16-bit elements.
template <typename T, int LO>
__device__ __forceinline__ uint32_t values2(uint32_t w, float s) {
    return pack2<T>(static_cast<float>(static_cast<int8_t>(w >> (8 * LO))) * s,
                    static_cast<float>(static_cast<int8_t>(w >> (8 * LO + 8))) * s);
}

// The append's grid and lanes.
template <typename T, int D>
__global__ __launch_bounds__(512) void kv_read_kernel(KvView kv, uint16_t* k, uint16_t* v, const int* __restrict__ cu,
                                                      const int* __restrict__ starts, const int* __restrict__ table,
                                                      int max_pages, int total) {
    constexpr int C = D / 64;
    const int b = blockIdx.y, h = blockIdx.z >> 1;
    const bool is_v = blockIdx.z & 1;
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int ps = 1 << kv.ps_log2;
    const KvRows rows = kv_rows(cu, b, total);
    if (rows.count == 0) return;
    const int start = min(max(load_uniform(starts + b), 0), 1 << 30);
    uint16_t* x = (is_v ? v : k) + static_cast<size_t>(rows.first) * kv.hkv * D + static_cast<size_t>(h) * D;
    const int kg = lane >> 4, t = lane & 15;
    const uint32_t sel = quad_selector(lane);
    const int last = (start + rows.count - 1) >> kv.ps_log2;
    for (int pg = (start >> kv.ps_log2) + blockIdx.x; pg <= last; pg += gridDim.x) {
        const int t0 = pg << kv.ps_log2;
        const int lo = max(start - t0, 0), hi = min(start + rows.count - t0, ps);
        const int slot = wave * kSub + t;
        if (wave * kSub >= hi || wave * kSub + kSub <= lo) continue;
        const int page = pg < max_pages ? load_uniform(table + static_cast<size_t>(b) * max_pages + pg) : -1;
        const bool there = page >= 0 && page < kv.num_pages;
        const size_t ph = there ? static_cast<size_t>(page) * kv.hkv + h : 0;
        const uint8_t* mine = (is_v ? kv.vc : kv.kc) + ph * (static_cast<size_t>(ps) * D) +
                              static_cast<size_t>(wave) * kSub * D + lane * 16;
        u32x4 q[C];
#pragma unroll
        for (int c = 0; c < C; ++c) q[c] = there ? ld16(mine + 1024 * c) ^ kKvBias : u32x4{0, 0, 0, 0};
        const float s = (there ? load_uniform((is_v ? kv.vs : kv.ks) + ph) : 0.0f) / 127.0f;
        uint16_t* row = x + static_cast<ptrdiff_t>(t0 + slot - start) * kv.hkv * D + 16 * kg;
#pragma unroll
        for (int c = 0; c < C; ++c) {
            if (is_v) {
#pragma unroll
                for (int i = 0; i < 4; ++i) q[c][i] = quad_transpose(q[c][i], sel);
            }
            if (slot < lo || slot >= hi) continue;
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const uint32_t a = q[c][2 * j], d = q[c][2 * j + 1];
                st16(row + 64 * c + 8 * j, u32x4{values2<T, 0>(a, s), values2<T, 2>(a, s), values2<T, 0>(d, s),
                                                        values2<T, 2>(d, s)});
            }
        }
    }
}

// Page copies of up to 32 layers in a launch. Grid: pairs (strided over), K
// and V, layers.
constexpr int kCopyLayers = 32;
struct CopySet {
    uint8_t* codes[kCopyLayers][2];
    float* scales[kCopyLayers][2];
};

__global__ __launch_bounds__(256) void kv_copy_kernel(CopySet set, const int* __restrict__ src,
                                                      const int* __restrict__ dst, int count, int num_pages, int hkv,
                                                      uint32_t vecs) {
    uint8_t* codes = set.codes[blockIdx.z][blockIdx.y];
    float* scales = set.scales[blockIdx.z][blockIdx.y];
    for (int i = blockIdx.x; i < count; i += gridDim.x) {
        const int a = src[i], b = dst[i];
        if (a < 0 || a >= num_pages || b < 0 || b >= num_pages || a == b) continue;
        const uint8_t* from = codes + static_cast<size_t>(a) * vecs * 16;
        uint8_t* to = codes + static_cast<size_t>(b) * vecs * 16;
        for (uint32_t v0 = 0; v0 < vecs; v0 += 1024) {  // 4 pieces per thread in flight
            u32x4 x[4];
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t v = v0 + j * 256 + threadIdx.x;
                if (v < vecs) x[j] = ld16_stream(from + static_cast<size_t>(v) * 16);
            }
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const uint32_t v = v0 + j * 256 + threadIdx.x;
                if (v < vecs) st16_stream(to + static_cast<size_t>(v) * 16, x[j]);
            }
        }
        for (int h = threadIdx.x; h < hkv; h += 256)
            scales[static_cast<size_t>(b) * hkv + h] = scales[static_cast<size_t>(a) * hkv + h];
    }
}

// Pages that up to `most` consecutive tokens touch.
int pages_touched(int most, int ps) { return (most + ps - 2) / ps + 1; }

template <typename T, int D>
void launch_append(const dim3& grid, int threads, const KvView& kv, const void* k, const void* v, const int* cu,
                   const int* ctx, const int* table, int max_pages, int total, int* dropped) {
    kv_append_kernel<T, D><<<grid, dim3(threads), 0, stream()>>>(kv, static_cast<const uint16_t*>(k),
                                                                 static_cast<const uint16_t*>(v), cu, ctx, table,
                                                                 max_pages, total, dropped);
}

template <typename T>
int kv_append(const char* name, const ng_kv_int8_cache* cache, const void* k, const void* v, const void* cu,
              const void* ctx, const void* table, int batch, int max_pages, int total, int most, void* dropped) {
    if (kv_check_cache(name, cache) != 0) return -1;
    NG_REQUIRE(k && v, "%s: null pointer", name);
    if (kv_check_batch(name, cache, cu, ctx, table, batch, max_pages, total, most) != 0) return -1;
    NG_REQUIRE(aligned16(k) && aligned16(v), "%s: k and v must be 16-byte aligned", name);
    const dim3 grid(min(pages_touched(min(most, total), cache->page_size), 1 << 20), batch, 2 * cache->num_kv_heads);
    const int threads = cache->page_size / kSub * kWave;
    const auto call = [&](auto launch) {
        launch(grid, threads, kv_view(*cache), k, v, static_cast<const int*>(cu), static_cast<const int*>(ctx),
               static_cast<const int*>(table), max_pages, total, static_cast<int*>(dropped));
    };
    switch (cache->head_dim) {
        case 64: call(launch_append<T, 64>); break;
        case 128: call(launch_append<T, 128>); break;
        case 192: call(launch_append<T, 192>); break;
        default: call(launch_append<T, 256>); break;
    }
    NG_CHECK_LAUNCH(name);
    return 0;
}

template <typename T, int D>
void launch_read(const dim3& grid, int threads, const KvView& kv, void* k, void* v, const int* cu, const int* starts,
                 const int* table, int max_pages, int total) {
    kv_read_kernel<T, D><<<grid, dim3(threads), 0, stream()>>>(kv, static_cast<uint16_t*>(k), static_cast<uint16_t*>(v),
                                                               cu, starts, table, max_pages, total);
}

template <typename T>
int kv_read(const char* name, const ng_kv_int8_cache* cache, void* k, void* v, const void* cu, const void* starts,
            const void* table, int batch, int max_pages, int total, int most) {
    if (kv_check_cache(name, cache) != 0) return -1;
    NG_REQUIRE(k && v, "%s: null pointer", name);
    if (kv_check_batch(name, cache, cu, starts, table, batch, max_pages, total, most) != 0) return -1;
    NG_REQUIRE(aligned16(k) && aligned16(v), "%s: k and v must be 16-byte aligned", name);
    const dim3 grid(min(pages_touched(min(most, total), cache->page_size), 1 << 20), batch, 2 * cache->num_kv_heads);
    const int threads = cache->page_size / kSub * kWave;
    const auto call = [&](auto launch) {
        launch(grid, threads, kv_view(*cache), k, v, static_cast<const int*>(cu), static_cast<const int*>(starts),
               static_cast<const int*>(table), max_pages, total);
    };
    switch (cache->head_dim) {
        case 64: call(launch_read<T, 64>); break;
        case 128: call(launch_read<T, 128>); break;
        case 192: call(launch_read<T, 192>); break;
        default: call(launch_read<T, 256>); break;
    }
    NG_CHECK_LAUNCH(name);
    return 0;
}

}  // namespace
}  // namespace ng

using namespace ng;

extern "C" int ng_kv_int8_append(const ng_kv_int8_cache* cache, const void* k, const void* v, const void* cu_tokens,
                                 const void* context_lens, const void* page_table, int batch, int max_pages,
                                 int total_tokens, int max_tokens, void* d_dropped) {
    return kv_append<f16>("ng_kv_int8_append", cache, k, v, cu_tokens, context_lens, page_table, batch, max_pages,
                          total_tokens, max_tokens, d_dropped);
}

extern "C" int ng_bf16_kv_int8_append(const ng_kv_int8_cache* cache, const void* k, const void* v,
                                      const void* cu_tokens, const void* context_lens, const void* page_table,
                                      int batch, int max_pages, int total_tokens, int max_tokens, void* d_dropped) {
    return kv_append<bf16>("ng_bf16_kv_int8_append", cache, k, v, cu_tokens, context_lens, page_table, batch, max_pages,
                           total_tokens, max_tokens, d_dropped);
}

extern "C" int ng_kv_int8_read(const ng_kv_int8_cache* cache, void* k, void* v, const void* cu_tokens,
                               const void* starts, const void* page_table, int batch, int max_pages, int total_tokens,
                               int max_tokens) {
    return kv_read<f16>("ng_kv_int8_read", cache, k, v, cu_tokens, starts, page_table, batch, max_pages, total_tokens,
                        max_tokens);
}

extern "C" int ng_bf16_kv_int8_read(const ng_kv_int8_cache* cache, void* k, void* v, const void* cu_tokens,
                                    const void* starts, const void* page_table, int batch, int max_pages,
                                    int total_tokens, int max_tokens) {
    return kv_read<bf16>("ng_bf16_kv_int8_read", cache, k, v, cu_tokens, starts, page_table, batch, max_pages,
                         total_tokens, max_tokens);
}

extern "C" int ng_kv_int8_copy_pages(const ng_kv_int8_cache* caches, int num_caches, const void* src, const void* dst,
                                     int count) {
    const char* name = "ng_kv_int8_copy_pages";
    NG_REQUIRE(caches && src && dst, "%s: null pointer", name);
    NG_REQUIRE(num_caches >= 1 && num_caches <= 64, "%s: %d caches are outside 1..64", name, num_caches);
    NG_REQUIRE(count > 0, "%s: invalid count %d", name, count);
    NG_REQUIRE(count <= (1 << 30), "%s: count %d is above 2^30", name, count);
    for (int i = 0; i < num_caches; ++i) {
        if (kv_check_cache(name, &caches[i]) != 0) return -1;
        NG_REQUIRE(caches[i].num_pages == caches[0].num_pages && caches[i].num_kv_heads == caches[0].num_kv_heads &&
                       caches[i].head_dim == caches[0].head_dim && caches[i].page_size == caches[0].page_size,
                   "%s: cache %d has other sizes than cache 0", name, i);
    }
    const ng_kv_int8_cache& c = caches[0];
    const uint32_t vecs = static_cast<uint32_t>(static_cast<size_t>(c.num_kv_heads) * c.page_size * c.head_dim / 16);
    for (int l0 = 0; l0 < num_caches; l0 += kCopyLayers) {
        const int n = min(num_caches - l0, kCopyLayers);
        CopySet set{};
        for (int i = 0; i < n; ++i) {
            const ng_kv_int8_cache& x = caches[l0 + i];
            set.codes[i][0] = static_cast<uint8_t*>(x.k_codes);
            set.codes[i][1] = static_cast<uint8_t*>(x.v_codes);
            set.scales[i][0] = static_cast<float*>(x.k_scales);
            set.scales[i][1] = static_cast<float*>(x.v_scales);
        }
        kv_copy_kernel<<<dim3(min(count, 1 << 16), 2, n), dim3(256), 0, stream()>>>(
            set, static_cast<const int*>(src), static_cast<const int*>(dst), count, c.num_pages, c.num_kv_heads, vecs);
        NG_CHECK_LAUNCH(name);
    }
    return 0;
}
