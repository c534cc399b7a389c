// kv_cache.hpp - layout of the 8-bit paged key/value cache, shared by the
// kernels that write and read it (kv_cache.hip, kv_attention.hip).
//
// A page and head holds page_size x D codes as page_size / 16 sub-blocks of 16
// tokens, each D / 64 chunks of 1 KiB: 64 pieces of 16 bytes, one per lane of
// a wave, in the order in which a 16 x 16 x 32 MFMA takes its first operand, so
// that attention loads whole KiB straight into registers. A byte holds its code +
// 128, which v_perm turns into fp16 with one subtraction.
//   K: piece (kg, t) = 16 kg + t holds token t, d = 64 c + 16 kg + 0 .. 15.
//   V: piece (kg, q, r) = 16 kg + 4 q + r holds in dword i the tokens 4 q ..
//      4 q + 3 of d = 64 c + 16 kg + 4 i + r: K's order with each 4 x 4 block of
//      bytes transposed over the four lanes of a quad, which is how a wave
//      writes it.
#pragma once

#include "ng_common.hpp"
#include "../../include/kv_cache.h"

namespace ng {

constexpr int kSub = 16;                    // tokens of a sub-block
constexpr uint32_t kKvBias = 0x80808080u;  // codes to bytes and back

// A cache as the kernels take it; ps_log2: page_size = 1 << ps_log2.
struct KvView {
    uint8_t* kc;
    uint8_t* vc;
    float* ks;  // largest magnitudes; a value is code * that / 127
    float* vs;
    int num_pages, hkv, ps_log2;
};

inline bool kv_head_dim_ok(int D) { return D == 64 || D == 128 || D == 192 || D == 256; }
inline bool kv_page_ok(int p) { return p == 16 || p == 32 || p == 64 || p == 128; }
inline int kv_log2(int p) { return p == 16 ? 4 : p == 32 ? 5 : p == 64 ? 6 : 7; }

inline KvView kv_view(const ng_kv_int8_cache& c) {
    return KvView{static_cast<uint8_t*>(c.k_codes), static_cast<uint8_t*>(c.v_codes), static_cast<float*>(c.k_scales),
                  static_cast<float*>(c.v_scales), c.num_pages, c.num_kv_heads, kv_log2(c.page_size)};
}

inline int kv_check_cache(const char* name, const ng_kv_int8_cache* c) {
    NG_REQUIRE(c, "%s: null pointer", name);
    NG_REQUIRE(c->k_codes && c->v_codes && c->k_scales && c->v_scales, "%s: null pointer in the cache", name);
    NG_REQUIRE(c->num_pages > 0 && c->num_kv_heads > 0, "%s: invalid cache (pages=%d, heads=%d)", name, c->num_pages,
               c->num_kv_heads);
    NG_REQUIRE(c->num_kv_heads <= 32767, "%s: %d heads are too many", name, c->num_kv_heads);
    NG_REQUIRE(kv_head_dim_ok(c->head_dim), "%s: head_dim %d is not 64, 128, 192 or 256", name, c->head_dim);
    NG_REQUIRE(kv_page_ok(c->page_size), "%s: page_size %d is not 16, 32, 64 or 128", name, c->page_size);
    NG_REQUIRE(aligned16(c->k_codes) && aligned16(c->v_codes), "%s: codes must be 16-byte aligned", name);
    return 0;
}

// The batch arguments of the calls that go through a page table.
inline int kv_check_batch(const char* name, const ng_kv_int8_cache* c, const void* cu, const void* lens,
                          const void* table, int batch, int max_pages, int total, int most) {
    NG_REQUIRE(cu && lens && table, "%s: null pointer", name);
    NG_REQUIRE(batch > 0 && batch <= 65535, "%s: batch %d is outside 1..65535", name, batch);
    NG_REQUIRE(max_pages > 0 && total > 0 && most > 0, "%s: invalid sizes (max_pages=%d, tokens=%d, longest=%d)", name,
               max_pages, total, most);
    NG_REQUIRE(total < (1 << 30), "%s: 2^30 tokens or more", name);
    NG_REQUIRE(max_pages <= (1 << 30) / c->page_size, "%s: a table of more than 2^30 tokens", name);
    return 0;
}

// A load of memory that nothing writes while the kernel runs, at an address that
// is the same for the whole wave: scalar, so that it does not queue behind the
// vector loads in flight (a store to another array would otherwise forbid it).
template <typename X>
__device__ __forceinline__ X load_uniform(const X* p) {
    return *(const __attribute__((address_space(4))) X*)(reinterpret_cast<uintptr_t>(p));
}

// Sequence b's rows of a packed batch, whatever cu holds.
struct KvRows {
    int first, count;
};
__device__ __forceinline__ KvRows kv_rows(const int* cu, int b, int total) {
    const int a = min(max(load_uniform(cu + b), 0), total);
    return {a, max(min(load_uniform(cu + b + 1), total), a) - a};
}

// 4 x 4 bytes transposed over the four lanes of a quad: byte e of lane r's
// result is byte r of lane e's w. Its own inverse.
__device__ __forceinline__ uint32_t quad_transpose(uint32_t w, uint32_t sel) {
    const uint32_t a = dpp_u32<0x00>(w), b = dpp_u32<0x55>(w), c = dpp_u32<0xAA>(w), d = dpp_u32<0xFF>(w);
    const uint32_t lo = __builtin_amdgcn_perm(b, a, sel), hi = __builtin_amdgcn_perm(d, c, sel);
    return __builtin_amdgcn_perm(hi, lo, 0x05040100u);
}
// sel of lane r = lane % 4: byte r of the low operand, then byte r of the high one.
__device__ __forceinline__ uint32_t quad_selector(int lane) {
    return 0x0c0c0400u + 0x0101u * static_cast<uint32_t>(lane & 3);
}

}  // namespace ng
