// kv_attention.hip - attention over the 8-bit key/value cache (kv_cache.h; its
// layout: kv_cache.hpp).
//
// With a page's magnitudes k_s, v_s, codes k, v and x_j = c k_s (q . k_j):
//   out = 1/127 sum_j 2^(x_j - m) v_s v_j / sum_j 2^(x_j - m),  m a running
// maximum of the visible x_j (c holds log2(e) / 127), sums in 32 bits. One pass
// over the cache.
//
// Both products run on the matrix cores with the codes as exact fp16 integers:
//   S^T = K Q^T: rows are tokens, columns queries; the scale of a token's page
//     multiplies the 32-bit sums.
//   O^T = V^T P^T: a lane of S^T holds 4 tokens of one query, which are 4 of the 8
//     values of its second operand, so P goes from one product into the next
//     without leaving its lane. P's entries are 2^(x - m) v_s / u, u the
//     largest v_s that the row has met (the sums are rescaled when it grows, as
//     they are when m does): at most 1, as fp16, and lifted by a power of two into
//     fp16's upper range, so that a weight becomes subnormal only below 2^-29
//     (prompts 2^-21) and nothing below 2^-40 (2^-32): 10^5 small weights beside
//     a large one count. For single tokens an entry's rounding error is a second fp16
//     entry; prompts, where MFMAs are the bound, keep the first alone (11 bits).
//     The error against 64 bits, relative (4 x 4096 tokens, fp16): 0.00028 with the
//     first, 0.00021 with both, which is the output's own rounding; the second
//     costs 1.6-4.3% of a call's time (64 x 4096: 66.6 -> 67.8 us as a graph).
// The queries of all heads that share a key/value head, and of several tokens,
// are the columns: row r of a sequence and key/value head is head r % group of
// its token r / group.
//
// bf16 queries become fp16 times a power of two of their row, which loses
// nothing of elements within 2^-14 of the row's largest, and at most 2^-25 of
// that largest for the others.
#include "kv_cache.hpp"

#include <algorithm>

namespace ng {
namespace {

typedef _Float16 f16x8 __attribute__((ext_vector_type(8)));
typedef float f32x4 __attribute__((ext_vector_type(4)));
typedef float f32x16 __attribute__((ext_vector_type(16)));

constexpr float kNegInf = -__builtin_inff();
constexpr float kLeastUnit = 0x1p-124f;  // u of a row that has met nothing

struct AttnArgs {
    const int* cu;
    const int* lens;
    const int* table;
    int max_pages, total, hq, group;
    float scale;  // softmax_scale log2(e) / 127
    int window, sinks;
    int row_tile;       // rows that a block takes together
    int splits, chunk;  // slices of a sequence that there is room for; tiles of a slice
    float* part;        // their outputs [splits][total hq][D], then (m, l) [splits][total hq]
};

// Two codes (two bytes of a dword, which hold code + 128) as exact fp16 values:
// placed under an fp16 exponent of 2^10, 1152 subtracted.
template <uint32_t SEL>
__device__ __forceinline__ uint32_t codes2(uint32_t bytes) {
    const f16x2 bias = {static_cast<f16>(-1152.0f), static_cast<f16>(-1152.0f)};
    const f16x2 v = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, bytes, SEL)) + bias;
    return __builtin_bit_cast(uint32_t, v);
}
__device__ __forceinline__ f16x8 codes8(uint32_t lo, uint32_t hi) {
    return __builtin_bit_cast(f16x8, u32x4{codes2<0x04010400u>(lo), codes2<0x04030402u>(lo), codes2<0x04010400u>(hi),
                                           codes2<0x04030402u>(hi)});
}

// The larger of three (fmaxf would first make NaNs of either kind quiet, an
// operation for each of its operands; here a NaN loses either way).
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    __asm__("v_max3_f32 %0, %1, %2, %3" : "=v"(d) : "v"(a), "v"(b), "v"(c));
    return d;
}

// The tokens that a run of queries (positions p0 .. p1) sees, in tiles of 64:
// `lead` tiles from 0 on for the first tokens, then those from tile `from` on.
struct Tiles {
    int lead, from, count;
    __device__ __forceinline__ int tile(int i) const { return i < lead ? i : from + i - lead; }
};
__device__ __forceinline__ Tiles tiles_seen(int p0, int p1, int len, int window, int sinks) {
    const int end = (min(p1 + 1, len) + 63) >> 6;
    if (end <= 0) return {0, 0, 0};
    if (window == 0) return {0, 0, end};
    const int from = min(max(p0 - window + 1, 0) >> 6, end);
    const int lead = min((min(sinks, len) + 63) >> 6, from);
    return {lead, from, lead + end - from};
}

// How a row tile's tiles are shared out: slices of `chunk` tiles.
struct Slices {
    int chunk, count;
};
__device__ __forceinline__ Slices slices(const AttnArgs& a, int tiles) {
    const int chunk = max(a.chunk, (tiles + a.splits - 1) / a.splits);
    return {chunk, max((tiles + chunk - 1) / chunk, 1)};
}

// One sequence as a block sees it.
struct Seq {
    KvRows rows;
    int last;   // position of its last query
    int len;    // tokens that the table can hold of it
    const int* table;
};
__device__ __forceinline__ Seq sequence(const AttnArgs& a, const KvView& kv, int b) {
    Seq s;
    s.rows = kv_rows(a.cu, b, a.total);
    const int n = min(max(load_uniform(a.lens + b), 0), 1 << 30);
    s.last = n - 1;
    s.len = min(n, a.max_pages << kv.ps_log2);
    s.table = a.table + static_cast<size_t>(b) * a.max_pages;
    return s;
}

// A 16-token sub-block of a head (of a sequence that has tokens): byte offset of
// its codes, index of its scales, and whether there is such a page (if not, both
// name the first one, whose memory is there to be read).
struct Sub {
    size_t codes, scale;
    bool there;
};
__device__ __forceinline__ Sub sub_block(const KvView& kv, const Seq& s, int h, int token, int D) {
    int page = load_uniform(s.table + (min(token, s.len - 1) >> kv.ps_log2));
    const bool there = (token < s.len) & (page >= 0) & (page < kv.num_pages);
    page = there ? page : 0;
    const size_t ph = static_cast<size_t>(page) * kv.hkv + h;
    return {((ph << kv.ps_log2) + (token & ((1 << kv.ps_log2) - 1))) * D, ph, there};
}

// Values of the lane 32 away, and of the lanes 16, 32 and 48 away (those that
// hold a column of a 32 x 32 and of a 16 x 16 tile), joined with the lane's own.
template <typename F>
__device__ __forceinline__ float with_half(float v, F&& join) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    return join(as_float(r[0]), as_float(r[1]));
}
template <typename F>
__device__ __forceinline__ float with_rows(float v, F&& join) {
    const uint32_t b = __builtin_bit_cast(uint32_t, v);
    const auto r = __builtin_amdgcn_permlane16_swap(b, b, false, false);
    return with_half(join(as_float(r[0]), as_float(r[1])), join);
}
__device__ __forceinline__ float larger(float a, float b) { return max3(a, b, b); }
__device__ __forceinline__ float plus(float a, float b) { return a + b; }

// 2^(m - to) where to >= m may be -inf (nothing seen yet on either side).
__device__ __forceinline__ float decay(float m, float to) {
    return __builtin_amdgcn_exp2f(m - (to == kNegInf ? 0.0f : to));
}

// N pieces of 8 elements of a query row, piece j at row + at(j), as fp16
// operands; the lanes FROM (16 or 32) and its doubles away hold the rest of the
// row. Returns the factor that undoes bf16's scaling.
template <typename T, int N, int FROM, typename At>
__device__ __forceinline__ float load_row(const uint16_t* row, bool real, At&& at, f16x8 (&q)[N]) {
    u32x4 raw[N];
#pragma unroll
    for (int j = 0; j < N; ++j) raw[j] = real ? ld16(row + at(j)) : u32x4{0, 0, 0, 0};
    if constexpr (__is_same(T, f16)) {
#pragma unroll
        for (int j = 0; j < N; ++j) q[j] = __builtin_bit_cast(f16x8, raw[j]);
        return 1.0f;
    } else {
        uint32_t m = 0;
#pragma unroll
        for (int j = 0; j < N; ++j) m = absmax_bits8(raw[j], m);
#pragma unroll
        for (int off = FROM; off < kWave; off <<= 1)
            m = umax32(m, static_cast<uint32_t>(__shfl_xor(static_cast<int>(m), off, kWave)));
        const int e = max(static_cast<int>(m >> 7), 1) - 127;  // 2^e <= largest < 2^(e + 1)
        const float f = __builtin_ldexpf(1.0f, -e);
#pragma unroll
        for (int j = 0; j < N; ++j) {
            float x[8];
            unpack8<bf16>(raw[j], x);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] *= f;
            q[j] = __builtin_bit_cast(f16x8, pack8<f16>(x));
        }
        return __builtin_ldexpf(1.0f, e);
    }
}

// Few queries to a sequence: bound by reading the cache (64 sequences of up to
// 4096 tokens, 32 heads on 8, D = 128: 65 us, 5.3 TB/s; one of 131071: 44 us, 6.1
// TB/s, and 4-5 us for the join; 500 tokens: 6.9 us, latency). A block of four waves
// takes up to 16 rows and a slice of the tokens; a wave every fourth tile of
// 16 NB tokens, straight from memory into registers: K's codes of the next
// tile are requested when this tile's are used up, then V's, so that half a
// tile is always on its way. The waves' results are joined in LDS.
// Grid: slices, key/value heads x row tiles (strided over), batch.
constexpr int kDecodeWaves = 4;
constexpr float kDecodeLift = 0x1p15f;  // weights are at most 1

template <typename T, int D, int NB>
__global__ __launch_bounds__(kDecodeWaves * kWave) void kv_decode_kernel(uint16_t* out, const uint16_t* q, KvView kv,
                                                                         AttnArgs a) {
    constexpr int C = D / 64;
    constexpr int kPer = 4 / NB;  // steps of a 64-token tile
    __shared__ f32x4 s_o[kDecodeWaves - 1][D / 4][16];
    __shared__ float s_m[kDecodeWaves][16], s_l[kDecodeWaves][16];
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 15, kg = lane >> 4;
    const uint32_t koff = lane * 16, voff = (16 * (col >> 2) + 4 * kg + (col & 3)) * 16;
    const Seq s = sequence(a, kv, blockIdx.z);
    const int h = blockIdx.y % kv.hkv;
    const int R = s.rows.count * a.group;
    for (int r0 = blockIdx.y / kv.hkv * 16; r0 < R; r0 += static_cast<int>(gridDim.y) / kv.hkv * 16) {
        const int r = r0 + col;
        const bool real = r < R;
        const int i = r / a.group;
        const int p = real ? s.last - s.rows.count + 1 + i : -1;
        const int p0 = s.last - s.rows.count + 1 + r0 / a.group;
        const int p1 = s.last - s.rows.count + 1 + min(r0 + 15, R - 1) / a.group;
        const Tiles tl = tiles_seen(p0, p1, s.len, a.window, a.sinks);
        const Slices sl = slices(a, tl.count);
        if (static_cast<int>(blockIdx.x) >= sl.count) continue;
        const size_t row = static_cast<size_t>(s.rows.first + i) * a.hq + h * a.group + (r - i * a.group);
        f16x8 qf[2 * C];  // piece 2 c + j: d = 64 c + 16 kg + 8 j + 0 .. 7
        const float unscale = load_row<T, 2 * C, 16>(q + row * D, real, [&](int j) { return 64 * (j >> 1) + 16 * kg + 8 * (j & 1); }, qf);

        const int v0 = static_cast<int>(blockIdx.x) * sl.chunk, v1 = min(v0 + sl.chunk, tl.count);
        const int steps = max(v1 - v0, 0) * kPer;  // of the block; wave w takes step w, w + 4, ...
        const auto token_of = [&](int step) { return tl.tile(v0 + step / kPer) * 64 + step % kPer * (16 * NB); };
        u32x4 kr[NB][C], vr[NB][C];
        Sub sub[NB], nsub[NB];
        const auto find = [&](int step, Sub (&x)[NB]) {
            const int t0 = token_of(step);
#pragma unroll
            for (int t = 0; t < NB; ++t) x[t] = sub_block(kv, s, h, t0 + 16 * t, D);
        };
        const auto load_k = [&](const Sub (&x)[NB]) {
#pragma unroll
            for (int t = 0; t < NB; ++t)
#pragma unroll
                for (int c = 0; c < C; ++c) kr[t][c] = ld16_stream(kv.kc + x[t].codes + 1024 * c + koff);
        };
        const auto load_v = [&](const Sub (&x)[NB]) {
#pragma unroll
            for (int t = 0; t < NB; ++t)
#pragma unroll
                for (int c = 0; c < C; ++c) vr[t][c] = ld16_stream(kv.vc + x[t].codes + 1024 * c + voff);
        };
        float m = kNegInf, l = 0.0f, u = kLeastUnit;
        f32x4 acc[C][4];
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) acc[c][j] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        int step = wave;
        if (step < steps) {
            find(step, sub);
            load_k(sub);
            load_v(sub);
        }
        for (; step < steps; step += kDecodeWaves) {
            const bool more = step + kDecodeWaves < steps;
            if (more) find(step + kDecodeWaves, nsub);
            float ks[NB], vs[NB];
#pragma unroll
            for (int t = 0; t < NB; ++t) ks[t] = load_uniform(kv.ks + sub[t].scale), vs[t] = load_uniform(kv.vs + sub[t].scale);
            f32x4 x[NB];
#pragma unroll
            for (int t = 0; t < NB; ++t) {
                x[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                for (int c = 0; c < C; ++c) {
                    x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(kr[t][c][0], kr[t][c][1]), qf[2 * c], x[t], 0, 0, 0);
                    x[t] = __builtin_amdgcn_mfma_f32_16x16x32_f16(codes8(kr[t][c][2], kr[t][c][3]), qf[2 * c + 1], x[t], 0, 0, 0);
                }
            }
            if (more) load_k(nsub);
            // Scores; those of tokens that a row does not see become -inf.
            const int t0 = token_of(step);
            bool whole = (t0 + 16 * NB - 1 <= p0) & (t0 + 16 * NB <= s.len) &
                         ((a.window == 0) | (t0 > p1 - a.window) | (t0 + 16 * NB <= a.sinks));
#pragma unroll
            for (int t = 0; t < NB; ++t) whole = whole & sub[t].there;
            float sc[NB][4];
#pragma unroll
            for (int t = 0; t < NB; ++t) {
                const float f = ks[t] * a.scale * unscale;
#pragma unroll
                for (int e = 0; e < 4; ++e) sc[t][e] = x[t][e] * f;
            }
            float un = 0.0f;  // the largest v_s of pages with a token that the row sees
            if (whole) {
#pragma unroll
                for (int t = 0; t < NB; ++t) un = fmaxf(un, vs[t]);
            } else {
#pragma unroll
                for (int t = 0; t < NB; ++t) {
                    bool some = false;
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int j = t0 + 16 * t + 4 * kg + e;
                        const bool seen = sub[t].there & (j <= p) & (j < s.len) &
                                          ((a.window == 0) | (j > p - a.window) | (j < a.sinks));
                        sc[t][e] = seen ? sc[t][e] : kNegInf;
                        some |= seen;
                    }
                    vs[t] = some ? vs[t] : 0.0f;
                    un = fmaxf(un, vs[t]);
                }
                un = with_rows(un, larger);
            }
            un = fmaxf(un, u);
            float mx = m;
#pragma unroll
            for (int t = 0; t < NB; ++t) mx = max3(max3(sc[t][0], sc[t][1], sc[t][2]), sc[t][3], mx);
            mx = with_rows(mx, larger);
            const float base = mx == kNegInf ? 0.0f : mx;
            const float down = decay(m, mx);
            l *= down;
            // 4 / u, so that neither u / 4 nor its reciprocal is subnormal, which v_rcp_f32 takes for 0.
            const float inv_u = __builtin_amdgcn_rcpf(0.25f * un);
            const float fade = un > u ? down * (0.25f * u * inv_u) : down;
            if (__any(fade != 1.0f)) {
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j) acc[c][j] *= fade;
            }
            m = mx;
            u = un;
            uint32_t pp[NB][2], pl[NB][2];  // weights, and what their rounding left
#pragma unroll
            for (int t = 0; t < NB; ++t) {
                const float f = 0.25f * vs[t] * inv_u * kDecodeLift;
                float w[4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    w[e] = __builtin_amdgcn_exp2f(sc[t][e] - base);
                    l += w[e];
                    w[e] *= f;
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    pp[t][e] = pack2<f16>(w[2 * e], w[2 * e + 1]);
                    pl[t][e] = pack2<f16>(w[2 * e] - el_get<f16, 0>(pp[t][e]), w[2 * e + 1] - el_get<f16, 1>(pp[t][e]));
                }
            }
#pragma unroll
            for (int t = 0; t < NB; t += 2) {
                const f16x8 pb = __builtin_bit_cast(f16x8, u32x4{pp[t][0], pp[t][1], pp[t + 1][0], pp[t + 1][1]});
                const f16x8 rest = __builtin_bit_cast(f16x8, u32x4{pl[t][0], pl[t][1], pl[t + 1][0], pl[t + 1][1]});
#pragma unroll
                for (int c = 0; c < C; ++c)
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const f16x8 vt = codes8(vr[t][c][j], vr[t + 1][c][j]);
                        acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, rest, acc[c][j], 0, 0, 0);
                        acc[c][j] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vt, pb, acc[c][j], 0, 0, 0);
                    }
            }
            if (more) load_v(nsub);
#pragma unroll
            for (int t = 0; t < NB; ++t) sub[t] = nsub[t];
        }
        l = with_rows(l, plus);
        // Join the waves: lane (column, kg) of each holds d = 64 c + 16 kg + 4 j + e.
        if (kg == 0) {
            s_m[wave][col] = m;
            s_l[wave][col] = l;
        }
        __syncthreads();
        float M = s_m[0][col];
#pragma unroll
        for (int w = 1; w < kDecodeWaves; ++w) M = fmaxf(M, s_m[w][col]);
        float L = 0.0f;
#pragma unroll
        for (int w = 0; w < kDecodeWaves; ++w) L += s_l[w][col] * decay(s_m[w][col], M);
        // u / (127 L) first: u times the sums may pass fp32's range where the output does not.
        const float f = L == 0.0f ? 0.0f : decay(m, M) * (u / (127.0f * L));
#pragma unroll
        for (int c = 0; c < C; ++c)
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                acc[c][j] *= 1.0f / kDecodeLift;
                acc[c][j] *= f;
                if (wave > 0) s_o[wave - 1][16 * c + 4 * kg + j][col] = acc[c][j];
            }
        __syncthreads();
        if (wave == 0 && real) {
            const size_t all = static_cast<size_t>(a.total) * a.hq;
            const size_t slot = blockIdx.x * all + row;
#pragma unroll
            for (int c = 0; c < C; ++c) {
                float o[16];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
#pragma unroll
                    for (int w = 0; w < kDecodeWaves - 1; ++w) acc[c][j] += s_o[w][16 * c + 4 * kg + j][col];
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[4 * j + e] = acc[c][j][e];
                }
                if (sl.count > 1) {
                    float* to = a.part + slot * D + 64 * c + 16 * kg;
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        *reinterpret_cast<f32x4*>(to + 4 * j) = f32x4{o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]};
                } else {
                    uint16_t* to = out + row * D + 64 * c + 16 * kg;
#pragma unroll
                    for (int j = 0; j < 2; ++j) {
                        float y[8];
#pragma unroll
                        for (int e = 0; e < 8; ++e) y[e] = o[8 * j + e];
                        st16(to + 8 * j, pack8<T>(y));
                    }
                }
            }
            if (sl.count > 1 && kg == 0) {
                float* ml = a.part + a.splits * all * D + slot * 2;
                ml[0] = M;
                ml[1] = L;
            }
        }
        __syncthreads();  // LDS is free for the next row tile
    }
}

// Many queries to a sequence: bound by the power limit. 8192 tokens, 32 heads on
// 8, D = 128, causal: 570-625 us on MI355X (880-965 TFLOP/s; a plain product
// reaches 1090-1160 there) at 1.86 GHz, 468 us on zeros at full clock; without
// the reads of first operands 552 of 596 us, without conversion into LDS 518,
// without exponentials 551. A block of four waves takes 128 rows, 32 a wave (32
// x 32 x 16 MFMAs), and goes through tiles of 64 tokens. A tile's codes become
// fp16 once a block, on their way into LDS: while a tile is multiplied, the next
// one's codes, which arrived in registers a tile earlier, are converted into the
// other half of LDS, and the one after that is requested. Wave w brings sub-block w.
//   K in LDS: 16-byte pieces (d / 8, token), V: (sub-block, g, position of d),
//   a piece being the 8 tokens that lane half g of an MFMA's second operand
//   holds, quads g and 2 + g. d = 64 c + 16 kg + 4 i + r stands at position
//   64 c + 16 i + 4 kg + r, so that a wave's writes of one i are contiguous.
// Every MFMA of a wave has VALU work of its own beside it, in four phases:
//   scores of tokens 0-31     | K of the next tile converted
//   scores of tokens 32-63    | weights of tokens 0-31
//   V P of tokens 0-31        | weights of tokens 32-63
//   V P of tokens 32-63       | V of the next tile converted
// (left to the two waves of a SIMD to overlap, they did not: the waves fall
// into step, and MFMAs and VALU took 37% and 60% of the time one after the
// other.) A row's maximum is raised only when a score passes it by 2^8 (weights
// up to 2^8 then, exact all the same), so most tiles rescale nothing. v_s / u
// goes into the exponent, 2^(x - m + log2(v_s / u)), and out of it again for
// the sum, once for a sub-block.
// Grid: row tiles x key/value heads (the last rows, which see most, first; a
// head's blocks in the same L2 where 8 divides the heads), batch, slices.
constexpr int kPromptWaves = 4, kPromptRows = 32 * kPromptWaves;
constexpr float kLazy = 8.0f;
constexpr float kPromptLift = 7.0f;  // log2; weights are at most 2^kLazy
// Up to this many blocks, most of which are resident at once, those of all
// sequences that see most come first (three prompts of up to 1000 tokens, 768
// blocks: 40.3 -> 37.5 us; two of 1000: 37.7 -> 35.4), above it sequence by
// sequence, whose light blocks run beside the next one's heavy ones (two of 2000,
// 1024 blocks: 73 us against 89).
constexpr unsigned kMixBlocks = 768;

template <typename T, int D>
__global__ __launch_bounds__(kPromptWaves * kWave, D <= 128 ? 2 : 1) void kv_prompt_kernel(uint16_t* out,
                                                                                          const uint16_t* q, KvView kv,
                                                                                          AttnArgs a) {
    constexpr int C = D / 64, N = D / 16;  // MFMAs of a phase, dwords of K or V that a lane brings
    constexpr int kHalf = 64 * D * 2;       // bytes of a tile of K
    __shared__ __align__(1024) uint8_t lds[2][2 * kHalf];
    __shared__ __align__(16) float s_scale[2][2][32][4];  // of the sub-blocks: K's (< 0: no page), log2 of V's
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const int col = lane & 31, g = lane >> 5;
    const bool mixed = gridDim.x * gridDim.y <= kMixBlocks;
    const unsigned pos = blockIdx.y * gridDim.x + blockIdx.x;
    const int h = static_cast<int>((mixed ? pos : blockIdx.x) % kv.hkv);
    const int b = mixed ? pos / kv.hkv % gridDim.y : blockIdx.y;
    const int behind = mixed ? pos / (kv.hkv * gridDim.y) : blockIdx.x / kv.hkv;
    const Seq s = sequence(a, kv, b);
    const int R = s.rows.count * a.group, tiles = (R + kPromptRows - 1) / kPromptRows;
    const int first = s.last - s.rows.count + 1;  // position of the first query
    const int kput = ((2 * (lane >> 4)) * 64 + kSub * wave + (lane & 15)) * 16;
    const int vput = kHalf + ((2 * wave + ((lane >> 2) & 1)) * D + 4 * (lane >> 4) + (lane & 3)) * 16 + ((lane >> 3) & 1) * 8;
    for (int rt = tiles - 1 - behind; rt >= 0; rt -= static_cast<int>(gridDim.x) / kv.hkv) {
        const int r0 = rt * kPromptRows;
        const int p0 = first + r0 / a.group, p1 = first + min(r0 + kPromptRows - 1, R - 1) / a.group;
        const Tiles tl = tiles_seen(p0, p1, s.len, a.window, a.sinks);
        const Slices sl = slices(a, tl.count);
        if (static_cast<int>(blockIdx.z) >= sl.count) continue;
        const int v0 = static_cast<int>(blockIdx.z) * sl.chunk, v1 = min(v0 + sl.chunk, tl.count);
        // The wave's rows and their positions.
        const int rw = r0 + 32 * wave, r = rw + col;
        const bool real = r < R;
        const int i = r / a.group, p = real ? first + i : -1;
        const int pw0 = first + rw / a.group, pw1 = rw < R ? first + min(rw + 31, R - 1) / a.group : -1;
        const size_t row = static_cast<size_t>(s.rows.first + i) * a.hq + h * a.group + (r - i * a.group);
        f16x8 qf[D / 16];
        const float unscale = load_row<T, D / 16, 32>(q + row * D, real, [&](int j) { return 16 * j + 8 * g; }, qf);

        u32x4 kr[C], vr[C];
        float ks = -1.0f, vs = 0.0f;
        Sub sub;
        const auto find = [&](int v) { sub = sub_block(kv, s, h, tl.tile(min(v, v1 - 1)) * 64 + kSub * wave, D); };
        const auto request_k = [&] {  // of the sub-block in `sub`, and its scales
#pragma unroll
            for (int c = 0; c < C; ++c) kr[c] = ld16(kv.kc + sub.codes + 1024 * c + 16 * lane);
            ks = load_uniform(kv.ks + sub.scale);
            vs = load_uniform(kv.vs + sub.scale);
            ks = sub.there ? ks : -1.0f;
            vs = sub.there ? vs : 0.0f;
        };
        const auto request_v = [&] {
#pragma unroll
            for (int c = 0; c < C; ++c) vr[c] = ld16(kv.vc + sub.codes + 1024 * c + 16 * lane);
        };
        // Dword d of what was requested, as fp16 into LDS (after a slice's last tile once more, for nobody).
        u32x2 before;
        const auto put_k = [&](int half, int d) {
            const uint32_t w = kr[d >> 2][d & 3];
            const u32x2 y = {codes2<0x04010400u>(w), codes2<0x04030402u>(w)};
            if (d & 1)
                *reinterpret_cast<u32x4*>(lds[half] + kput + (d >> 2) * 8192 + ((d >> 1) & 1) * 1024) =
                    u32x4{before[0], before[1], y[0], y[1]};
            before = y;
        };
        const auto put_v = [&](int half, int d) {
            const uint32_t w = vr[d >> 2][d & 3];
            *reinterpret_cast<u32x2*>(lds[half] + vput + (d >> 2) * 1024 + (d & 3) * 256) =
                u32x2{codes2<0x04010400u>(w), codes2<0x04030402u>(w)};
        };
        const auto put_scales = [&](int half) {
            s_scale[half][g][col][wave] = g == 0 ? ks : __builtin_amdgcn_logf(vs);
        };

        float m = kNegInf, l = 0.0f, lu = -126.0f;  // lu: log2 u
        f32x16 acc[D / 32];
#pragma unroll
        for (int b = 0; b < D / 32; ++b) acc[b] = f32x16{};
        if (v0 < v1) {
            find(v0);
            request_k();
            request_v();
#pragma unroll
            for (int d = 0; d < N; ++d) put_k(0, d), put_v(0, d);
            put_scales(0);
            find(v0 + 1);
            request_k();
            request_v();
            find(v0 + 2);
        }
        __syncthreads();
        for (int v = v0; v < v1; ++v) {
            const int half = (v - v0) & 1;
            const int t0 = tl.tile(v) * 64;
            // First operands of the tile's 4 N MFMAs in order, read three ahead.
            const uint8_t *kb = lds[half] + (g * 64 + col) * 16, *vb = lds[half] + kHalf + (g * D + col) * 16;
            f16x8 ring[4];
            const auto read = [&](int j) {
                if (j >= 4 * N) return;
                const int b = j / N % 2, d = j % N;
                const uint8_t* at = j < 2 * N ? kb + (2 * d * 64 + 32 * b) * 16
                                              : vb + (2 * (2 * b + d / (D / 32)) * D + 32 * (d % (D / 32))) * 16;
                ring[j & 3] = *reinterpret_cast<const f16x8*>(at);
            };
            read(0), read(1), read(2);
            const f32x4 ks4 = *reinterpret_cast<const f32x4*>(s_scale[half][0][col]);
            const f32x4 lv4 = *reinterpret_cast<const f32x4*>(s_scale[half][1][col]);
            put_scales(half ^ 1);
            __builtin_amdgcn_sched_barrier(0);
            f32x16 x = f32x16{}, y = f32x16{};
#pragma unroll
            for (int d = 0; d < N; ++d) {
                read(d + 3);
                x = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[d & 3], qf[d], x, 0, 0, 0);
                put_k(half ^ 1, d);
                __builtin_amdgcn_sched_barrier(0);
            }
            request_k();
            bool whole = (t0 + 63 <= pw0) & (t0 + 64 <= s.len) &
                         ((a.window == 0) | (t0 > pw1 - a.window) | (t0 + 64 <= a.sinks));
            const float ksv[4] = {ks4[0], ks4[1], ks4[2], ks4[3]};
            float lv[4] = {lv4[0], lv4[1], lv4[2], lv4[3]}, f[4];
#pragma unroll
            for (int b = 0; b < 4; ++b) {
                // A sub-block's factor is kept above 0 so that -inf stays -inf.
                f[b] = fmaxf(ksv[b] * a.scale * unscale, 0x1p-126f);
            }
            const float least = fminf(fminf(ksv[0], ksv[1]), fminf(ksv[2], ksv[3]));
            whole = whole & (__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, least)) >= 0);
            // Token of score e of half b: t0 + 32 b + 8 (e / 4) + 4 g + e % 4, of sub-block 2 b + e / 8. Scores that the
            // row does not see become -inf; whether its maximum or u have to grow for the others.
            float mx, lx;
            const auto look = [&](int b, const f32x16& x, float (&sc)[16]) {
#pragma unroll
                for (int e = 0; e < 16; ++e) sc[e] = x[e];
                if (!whole) {
#pragma unroll
                    for (int n = 0; n < 2; ++n) {
                        bool some = false;
#pragma unroll
                        for (int e = 8 * n; e < 8 * n + 8; ++e) {
                            const int j = t0 + 32 * b + 8 * (e >> 2) + 4 * g + (e & 3);
                            const bool seen = (ksv[2 * b + n] >= 0.0f) & (j <= p) & (j < s.len) &
                                              ((a.window == 0) | (j > p - a.window) | (j < a.sinks));
                            sc[e] = seen ? sc[e] : kNegInf;
                            some |= seen;
                        }
                        lv[2 * b + n] = some ? lv[2 * b + n] : kNegInf;
                    }
                }
                float top[2];
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float* c = sc + 8 * n;
                    top[n] = max3(max3(c[0], c[1], c[2]), max3(c[3], c[4], c[5]), max3(c[6], c[7], c[7])) * f[2 * b + n];
                }
                mx = with_half(larger(top[0], top[1]), larger);
                lx = larger(lv[2 * b], lv[2 * b + 1]);
                if (!whole) lx = with_half(lx, larger);
                return __any((mx > m + kLazy) | (lx > lu));
            };
            const auto rescale = [&] {
                const float to = mx > m + kLazy ? mx : m;
                const float down = decay(m, to);
                const float fade = down * __builtin_amdgcn_exp2f(fminf(lu - lx, 0.0f));
                l *= down;
#pragma unroll
                for (int b = 0; b < D / 32; ++b) acc[b] *= fade;
                m = to;
                lu = fmaxf(lu, lx);
            };
            // Weights of the scores [16 d / N, 16 (d + 1) / N) of half b; log2(v_s / u) is kept where its inverse is
            // finite: below, V's part is nothing beside what u stands for.
            float off[2], back[2], w[16];
            const auto begin = [&](int b) {
                const float base = m == kNegInf ? 0.0f : m;
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    const float d = fmaxf(lv[2 * b + n] - lu, -60.0f) + kPromptLift;
                    off[n] = d - base;
                    back[n] = __builtin_amdgcn_exp2f(-d);
                }
            };
            const auto weigh = [&](int b, int d, const float (&sc)[16], uint32_t (&pk)[8]) {
#pragma unroll
                for (int e = 16 * d / N; e < 16 * (d + 1) / N; ++e) {
                    const int n = e >> 3;
                    w[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(sc[e], f[2 * b + n], off[n]));
                    if (e & 1) {
                        pk[e >> 1] = __builtin_bit_cast(uint32_t, __builtin_convertvector(f32x2{w[e - 1], w[e]}, f16x2));
                        w[e] += w[e - 1];
                        if ((e & 7) != 1) w[e] += w[e - 2];
                        if ((e & 7) == 7) l = __builtin_fmaf(w[e], back[n], l);
                    }
                }
            };
            float sc[16], sd[16];
            uint32_t pa[8], pb[8];
            const auto operand = [](const uint32_t (&pk)[8], int n) {
                return __builtin_bit_cast(f16x8, u32x4{pk[4 * n], pk[4 * n + 1], pk[4 * n + 2], pk[4 * n + 3]});
            };
            const auto add = [&](int d, int j, const uint32_t (&pk)[8]) {
                acc[d % (D / 32)] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[j & 3], operand(pk, d / (D / 32)),
                                                                           acc[d % (D / 32)], 0, 0, 0);
            };
            if (look(0, x, sc)) rescale();
            begin(0);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 0; d < N; ++d) {
                read(N + d + 3);
                y = __builtin_amdgcn_mfma_f32_32x32x16_f16(ring[(N + d) & 3], qf[d], y, 0, 0, 0);
                weigh(0, d, sc, pa);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int k = 0; k < 8; ++k) __asm__ volatile("" : "+v"(pa[k]));  // weighed here, not where it is used
            if (look(1, y, sd)) {
                // What is weighed already counts under the old maximum and u.
#pragma unroll
                for (int d = 0; d < N; ++d) {
                    const f16x8 first = *reinterpret_cast<const f16x8*>(vb + (2 * (d / (D / 32)) * D + 32 * (d % (D / 32))) * 16);
                    acc[d % (D / 32)] = __builtin_amdgcn_mfma_f32_32x32x16_f16(first, operand(pa, d / (D / 32)),
                                                                               acc[d % (D / 32)], 0, 0, 0);
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) pa[k] = 0;
                rescale();
            }
            begin(1);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int d = 0; d < N; ++d) {
                read(2 * N + d + 3);
                add(d, 2 * N + d, pa);
                weigh(1, d, sd, pb);
                __builtin_amdgcn_sched_barrier(0);
            }
#pragma unroll
            for (int d = 0; d < N; ++d) {
                read(3 * N + d + 3);
                add(d, 3 * N + d, pb);
                put_v(half ^ 1, d);
                __builtin_amdgcn_sched_barrier(0);
            }
            request_v();
            find(v + 3);
            __syncthreads();
        }
        l = with_half(l, plus);
        if (real) {
            const float inv = l == 0.0f ? 0.0f : __builtin_amdgcn_exp2f(lu) / (127.0f * l);
            const size_t all = static_cast<size_t>(a.total) * a.hq, slot = blockIdx.z * all + row;
            // acc[b][4 n + e] is position 32 b + 8 n + 4 g + e: i = 2 (b % 2) + n / 2, kg = 2 (n % 2) + g.
#pragma unroll
            for (int c = 0; c < C; ++c)
#pragma unroll
                for (int n = 0; n < 2; ++n) {
                    float o[16];
#pragma unroll
                    for (int j = 0; j < 4; ++j)
#pragma unroll
                        for (int e = 0; e < 4; ++e) o[4 * j + e] = acc[2 * c + (j >> 1)][4 * (2 * (j & 1) + n) + e] * 0x1p-7f * inv;
                    const int d = 64 * c + 16 * (2 * n + g);
                    if (sl.count > 1) {
#pragma unroll
                        for (int j = 0; j < 4; ++j)
                            *reinterpret_cast<f32x4*>(a.part + slot * D + d + 4 * j) =
                                f32x4{o[4 * j], o[4 * j + 1], o[4 * j + 2], o[4 * j + 3]};
                    } else {
#pragma unroll
                        for (int j = 0; j < 2; ++j) {
                            float y[8];
#pragma unroll
                            for (int e = 0; e < 8; ++e) y[e] = o[8 * j + e];
                            st16(out + row * D + d + 8 * j, pack8<T>(y));
                        }
                    }
                }
            if (sl.count > 1 && g == 0) {
                float* ml = a.part + a.splits * all * D + slot * 2;
                ml[0] = m;
                ml[1] = l;
            }
        }
    }
}

// Joins the slices of a row: out = sum_s l_s 2^(m_s - M) o_s / sum_s l_s 2^(m_s - M).
// WAVES waves a row, wave w the slices w, w + WAVES, ..., eight on their way at a
// time (one after the other took 37 us for 32 rows of 128 slices, longer than
// the attention itself); a block has four waves, so 4 / WAVES rows. Rows of one
// slice are done already. Grid: rows of a sequence (strided over), batch.
constexpr int kJoinWaves = 4;

template <typename T, int D, int WAVES>
__global__ __launch_bounds__(kJoinWaves * kWave) void kv_join_kernel(uint16_t* out, KvView kv, AttnArgs a) {
    constexpr int C = D / 64, kRows = kJoinWaves / WAVES;
    __shared__ float s_o[kJoinWaves][D];
    const Seq s = sequence(a, kv, blockIdx.y);
    const int lane = threadIdx.x & (kWave - 1);
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x / kWave);
    const size_t all = static_cast<size_t>(a.total) * a.hq;
    const int rows = s.rows.count * a.hq;
    for (int first = blockIdx.x * kRows; first < rows; first += gridDim.x * kRows) {
        const int rr = min(first + wave / WAVES, rows - 1);  // a block's last rows may be the same one
        const int i = rr / a.hq, hh = rr - i * a.hq;
        const int r = i * a.group + hh % a.group, r0 = r & -a.row_tile, R = s.rows.count * a.group;
        const int p0 = s.last - s.rows.count + 1 + r0 / a.group;
        const int p1 = s.last - s.rows.count + 1 + min(r0 + a.row_tile - 1, R - 1) / a.group;
        const int n = slices(a, tiles_seen(p0, p1, s.len, a.window, a.sinks).count).count;
        if (n == 1) continue;  // the whole block's where WAVES is 4; a wave's own otherwise, which waits for nobody
        const size_t row = static_cast<size_t>(s.rows.first) * a.hq + rr;
        const float* ml = a.part + a.splits * all * D + row * 2;
        const float* po = a.part + row * D + lane;
        float M = kNegInf;
        for (int x = lane; x < n; x += kWave) M = fmaxf(M, ml[x * all * 2]);
        M = wave_max_f32(M);
        float L = 0.0f, o[C];
#pragma unroll
        for (int c = 0; c < C; ++c) o[c] = 0.0f;
        for (int x0 = 0; x0 < n; x0 += kWave) {
            // 64 slices' weights, one to a lane.
            const int mine = x0 + lane, end = min(n - x0, kWave);
            const float w = mine < n ? ml[mine * all * 2 + 1] * decay(ml[mine * all * 2], M) : 0.0f;
            L += wave_sum_f32(w);
            for (int x = wave % WAVES; x < end; x += 8 * WAVES) {
                float v[8][C];
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int y = min(x + k * WAVES, end - 1);
#pragma unroll
                    for (int c = 0; c < C; ++c) v[k][c] = po[(x0 + y) * all * D + 64 * c];
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const int y = x + k * WAVES;
                    const float f = y < end ? __shfl(w, y, kWave) : 0.0f;
#pragma unroll
                    for (int c = 0; c < C; ++c) o[c] += f * v[k][c];
                }
            }
        }
        const float inv = L == 0.0f ? 0.0f : 1.0f / L;
        if constexpr (WAVES == 1) {
#pragma unroll
            for (int c = 0; c < C; ++c) out[row * D + 64 * c + lane] = from_f32<T>(o[c] * inv);
        } else {
#pragma unroll
            for (int c = 0; c < C; ++c) s_o[wave][64 * c + lane] = o[c];
            __syncthreads();
            for (int d = threadIdx.x; d < D; d += kJoinWaves * kWave) {
                float v = 0.0f;
#pragma unroll
                for (int w = 0; w < kJoinWaves; ++w) v += s_o[w][d];
                out[row * D + d] = from_f32<T>(v * inv);
            }
            __syncthreads();
        }
    }
}

// ---- host side ---------------------------------------------------------------

// Sequences of at least kPromptFrom rows take the prompt kernel.
constexpr int kPromptFrom = 33;
// Slices worth having with few queries: two blocks to a CU (that many are
// resident; 64 sequences of up to 4096 tokens: 67 us with 512 blocks in one
// slice, 75-80 us with 1024 in two, and the join), a tile to a wave at least.
// Below 1024 tokens the join costs more than it saves (500 tokens: 7.4 us in
// one slice, 9.7 in two; 4096 tokens of one sequence: 13 us in 16 slices, 15 in 8).
constexpr int kBlocksWanted = 512, kTilesLeast = 4;
struct Plan {
    bool prompt;
    int row_tile, row_tiles, splits, chunk;
};

size_t slice_bytes(size_t rows, int D) { return rows * (D + 2) * sizeof(float); }

// Slices worth having with many queries, from how long a launch would take: a
// tile of 64 tokens at D = 128 takes a block 1.4 us where it has a CU to
// itself and 2.4 us where two share one (as many as are resident up to D =
// 128); the join, 5 us and its traffic at 4 TB/s. A prompt from its first
// token on sees half its tiles on average. (512 queries behind 8000 tokens, 8
// heads: 178 us in one slice, 122 in two, 106 in four; a prompt of 1000, 32
// heads: 31 us in one slice, 50 in two.)
int prompt_splits(int D, long long blocks, long long rows, double average, int tiles) {
    const int resident = D <= 128 ? 512 : 256;
    int best = 1;
    double least = 0.0;
    for (int s = 1; s <= 64 && s <= std::max(tiles / kTilesLeast, 1); ++s) {
        const int chunk = (tiles + s - 1) / s;
        const double each = (blocks * s <= 256 ? 1.4 : D <= 128 ? 2.4 : 1.4) * D / 128;
        double t = std::max(chunk * each, average * static_cast<double>(blocks) / resident * each);
        if (s > 1) t += 5.0 + static_cast<double>(s) * 2.0 * static_cast<double>(slice_bytes(rows, D)) / 4e6;
        if (s == 1 || t < least) {
            best = s;
            least = t;
        }
    }
    return best;
}

Plan plan(int hkv, int group, int D, int batch, int max_q, int max_kv, int window, int sinks) {
    Plan p;
    const long long rows = static_cast<long long>(max_q) * group;
    p.prompt = rows >= kPromptFrom;
    p.row_tile = p.prompt ? kPromptRows : 16;
    p.row_tiles = static_cast<int>(std::min((rows + p.row_tile - 1) / p.row_tile, 1ll << 30));
    // Tiles that a block's rows see at most: all, or the window of each of its tokens and the first tokens.
    int tiles = (std::min(max_kv, 1 << 30) + 63) / 64;
    double average = std::max(tiles - max_q / 128.0, tiles * 0.5);
    const long long seen = (static_cast<long long>(window) + p.row_tile / group + 127) / 64 + (static_cast<long long>(sinks) + 63) / 64;
    if (window > 0 && seen < tiles) average = tiles = static_cast<int>(seen);
    const long long blocks = static_cast<long long>(batch) * hkv * p.row_tiles;
    const long long want = (kBlocksWanted + blocks - 1) / blocks;
    const int most = tiles < 4 * kTilesLeast ? 1 : tiles / kTilesLeast;
    p.splits = p.prompt ? prompt_splits(D, blocks, rows * hkv * batch, average, tiles)
                        : static_cast<int>(std::min<long long>(want, most));
    p.chunk = (tiles + p.splits - 1) / p.splits;
    p.splits = (tiles + p.chunk - 1) / p.chunk;
    return p;
}

template <typename T, int D>
void launch_attention(const Plan& p, int batch, uint16_t* out, const uint16_t* q, const KvView& kv, const AttnArgs& a,
                      int max_q) {
    constexpr int NB = D <= 128 ? 4 : 2;
    const int y = std::min(p.row_tiles, std::max(1, 65535 / kv.hkv)) * kv.hkv;
    if (p.prompt)
        kv_prompt_kernel<T, D><<<dim3(y, batch, p.splits), dim3(kPromptWaves * kWave), 0, stream()>>>(out, q, kv, a);
    else
        kv_decode_kernel<T, D, NB><<<dim3(p.splits, y, batch), dim3(kDecodeWaves * kWave), 0, stream()>>>(out, q, kv, a);
    if (p.splits > 1) {
        const long long rows = static_cast<long long>(max_q) * a.hq;
        const auto grid = [&](int per) { return dim3(static_cast<unsigned>(std::min<long long>((rows + per - 1) / per, 1 << 20)), batch); };
        if (p.splits <= 8)
            kv_join_kernel<T, D, 1><<<grid(kJoinWaves), dim3(kJoinWaves * kWave), 0, stream()>>>(out, kv, a);
        else
            kv_join_kernel<T, D, kJoinWaves><<<grid(1), dim3(kJoinWaves * kWave), 0, stream()>>>(out, kv, a);
    }
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
    NG_REQUIRE(scale >= 0.0f && __builtin_isfinite(scale * 1.4426950408889634f),
               "%s: softmax_scale must be >= 0 and below FLT_MAX / log2(e)", name);
    NG_REQUIRE(window >= 0 && sinks >= 0, "%s: window and sinks must be >= 0", name);
    NG_REQUIRE(aligned16(out) && aligned16(q) && aligned16(workspace), "%s: pointers must be 16-byte aligned", name);
    NG_REQUIRE(static_cast<long long>(total) * hq <= (1ll << 30), "%s: more than 2^30 query rows", name);
    const size_t bytes = static_cast<size_t>(total) * hq * cache->head_dim * 2;
    NG_REQUIRE(out == q || static_cast<char*>(out) + bytes <= static_cast<const char*>(q) ||
                   static_cast<const char*>(q) + bytes <= static_cast<char*>(out),
               "%s: out overlaps q without being q", name);
    max_q = std::min(max_q, total);
    AttnArgs a{static_cast<const int*>(cu), static_cast<const int*>(lens), static_cast<const int*>(table), max_pages,
               total, hq, hq / cache->num_kv_heads, scale * static_cast<float>(1.4426950408889634 / 127.0), std::min(window, 1 << 30), sinks,
               16, 1, 1, static_cast<float*>(workspace)};
    Plan p = plan(cache->num_kv_heads, a.group, cache->head_dim, batch, max_q, max_kv, a.window, sinks);
    const size_t rows = static_cast<size_t>(total) * hq;
    const size_t room = workspace == nullptr ? 0 : workspace_bytes / slice_bytes(rows, cache->head_dim);
    if (room < static_cast<size_t>(p.splits)) {
        const int tiles = p.chunk * p.splits;
        p.splits = std::max<int>(static_cast<int>(room), 1);
        p.chunk = (tiles + p.splits - 1) / p.splits;
    }
    a.row_tile = p.row_tile;
    a.splits = p.splits;
    a.chunk = p.chunk;
    const KvView kv = kv_view(*cache);
    uint16_t* o = static_cast<uint16_t*>(out);
    const uint16_t* x = static_cast<const uint16_t*>(q);
    switch (cache->head_dim) {
        case 64: launch_attention<T, 64>(p, batch, o, x, kv, a, max_q); break;
        case 128: launch_attention<T, 128>(p, batch, o, x, kv, a, max_q); break;
        case 192: launch_attention<T, 192>(p, batch, o, x, kv, a, max_q); break;
        default: launch_attention<T, 256>(p, batch, o, x, kv, a, max_q); break;
    }
    NG_CHECK_LAUNCH(name);
    return 0;
}

}  // namespace
}  // namespace ng

using namespace ng;

extern "C" size_t ng_kv_int8_attention_workspace(const ng_kv_int8_cache* cache, int num_q_heads, int batch,
                                                 int max_q_len, int max_kv_len) {
    if (cache == nullptr || cache->num_kv_heads <= 0 || !kv_head_dim_ok(cache->head_dim) || num_q_heads <= 0 ||
        num_q_heads % cache->num_kv_heads != 0 || batch <= 0 || max_q_len <= 0 || max_kv_len <= 0)
        return 0;
    const Plan p = plan(cache->num_kv_heads, num_q_heads / cache->num_kv_heads, cache->head_dim, batch,
                        max_q_len, max_kv_len, 0, 0);
    if (p.splits <= 1) return 0;
    return p.splits * slice_bytes(static_cast<size_t>(batch) * max_q_len * num_q_heads, cache->head_dim);
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
