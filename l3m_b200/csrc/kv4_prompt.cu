// Attention of prompt chunks over the paged 4-bit cache on the fifth-generation tensor cores: the variant of
// l3m_kv4_attend_dev for thousands of query rows (the rule is prompt_fits() below). bf16 queries and
// results, head dims of 2 or 4 blocks.
//
// One CTA takes 256 rows (query, head of the group) of one request and kv head, as two tiles of 128, over the whole
// context, 128 tokens widened at a time and multiplied 64 at a time:
//   8 warps  widen a step's codes to f16 in shared memory, 4 the keys (K-major), 4 the values (as they lie, MN-major), swizzled
//            by 128 bytes, two buffers each, the next step's codes under way in registers;
//   2 warps  issue the products, one for each tile: S = Q K^T (both operands in shared memory) and O += P V (P in tensor
//            memory); one warp for both was the longest chain;
//   8 warps  one thread a row: S from tensor memory, softmax against the row's reference, P back as f16 over S's columns.
// S has two halves of 64 tokens a tile, so that the next half's scores are formed while one goes through the softmax, and the two
// tiles alternate. Tensor memory: S (then P) of tile t, half u at columns 128 t + 64 u, O of tile t at 256 + t * head_dim: all 512
// columns, one CTA an SM.
//
// Scales. A widened value is an f16 number, code times scale, rounded once; scales are first multiplied by a power of two that
// brings the context's largest near 2^11 (found in a first pass over the scales alone: 1/9 of the cache), undone in the scores'
// factor and in the result. Where the smallest would then lose bits (kReach below), plain_rows() takes the CTA's rows. Queries are brought to 2^10 by row. P is 2^14 at most: the reference moves when a score
// passes it by 14 (then to 10 below the largest), which multiplies O by a power of two.
//
// Bound: the tensor pipe inside a CTA (75% of its rate while one runs), the last wave of CTAs outside. 2 chunks of 1024 over up to
// 6000 tokens, 32 heads to 8 of 128, q4_0: 226 to 242 us for 144 GFLOP, 600 to 640 TFLOP/s, on 256 CTAs in two waves. Even shares of the context
// for one CTA an SM, joined behind, took 336 us: their loop leaves the softmax too few registers, and each share starts anew.
//
// Every wait has a limit; a wait that gives up sets a status bit and the CTA's rows become NaN.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include "kv4.cuh"
#include "kv4_prompt.h"

namespace l3m {
namespace {

constexpr int kSms = 148;                               // of a B200; not asked of the device, so that the scratch's size is the arguments' alone
constexpr int kRows = 128, kStep = 128, kHalf = 64;     // rows of a tile, tokens that are widened at a time, tokens of a product
constexpr int kSoftWarps = 8, kWideWarps = 8;          // half of the latter for keys, half for values
constexpr int kPromptThreads = 32 * (kSoftWarps + kWideWarps + 2);

struct PromptArgs {
    l3m_kv4_attend a;
    Kv4Dev c;
    int group, row_tiles, vec;
};

// ---- mbarriers, tensor memory, products

__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }
__device__ __forceinline__ void bar_init(uint64_t *b, int count) { asm volatile("mbarrier.init.shared.b64 [%0], %1;" ::"r"(smem_u32(b)), "r"(count) : "memory"); }
__device__ __forceinline__ void bar_arrive(uint64_t *b) { asm volatile("mbarrier.arrive.shared.b64 _, [%0];" ::"r"(smem_u32(b)) : "memory"); }
// True once the barrier's phase `parity` has completed; false if that did not happen within two seconds.
__device__ __forceinline__ bool bar_wait(uint64_t *b, uint32_t parity) {
    const uint32_t at = smem_u32(b);
    unsigned long long begun = 0;
    for (;;) {
        uint32_t ok;
        asm volatile("{ .reg .pred p;\n mbarrier.try_wait.parity.shared.b64 p, [%1], %2, 1000;\n selp.u32 %0, 1, 0, p; }" : "=r"(ok) : "r"(at), "r"(parity) : "memory");
        if (ok) return true;
        unsigned long long now;
        asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(now));
        if (!begun) begun = now;
        if (now - begun > 2000000000ull) return false;
    }
}
// The same for a whole warp, which has to stay together.
__device__ __forceinline__ bool warp_wait(uint64_t *b, uint32_t parity) { return __all_sync(0xffffffffu, bar_wait(b, parity)); }
__device__ __forceinline__ void tc_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
// The products' operands are uniform over the warp and one lane issues: the whole warp runs this code, so that the
// operands can stay in uniform registers (issued from a divergent branch a product took 125 cycles, whatever its size).
__device__ __forceinline__ uint32_t elect_one() {
    uint32_t is;
    asm volatile("{ .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p; }" : "=r"(is));
    return is;
}
__device__ __forceinline__ void tc_commit(uint32_t lead, uint32_t bar) {
    asm volatile("{ .reg .pred l;\n setp.ne.u32 l, %1, 0;\n @l tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0]; }" ::"r"(bar), "r"(lead) : "memory");
}
// Shared-memory operand of rows of 128 bytes swizzled by 128, groups of 8 rows 1024 bytes apart. Low word: address, and the bytes between
// blocks of 64 elements where those run along the product's M or N (values; unused where they run along K).
constexpr uint32_t kOperandHigh = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t operand(uint32_t at, uint32_t lead) { return (at >> 4 & 0x3fff) | (lead >> 4) << 16; }
// d (tensor memory) = or += a . b, f16 operands, f32 accumulators; a in shared or in tensor memory.
__device__ __forceinline__ void mma_ss(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{ .reg .pred l, p;\n .reg .b64 x, y;\n setp.ne.u32 l, %6, 0;\n setp.ne.u32 p, %4, 0;\n mov.b64 x, {%1, %5};\n mov.b64 y, {%2, %5};\n"
                 " @l tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p; }" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(add), "n"(kOperandHigh), "r"(lead) : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t lead, uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, uint32_t add) {
    asm volatile("{ .reg .pred l, p;\n .reg .b64 y;\n setp.ne.u32 l, %6, 0;\n setp.ne.u32 p, %4, 0;\n mov.b64 y, {%2, %5};\n"
                 " @l tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p; }" ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(add), "n"(kOperandHigh), "r"(lead) : "memory");
}
__device__ __forceinline__ void tmem_load32(uint32_t *r, uint32_t at) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, "
        "%29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
          "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(at));
}
__device__ __forceinline__ void tmem_load16(uint32_t *r, uint32_t at) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
                 : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]),
                   "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
                 : "r"(at));
}
__device__ __forceinline__ void tmem_store16(uint32_t at, const uint32_t *r) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(at), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
                 "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
                 : "memory");
}
// wait::ld with the loaded registers as operands, so that no use of them moves above it.
template <int N> __device__ __forceinline__ void tmem_wait_ld(uint32_t *r) {
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
    for (int i = 0; i < N; i++) asm volatile("" : "+r"(r[i]));
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two at a time: z = (x, y) * m + c; s += (x, y).
__device__ __forceinline__ void fma_two(float *z, float x, float y, float m, float c) {
    asm("{ .reg .b64 a, b, d;\n mov.b64 a, {%2, %3};\n mov.b64 b, {%4, %4};\n mov.b64 d, {%5, %5};\n fma.rn.f32x2 d, a, b, d;\n mov.b64 {%0, %1}, d; }" : "=f"(z[0]), "=f"(z[1]) : "f"(x), "f"(y), "f"(m), "f"(c));
}
__device__ __forceinline__ void add_two(float *s, float x, float y) {
    asm("{ .reg .b64 a, b;\n mov.b64 a, {%0, %1};\n mov.b64 b, {%2, %3};\n add.rn.f32x2 a, a, b;\n mov.b64 {%0, %1}, a; }" : "+f"(s[0]), "+f"(s[1]) : "f"(x), "f"(y));
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*(const __half2 *)&a, *(const __half2 *)&b);
    return *(const uint32_t *)&r;
}
__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }   // 2^e, -126 <= e <= 127
// x * 2^e for any e that a result needs: two factors.
__device__ __forceinline__ float scale2(float x, int e) {
    const int h = max(min(e, 240), -240) / 2;
    return x * exp2i(h) * exp2i(max(min(e, 240), -240) - h);
}
__device__ __forceinline__ uint32_t e2m1_pair(uint32_t w) {
    uint32_t d;
    asm("{ .reg .b8 c, z0, z1, z2;\n mov.b32 {c, z0, z1, z2}, %1;\n cvt.rn.f16x2.e2m1x2 %0, c; }" : "=r"(d) : "r"(w));
    return d;
}

// The 8 codes of a word as four f16 pairs, times the scales' pairs: q4_0 pairs nibbles k and k + 4 (s[0] twice), mxfp4
// the two of byte k (s[0] for bytes 0 and 1, s[1] for 2 and 3).
template <int MX> __device__ __forceinline__ uint4 widen(uint32_t w, uint32_t s0, uint32_t s1) {
    uint32_t f[4];
    if (MX) {
        f[0] = e2m1_pair(w); f[1] = e2m1_pair(w >> 8);
        f[2] = e2m1_pair(w >> 16); f[3] = e2m1_pair(w >> 24);
        return make_uint4(mul2(f[0], s0), mul2(f[1], s0), mul2(f[2], s1), mul2(f[3], s1));
    }
    // 1024 + n, and 1024 + 16 n four bits higher, are numbers whose last bits are the code's
    const uint32_t y = w >> 8;
    f[0] = (w & 0x000f000fu) | 0x64006400u; f[1] = (w & 0x00f000f0u) | 0x64006400u;
    f[2] = (y & 0x000f000fu) | 0x64006400u; f[3] = (y & 0x00f000f0u) | 0x64006400u;
    const __half2 off = __halves2half2(__ushort_as_half(0xe408), __ushort_as_half(0xe408));   // -1032
    const __half2 s16 = __halves2half2(__ushort_as_half(0x2c00), __ushort_as_half(0x2c00));   // 1/16
    const __half2 o16 = __halves2half2(__ushort_as_half(0xd480), __ushort_as_half(0xd480));   // -72
#pragma unroll
    for (int k = 0; k < 4; k++) {
        const __half2 h = *(const __half2 *)&f[k];
        const __half2 r = k % 2 ? __hfma2(h, s16, o16) : __hadd2(h, off);
        f[k] = *(const uint32_t *)&r;
    }
    return make_uint4(mul2(f[0], s0), mul2(f[1], s0), mul2(f[2], s0), mul2(f[3], s0));
}

template <int NG>
struct Smem {
    static constexpr int DP = 32 * NG, TILE = kRows * DP * 2;   // one operand tile of 128 rows
    uint8_t q[2][TILE], k[2][TILE], v[2][TILE];
    uint64_t k_full[2], v_full[2], k_empty[2], v_empty[2];
    uint64_t s_full[2][2], p_full[2][2], pv_done[2], end[2];   // [tile][half]
    uint32_t tmem, bad[4][4];             // tokens of a step in no page of the cache, a ring of four steps
    int k_top, v_top, k_low, v_low;       // the largest and the smallest exponent of the scales
};

// One token's keys or values as they lie in the cache.
template <int NG, int MX>
struct Codes {
    uint32_t w[4 * NG], sc[MX ? 1 : NG / 2];
    bool there;
};

// What a CTA does: its request, kv head and first row. The last rows first, they see most.
__device__ __forceinline__ void place(const PromptArgs &p, int &r, int &h, int &row0) {
    const int x = blockIdx.x, per_req = p.c.n_kv * p.row_tiles;
    r = x / per_req;
    h = (x - r * per_req) / p.row_tiles;
    row0 = (p.row_tiles - 1 - (x - r * per_req - h * p.row_tiles)) * 2 * kRows;
}

// A CTA's rows in 32 bits, for contexts whose scales lie further apart than widened numbers reach. A warp takes 8 rows at a time over the whole
// context, 32 tokens at a step: a lane forms one token's scores, then sums 4 dims of the values. It decodes a token for 8 rows, not 256, without
// tensor cores: 2 chunks of 1024 over 6000 tokens, 32 heads to 8 of 128, mxfp4, 19 ms in place of 248 us. buf: 8 rows' queries and probabilities a warp.
template <int NG, int MX>
__device__ __noinline__ void plain_rows(const PromptArgs &p, int k_up, int v_up, float *buf) {
    constexpr int R = 8, DP = 32 * NG, SB = MX ? 1 : 2, kWarps = kPromptThreads / 32;
    static_assert(kWarps * R * (DP + 32) * 4 <= 4 * kRows * DP * 2, "the warps' buffers fit the operands'");
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    int r, h, row0;
    place(p, r, h, row0);
    const Queries rq = queries_of(p.a, r);
    const int rows = min(rq.nq * p.group - row0, 2 * kRows);
    float *q = buf + warp * R * (DP + 32), *prob = q + R * DP;
    const int32_t *table = p.a.tables + (size_t)r * p.a.max_blocks;
    // A scale's value times 2^up; 0 for what is not finite.
    auto scale = [&](const uint8_t *at, int up) -> float {
        if (MX) return *at == 255 ? 0.0f : scale2(exp2i(*at - 127), up);
        const uint32_t x = *(const uint16_t *)at;
        return (x & 0x7c00) == 0x7c00 ? 0.0f : scale2(__half2float(__ushort_as_half((unsigned short)x)), up);
    };
    auto code = [](uint32_t n) -> float {
        if (!MX) return (float)(int)n - 8.0f;
        const float m = (float)(0xC8643210u >> 4 * (n & 7) & 15) * 0.5f;
        return n & 8 ? -m : m;
    };
    for (int g0 = warp * R; g0 < rows; g0 += kWarps * R) {
        int at[R];                                                           // the rows' positions
        float mult[R], m[R], l[R], o[R][4];
        __syncwarp();
#pragma unroll
        for (int i = 0; i < R; i++) {
            const int row = row0 + g0 + i, qi = row / p.group, head = h * p.group + row - qi * p.group;
            const bool live = g0 + i < rows;
            const __nv_bfloat16 *src = (const __nv_bfloat16 *)p.a.q + (size_t)(rq.start + qi) * p.a.q_ld + (size_t)head * p.c.dim;
            float x[NG], top = 0.0f;
#pragma unroll
            for (int j = 0; j < NG; j++) {
                x[j] = live && 32 * j + lane < p.c.dim ? __bfloat162float(src[32 * j + lane]) : 0.0f;
                top = fmaxf(top, fabsf(x[j]));
            }
#pragma unroll
            for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
            const int up = top > 0.0f ? 9 - max(min(ilogbf(top), 127), -149) : 0;
#pragma unroll
            for (int j = 0; j < NG; j++) q[i * DP + 32 * j + lane] = scale2(x[j], up);
            mult[i] = scale2(p.a.scale * 1.4426950408889634f, -up - k_up);
            at[i] = live ? rq.at + qi : -1;
            m[i] = -INFINITY;
            l[i] = 0.0f;
#pragma unroll
            for (int d = 0; d < 4; d++) o[i][d] = 0.0f;
        }
        __syncwarp();
        const int i1 = min(g0 + R, rows) - 1, first = rq.at + (row0 + g0) / p.group, last = rq.at + (row0 + i1) / p.group;
        const int lo = p.a.window ? max(0, first - p.a.window + 1) : 0, hi = last + 1;
#pragma unroll 1
        for (int t0 = lo & ~31; t0 < hi; t0 += 32) {
            const int tok = t0 + lane;
            const uint8_t *tile = nullptr;
            if (tok >= lo && tok < hi) {
                const int blk = tok / p.c.page, off = tok - blk * p.c.page, id = table[blk];
                if (id >= 0 && id < p.c.n_pages) tile = p.c.data + p.c.tile_at(id, h, off / kKvTile);
                else if (p.a.status) atomicOr((int *)p.a.status, L3M_KV4_BAD_PAGE);
            }
            const int row16 = tok % p.c.page % kKvTile;
            float s[R];
#pragma unroll
            for (int i = 0; i < R; i++) s[i] = 0.0f;
            if (tile) {
#pragma unroll 1
                for (int j = 0; j < NG; j++) {
                    const float d = scale(tile + 512 * NG + (row16 * NG + j) * SB, k_up);
                    float acc[R];
#pragma unroll
                    for (int i = 0; i < R; i++) acc[i] = 0.0f;
#pragma unroll 1
                    for (int t = 0; t < 4; t++) {
                        const uint32_t w = ((const uint32_t *)(tile + row16 * 16 * NG))[t * NG + j];
                        float c[8];
#pragma unroll
                        for (int e = 0; e < 8; e++) c[e] = code(w >> 4 * e & 15);
#pragma unroll
                        for (int i = 0; i < R; i++) {
                            const float4 a = *(const float4 *)(q + i * DP + 32 * j + 8 * t), b = *(const float4 *)(q + i * DP + 32 * j + 8 * t + 4);
                            acc[i] = fmaf(a.x, c[0], fmaf(a.y, c[1], fmaf(a.z, c[2], fmaf(a.w, c[3], acc[i]))));
                            acc[i] = fmaf(b.x, c[4], fmaf(b.y, c[5], fmaf(b.z, c[6], fmaf(b.w, c[7], acc[i]))));
                        }
                    }
#pragma unroll
                    for (int i = 0; i < R; i++) s[i] = fmaf(acc[i], d, s[i]);
                }
            }
#pragma unroll
            for (int i = 0; i < R; i++) {
                const bool seen = tile && tok <= at[i] && !(p.a.window && tok <= at[i] - p.a.window);
                const float z = seen ? s[i] * mult[i] : -INFINITY;
                float top = z;
#pragma unroll
                for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                if (top > m[i]) {
                    const float f = m[i] == -INFINITY ? 0.0f : ex2(m[i] - top);
                    m[i] = top;
                    l[i] *= f;
#pragma unroll
                    for (int d = 0; d < 4; d++) o[i][d] *= f;
                }
                const float e = seen ? ex2(z - m[i]) : 0.0f;
                l[i] += e;
                prob[i * 32 + lane] = e;
            }
            __syncwarp();
            // the values: lane = 4 dims, part lane / NG of block lane % NG
#pragma unroll 1
            for (int t = 0; t < 32; t++) {
                const uint8_t *from = (const uint8_t *)__shfl_sync(0xffffffffu, (unsigned long long)tile, t);
                if (!from || lane >= 8 * NG) continue;
                const int vrow = (t0 + t) % p.c.page % kKvTile, j = lane % NG;
                const uint32_t w = ((const uint16_t *)(from + 256 * NG + vrow * 16 * NG))[lane];
                const float d = scale(from + 512 * NG + kKvTile * NG * SB + (vrow * NG + j) * SB, v_up);
                float v[4];
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = code(w >> 4 * e & 15) * d;
#pragma unroll
                for (int i = 0; i < R; i++)
#pragma unroll
                    for (int e = 0; e < 4; e++) o[i][e] = fmaf(prob[i * 32 + t], v[e], o[i][e]);
            }
            __syncwarp();
        }
#pragma unroll
        for (int i = 0; i < R; i++) {
            float total = l[i];
#pragma unroll
            for (int d = 16; d; d >>= 1) total += __shfl_xor_sync(0xffffffffu, total, d);
            const int row = row0 + g0 + i, qi = row / p.group, head = h * p.group + row - qi * p.group, d0 = 32 * (lane % NG) + 4 * (lane / NG);
            if (g0 + i >= rows || lane >= 8 * NG || d0 >= p.c.dim) continue;
            __nv_bfloat16 *dst = (__nv_bfloat16 *)p.a.out + (size_t)(rq.start + qi) * p.a.out_ld + (size_t)head * p.c.dim + d0;
            const float inv = total != 0.0f ? 1.0f / total : 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) dst[e] = __float2bfloat16_rn(inv == 0.0f ? 0.0f : scale2(o[i][e] * inv, -v_up));
        }
    }
}

template <int NG, int MX>
__global__ void __launch_bounds__(kPromptThreads, 1) prompt_kernel(const __grid_constant__ PromptArgs p) {
    typedef Smem<NG> S;
    constexpr int DP = S::DP, SB = MX ? 1 : 2;
    extern __shared__ uint8_t raw[];
    S &s = *(S *)(((uintptr_t)raw + 1023) & ~(uintptr_t)1023);
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    asm volatile("griddepcontrol.wait;" ::: "memory");

    int r, h, row0;
    place(p, r, h, row0);
    const Queries rq = queries_of(p.a, r);
    const int start = rq.start, nq = rq.nq;
    const int rows = nq * p.group - row0;                                  // rows left from this CTA's first
    if (rows <= 0) return;
    const int tiles = rows > kRows ? 2 : 1;
    const int i0 = row0 / p.group, i1 = min((row0 + 2 * kRows - 1) / p.group, nq - 1), first = rq.at + i0, last = rq.at + i1;   // the rows' positions
    const int lo_any = p.a.window ? max(0, first - p.a.window + 1) : 0, hi_any = max(last + 1, 0);      // seen by some row
    const int whole_lo = p.a.window ? last - p.a.window + 1 : 0, whole_hi = first + 1;                  // seen by every row
    const int t0 = lo_any / kStep * kStep, steps = hi_any > lo_any ? (hi_any - t0 + kStep - 1) / kStep : 0, halves = hi_any > lo_any ? (hi_any - t0 + kHalf - 1) / kHalf : 0;
    const int32_t *table = p.a.tables + (size_t)r * p.a.max_blocks;

    if (tid == 0) {
        for (int b = 0; b < 2; b++) {
            bar_init(&s.k_full[b], kStep);
            bar_init(&s.v_full[b], kStep);
            bar_init(&s.k_empty[b], tiles);
            bar_init(&s.v_empty[b], tiles);
            for (int u = 0; u < 2; u++) {
                bar_init(&s.s_full[b][u], 1);
                bar_init(&s.p_full[b][u], kRows);
            }
            bar_init(&s.pv_done[b], 1);
            bar_init(&s.end[b], 1);
        }
        s.k_top = s.v_top = 0;
        s.k_low = s.v_low = 1 << 20;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    if (warp == kSoftWarps + kWideWarps) {
        asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], 512;" ::"r"(smem_u32(&s.tmem)) : "memory");
        asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
    }
    __syncthreads();

    // The row of token tok: where its tile is, null if its page is none of the cache's.
    auto tile_of = [&](int tok) -> const uint8_t * {
        const int blk = tok / p.c.page, off = tok - blk * p.c.page, id = table[blk];
        return id >= 0 && id < p.c.n_pages ? p.c.data + p.c.tile_at(id, h, off / kKvTile) : nullptr;
    };

    // ---- the scales' exponents, while the softmax's warps bring in the queries
    if (warp >= kSoftWarps) {
        // Largest and smallest in 16-bit pairs: e8m0 bytes, or the bits of f16 numbers without their signs. A scale of 0 or one that is not finite sets
        // nothing for the rest: a pass that meets one is done again one by one.
        uint32_t kt = 0, vt = 0, kl = 0, vl = 0, odd = 0;
        auto count = [&](uint32_t x, uint32_t &top, uint32_t &low) {
            if (MX) {
                odd |= (((x - 0x01010101u) & ~x) | ((~x - 0x01010101u) & x)) & 0x80808080u;
                const uint32_t y = x & 0x00ff00ffu, z = x >> 8 & 0x00ff00ffu;
                top = __vmaxu2(top, __vmaxu2(y, z));
                low = __vminu2(low, __vminu2(y, z));
            } else {
                x &= 0x7fff7fffu;
                odd |= ((x + 0x04000400u) | ((x - 0x00010001u) & ~x)) & 0x80008000u;
                top = __vmaxu2(top, x);
                low = __vminu2(low, x);
            }
        };
        auto count_good = [](uint32_t x, uint32_t &top, uint32_t &low) {
#pragma unroll
            for (int k = 0; k < 32; k += 8 * SB) {
                const uint32_t e = x >> k & (MX ? 0xff : 0x7fff);
                if (e && e < (MX ? 255 : 0x7c00)) top = __vmaxu2(top, e), low = __vminu2(low, e | 0xffff0000u);
            }
        };
        auto scan = [&](auto each) {
            kt = vt = odd = 0;
            kl = vl = ~0u;
#pragma unroll 8
            for (int tok = lo_any + tid - 32 * kSoftWarps; tok < hi_any; tok += kPromptThreads - 32 * kSoftWarps) {
                const uint8_t *tile = tile_of(tok);
                if (!tile) continue;
                const int row = tok % p.c.page % kKvTile;
                const uint8_t *ks = tile + 512 * NG + row * NG * SB, *vs = ks + kKvTile * NG * SB;
                if constexpr (NG * SB == 2) {                                // two bytes, twice
                    each(*(const uint16_t *)ks * 0x00010001u, kt, kl);
                    each(*(const uint16_t *)vs * 0x00010001u, vt, vl);
                } else {
#pragma unroll
                    for (int i = 0; i < NG * SB / 4; i++) {
                        each(((const uint32_t *)ks)[i], kt, kl);
                        each(((const uint32_t *)vs)[i], vt, vl);
                    }
                }
            }
        };
        scan(count);
        if (odd) scan(count_good);
        auto exponent = [](uint32_t x) { return MX || x >= 0x400 ? (int)(MX ? x : x >> 10) : 22 - __clz(x); };      // an f16 subnormal's by its highest bit, -9 .. 0
        kt = __reduce_max_sync(0xffffffffu, max(kt & 0xffff, kt >> 16));
        vt = __reduce_max_sync(0xffffffffu, max(vt & 0xffff, vt >> 16));
        kl = __reduce_min_sync(0xffffffffu, min(kl & 0xffff, kl >> 16));
        vl = __reduce_min_sync(0xffffffffu, min(vl & 0xffff, vl >> 16));
        if (lane == 0) {
            if (kt) {
                atomicMax(&s.k_top, max(exponent(kt), 0));
                atomicMin(&s.k_low, exponent(kl));
            }
            if (vt) {
                atomicMax(&s.v_top, max(exponent(vt), 0));
                atomicMin(&s.v_low, exponent(vl));
            }
        }
    }
    const int tile = warp / 4;                                              // of a softmax warp
    const int row = tile * kRows + (warp & 3) * 32 + lane, qi = (row0 + row) / p.group, head = h * p.group + (row0 + row) % p.group;
    const bool live = warp < kSoftWarps && row < rows;
    const int at = live ? rq.at + qi : -1;
    int up = 0;
    if (warp < kSoftWarps && tile < tiles) {
        // ---- this thread's query, in the order in which the keys' codes come out of their words
        const __nv_bfloat16 *src = (const __nv_bfloat16 *)p.a.q + (size_t)(start + qi) * p.a.q_ld + (size_t)head * p.c.dim;
        auto piece = [&](int c) {                                            // 8 dims
            uint4 v = make_uint4(0, 0, 0, 0);
            if (live && c * 8 < p.c.dim) {
                if (p.vec) {
                    v = *(const uint4 *)(src + c * 8);
                } else {
                    const uint16_t *hw = (const uint16_t *)src + c * 8;
                    v = make_uint4(hw[0] | (uint32_t)hw[1] << 16, hw[2] | (uint32_t)hw[3] << 16, hw[4] | (uint32_t)hw[5] << 16, hw[6] | (uint32_t)hw[7] << 16);
                }
            }
            return v;
        };
        float top = 0.0f;
#pragma unroll 4
        for (int c = 0; c < DP / 8; c++) {
            const uint4 v = piece(c);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
#pragma unroll
            for (int e = 0; e < 4; e++) top = fmaxf(top, fmaxf(fabsf(__uint_as_float(w[e] << 16)), fabsf(__uint_as_float(w[e] & 0xffff0000u))));
        }
        up = top > 0.0f ? 9 - max(min(ilogbf(top), 127), -149) : 0;        // |q| * 2^up < 2^10
        const float f0 = exp2i(up / 2), f1 = exp2i(up - up / 2);
        const int rr = row & (kRows - 1);
#pragma unroll 4
        for (int c = 0; c < DP / 8; c++) {
            const uint4 v = piece(c);
            const uint32_t w[4] = {v.x, v.y, v.z, v.w};
            float e[8];
#pragma unroll
            for (int i = 0; i < 4; i++) {
                e[2 * i] = __uint_as_float(w[i] << 16) * f0 * f1;
                e[2 * i + 1] = __uint_as_float(w[i] & 0xffff0000u) * f0 * f1;
            }
            const uint4 f = MX ? make_uint4(pack_f16(e[0], e[1]), pack_f16(e[2], e[3]), pack_f16(e[4], e[5]), pack_f16(e[6], e[7]))
                               : make_uint4(pack_f16(e[0], e[4]), pack_f16(e[1], e[5]), pack_f16(e[2], e[6]), pack_f16(e[3], e[7]));
            *(uint4 *)(s.q[tile] + c / 8 * (kRows * 128) + rr * 128 + ((c % 8 ^ rr & 7) << 4)) = f;
        }
        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");        // the products read what was written here
    }
    __syncthreads();
    const uint32_t tmem = s.tmem;
    // q4_0: d < 2^(top - 14), brought below 2^11. mxfp4: 2^(top - 127), brought to 2^11.
    const int k_up = MX ? 11 + 127 - s.k_top : 25 - s.k_top, v_up = MX ? 11 + 127 - s.v_top : 25 - s.v_top;
    // What f16 holds below the largest without loss: mxfp4's numbers of two bits down to 2^-24 (0.5 times 2^-34 of the largest scale 2^11), q4_0's
    // code times scale with 11 bits down to 2^-14 (a scale of 2^-24 of the largest)
    constexpr int kReach = MX ? 34 : 24;
    bool ok = true;

    if (s.k_top - s.k_low > kReach && s.k_low <= s.k_top || s.v_top - s.v_low > kReach && s.v_low <= s.v_top) {
        plain_rows<NG, MX>(p, k_up, v_up, (float *)s.k);
    } else if (warp >= kSoftWarps && warp < kSoftWarps + kWideWarps) {
        // ---- widening: thread = token of the step
        const int tk = tid & (kStep - 1);
        const bool values = warp >= kSoftWarps + kWideWarps / 2;
        const int by = values ? v_up : k_up, code_at = values ? 256 * NG : 0, scale_at = 512 * NG + (values ? kKvTile * NG * SB : 0);
        typedef Codes<NG, MX> C;
        // A token's tile is found a step before its codes are read, its codes are read a step before they are widened.
        auto find = [&](int j) -> const uint8_t * {
            const int tok = t0 + j * kStep + tk;
            return j < steps && tok >= lo_any && tok < hi_any ? tile_of(tok) : nullptr;
        };
        auto fetch = [&](C &c, const uint8_t *tl, int j) {
            c.there = tl != nullptr;
            if (!tl) return;
            const int row16 = (t0 + j * kStep + tk) % p.c.page % kKvTile;
            const uint8_t *codes = tl + code_at + row16 * 16 * NG, *sc = tl + scale_at + row16 * NG * SB;
#pragma unroll
            for (int i = 0; i < NG; i++) {
                const uint4 a = __ldg((const uint4 *)codes + i);
                c.w[4 * i] = a.x; c.w[4 * i + 1] = a.y; c.w[4 * i + 2] = a.z; c.w[4 * i + 3] = a.w;
            }
            if (MX) {
                c.sc[0] = NG == 4 ? *(const uint32_t *)sc : *(const uint16_t *)sc;
            } else {
#pragma unroll
                for (int i = 0; i < NG / 2; i++) c.sc[i] = ((const uint32_t *)sc)[i];
            }
        };
        // Block j's scale brought up by 2^by. edge: what is not finite counts as 0.
        auto scale_of = [&](const C &c, int j, bool edge) -> float {
            if (MX) {
                const int bits = (int)(c.sc[0] >> (8 * j) & 0xff), e = bits + by - 127;
                return e < -24 || (edge && bits == 255) ? 0.0f : exp2i(min(e, 15));
            }
            uint32_t hbits = c.sc[j / 2] >> (16 * (j % 2)) & 0xffff;
            if (edge && (hbits & 0x7c00) == 0x7c00) hbits = 0;
            return scale2(__half2float(__ushort_as_half((unsigned short)hbits)), by);
        };
        C cur, next;
        fetch(cur, find(0), 0);
        const uint8_t *ahead = find(1);
        for (int j = 0; j < steps && ok; j++) {
            const int b = j & 1, tok0 = t0 + j * kStep, sw = tk & 7;
            const bool edge = tok0 < whole_lo || tok0 + kStep > whole_hi;
            fetch(next, ahead, j + 1);
            ahead = find(j + 2);
            if (j >= 2) ok = warp_wait(values ? &s.v_empty[b] : &s.k_empty[b], (j / 2 - 1) & 1);
            uint8_t *dst = (values ? s.v[b] : s.k[b]) + tk * 128;
            if (!values) {
                const bool wanted = tok0 + tk >= lo_any && tok0 + tk < hi_any;
                const uint32_t miss = __ballot_sync(0xffffffffu, wanted && !cur.there);
                if (lane == 0) s.bad[j & 3][warp - kSoftWarps] = miss;
                if (wanted && !cur.there && p.a.status) atomicOr((int *)p.a.status, L3M_KV4_BAD_PAGE);
#pragma unroll
                for (int g = 0; g < NG; g++) {
                    const float d = cur.there ? scale_of(cur, g, edge) : 0.0f;
                    const uint32_t d2 = pack_f16(d, d);
#pragma unroll
                    for (int t = 0; t < 4; t++) {
                        const uint4 v = cur.there ? widen<MX>(cur.w[t * NG + g], d2, d2) : make_uint4(0, 0, 0, 0);
                        const int c = 4 * g + t;
                        *(uint4 *)(dst + c / 8 * (kRows * 128) + ((c % 8 ^ sw) << 4)) = v;
                    }
                }
            } else {
#pragma unroll
                for (int q2 = 0; q2 < NG / 2; q2++) {
                    const float d0 = cur.there ? scale_of(cur, 2 * q2, edge) : 0.0f, d1 = cur.there ? scale_of(cur, 2 * q2 + 1, edge) : 0.0f;
                    const uint32_t s0 = MX ? pack_f16(d0, d0) : pack_f16(d0, d1), s1 = pack_f16(d1, d1);
#pragma unroll
                    for (int g = 0; g < 8; g++) {
                        const int c = g * (NG / 2) + q2;
                        const uint4 v = cur.there ? widen<MX>(cur.w[c], s0, s1) : make_uint4(0, 0, 0, 0);
                        *(uint4 *)(dst + c / 8 * (kRows * 128) + ((c % 8 ^ sw) << 4)) = v;
                    }
                }
            }
            asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
            bar_arrive(values ? &s.v_full[b] : &s.k_full[b]);
            cur = next;
        }
    } else if (warp >= kSoftWarps + kWideWarps) {
        // ---- the products of tile t
        const uint32_t t = __shfl_sync(0xffffffffu, warp - kSoftWarps - kWideWarps, 0);
        if (steps && t < tiles) {
            const uint32_t lead = elect_one(), nh = __shfl_sync(0xffffffffu, halves, 0);
            constexpr uint32_t base = 1u << 4 | (kRows / 16) << 24;         // f32 accumulators, f16 operands, M 128
            constexpr uint32_t qk = base | (kHalf / 8) << 17, pv = base | (DP / 8) << 17 | 1u << 16;   // N; bit 16: b runs along N
            constexpr uint32_t kBlock = kRows * 128 >> 4, kHalfRows = kHalf * 128 >> 4, kTile = S::TILE >> 4;   // in the operands' units
            const uint32_t q0 = operand(smem_u32(s.q), 16), k0 = operand(smem_u32(s.k), 16), v0 = operand(smem_u32(s.v), kRows * 128);
            const uint32_t s_bar = smem_u32(s.s_full), pv_bar = smem_u32(s.pv_done), ke_bar = smem_u32(s.k_empty), ve_bar = smem_u32(s.v_empty);
            // Half u's scores, two halves ahead of the softmax. All of tensor memory is this CTA's: it begins at 0.
            auto score = [&](uint32_t u) {
                const uint32_t qa = q0 + t * kTile, ka = k0 + (u / 2 & 1) * kTile + (u & 1) * kHalfRows, d = t * 128 + (u & 1) * kHalf;
#pragma unroll
                for (int c = 0; c < DP / 16; c++) mma_ss(lead, d, qa + c / 4 * kBlock + c % 4 * 2, ka + c / 4 * kBlock + c % 4 * 2, qk, c > 0);
                tc_commit(lead, s_bar + (t * 2 + (u & 1)) * 8);
                if (u & 1 || u == nh - 1) tc_commit(lead, ke_bar + (u / 2 & 1) * 8);
            };
            ok = tmem == 0 && warp_wait(&s.k_full[0], 0);
            tc_after();
            for (uint32_t u = 0; u < min(2u, nh) && ok; u++) score(u);
            for (uint32_t u = 0; u < nh && ok; u++) {
                if (!(u & 1)) ok = warp_wait(&s.v_full[u / 2 & 1], u / 4 & 1);
                ok = ok && warp_wait(&s.p_full[t][u & 1], u / 2 & 1);
                if (!ok) break;
                tc_after();
                const uint32_t va = v0 + (u / 2 & 1) * kTile + (u & 1) * kHalfRows, pa = t * 128 + (u & 1) * kHalf;
#pragma unroll
                for (int c = 0; c < kHalf / 16; c++) mma_ts(lead, 256 + t * DP, pa + c * 8, va + c * (2048 >> 4), pv, u > 0 || c > 0);
                tc_commit(lead, pv_bar + t * 8);
                if (u & 1 || u == nh - 1) tc_commit(lead, ve_bar + (u / 2 & 1) * 8);
                if (u + 2 >= nh) continue;
                if (!(u & 1)) ok = warp_wait(&s.k_full[(u + 2) / 2 & 1], (u + 2) / 4 & 1);
                ok = ok && warp_wait(&s.pv_done[t], u & 1);                  // S of half u + 2 takes the columns of P of half u
                if (!ok) break;
                tc_after();
                score(u + 2);
            }
            // Nothing of this warp's is under way when the CTA ends, whatever ended the loop
            tc_commit(lead, smem_u32(&s.end[t]));
            ok = warp_wait(&s.end[t], 0) && ok;
        }
    } else if (tile < tiles) {
        // ---- softmax: thread = row
        const uint32_t mine = tmem + tile * 128 + ((uint32_t)(warp & 3) << 21);     // lane 32 * (warp % 4) in the upper half
        const uint32_t mine_o = tmem + 256 + tile * DP + ((uint32_t)(warp & 3) << 21);
        const float mult = scale2(p.a.scale * 1.4426950408889634f, -up - k_up);
        float ref = 0.0f, sum = 0.0f;
        bool fresh = true;                                                   // the row has seen nothing yet
        const int low = p.a.window ? at - p.a.window + 1 : 0;
        for (int u = 0; u < halves && ok; u++) {
            ok = warp_wait(&s.s_full[tile][u & 1], u / 2 & 1);
            if (!ok) break;
            tc_after();
            const int tok0 = t0 + u * kHalf;
            const uint32_t here = mine + (u & 1) * kHalf;
            const uint32_t bad0 = s.bad[u / 2 & 3][u % 2 * 2], bad1 = s.bad[u / 2 & 3][u % 2 * 2 + 1];
            uint32_t v[64];
            tmem_load32(v, here);
            tmem_load32(v + 32, here + 32);
            tmem_wait_ld<64>(v);
            float z[64], top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
            for (int i = 0; i < 64; i += 2) fma_two(z + i, __uint_as_float(v[i]), __uint_as_float(v[i + 1]), mult, -ref);
            if (tok0 < whole_lo || tok0 + kHalf > whole_hi || (bad0 | bad1)) {
                // the tokens of this half that the row sees
                const int from = low - tok0, to = at - tok0;
                unsigned long long seen = ~((unsigned long long)bad1 << 32 | bad0);
                seen &= to < 0 ? 0ull : to > 62 ? ~0ull : (2ull << to) - 1ull;
                seen &= from > 63 ? 0ull : from < 1 ? ~0ull : ~0ull << from;
                const uint32_t lo32 = (uint32_t)seen, hi32 = (uint32_t)(seen >> 32);
#pragma unroll
                for (int i = 0; i < 64; i++) z[i] = (i < 32 ? lo32 >> i : hi32 >> (i - 32)) & 1 ? z[i] : -INFINITY;
            }
#pragma unroll
            for (int i = 0; i < 64; i += 2) top[i / 2 % 4] = max3(top[i / 2 % 4], z[i], z[i + 1]);
            const float high = fmaxf(fmaxf(top[0], top[1]), fmaxf(top[2], top[3]));
            const bool move = high > 14.0f || (fresh && high > -INFINITY);
            if (__any_sync(0xffffffffu, move)) {
                // Rows whose reference is passed: a new one, a whole number above the old, 10 below the largest
                float by = 0.0f;
                if (move) by = ceilf(high) - 10.0f;
                const float f = fresh ? 1.0f : ex2(-by);
                ref += by;
                fresh = fresh && !move;
                sum *= f;
                if (u > 0) {
                    ok = warp_wait(&s.pv_done[tile], (u - 1) & 1) && ok;
                    tc_after();
#pragma unroll 1
                    for (int d = 0; d < DP; d += 16) {
                        uint32_t o[16];
                        tmem_load16(o, mine_o + d);
                        tmem_wait_ld<16>(o);
#pragma unroll
                        for (int i = 0; i < 16; i++) o[i] = __float_as_uint(__uint_as_float(o[i]) * f);
                        tmem_store16(mine_o + d, o);
                    }
                }
#pragma unroll
                for (int i = 0; i < 64; i++) z[i] -= by;
            }
            float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int i = 0; i < 32; i++) {
                const float e0 = ex2(z[2 * i]), e1 = ex2(z[2 * i + 1]);
                add_two(part + i % 2 * 2, e0, e1);
                v[i] = pack_f16(e0, e1);
            }
            sum += part[0] + part[1] + (part[2] + part[3]);
            if (u > 0 && u == halves - 1) {
                // The products before the last, while the last wait for this warp's P: a parity tells one phase from the next, not from the one behind that
                ok = warp_wait(&s.pv_done[tile], (u - 1) & 1) && ok;
            }
            tmem_store16(here, v);
            tmem_store16(here + 16, v + 16);
            tmem_wait_st();
            tc_before();
            bar_arrive(&s.p_full[tile][u & 1]);
        }
        // ---- the rows' results
        if (halves) ok = warp_wait(&s.pv_done[tile], (halves - 1) & 1) && ok;
        tc_after();
        const float inv = sum != 0.0f ? 1.0f / sum : 0.0f;
        __nv_bfloat16 *dst = (__nv_bfloat16 *)p.a.out + (size_t)(start + qi) * p.a.out_ld + (size_t)head * p.c.dim;
#pragma unroll
        for (int c = 0; c < DP / 16; c++) {                                  // 16 columns: 4 dims of each of 4 (2) blocks
            uint32_t o[16];
            if (steps) {
                tmem_load16(o, mine_o + 16 * c);
                tmem_wait_ld<16>(o);
            }
#pragma unroll
            for (int q4 = 0; q4 < 4; q4++) {
                float e[4];
                int d;
                if (NG == 4) {                                               // one part g = c: block q4
                    d = 32 * q4 + 4 * c;
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int col = MX ? q4 / 2 * 8 + q4 % 2 * 4 + k : q4 / 2 * 8 + 2 * k + q4 % 2;
                        e[k] = __uint_as_float(o[col]);
                    }
                } else {                                                     // two parts g = 2 c, 2 c + 1: blocks 0 and 1
                    d = 32 * (q4 % 2) + 4 * (2 * c + q4 / 2);
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        const int col = q4 / 2 * 8 + (MX ? q4 % 2 * 4 + k : 2 * k + q4 % 2);
                        e[k] = __uint_as_float(o[col]);
                    }
                }
                if (!live || d >= p.c.dim) continue;
#pragma unroll
                for (int k = 0; k < 4; k++) e[k] = !ok ? __uint_as_float(0x7fffffffu) : inv == 0.0f ? 0.0f : scale2(e[k] * inv, -v_up);
                if (p.vec) {
                    __nv_bfloat162 two[2] = {__floats2bfloat162_rn(e[0], e[1]), __floats2bfloat162_rn(e[2], e[3])};
                    *(uint2 *)(dst + d) = *(const uint2 *)two;
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++) dst[d + k] = __float2bfloat16_rn(e[k]);
                }
            }
        }
    }
    if (!ok && p.a.status) atomicOr((int *)p.a.status, L3M_KV4_TIMEOUT);
    tc_before();
    __syncthreads();
    if (warp == kSoftWarps + kWideWarps) {
        tc_after();
        asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, 512;" ::"r"(tmem) : "memory");
    }
}

template <int NG, int MX>
cudaError_t launch(const PromptArgs &p, cudaStream_t s) {
    const int smem = (int)sizeof(Smem<NG>) + 1024;
    cudaError_t e = cudaFuncSetAttribute(prompt_kernel<NG, MX>, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
    if (e != cudaSuccess) return e;
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)((long long)p.a.n_req * p.c.n_kv * p.row_tiles));
    cfg.blockDim = dim3(kPromptThreads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, prompt_kernel<NG, MX>, p);
}

}  // namespace

// When: a CTA here takes as long for one row as for 256, and the CTAs run in waves of one an SM; the kernel of kv4_attend.cu takes time by
// the row, whichever request or head it is of. Measured, contexts of 512 to 16384, the rows at which both take as long:
// 5300 to 7600 a wave at a head dim of 128, 10000 to 13700 at 64. At 16384 tokens, 8 kv heads and 128 dims: 1024 rows a head of one request 393 us here and
// 525 there, of 8 requests 789 and 3988; 256 rows of 2 requests 395 and 278, of one 391 and 151.
bool prompt_fits(const l3m_kv4 *c, const l3m_kv4_attend *a) {
    const int ng = (c->head_dim + kKvBlock - 1) / kKvBlock;
    if (a->dtype != L3M_DT_BF16 || (ng != 2 && ng != 4) || a->n_req > 1 << 20) return false;
    const long long rows = (long long)a->max_q * (a->n_heads / c->n_kv_heads), lines = (long long)a->n_req * c->n_kv_heads;
    if (rows >= 1 << 24 || lines >= 1 << 30) return false;
    const long long ctas = (rows + 2 * kRows - 1) / (2 * kRows) * lines, waves = (ctas + kSms - 1) / kSms;
    return rows && lines && ctas < 0x7fffffff && rows * lines >= waves * (ng == 4 ? 6400 : 12500);
}

cudaError_t prompt_attend(const l3m_kv4 *c, const l3m_kv4_attend *a, cudaStream_t s) {
    PromptArgs p = {*a, kv4_dev(c), a->n_heads / c->n_kv_heads, 0, 0};
    p.row_tiles = (int)(((long long)a->max_q * p.group + 2 * kRows - 1) / (2 * kRows));
    p.vec = !(((uintptr_t)a->q | (uintptr_t)a->out) & 15) && (a->q_ld | a->out_ld) % 8 == 0;
    const bool mx = c->dtype == L3M_DT_MXFP4;
    if (p.c.ng == 2) return mx ? launch<2, 1>(p, s) : launch<2, 0>(p, s);
    return mx ? launch<4, 1>(p, s) : launch<4, 0>(p, s);
}

}  // namespace l3m
