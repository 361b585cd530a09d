// Attention over the paged 4-bit cache (l3m_kv4_attend_dev; contract in include/l3m_kernels.h, layout in
// kv4.cuh).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <cmath>
#include <cstdio>
#include "kv4.cuh"
#include "kv4_prompt.h"

using namespace l3m;

extern "C" int l3m_error_msg(const char *msg);
extern "C" int l3m_error_cuda(int e, const char *what);

namespace {

int refuse(const char *entry, const char *why) {
    char msg[200];
    snprintf(msg, sizeof msg, "%s: %s", entry, why);
    return l3m_error_msg(msg);
}

struct AttendArgs {
    l3m_kv4_attend a;
    Kv4Dev c;
    int group, row_tiles;                 // query heads per kv head; row tiles of a request with max_q queries
    int split;                            // 1: workers share all tiles out evenly, 0: a worker takes whole segments
    float *part;                          // [workers][2] partial results of [rows][Dp + 2] floats: values, then reference and sum
    int4 *desc;                           // [workers][2]: the segment whose last piece the worker did: where it began, head, row tile; its request's first row and rows
};

// ---- warp pieces

__device__ __forceinline__ uint32_t prmt(uint32_t a, uint32_t b, uint32_t sel) {
    uint32_t d;
    asm("prmt.b32 %0, %1, %2, %3;" : "=r"(d) : "r"(a), "r"(b), "r"(sel));
    return d;
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// Two floats rounded to f16 (lo in the low half).
__device__ __forceinline__ uint32_t pack_f16(float lo, float hi) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
    return d;
}
__device__ __forceinline__ float2 unpack_f16(uint32_t v) {
    const __half2 h = *(const __half2 *)&v;
    return __half22float2(h);
}
// The 8x8 f16 matrix held as accumulators are (row lane / 4, columns 2 * (lane % 4)), transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t v) {
    uint32_t d;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}
__device__ __forceinline__ void mma(float *c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t mul2(uint32_t a, uint32_t b) {
    const __half2 r = __hmul2(*(const __half2 *)&a, *(const __half2 *)&b);
    return *(const uint32_t *)&r;
}
// The two e2m1 codes of byte K (the low nibble first) as f16.
template <int K> __device__ __forceinline__ uint32_t e2m1_pair(uint32_t w) {
    uint32_t d;
    asm("{ .reg .b8 c, z0, z1, z2;\n mov.b32 {c, z0, z1, z2}, %1;\n cvt.rn.f16x2.e2m1x2 %0, c; }" : "=r"(d) : "r"(w >> (8 * K)));
    return d;
}

// N 32-bit words from shared memory in the widest accesses that N words' alignment allows.
template <int N> __device__ __forceinline__ void lds_words(uint32_t *w, const uint8_t *p) {
    if constexpr (N % 4 == 0) {
#pragma unroll
        for (int i = 0; i < N / 4; i++) {
            const uint4 v = ((const uint4 *)p)[i];
            w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
        }
    } else if constexpr (N % 2 == 0) {
#pragma unroll
        for (int i = 0; i < N / 2; i++) {
            const uint2 v = ((const uint2 *)p)[i];
            w[2 * i] = v.x; w[2 * i + 1] = v.y;
        }
    } else {
#pragma unroll
        for (int i = 0; i < N; i++) w[i] = ((const uint32_t *)p)[i];
    }
}
// N 16-bit values, two to a word.
template <int N> __device__ __forceinline__ void lds_halves(uint32_t *w, const uint8_t *p) {
    if constexpr (N % 2 == 0) {
        lds_words<N / 2>(w, p);
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 2) w[i / 2] = ((const uint16_t *)p)[i] | (i + 1 < N ? (uint32_t)((const uint16_t *)p)[i + 1] << 16 : 0u);
    }
}
// N bytes, four to a word.
template <int N> __device__ __forceinline__ void lds_bytes(uint32_t *w, const uint8_t *p) {
    if constexpr (N % 4 == 0) {
        lds_words<N / 4>(w, p);
    } else {
#pragma unroll
        for (int i = 0; i < (N + 3) / 4; i++) w[i] = 0;
#pragma unroll
        for (int i = 0; i < N; i++) w[i / 4] |= (uint32_t)p[i] << (8 * (i % 4));
    }
}
// Halves h of a (low) and of b (high).
__device__ __forceinline__ uint32_t pair_of(const uint32_t *a, const uint32_t *b, int h) { return prmt(a[h / 2], b[h / 2], h % 2 ? 0x7632 : 0x5410); }

__device__ __forceinline__ float exp2i(int e) { return __int_as_float((e + 127) << 23); }   // 2^e, -126 <= e <= 127

__device__ __forceinline__ float load_f32(const float *p) { return *p; }
__device__ __forceinline__ float load_f32(const __nv_bfloat16 *p) { return __bfloat162float(*p); }
__device__ __forceinline__ void store_f32(float *p, float x) { *p = x; }
__device__ __forceinline__ void store_f32(__nv_bfloat16 *p, float x) { *p = __float2bfloat16_rn(x); }

constexpr int kStages = 4;               // tiles of a warp's ring: two pairs
constexpr int kMaxSms = 160;
constexpr float kFloor = -1e30f;         // the reference of a row that has seen nothing

constexpr int kCtas = 2;                 // resident CTAs per SM
// Warps of a CTA: as many as the registers of a variant allow: 12 on an SM at 166 each, 8 at 255. (Of the latter, one CTA of 6 warps
// took 103 us where two of 4 take 81, one of 4 108: 32 requests of 1000 tokens, 5 queries each, f32, 32 heads to 8 of 128.)
constexpr int warps_of(int ng, int nt) { return ng * nt <= 5 ? 6 : 4; }

constexpr int kMostBase = 4;             // bf16 results over q4_0: the window's base up to which one pass serves, scales below 32

template <typename T, int NG, int NT>
__device__ __noinline__ void far_tiles(const AttendArgs &p, uint8_t *smem, int r, int h, int rt, Queries rq, int a, int b);

// One piece of a segment (request r, kv head h, row tile rt): cache tiles [a, b), by the CTA's warps. Scores are
// computed transposed, S^T = K Q^T (16 tokens x 8 rows a product), so that a decode step's few rows pad to 8, not 16, and
// O^T = V^T P^T follows from it with one 8x8 transposition per 8 tokens. Each warp keeps its own softmax reference and
// sums over its pairs of tiles, every kWarps-th of the piece; the warps are joined at the end.
//
// Codes go into the products as the integers they are, so that the cache's values suffer no rounding. For q4_0 and bf16 results a
// nibble in the low byte of a half is an f16 subnormal, n * 2^-24 (or n * 2^-20 four bits higher): one mask, no conversion. Its offset
// of 8 is taken off the sum instead: scores start at -8 sum(q), and the sum of P times scale, which the values' offset multiplies,
// comes from one more product with ones. Float results use n - 8 itself (one more f16 operation), so that nothing cancels.
// What that costs: the tensor cores align a product's terms by their exponents and cut them off 24 bits below the largest, and a subnormal's exponent counts as
// -14, so a step of 16 tokens loses up to 2^-14 of P times scale (in units of a code, most often 2^-15), 2^-17 of the codes' sums; settle() keeps what
// the sums themselves lose from growing with the context.
// A key's scale multiplies its block's score; a value's scale multiplies P. Queries are scaled to 2^10 by a power of two, so f16 holds
// them (bf16 exactly, float as two f16 of 22 bits); P is held up to 2^14, rounded to f16 for bf16 results and
// split in two f16 for float ones.
template <typename T, int MX, int NG, int NT>
struct Worker {
    static constexpr int kWarps = warps_of(NG, NT), kThreads = 32 * kWarps;
    static constexpr bool PREC = sizeof(T) == 4;
    static constexpr bool SUBN = !PREC && !MX;
    static constexpr int NR = 8 * NT, DP = 32 * NG, SB = MX ? 1 : 2;
    static constexpr int TB = NG * (512 + 32 * SB);
    static constexpr int RING = kStages * TB;
    static constexpr int LD = DP + 4, BUF = kWarps * NR * LD * 4;          // the warps' results, [warp][row][LD]: values, reference, sum
    // q4_0's bf16 results keep them beside the ring, as a warp may come back to its tiles (run()); the others in its place.
    static constexpr int BUF_AT = SUBN ? kWarps * RING : 0;
    static constexpr int SMEM = (BUF_AT + BUF > kWarps * RING ? BUF_AT + BUF : kWarps * RING) + (SUBN ? kWarps * (int)sizeof(AttendArgs) : 0);
    static constexpr int QP = PREC ? 2 : 1;
    static constexpr int NG2 = NG + NG % 2;                                  // blocks, in pairs
    static constexpr int SW = MX ? (NG + 3) / 4 : (NG + 1) / 2;              // words of a row's scales

    const AttendArgs &p;
    uint8_t *smem;
    int warp, lane, g, t;
    uint32_t q[QP][NT][NG][4];            // B fragments of the rows: [high, low part][row][block][2 steps x 2]
    uint32_t c0[SUBN ? NT : 1][2];        // the offset's part of the scores as a B fragment: -sum(q) / 2^8 of block k, and its rest, against the keys' scales
    float mult[NT][2];
    int pos[NT][2];
    float ref[NT][2], sum[NT][2];
    float o[NT][NG][2][4];
    float w[SUBN ? NT : 1][SUBN ? (NG + 1) / 2 : 1][4];                       // two blocks' sums of P times scale: rows 0-7 block 2i, rows 8-15 block 2i + 1
    // The window of the values' scales that a step's products take as they come: exponents base .. base + 15. mxfp4: a base for each block,
    // four to a word; the block's sums are in units of 2^(base - 113). q4_0: one base for all blocks, which lowers P's limit. For bf16 results P itself
    // is held in f16, so that with a base above 4 (scales of 32 and more) it would have too few bits: the rows are then done again, see run().
    uint32_t base4[MX ? SW : 1];
    int base;
    bool begun;
    static constexpr int kFirstBase = 115;                                   // scales of 2^-12 to 2^3, as activations have them; another window costs the first step a little

    __device__ Worker(const AttendArgs &args, uint8_t *sm) : p(args), smem(sm) {
        warp = threadIdx.x >> 5;
        lane = threadIdx.x & 31;
        g = lane >> 2;
        t = lane & 3;
    }
    // Row r of a 16-token product is token tau(r): a warp's reads of keys (rows g) and of values (tokens of k = 2t, 2t + 1) then spread over the banks.
    __device__ static int tau(int r) { return (r & 8) | (r & 1 ? 4 + (((r >> 1) & 3) ^ 1) : (r >> 1) & 3); }

    __device__ __forceinline__ void load_rows(int start, int nq, int first, int h, int rt) {
        float m8[NT], cs[NT][NG];
        const float log2e = 1.4426950408889634f;
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const int row = rt * NR + n * 8 + g, i = row / p.group, head = h * p.group + row - i * p.group;
            const T *src = (const T *)p.a.q + (size_t)(start + i) * p.a.q_ld + (size_t)head * p.c.dim;
            float x[NG][8], top = 0.0f;
#pragma unroll
            for (int j = 0; j < NG; j++)
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    const int d = 32 * j + 8 * t;
                    x[j][e] = i < nq && d < p.c.dim ? load_f32(src + d + e) : 0.0f;
                    top = fmaxf(top, fabsf(x[j][e]));
                }
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
            top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
            const int up = top > 0.0f ? 9 - max(min(ilogbf(top), 127), -149) : 0;      // |x| * 2^up < 2^10
            const float up0 = exp2i(up / 2), up1 = exp2i(up - up / 2);
            m8[n] = ldexpf(p.a.scale * log2e, (SUBN ? 24 : 0) - up);
#pragma unroll
            for (int j = 0; j < NG; j++) {
                float s = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) x[j][e] = x[j][e] * up0 * up1;
                if (SUBN) {
                    // The fragments hold nibbles 2k and 2k + 4, then 16 times nibbles 2k + 1 and 2k + 5.
#pragma unroll
                    for (int k = 0; k < 2; k++) {
                        q[0][n][j][2 * k] = pack_f16(x[j][2 * k], x[j][2 * k + 4]);
                        q[0][n][j][2 * k + 1] = pack_f16(x[j][2 * k + 1] * 0.0625f, x[j][2 * k + 5] * 0.0625f);
                        const float2 a = unpack_f16(q[0][n][j][2 * k]), b = unpack_f16(q[0][n][j][2 * k + 1]);
                        s += a.x + a.y + 16.0f * (b.x + b.y);
                    }
                } else {
#pragma unroll
                    for (int k = 0; k < 4; k++) {
                        // q4_0: nibbles k and k + 4 make a pair; mxfp4: the two of a byte
                        const float a = x[j][MX ? 2 * k : k], b = x[j][MX ? 2 * k + 1 : k + 4];
                        q[0][n][j][k] = pack_f16(a, b);
                        const float2 back = unpack_f16(q[0][n][j][k]);
                        if (PREC) q[QP - 1][n][j][k] = pack_f16(a - back.x, b - back.y);
                    }
                }
                cs[n][j] = s;
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++) {
            if (SUBN) {
#pragma unroll
                for (int j = 0; j < NG; j++) {
                    cs[n][j] += __shfl_xor_sync(0xffffffffu, cs[n][j], 1);
                    cs[n][j] += __shfl_xor_sync(0xffffffffu, cs[n][j], 2);
                }
                // k = 0 .. NG2 - 1: the blocks' high parts, k = NG2 .. 2 NG2 - 1: what f16 leaves of them
                float k4[4];
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const int k = 2 * t + (i & 1) + (i & 2 ? 8 : 0);
                    float hi = 0.0f;
#pragma unroll
                    for (int j = 0; j < NG; j++) hi = k % NG2 == j && k < 2 * NG2 ? cs[n][j] * -0x1p-8f : hi;
                    const float rest = hi - __half2float(__float2half_rn(hi));
                    k4[i] = k < NG2 ? hi : rest;
                }
                c0[SUBN ? n : 0][0] = pack_f16(k4[0], k4[1]);
                c0[SUBN ? n : 0][1] = pack_f16(k4[2], k4[3]);
            }
#pragma unroll
            for (int c = 0; c < 2; c++) {
                mult[n][c] = __shfl_sync(0xffffffffu, m8[n], 8 * t + 4 * c);
                const int i = (rt * NR + n * 8 + 2 * t + c) / p.group;
                pos[n][c] = i < nq ? first + i : -1;
                ref[n][c] = kFloor;
                sum[n][c] = 0.0f;
            }
#pragma unroll
            for (int j = 0; j < NG; j++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    o[n][j][0][e] = o[n][j][1][e] = 0.0f;
                    if (SUBN) w[n][j / 2][e] = 0.0f;
                }
        }
        base = PREC && !MX ? -16 : 0;
#pragma unroll
        for (int i = 0; i < (MX ? SW : 1); i++) base4[i] = 0x01010101u * kFirstBase;
        begun = false;
    }

    __device__ __forceinline__ void scale_rows(int n, float f0, float f1) {
#pragma unroll
        for (int j = 0; j < NG; j++) {
#pragma unroll
            for (int m = 0; m < 2; m++) {
                o[n][j][m][0] *= f0; o[n][j][m][1] *= f1;
                o[n][j][m][2] *= f0; o[n][j][m][3] *= f1;
            }
            if (SUBN) {
                w[n][j / 2][j % 2 * 2] *= f0; w[n][j / 2][j % 2 * 2 + 1] *= f1;
            }
        }
    }

    // U tiles in shared memory, neighbours in the context. EDGE: some row does not see some of their tokens, which begin at tok0;
    // [lo_any, hi_any) is seen by some row. False: their scales do not fit the window, and the tiles have to come one by one, EDGE.
    template <bool EDGE, int U, bool FAR = false> __device__ __forceinline__ bool step(const uint8_t *sm, int tok0, int lo_any, int hi_any) {
        const int ra = tau(g), t0 = PREC ? ra : t, t1 = 4 + (t ^ 1);
        constexpr int KS = 512 * NG, VS = KS + 16 * NG * SB;
        // ---- scores
        float s[U][NT][4];
#pragma unroll
        for (int u = 0; u < U; u++) {
            const uint8_t *tl = sm + u * TB;
            uint32_t ka[NG], kb[NG], sa[SW], sb[SW];
            lds_words<NG>(ka, tl + ra * 16 * NG + t * 4 * NG);
            lds_words<NG>(kb, tl + (ra + 8) * 16 * NG + t * 4 * NG);
            if (MX) {
                lds_bytes<NG>(sa, tl + KS + ra * NG);
                lds_bytes<NG>(sb, tl + KS + (ra + 8) * NG);
            } else {
                lds_halves<NG>(sa, tl + KS + ra * NG * 2);
                lds_halves<NG>(sb, tl + KS + (ra + 8) * NG * 2);
            }
#pragma unroll
            for (int n = 0; n < NT; n++) {
                s[u][n][0] = s[u][n][1] = s[u][n][2] = s[u][n][3] = 0.0f;
                if (SUBN) {
                    // A: the scales of rows g and g + 8, columns 2t, 2t + 1 (+ 8): blocks 2t % NG2 and the next
                    uint32_t f[4] = {0, 0, 0, 0};
                    if constexpr (NG % 2 == 0) {
                        const uint8_t *row = tl + KS + ra * NG * 2;
                        if (t < NG) f[0] = *(const uint32_t *)(row + t % (NG / 2) * 4), f[1] = *(const uint32_t *)(row + 16 * NG + t % (NG / 2) * 4);
                        if (NG > 4 && t + 4 < NG) f[2] = *(const uint32_t *)(row + (t + 4) % (NG / 2) * 4), f[3] = *(const uint32_t *)(row + 16 * NG + (t + 4) % (NG / 2) * 4);
                    } else {
#pragma unroll
                        for (int i = 0; i < SW; i++) {
                            const bool lo = t < NG2 && t % (NG2 / 2) == i, hi = t + 4 < NG2 && (t + 4) % (NG2 / 2) == i;
                            f[0] = lo ? sa[i] : f[0]; f[1] = lo ? sb[i] : f[1];
                            f[2] = hi ? sa[i] : f[2]; f[3] = hi ? sb[i] : f[3];
                        }
                    }
                    mma(s[u][n], f[0], f[1], f[2], f[3], c0[SUBN ? n : 0][0], c0[SUBN ? n : 0][1]);
#pragma unroll
                    for (int e = 0; e < 4; e++) s[u][n][e] *= 0x1p-13f;       // 8 * 2^-24 * 2^8
                }
            }
#pragma unroll
            for (int j = 0; j < NG; j++) {
                uint32_t fa[4], fb[4];
                codes4(fa, ka[j]);
                codes4(fb, kb[j]);
                float da, db;
                if (MX) {
                    da = __uint_as_float((sa[j / 4] >> (8 * (j % 4)) & 0xff) << 23);
                    db = __uint_as_float((sb[j / 4] >> (8 * (j % 4)) & 0xff) << 23);
                } else {
                    const float2 a2 = unpack_f16(sa[j / 2]), b2 = unpack_f16(sb[j / 2]);
                    da = j % 2 ? a2.y : a2.x;
                    db = j % 2 ? b2.y : b2.x;
                }
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    float acc[4];
                    if (PREC) {
                        acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
                        mma(acc, fa[0], fb[0], fa[1], fb[1], q[QP - 1][n][j][0], q[QP - 1][n][j][1]);
                        mma(acc, fa[2], fb[2], fa[3], fb[3], q[QP - 1][n][j][2], q[QP - 1][n][j][3]);
                        mma(acc, fa[0], fb[0], fa[1], fb[1], q[0][n][j][0], q[0][n][j][1]);
                    } else {
                        acc[0] = acc[1] = acc[2] = acc[3] = 0.0f;
                        mma(acc, fa[0], fb[0], fa[1], fb[1], q[0][n][j][0], q[0][n][j][1]);
                    }
                    mma(acc, fa[2], fb[2], fa[3], fb[3], q[0][n][j][2], q[0][n][j][3]);
                    s[u][n][0] = fmaf(acc[0], da, s[u][n][0]);
                    s[u][n][1] = fmaf(acc[1], da, s[u][n][1]);
                    s[u][n][2] = fmaf(acc[2], db, s[u][n][2]);
                    s[u][n][3] = fmaf(acc[3], db, s[u][n][3]);
                }
            }
            if (EDGE) {
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const int tok = tok0 + u * kKvTile + ra + (e & 2 ? 8 : 0), at = pos[n][e & 1];
                        if (tok > at || (p.a.window && tok <= at - p.a.window)) s[u][n][e] = -INFINITY;
                    }
            }
        }
        // ---- the values' scales: of this lane's tokens as P's transposed pairs want them, or (float results) as the scores lie
        uint32_t v[U][4][SW];
        auto load_scales = [&]() {
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    if (PREC && k % 2) {
#pragma unroll
                        for (int i = 0; i < SW; i++) v[u][k][i] = 0;
                        continue;
                    }
                    const int row = (k % 2 ? t1 : t0) + (k / 2) * 8;
                    if (MX) lds_bytes<NG>(v[u][k], sm + u * TB + VS + row * NG);
                    else lds_halves<NG>(v[u][k], sm + u * TB + VS + row * NG * 2);
                    if (EDGE) harmless(v[u][k], tok0 + u * kKvTile + row, lo_any, hi_any);
                }
        };
        auto relative = [&]() {                                              // mxfp4: bytes 0 .. 15 are in the window
            if (MX) {
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int k = 0; k < 4; k += PREC ? 2 : 1)
#pragma unroll
                        for (int i = 0; i < SW; i++) v[u][k][i] = EDGE && v[u][k][i] == kGone ? 0 : v[u][k][i] - base4[MX ? i : 0];
            }
        };
        load_scales();
        relative();
        // ---- does the reference still hold, do the scales lie in the window?
        bool far = !FAR && outside<U>(v);
        float lim = limit(), z[U][NT][4], high = kFloor;         // the exponents of P
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    z[u][n][e] = EDGE && s[u][n][e] == -INFINITY ? -INFINITY : fmaf(s[u][n][e], mult[n][e & 1], -ref[n][e & 1]);
                    high = fmaxf(high, z[u][n][e]);
                }
        if (__any_sync(0xffffffffu, far || high > lim)) {
            if (MX && __any_sync(0xffffffffu, far)) {
                load_scales();
                uint32_t top[SW];
#pragma unroll
                for (int i = 0; i < SW; i++) {
                    top[i] = 0;
#pragma unroll
                    for (int u = 0; u < U; u++)
#pragma unroll
                        for (int k = 0; k < 4; k += PREC ? 2 : 1) top[i] = __vmaxu4(top[i], EDGE && v[u][k][i] == kGone ? 0 : v[u][k][i]);
#pragma unroll
                    for (int d = 1; d < 32; d <<= 1) top[i] = __vmaxu4(top[i], __shfl_xor_sync(0xffffffffu, top[i], d));
                }
#pragma unroll
                for (int j = 0; j < NG; j++) {                               // a block whose base moves gets room for three more below the window's end
                    const int at = 8 * (j % 4), have = base4[MX ? j / 4 : 0] >> at & 0xff, most = min((int)(top[j / 4] >> at & 0xff), 254);
                    if (most > have + 15 || (!begun && most < have)) {
                        const int to = max(min(most - 12, 239), 0);
                        base4[MX ? j / 4 : 0] += (uint32_t)(to - have) << at;
                        const float f = !begun || to - have > 126 ? 0.0f : exp2i(have - to);
#pragma unroll
                        for (int n = 0; n < NT; n++)
#pragma unroll
                            for (int e = 0; e < 4; e++) {
                                o[n][j][0][e] *= f;
                                o[n][j][1][e] *= f;
                            }
                    }
                }
                relative();
            } else if (!MX && !FAR && __any_sync(0xffffffffu, far)) {
                uint32_t top = 0;
#pragma unroll
                for (int u = 0; u < U; u++)
#pragma unroll
                    for (int k = 0; k < 4; k += PREC ? 2 : 1)
#pragma unroll
                        for (int i = 0; i < SW; i++) top = max(top, max(v[u][k][i] >> 10 & 31, v[u][k][i] >> 26 & 31));
                base = max(base, (int)__reduce_max_sync(0xffffffffu, top) - 15);
                lim = limit();                                               // raising base lowers it
            }
            begun = true;
            if (!SUBN) far = __any_sync(0xffffffffu, outside<U>(v));
#pragma unroll
            for (int n = 0; n < NT; n++) {
                float f[2];
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    float m = -INFINITY;
#pragma unroll
                    for (int u = 0; u < U; u++)
#pragma unroll
                        for (int e = c; e < 4; e += 2)
                            if (!(EDGE && s[u][n][e] == -INFINITY)) m = fmaxf(m, s[u][n][e] * mult[n][c]);
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 4));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 8));
                    m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, 16));
                    f[c] = 1.0f;
                    if (m - ref[n][c] > lim) {
                        const float to = m - lim + 2.0f;                     // room for 2^2 before the next move: more costs P bits where scales are small
                        f[c] = ex2(ref[n][c] - to);
                        ref[n][c] = to;
                    }
#pragma unroll
                    for (int u = 0; u < U; u++)
#pragma unroll
                        for (int e = c; e < 4; e += 2) z[u][n][e] = EDGE && s[u][n][e] == -INFINITY ? -INFINITY : fmaf(s[u][n][e], mult[n][c], -ref[n][c]);
                    sum[n][c] *= f[c];
                }
                scale_rows(n, f[0], f[1]);
            }
        }
        // ---- probabilities and values
        if constexpr (EDGE && U == 1 && (!SUBN || FAR)) {
            if (FAR || far) {
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) z[0][n][e] = ex2(z[0][n][e]);
                    sum[n][0] += z[0][n][0] + z[0][n][2];
                    sum[n][1] += z[0][n][1] + z[0][n][3];
                }
                far_values(sm, z[0], tok0, lo_any, hi_any);
                return true;
            }
        } else if (!SUBN && far) {
            return false;                                                    // nothing has been added yet
        }
        if constexpr (!FAR) {
#pragma unroll
            for (int u = 0; u < U; u++) {
                uint32_t pb[NT][2];
#pragma unroll
                for (int n = 0; n < NT; n++) {
#pragma unroll
                    for (int e = 0; e < 4; e++) z[u][n][e] = ex2(z[u][n][e]);
                    sum[n][0] += z[u][n][0] + z[u][n][2];
                    sum[n][1] += z[u][n][1] + z[u][n][3];
                    if (!PREC) {
                        pb[n][0] = transpose8(pack_f16(z[u][n][0], z[u][n][1]));
                        pb[n][1] = transpose8(pack_f16(z[u][n][2], z[u][n][3]));
                    }
                }
                uint32_t c[4][(NG + 1) / 2];
                const uint8_t *vc = sm + u * TB + 256 * NG + g * 2 * NG;
                lds_halves<NG>(c[0], vc + t * 16 * NG);
                lds_halves<NG>(c[1], vc + t1 * 16 * NG);
                lds_halves<NG>(c[2], vc + (t + 8) * 16 * NG);
                lds_halves<NG>(c[3], vc + (t1 + 8) * 16 * NG);
#pragma unroll
                for (int j = 0; j < NG; j++) {
                    uint32_t fa[4], fb[4];
                    value4(fa, c[0], c[1], j);
                    value4(fb, c[2], c[3], j);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        if (PREC) {
                            float d0, d1;
                            if (MX) {
                                d0 = rel_f32(v[u][0][j / 4] >> (8 * (j % 4)) & 0xff);
                                d1 = rel_f32(v[u][2][j / 4] >> (8 * (j % 4)) & 0xff);
                            } else {
                                const float2 a2 = unpack_f16(v[u][0][j / 2]), b2 = unpack_f16(v[u][2][j / 2]);
                                d0 = j % 2 ? a2.y : a2.x;
                                d1 = j % 2 ? b2.y : b2.x;
                            }
                            const float x0 = z[u][n][0] * d0, x1 = z[u][n][1] * d0, x2 = z[u][n][2] * d1, x3 = z[u][n][3] * d1;
                            const uint32_t h0 = pack_f16(x0, x1), h1 = pack_f16(x2, x3);
                            const float2 u0 = unpack_f16(h0), u1 = unpack_f16(h1);
                            const uint32_t l0 = transpose8(pack_f16(x0 - u0.x, x1 - u0.y)), l1 = transpose8(pack_f16(x2 - u1.x, x3 - u1.y));
                            const uint32_t b0 = transpose8(h0), b1 = transpose8(h1);
#pragma unroll
                            for (int m = 0; m < 2; m++) {                        // a tile's sum by itself: the accumulator of a product is truncated, not rounded
                                float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                                mma(acc, fa[2 * m], fa[2 * m + 1], fb[2 * m], fb[2 * m + 1], l0, l1);
                                mma(acc, fa[2 * m], fa[2 * m + 1], fb[2 * m], fb[2 * m + 1], b0, b1);
#pragma unroll
                                for (int e = 0; e < 4; e++) o[n][j][m][e] += acc[e];
                            }
                        } else {
                            uint32_t d0, d1;
                            if (MX) {
                                d0 = rel_f16(v[u][0], v[u][1], j);
                                d1 = rel_f16(v[u][2], v[u][3], j);
                            } else {
                                d0 = pair_of(v[u][0], v[u][1], j);
                                d1 = pair_of(v[u][2], v[u][3], j);
                            }
                            const uint32_t b0 = mul2(pb[n][0], d0), b1 = mul2(pb[n][1], d1);
                            mma(o[n][j][0], fa[0], fa[1], fb[0], fb[1], b0, b1);
                            mma(o[n][j][1], fa[2], fa[3], fb[2], fb[3], b0, b1);
                            if (SUBN) {
                                constexpr uint32_t one = 0x3c003c00u;
                                const uint32_t up = j % 2 ? 0 : one, down = j % 2 ? one : 0;
                                mma(w[SUBN ? n : 0][SUBN ? j / 2 : 0], up, down, up, down, b0, b1);
                            }
                        }
                    }
                }
            }
        }
        return true;
    }
    // A word's 8 codes as four pairs.
    __device__ __forceinline__ static void codes4(uint32_t *f, uint32_t x) {
        if (MX) {
            f[0] = e2m1_pair<0>(x); f[1] = e2m1_pair<1>(x);
            f[2] = e2m1_pair<2>(x); f[3] = e2m1_pair<3>(x);
        } else {
            const uint32_t y = x >> 8;                                       // n0 and 16 n1 of the low bytes, then of the high ones
            f[0] = x & 0x000f000fu; f[1] = x & 0x00f000f0u;
            f[2] = y & 0x000f000fu; f[3] = y & 0x00f000f0u;
            if (!SUBN) whole(f);
        }
    }
    // Block j's 4 codes of two tokens as four pairs of the same dim.
    __device__ __forceinline__ static void value4(uint32_t *f, const uint32_t *a, const uint32_t *b, int j) {
        if (MX) {
            const uint32_t wa = a[j / 2], wb = b[j / 2];
            const uint32_t x0 = j % 2 ? e2m1_pair<2>(wa) : e2m1_pair<0>(wa), y0 = j % 2 ? e2m1_pair<2>(wb) : e2m1_pair<0>(wb);
            const uint32_t x1 = j % 2 ? e2m1_pair<3>(wa) : e2m1_pair<1>(wa), y1 = j % 2 ? e2m1_pair<3>(wb) : e2m1_pair<1>(wb);
            f[0] = prmt(x0, y0, 0x5410); f[1] = prmt(x0, y0, 0x7632);
            f[2] = prmt(x1, y1, 0x5410); f[3] = prmt(x1, y1, 0x7632);
        } else {
            if (SUBN) {                                                      // y = n0 + 16 n1 and n0 of the low bytes, then of the high ones
                const uint32_t x = pair_of(a, b, j);
                f[0] = x & 0x00ff00ffu; f[1] = x & 0x000f000fu;
                f[2] = prmt(x, 0, 0x4341); f[3] = f[2] & 0x000f000fu;
            } else {
                const uint32_t x = pair_of(a, b, j), y = x >> 8;
                f[0] = x & 0x000f000fu; f[1] = x & 0x00f000f0u;
                f[2] = y & 0x000f000fu; f[3] = y & 0x00f000f0u;
                whole(f);
            }
        }
    }
    // n -> n - 8 in f16: 1024 + n (or 1024 + 16 n) is a number whose last bits are n.
    __device__ __forceinline__ static void whole(uint32_t *f) {
        const __half2 off = __halves2half2(__ushort_as_half(0xe408), __ushort_as_half(0xe408));   // -1032
        const __half2 s16 = __halves2half2(__ushort_as_half(0x2c00), __ushort_as_half(0x2c00));   // 1/16
        const __half2 o16 = __halves2half2(__ushort_as_half(0xd480), __ushort_as_half(0xd480));   // -72
#pragma unroll
        for (int k = 0; k < 4; k++) {
            uint32_t x = f[k] | 0x64006400u;
            const __half2 h = *(const __half2 *)&x;
            const __half2 r = k % 2 ? __hfma2(h, s16, o16) : __hadd2(h, off);
            f[k] = *(const uint32_t *)&r;
        }
    }
    // mxfp4 scales in the window, e above its base: 2^(e - 14), 2^-14 to 2.
    __device__ __forceinline__ static float rel_f32(uint32_t e) { return __uint_as_float((e + 113u) << 23); }
    __device__ __forceinline__ static uint32_t rel_f16(const uint32_t *a, const uint32_t *b, int j) {
        const uint32_t x = prmt(a[j / 4], b[j / 4], j % 4 < 2 ? 0x5410 : 0x7632);      // two blocks' bytes of both tokens
        const uint32_t e = j % 2 ? prmt(x, 0, 0x4341) : x & 0x00ff00ffu;
        return e * 1024u + 0x04000400u;
    }
    // The largest exponent of P: P times a scale has to stay below 2^16 in the products' f16.
    __device__ __forceinline__ float limit() const { return MX ? 14.0f : 14.0f - (float)base; }

    // Does some scale of this lane's tokens lie outside the window? mxfp4: bytes 0 .. 15 above the base. q4_0: the exponents of f16 scales, for
    // bf16 results those above the window alone (scales of 2 and more, mostly none): below it P times scale has its 11 bits down to 2^-14.
    template <int U> __device__ __forceinline__ bool outside(const uint32_t (&v)[U][4][SW]) const {
        uint32_t any = 0;
#pragma unroll
        for (int u = 0; u < U; u++)
#pragma unroll
            for (int k = 0; k < 4; k += PREC ? 2 : 1)
#pragma unroll
                for (int i = 0; i < SW; i++) {
                    // a difference below 0 shows in its own high bits, whatever it borrows from the next one
                    if (MX) any |= v[u][k][i] & (0xf0f0f0f0u >> (NG - 4 * i < 4 ? 8 * (4 * i + 4 - NG) : 0));
                    else if (PREC) any |= ((v[u][k][i] & 0x7fff7fffu) - (uint32_t)base * 0x04000400u) & (NG - 2 * i < 2 ? 0x0000c000u : 0xc000c000u);
                    else any |= v[u][k][i] & 0x40004000u;
                }
        if (SUBN && any && base > 0) {
            any = 0;
#pragma unroll
            for (int u = 0; u < U; u++)
#pragma unroll
                for (int k = 0; k < 4; k++)
#pragma unroll
                    for (int i = 0; i < SW; i++) any = __vmaxu2(any, v[u][k][i] & 0x7fff7fffu);
            return (int)max(any >> 10 & 31, any >> 26) > base + 15;
        }
        return any != 0;
    }

    // What must not meet the zeros of rows that do not see token tok: a scale that is not finite counts as 0, and so does the scale of a token that
    // no row sees (mxfp4: kGone, as good as any in the window then).
    static constexpr uint32_t kGone = 0xffffffffu;
    __device__ __forceinline__ static void harmless(uint32_t *v, int tok, int lo_any, int hi_any) {
        const bool gone = tok < lo_any || tok >= hi_any;
#pragma unroll
        for (int i = 0; i < SW; i++) {
            uint32_t &x = v[i];
            if (MX) {
#pragma unroll
                for (int k = 0; k < 32; k += 8)
                    if ((x >> k & 0xff) == 0xff) x &= ~(0xffu << k);
                if (gone) x = kGone;
            } else {
                if ((x & 0x7c00u) == 0x7c00u) x &= 0xffff0000u;
                if ((x & 0x7c000000u) == 0x7c000000u) x &= 0x0000ffffu;
                if (gone) x = 0;
            }
        }
    }

    // A tile whose scales the window does not hold: its values' products by sixteen exponents at a time, each level's scales brought up to the
    // window (or down to it: q4_0 scales of 2 and more for bf16 results) and its sums added in 32 bits. So no scale is lost beside
    // a larger one of another token, or one that some rows do not see (mxfp4's blocks have windows of their own). 64 requests to 8192 tokens, 32 heads
    // to 8 of 128, bf16, mxfp4: 133 us where no tile comes here (136 with blocks 2^40 apart), 516 where all do, a token in 16 being 2^20 above the
    // others. There are eight levels: what is 2^-112 of the block's largest scale counts as 0, and the sums' 32 bits keep no more.
    __device__ __forceinline__ void far_values(const uint8_t *tl, const float (&zz)[NT][4], int tok0, int lo_any, int hi_any) {
        const int ra = tau(g), t1 = 4 + (t ^ 1);
        constexpr int VS = 512 * NG + 16 * NG * SB;
        uint32_t pb[NT][2];
        if (!PREC) {
#pragma unroll
            for (int n = 0; n < NT; n++) {
                pb[n][0] = transpose8(pack_f16(zz[n][0], zz[n][1]));
                pb[n][1] = transpose8(pack_f16(zz[n][2], zz[n][3]));
            }
        }
        bool more = true;
#pragma unroll 1
        for (int lev = SUBN ? -1 : 0; lev < 8 && __any_sync(0xffffffffu, more); lev++) {
            const float up = exp2i(16 * lev), down = exp2i(-16 * lev);
            more = SUBN && lev < 0;
            // A scale brought to the window, as a float; 0 outside this level
            auto scale = [&](int row, int j) -> float {
                const int low = (MX ? (int)(base4[MX ? j / 4 : 0] >> (8 * (j % 4)) & 0xff) : base) - 16 * lev;      // exponents low .. low + 15
                if (tok0 + row < lo_any || tok0 + row >= hi_any) return 0.0f;
                if (MX) {
                    const int e = tl[VS + row * NG + j];
                    if (e == 255) return 0.0f;
                    more |= e > 0 && e < low;
                    return e >= low && e <= low + 15 ? exp2i(e - low - 14) : 0.0f;
                }
                const uint32_t x = *(const uint16_t *)(tl + VS + (row * NG + j) * 2);
                const int e = x >> 10 & 31;
                if (e == 31) return 0.0f;
                more |= (x & 0x7fff) && e < low;
                return e >= low && e <= low + 15 ? __half2float(__ushort_as_half((unsigned short)x)) * up : 0.0f;
            };
            uint32_t c[4][(NG + 1) / 2];
            const uint8_t *vc = tl + 256 * NG + g * 2 * NG;
            lds_halves<NG>(c[0], vc + t * 16 * NG);
            lds_halves<NG>(c[1], vc + t1 * 16 * NG);
            lds_halves<NG>(c[2], vc + (t + 8) * 16 * NG);
            lds_halves<NG>(c[3], vc + (t1 + 8) * 16 * NG);
#pragma unroll
            for (int j = 0; j < NG; j++) {
                uint32_t fa[4], fb[4];
                value4(fa, c[0], c[1], j);
                value4(fb, c[2], c[3], j);
                uint32_t s0 = 0, s1 = 0;
                float d0 = 0.0f, d1 = 0.0f;
                if (PREC) {
                    d0 = scale(ra, j);
                    d1 = scale(ra + 8, j);
                } else {
                    s0 = pack_f16(scale(t, j), scale(t1, j));
                    s1 = pack_f16(scale(t + 8, j), scale(t1 + 8, j));
                }
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    uint32_t b0, b1, l0 = 0, l1 = 0;
                    if (PREC) {
                        const float x0 = zz[n][0] * d0, x1 = zz[n][1] * d0, x2 = zz[n][2] * d1, x3 = zz[n][3] * d1;
                        const uint32_t h0 = pack_f16(x0, x1), h1 = pack_f16(x2, x3);
                        const float2 u0 = unpack_f16(h0), u1 = unpack_f16(h1);
                        l0 = transpose8(pack_f16(x0 - u0.x, x1 - u0.y));
                        l1 = transpose8(pack_f16(x2 - u1.x, x3 - u1.y));
                        b0 = transpose8(h0);
                        b1 = transpose8(h1);
                    } else {
                        b0 = mul2(pb[n][0], s0);
                        b1 = mul2(pb[n][1], s1);
                    }
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        if (PREC) mma(acc, fa[2 * m], fa[2 * m + 1], fb[2 * m], fb[2 * m + 1], l0, l1);
                        mma(acc, fa[2 * m], fa[2 * m + 1], fb[2 * m], fb[2 * m + 1], b0, b1);
#pragma unroll
                        for (int e = 0; e < 4; e++) o[n][j][m][e] = fmaf(acc[e], down, o[n][j][m][e]);
                    }
                    if (SUBN) {
                        constexpr uint32_t one = 0x3c003c00u;
                        const uint32_t hi = j % 2 ? 0 : one, lo = j % 2 ? one : 0;
                        float acc[4] = {0.0f, 0.0f, 0.0f, 0.0f};
                        mma(acc, hi, lo, hi, lo, b0, b1);
#pragma unroll
                        for (int e = 0; e < 4; e++) w[SUBN ? n : 0][SUBN ? j / 2 : 0][e] = fmaf(acc[e], down, w[SUBN ? n : 0][SUBN ? j / 2 : 0][e]);
                    }
                }
            }
        }
    }

    // Cache tiles [a, b) of request r's head h into the rows' sums.
    __device__ __forceinline__ void run(int r, int h, int rt, const Queries &rq, int a, int b) {
        tiles<false>(r, h, rt, rq, a, b);
        if constexpr (SUBN) {
            dump();
            // The rows of a cache with such scales, rare as they are, take their tiles twice. As a case of the loop this cost all others 5% (64 requests to 8192
            // tokens, 32 heads to 8 of 128), as a second loop in this function 3%, as it is 1.5%.
            if (base > kMostBase) {
                // (from a copy: a kernel that gives its parameters' address away reads them more slowly, 1.2% of the same case)
                AttendArgs *copy = (AttendArgs *)(smem + BUF_AT + BUF) + warp;
                if (lane == 0) *copy = p;
                __syncwarp();
                far_tiles<T, NG, NT>(*copy, smem, r, h, rt, rq, a, b);
            }
        }
    }

    // FAR: one tile at a time, all of them by far_values().
    template <bool FAR> __device__ __forceinline__ void tiles(int r, int h, int rt, const Queries &rq, int a, int b) {
        const int32_t *table = p.a.tables + (size_t)r * p.a.max_blocks;
        const int i0 = rt * NR / p.group, i1 = min((rt * NR + NR - 1) / p.group, rq.nq - 1);
        const int first = rq.at + i0, last = rq.at + i1;                     // the rows' positions
        const int lo_any = p.a.window ? first - p.a.window + 1 : 0, hi_any = last + 1;
        const int whole_lo = p.a.window ? last - p.a.window + 1 : 0, whole_hi = first + 1;   // seen by every row
        uint8_t *ring = smem + warp * RING;
        const int pairs = (b - a + 1) / 2, n = warp < pairs ? (pairs - warp + kWarps - 1) / kWarps : 0;      // this warp's pairs of tiles: warp, warp + kWarps, ...
        int where = -1;                                                      // lane i: the number in the cache of tile i % 2 of pair 16 * (k / 16) + i / 2
        auto locate = [&](int k) {
            const int tl = a + 2 * (warp + (k + lane / 2) * kWarps) + lane % 2;
            where = -1;
            if (tl < b) {
                const int blk = tl / p.c.tiles, id = table[blk];
                if (id >= 0 && id < p.c.n_pages) where = (id * p.c.n_kv + h) * p.c.tiles + tl - blk * p.c.tiles;
                else if (p.a.status) atomicOr((int *)p.a.status, L3M_KV4_BAD_PAGE);
            }
        };
        uint32_t good = 0;                                                   // which of the ring's tiles are there
        auto fetch = [&](int k) {
            if (k < n) {
                if (k % 16 == 0) locate(k);
                const int st = k % 2 * 2;
                good &= ~(3u << st);
#pragma unroll
                for (int u = 0; u < 2; u++) {
                    const int from = __shfl_sync(0xffffffffu, where, k % 16 * 2 + u);
                    if (from >= 0) {
                        good |= 1u << (st + u);
                        const uint8_t *src = p.c.data + (size_t)from * TB + lane * 16;
                        const uint32_t dst = (uint32_t)__cvta_generic_to_shared(ring + (st + u) * TB) + lane * 16;
#pragma unroll
                        for (int c = 0; c < TB; c += 512)
                            if (c + 512 <= TB || c + lane * 16 < TB)
                                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst + c), "l"(src + c) : "memory");
                    }
                }
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
        fetch(0);                                                            // under way while the rows are read
        load_rows(rq.start, rq.nq, rq.at, h, rt);
        for (int k = 0; k < n; k++) {
            fetch(k + 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
            __syncwarp();
            const int st = k % 2 * 2, tok0 = (a + 2 * (warp + k * kWarps)) * kKvTile;
            const uint32_t both = good >> st & 3;
            if (FAR || !(both == 3 && tok0 >= whole_lo && tok0 + 2 * kKvTile <= whole_hi && step<false, 2>(ring + st * TB, tok0, lo_any, hi_any))) {
#pragma unroll 1
                for (int u = 0; u < 2; u++)
                    if (both >> u & 1) step<true, 1, FAR>(ring + (st + u) * TB, tok0 + u * kKvTile, lo_any, hi_any);
            }
            __syncwarp();
            if (SUBN && k % 32 == 31) settle();
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }

    // The offset of the codes so far taken off the sums. A product truncates what it adds to, by up to 2^-23 of it: sums that held the codes of a whole
    // share would lose more the longer it is. So they hold values, and the codes (up to 255 where a value has 8) of 32 steps at most.
    __device__ __forceinline__ void settle() {
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int j = 0; j < NG; j++)
#pragma unroll
                for (int c = 0; c < 2; c++) {
                    float &sum8 = w[SUBN ? n : 0][SUBN ? j / 2 : 0][j % 2 * 2 + c];
#pragma unroll
                    for (int m = 0; m < 2; m++) {
                        o[n][j][m][c] = fmaf(sum8, -8.0f * 17.0f * 0x1p-24f, o[n][j][m][c]);
                        o[n][j][m][2 + c] = fmaf(sum8, -8.0f * 0x1p-24f, o[n][j][m][2 + c]);
                    }
                    sum8 = 0.0f;
                }
    }

    // This warp's results for the join.
    __device__ __forceinline__ void dump() const {
        float *buf = (float *)(smem + BUF_AT);
#pragma unroll
        for (int n = 0; n < NT; n++) {
#pragma unroll
            for (int c = 0; c < 2; c++) {
                float s = sum[n][c];
                s += __shfl_xor_sync(0xffffffffu, s, 4);
                s += __shfl_xor_sync(0xffffffffu, s, 8);
                s += __shfl_xor_sync(0xffffffffu, s, 16);
                float *row = buf + (warp * NR + n * 8 + 2 * t + c) * LD;
                if (g == 0) {
                    row[DP] = ref[n][c];
                    row[DP + 1] = s;
                }
#pragma unroll
                for (int j = 0; j < NG; j++) {
                    float v[4] = {o[n][j][0][c], o[n][j][0][2 + c], o[n][j][1][c], o[n][j][1][2 + c]};
                    if (SUBN) {
                        const float off = w[SUBN ? n : 0][SUBN ? j / 2 : 0][j % 2 * 2 + c] * 8.0f;
                        const float hi0 = fmaf(v[0] - v[1], 0x1p20f, -off), hi1 = fmaf(v[2] - v[3], 0x1p20f, -off);
                        v[0] = fmaf(v[1], 0x1p24f, -off); v[1] = hi0;
                        v[2] = fmaf(v[3], 0x1p24f, -off); v[3] = hi1;
                    }
                    if (MX) {
                        const float unit = exp2i((int)(base4[MX ? j / 4 : 0] >> (8 * (j % 4)) & 0xff) - 113);
                        v[0] *= unit, v[1] *= unit, v[2] *= unit, v[3] *= unit;
                    }
                    *(float4 *)(row + 32 * j + 4 * g) = make_float4(v[0], v[1], v[2], v[3]);
                }
            }
        }
    }

    // The warps' results joined; the rows' outputs, or a partial result.
    __device__ __forceinline__ void finish(int start, int nq, int h, int rt, float *part) {
        const float *buf = (const float *)(smem + BUF_AT);
        if constexpr (!SUBN) {
            __syncthreads();                                                 // every warp is done with the ring
            dump();
        }
        __syncthreads();
        constexpr int PER = DP / 4;
        for (int i = threadIdx.x; i < NR * PER; i += kThreads) {
            const int row = i / PER, d = (i - row * PER) * 4;
            float m = kFloor, l = 0.0f;
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
            for (int k = 0; k < kWarps; k++) m = fmaxf(m, buf[(k * NR + row) * LD + DP]);
#pragma unroll
            for (int k = 0; k < kWarps; k++) {
                const float *from = buf + (k * NR + row) * LD;
                const float f = ex2(from[DP] - m);
                const float4 x = *(const float4 *)(from + d);
                l = fmaf(from[DP + 1], f, l);
                v.x = fmaf(x.x, f, v.x); v.y = fmaf(x.y, f, v.y); v.z = fmaf(x.z, f, v.z); v.w = fmaf(x.w, f, v.w);
            }
            if (part) {
                float *to = part + row * (DP + 4);
                *(float4 *)(to + d) = v;
                if (d == 0) *(float2 *)(to + DP) = make_float2(m, l);
            } else {
                put(start, nq, h, rt, row, d, v, l);
            }
        }
        __syncthreads();                                                     // the buffer is the next piece's ring
    }

    __device__ __forceinline__ void put(int start, int nq, int h, int rt, int row8, int d, float4 v, float l) const {
        const int row = rt * NR + row8, i = row / p.group;
        if (i >= nq || d >= p.c.dim) return;
        T *dst = (T *)p.a.out + (size_t)(start + i) * p.a.out_ld + (size_t)(h * p.group + row - i * p.group) * p.c.dim + d;
        const float f = l != 0.0f ? 1.0f / l : 0.0f;
        store_f32(dst, v.x * f);
        store_f32(dst + 1, v.y * f);
        store_f32(dst + 2, v.z * f);
        store_f32(dst + 3, v.w * f);
    }
};

// A warp's share of a piece again, all of it by far_values(): q4_0 and bf16 results.
template <typename T, int NG, int NT>
__device__ __noinline__ void far_tiles(const AttendArgs &p, uint8_t *smem, int r, int h, int rt, Queries rq, int a, int b) {
    Worker<T, 0, NG, NT> w(p, smem);
    w.template tiles<true>(r, h, rt, rq, a, b);
    w.dump();
}

struct Request : Queries { int lo, tiles, rts; };                 // cache tiles [lo, lo + tiles), row tiles

__device__ __forceinline__ Request request_of(const AttendArgs &p, int r, int nr) {
    Request q;
    (Queries &)q = queries_of(p.a, r);
    const int lo = p.a.window && q.at > 0 ? max(0, q.at - p.a.window + 1) : 0;
    q.lo = lo / kKvTile;
    q.tiles = max(1, (q.kv + kKvTile - 1) / kKvTile - q.lo);     // one at least: a request whose queries see nothing has rows to write
    q.rts = (q.nq * p.group + nr - 1) / nr;
    return q;
}

template <int kWarps> __device__ long long block_sum_scan(long long v, long long *ws, long long *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    for (int o = 1; o < 32; o <<= 1) {
        const long long u = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += u;
    }
    if (lane == 31) ws[warp] = v;
    __syncthreads();
    long long all = 0;
    for (int k = 0; k < kWarps; k++) {
        if (k < warp) v += ws[k];
        all += ws[k];
    }
    *total = all;
    __syncthreads();
    return v;
}

// Bound: instructions beside memory. 64 requests to 8192 tokens, 32 heads to 8 of 128, bf16, q4_0: 107 us for 403 MB, 3.8 TB/s (the
// same loads without the arithmetic took 75 us, the arithmetic on one tile over and over 99, before it had the codes' exact halves and settle());
// one request of 250001, 16 heads to 2: 34.6 us for 72 MB, of which 19 at the rate above and the rest the fixed chain of shares and join.
template <typename T, int MX, int NG, int NT>
__global__ void __launch_bounds__(32 * warps_of(NG, NT), kCtas) attend_kernel(const __grid_constant__ AttendArgs p) {
    typedef Worker<T, MX, NG, NT> W;
    constexpr int kWarps = W::kWarps, kThreads = W::kThreads;
    extern __shared__ __align__(16) uint8_t smem[];
    W w(p, smem);
    const int n_req = p.a.n_req, heads = p.c.n_kv;
    asm volatile("griddepcontrol.wait;" ::: "memory");                      // what ran before on the stream is done and visible
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");          // the join's CTAs take this one's place as it ends, and wait for all
    // All segments' cache tiles in one line, request by request, head by head, row tile by row tile: a worker's share is [u0, u1).
    // Not split, the line is of segments (the same number for each request), and a worker takes every gridDim.x-th.
    __shared__ long long ws[kWarps];
    __shared__ long long found_at;
    __shared__ int found;
    const int per_req = heads * p.row_tiles;
    long long share = 1, u0 = blockIdx.x, u1 = (long long)n_req * per_req, at = 0;
    int r = 0;
    if (p.split) {
        long long total = 0;
        for (int c = 0; c < n_req; c += kThreads) {
            const int i = c + threadIdx.x;
            long long n = 0, sum;
            if (i < n_req) {
                const Request q = request_of(p, i, W::NR);
                n = (long long)q.tiles * q.rts * heads;
            }
            block_sum_scan<W::kWarps>(n, ws, &sum);
            total += sum;
        }
        share = (total + gridDim.x - 1) / gridDim.x;
        share = (share + 2 * kWarps - 1) / (2 * kWarps) * (2 * kWarps);
        u0 = share * blockIdx.x;
        u1 = min(u0 + share, total);
        long long base = 0;
        for (int c = 0; c < n_req && u0 < u1; c += kThreads) {
            const int i = c + threadIdx.x;
            long long n = 0, sum;
            if (i < n_req) {
                const Request q = request_of(p, i, W::NR);
                n = (long long)q.tiles * q.rts * heads;
            }
            const long long upto = base + block_sum_scan<W::kWarps>(n, ws, &sum);
            if (upto - n <= u0 && u0 < upto) {
                found = i;
                found_at = upto - n;
            }
            base += sum;
            if (u0 < base) break;
        }
        __syncthreads();
        if (u0 < u1) {
            r = found;
            at = found_at;
        }
    }
    int4 desc = make_int4(-1, 0, 0, 0), desc2 = make_int4(0, 0, 0, 0);
    while (u0 < u1) {
        if (!p.split) {
            r = (int)(u0 / per_req);
            at = (long long)r * per_req;
        }
        const Request q = request_of(p, r, W::NR);
        int x, off = 0, len = q.tiles, rts = p.row_tiles;
        if (p.split) {
            const long long n = (long long)q.tiles * q.rts * heads;
            if (u0 >= at + n) {
                at += n;
                r++;
                continue;
            }
            x = (int)((u0 - at) / q.tiles);
            off = (int)(u0 - at - (long long)x * q.tiles);
            len = (int)min((long long)(q.tiles - off), u1 - u0);
            rts = q.rts;
        } else {
            x = (int)(u0 - at);
        }
        const int h = x / rts, rt = x - h * rts;
        if (rt < q.rts) {
            const int last = q.at + min((rt * W::NR + W::NR - 1) / p.group, q.nq - 1), top = last >= 0 ? last / kKvTile + 1 : 0;
            const bool begins = off == 0, ends = off + len == q.tiles;
            w.run(r, h, rt, q, q.lo + off, min(q.lo + off + len, top));
            w.finish(q.start, q.nq, h, rt, begins && ends ? nullptr : p.part + ((size_t)blockIdx.x * 2 + (begins ? 1 : 0)) * W::NR * (W::DP + 4));
            if (!begins && ends) {
                desc = make_int4((int)((u0 - off) / share), h, rt, 0);
                desc2 = make_int4(q.start, q.nq, 0, 0);
            }
        }
        u0 += p.split ? len : gridDim.x;
    }
    if (p.split && threadIdx.x == 0) {
        p.desc[2 * blockIdx.x] = desc;
        p.desc[2 * blockIdx.x + 1] = desc2;
    }
}

// The pieces of the segments that several workers shared, joined: CTA (w, y) does `rows` rows of the segment that ends
// in worker w. Its threads are [part][row][4 dims]: with few rows they take the pieces apart as well.
constexpr int kJoinThreads = 512;

template <typename T, int MX, int NG, int NT>
__global__ void __launch_bounds__(kJoinThreads) join_kernel(const __grid_constant__ AttendArgs p, int rows) {
    typedef Worker<T, MX, NG, NT> W;
    constexpr int LD = W::DP + 4, SIZE = W::NR * LD, PER = W::DP / 4;
    __shared__ float4 sv[kJoinThreads];
    __shared__ float2 sml[kJoinThreads];
    asm volatile("griddepcontrol.wait;" ::: "memory");                      // the workers are done and their pieces visible
    const int4 d = p.desc[2 * blockIdx.x], d2 = p.desc[2 * blockIdx.x + 1];
    if (d.x < 0) return;
    const int items = rows * PER, parts = max(1, kJoinThreads / items), n = blockIdx.x - d.x + 1;
    for (int base = 0; base < items; base += kJoinThreads) {                 // one turn where parts > 1
        const int it = parts > 1 ? threadIdx.x % items : base + threadIdx.x, part = parts > 1 ? threadIdx.x / items : 0;
        const int row = blockIdx.y * rows + it / PER, at = it % PER * 4;
        const bool on = it < items && part < parts;
        auto piece = [&](int k) { return p.part + ((size_t)(d.x + k) * 2 + (k == 0 ? 1 : 0)) * SIZE + (size_t)row * LD; };
        float m = kFloor, l = 0.0f;
        float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        if (on) {
            for (int k = part; k < n; k += 4 * parts) {                      // four pieces' loads at a time
                float2 ml[4];
                float4 x[4];
                float to = m;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    ml[i] = make_float2(kFloor, 0.0f);
                    x[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
                    if (k + i * parts < n) {
                        const float *from = piece(k + i * parts);
                        ml[i] = *(const float2 *)(from + W::DP);
                        x[i] = *(const float4 *)(from + at);
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; i++) to = fmaxf(to, ml[i].x);
                float f = ex2(m - to);
                m = to;
                l *= f;
                v.x *= f; v.y *= f; v.z *= f; v.w *= f;
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    f = ex2(ml[i].x - m);
                    l = fmaf(ml[i].y, f, l);
                    v.x = fmaf(x[i].x, f, v.x); v.y = fmaf(x[i].y, f, v.y); v.z = fmaf(x[i].z, f, v.z); v.w = fmaf(x[i].w, f, v.w);
                }
            }
        }
        if (parts > 1) {
            sv[threadIdx.x] = v;
            sml[threadIdx.x] = make_float2(m, l);
            __syncthreads();
            if (on && part == 0) {
                float top = m;
                for (int k = 1; k < parts; k++) top = fmaxf(top, sml[k * items + it].x);
                float f = ex2(m - top);
                l *= f;
                v.x *= f; v.y *= f; v.z *= f; v.w *= f;
                for (int k = 1; k < parts; k++) {
                    const float2 ml = sml[k * items + it];
                    const float4 x = sv[k * items + it];
                    f = ex2(ml.x - top);
                    l = fmaf(ml.y, f, l);
                    v.x = fmaf(x.x, f, v.x); v.y = fmaf(x.y, f, v.y); v.z = fmaf(x.z, f, v.z); v.w = fmaf(x.w, f, v.w);
                }
            }
        }
        if (on && part == 0) {
            W w(p, nullptr);
            w.put(d2.x, d2.y, d.y, d.z, row, at, v, l);
        }
    }
}

// Cached tokens from which the line is cut into even shares, whose pieces a second kernel joins. One token each, 32 heads to 8 of
// 128, bf16, alone on the GPU: 1 request of 768 tokens 19.5 us cut and 15.3 whole, of 1024 19.5 and 16.4, of 2048 19.5 and 22.9; f32 of 1024
// 21.5 and 22.5. Longer contexts, and those of uneven lengths, gain more the longer they are: a request of 100000 takes 48 us.
constexpr int kSplitFrom = 1024;

// Blocks of 8 rows that share a tile's codes, 1 or 2. Two take 5/3 of one's time and fewer warps fit an SM, so they are for rows that
// fill them, and work enough. Measured, one and two, 32 heads to 8 of 128, f32: 1024 rows of one request over 4096 tokens
// 241 and 201 us; 16 rows of 16 requests over 2000 (16000 tiles) 53 and 49, of 8 requests 37 and 39; 20 rows of 32 requests over 1000 71 and 82.
// With 16 heads to 4 of 96: 16 rows of 8 requests over 8192 (16400 tiles) 45 and 47, over 2000 27 and 35.
int row_blocks(const l3m_kv4 *c, const l3m_kv4_attend *a) {
    const long long rows = (long long)a->max_q * (a->n_heads / c->n_kv_heads), one = (rows + 7) / 8, two = (rows + 15) / 16;
    const double span = a->window ? std::min((double)a->max_kv, (double)a->window + a->max_q) : (double)a->max_kv;
    const double tiles = (double)a->n_req * c->n_kv_heads * two * (span / kKvTile);
    return 3 * one > 5 * two && tiles >= 20000 && (c->head_dim + 31) / 32 <= 4 ? 2 : 1;
}

size_t part_floats(int nr, int ng) { return (size_t)2 * nr * (32 * ng + 4); }

int sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) return 148;
    return std::min(sms, kMaxSms);
}

template <typename T, int MX, int NG, int NT>
cudaError_t launch(AttendArgs p, cudaStream_t s) {
    typedef Worker<T, MX, NG, NT> W;
    cudaError_t e = cudaFuncSetAttribute(attend_kernel<T, MX, NG, NT>, cudaFuncAttributeMaxDynamicSharedMemorySize, W::SMEM);
    if (e != cudaSuccess) return e;
    const int workers = sm_count() * kCtas;
    p.row_tiles = (int)(((long long)p.a.max_q * p.group + W::NR - 1) / W::NR);
    p.split = p.a.max_kv > kSplitFrom;
    p.desc = (int4 *)p.a.scratch;
    p.part = (float *)((char *)p.a.scratch + (size_t)kMaxSms * kCtas * 2 * sizeof(int4));
    const long long segs = (long long)p.a.n_req * p.c.n_kv * p.row_tiles;
    const int grid = p.split ? workers : (int)std::min<long long>(segs, 1 << 20);
    // Both launches are programmatic: their CTAs may come up while what precedes them drains, and wait for it.
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(W::kThreads);
    cfg.dynamicSmemBytes = W::SMEM;
    cfg.stream = s;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    e = cudaLaunchKernelEx(&cfg, attend_kernel<T, MX, NG, NT>, p);
    if (e != cudaSuccess || !p.split) return e;
    const int rows = workers > 8 * segs ? 1 : W::NR;                         // a row per CTA where a segment has many pieces
    cfg.gridDim = dim3(workers, W::NR / rows);
    cfg.blockDim = dim3(kJoinThreads);
    cfg.dynamicSmemBytes = 0;
    return cudaLaunchKernelEx(&cfg, join_kernel<T, MX, NG, NT>, p, rows);
}

template <typename T, int MX, int NT>
cudaError_t by_blocks(const AttendArgs &p, cudaStream_t s) {
    switch (p.c.ng) {
    case 1: return launch<T, MX, 1, NT>(p, s);
    case 2: return launch<T, MX, 2, NT>(p, s);
    case 3: return launch<T, MX, 3, NT>(p, s);
    case 4: return launch<T, MX, 4, NT>(p, s);
    default: break;
    }
    if constexpr (NT == 1) {
        switch (p.c.ng) {
        case 5: return launch<T, MX, 5, 1>(p, s);
        case 6: return launch<T, MX, 6, 1>(p, s);
        case 7: return launch<T, MX, 7, 1>(p, s);
        default: return launch<T, MX, 8, 1>(p, s);
        }
    }
    return cudaErrorInvalidValue;
}

const char *attend_error(const l3m_kv4 *c, const l3m_kv4_attend *a) {
    if (const char *why = kv4_shape_error(c)) return why;
    if (!a) return "arguments are required";
    if (a->dtype != L3M_DT_F32 && a->dtype != L3M_DT_BF16) return "dtype must be f32 or bf16";
    if (a->n_heads < 1 || a->n_heads > 65535 || a->n_heads % c->n_kv_heads) return "n_heads must be a positive multiple of n_kv_heads";
    if (a->n_req < 0 || a->max_blocks < 0 || a->max_q < 0 || a->max_kv < 0 || a->window < 0 || a->max_rows < 0) return "a count is negative";
    if ((int64_t)a->max_q * a->n_heads > 1 << 30) return "max_q * n_heads must be at most 2^30";
    if (a->max_kv > (int64_t)a->max_blocks * c->page) return "max_kv must not exceed max_blocks * page";
    return nullptr;
}

}  // namespace

extern "C" {

L3M_API size_t l3m_kv4_attend_scratch(const l3m_kv4 *cache, const l3m_kv4_attend *a) {
    if (attend_error(cache, a)) return 0;
    if (a->max_kv <= kSplitFrom || prompt_fits(cache, a)) return 16;
    const int ng = (cache->head_dim + kKvBlock - 1) / kKvBlock, nt = row_blocks(cache, a);
    return (size_t)kMaxSms * kCtas * (2 * sizeof(int4) + part_floats(8 * nt, ng) * sizeof(float));
}

L3M_API int l3m_kv4_attend_dev(const l3m_kv4 *cache, const l3m_kv4_attend *a, void *stream) {
    const char *me = "l3m_kv4_attend_dev";
    if (const char *why = attend_error(cache, a)) return refuse(me, why);
    if (const char *why = kv4_error(cache)) return refuse(me, why);
    if (!(std::fabs(a->scale) < 0x1p127f)) return refuse(me, "scale must be finite and below 2^127");
    if (!a->n_req || !a->max_q) return 0;
    if (!a->q || !a->out || !a->q_start || !a->kv_len || (a->max_blocks && !a->tables)) return refuse(me, "a pointer is missing");
    const int64_t width = (int64_t)a->n_heads * cache->head_dim;
    if (a->q_ld < width || a->out_ld < width) return refuse(me, "a token stride is smaller than its heads");
    if (((uintptr_t)a->q | (uintptr_t)a->out) & (a->dtype == L3M_DT_F32 ? 3 : 1) || ((uintptr_t)a->q_start | (uintptr_t)a->kv_len | (uintptr_t)a->tables | (uintptr_t)a->status) & 3)
        return refuse(me, "a pointer is not aligned to its type");
    if (!a->scratch || a->scratch_bytes < l3m_kv4_attend_scratch(cache, a) || ((uintptr_t)a->scratch & 15)) return refuse(me, "scratch is too small or not 16-byte aligned");
    l3m_kv4_attend b = *a;
    if (b.window >= b.max_kv) b.window = 0;                                  // it leaves nothing out
    AttendArgs p = {b, kv4_dev(cache), a->n_heads / cache->n_kv_heads, 0, 0, nullptr, nullptr};
    const int mx = cache->dtype == L3M_DT_MXFP4, two = row_blocks(cache, a) == 2;
    const cudaStream_t s = (cudaStream_t)stream;
    cudaError_t e;
    if (prompt_fits(cache, a)) {
        e = prompt_attend(cache, &b, s);
    } else if (a->dtype == L3M_DT_F32) {
        if (mx) e = two ? by_blocks<float, 1, 2>(p, s) : by_blocks<float, 1, 1>(p, s);
        else e = two ? by_blocks<float, 0, 2>(p, s) : by_blocks<float, 0, 1>(p, s);
    } else {
        if (mx) e = two ? by_blocks<__nv_bfloat16, 1, 2>(p, s) : by_blocks<__nv_bfloat16, 1, 1>(p, s);
        else e = two ? by_blocks<__nv_bfloat16, 0, 2>(p, s) : by_blocks<__nv_bfloat16, 0, 1>(p, s);
    }
    return e == cudaSuccess ? 0 : l3m_error_cuda(e, me);
}

}  // extern "C"
