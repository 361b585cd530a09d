// The paged 4-bit key/value cache: a step's bookkeeping (l3m_kv4_plan_dev), the pass that norms,
// rotates and stores a step's queries, keys and values (l3m_qkv_rope_dev), and the read-back
// (l3m_kv4_load_dev). Contracts in include/l3m_kernels.h, layout in kv4.cuh.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <algorithm>
#include <cfloat>
#include <cmath>
#include <cstdio>
#include <type_traits>
#include "kv4.cuh"

using namespace l3m;

extern "C" int l3m_error_msg(const char *msg);
extern "C" int l3m_error_cuda(int e, const char *what);

namespace {

int refuse(const char *entry, const char *why) {
    char msg[200];
    snprintf(msg, sizeof msg, "%s: %s", entry, why);
    return l3m_error_msg(msg);
}

int launched(cudaError_t e, const char *entry) {
    return e == cudaSuccess ? 0 : l3m_error_cuda(e, entry);
}

// ---- plan

constexpr int kPlanThreads = 1024;
constexpr int kPlanMaxReq = 16384;
constexpr size_t plan_smem(int n_req) { return (size_t)3 * (n_req + 1) * 4 + n_req; }

struct PlanArgs {
    l3m_kv4_plan a;
};

struct Sums { long long gone, rows, pages; };          // pages returned, rows of q, pages wanted

__device__ __forceinline__ Sums add(const Sums &a, const Sums &b) { return {a.gone + b.gone, a.rows + b.rows, a.pages + b.pages}; }

// Inclusive sums over the block; `total` gets the block's. ws: one entry per warp, free again when this returns.
__device__ Sums block_scan(Sums v, Sums *ws, Sums *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const Sums u = {__shfl_up_sync(0xffffffffu, v.gone, o), __shfl_up_sync(0xffffffffu, v.rows, o), __shfl_up_sync(0xffffffffu, v.pages, o)};
        if (lane >= o) v = add(v, u);
    }
    if (lane == 31) ws[warp] = v;
    __syncthreads();
    Sums all = {0, 0, 0}, before = {0, 0, 0};
    for (int k = 0; k < warps; k++) {
        if (k == warp) before = all;
        all = add(all, ws[k]);
    }
    *total = all;
    __syncthreads();
    return add(v, before);
}

// The last index i of sorted a[0..n) with a[i] <= x (a[0] <= x is the caller's promise).
__device__ int last_not_above(const int *a, int n, int x) {
    int lo = 0, hi = n;
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (a[mid] <= x) lo = mid;
        else hi = mid;
    }
    return lo;
}

__device__ __forceinline__ bool bad_lengths(const l3m_kv4_plan &a, long long kv, long long count) {
    return kv < 0 || (kv + count + a.page - 1) / a.page > a.max_blocks || kv + count + a.page > 0x7fffffff;
}

// Every CTA sums the requests' lengths for itself (a few microseconds at most: they fit one SM's
// shared memory), so the CTAs need nothing from each other; then they share out the rows of slot and
// pos, the new table entries and the returned pages. A page that comes off the stack above its old
// top is one that an ended request returns in this call: it is read from that request's table row,
// which nobody writes, not from the stack, which another CTA may still be writing.
// Bound: the chain of a launch, the lengths' loads, the scan and a table read. 24 decoding requests 6.9 us, 512 requests with 128 new prompts
// (2.2 MB written) 11.9 us, of which the rows' binary search is the larger part of the difference.
__global__ void __launch_bounds__(kPlanThreads) plan_kernel(const __grid_constant__ PlanArgs p) {
    const l3m_kv4_plan &a = p.a;
    extern __shared__ int sh[];
    const int n = a.n_req;
    int *gone = sh, *used = sh + (n + 1), *start = sh + 2 * (n + 1);      // exclusive sums: pages returned, pages taken, rows
    uint8_t *ok = (uint8_t *)(sh + 3 * (n + 1));
    __shared__ Sums ws[32];
    __shared__ int left_s;
    const int tid = threadIdx.x;
    int status = 0;
    asm volatile("griddepcontrol.wait;" ::: "memory");                      // what ran before on the stream is done and visible

    const int free0 = *a.n_free;
    const int old_top = min(max(free0, 0), a.n_pages);
    if (free0 != old_top) status |= L3M_KV4_BAD_LENGTH;

    // Running sums over the requests of what ended ones return and of what the others bring and want.
    Sums base = {0, 0, 0};
    for (int c = 0; c < n; c += blockDim.x) {
        const int r = c + tid;
        Sums v = {0, 0, 0}, sum;
        if (r < n) {
            const long long kv = a.kv_len[r], fresh = a.new_len[r], count = fresh > 0 ? fresh : 0;
            const long long held = (kv + a.page - 1) / a.page, after = (kv + count + a.page - 1) / a.page;
            if (fresh < 0 && kv >= 0 && held <= a.max_blocks) v.gone = held;
            v.rows = count;
            if (!bad_lengths(a, kv, count)) v.pages = after - held;
        }
        const Sums upto = add(base, block_scan(v, ws, &sum));
        if (r < n) {
            gone[r] = (int)min(upto.gone - v.gone, (long long)a.n_pages);
            start[r] = (int)min(upto.rows - v.rows, 0x7fffffffLL);
            used[r] = (int)min(upto.pages - v.pages, 0x7fffffffLL);
        }
        base = add(base, sum);
    }
    if (base.gone > a.n_pages - old_top) {                                // more pages than the pool has: the excess is dropped
        status |= L3M_KV4_BAD_LENGTH;
        base.gone = a.n_pages - old_top;
    }
    const int n_gone = (int)base.gone, top = old_top + n_gone;
    if (tid == 0) {
        gone[n] = n_gone;
        start[n] = (int)min(base.rows, 0x7fffffffLL);
        used[n] = (int)min(base.pages, 0x7fffffffLL);
        left_s = top;
        if (blockIdx.x == 0) a.q_start[0] = 0;
    }
    __syncthreads();
    for (int r = tid; r < n; r += blockDim.x) {
        const long long kv = a.kv_len[r], fresh = a.new_len[r], count = fresh > 0 ? fresh : 0;
        const bool bad = bad_lengths(a, kv, count);
        const int pages_upto = used[r + 1], rows_upto = start[r + 1];
        const long long need = bad ? 0 : (kv + count + a.page - 1) / a.page - (kv + a.page - 1) / a.page;
        const bool pages_ok = need == 0 || pages_upto <= top, rows_ok = rows_upto <= a.max_tokens;
        const bool served = !bad && fresh >= 0 && pages_ok && rows_ok;
        if (bad) status |= L3M_KV4_BAD_LENGTH;
        if (!pages_ok) status |= L3M_KV4_NO_PAGES;
        if (count && !rows_ok) status |= L3M_KV4_NO_ROOM;
        ok[r] = served;
        if (blockIdx.x == 0) {
            a.q_start[r + 1] = rows_upto;
            a.kv_total[r] = served ? (int)(kv + count) : 0;
        }
        if (served && need) atomicMin(&left_s, top - pages_upto);
    }
    __syncthreads();
    if (blockIdx.x == 0) {
        if (tid == 0) *a.n_free_out = left_s;
        if (status && a.status) atomicOr((int *)a.status, status);
    }
    const int taken = top - left_s;
    const int step = gridDim.x * blockDim.x, first = blockIdx.x * blockDim.x + tid;
    auto returned = [&](int i) {                                          // the i-th returned page
        const int r = last_not_above(gone, n, i);
        return a.tables[(size_t)r * a.max_blocks + (i - gone[r])];
    };
    auto popped = [&](int i) {                                            // the i-th page off the stack
        const int at = top - 1 - i;
        return at < old_top ? a.free_pages[at] : returned(at - old_top);
    };
    for (int i = first; i < n_gone; i += step) a.free_pages[old_top + i] = returned(i);
    for (int i = first; i < taken; i += step) {
        const int r = last_not_above(used, n, i);
        if (!ok[r]) continue;
        const int block = (a.kv_len[r] + a.page - 1) / a.page + (i - used[r]);
        a.tables[(size_t)r * a.max_blocks + block] = popped(i);
    }
    const int total = min(start[n], a.max_tokens);
    for (int t = first; t < a.max_tokens; t += step) {
        int pos = -1, slot = -1;
        if (t < total) {
            const int r = last_not_above(start, n, t);
            if (ok[r]) {
                const int kv = a.kv_len[r], held = (kv + a.page - 1) / a.page;
                pos = kv + (t - start[r]);
                const int block = pos / a.page;
                const int id = block < held ? a.tables[(size_t)r * a.max_blocks + block] : popped(used[r] + block - held);
                if (id >= 0 && id < a.n_pages) slot = id * a.page + (pos - block * a.page);
                else if (a.status) atomicOr((int *)a.status, L3M_KV4_BAD_PAGE);
            }
        }
        a.pos[t] = pos;
        a.slot[t] = slot;
    }
}

// ---- qkv

constexpr int kQkvThreads = 256;

__device__ __forceinline__ float to_f32(float x) { return x; }
__device__ __forceinline__ float to_f32(__nv_bfloat16 x) { return __bfloat162float(x); }

// 8 values at p as they lie in memory: one or two 16-byte accesses where every row starts 16-byte aligned (VEC), else one by one.
template <typename T> struct Raw8;
template <> struct Raw8<float> {
    float4 a, b;
    template <bool VEC> __device__ __forceinline__ void load(const float *p) {
        if (VEC) {
            a = ((const float4 *)p)[0];
            b = ((const float4 *)p)[1];
        } else {
            a = make_float4(p[0], p[1], p[2], p[3]);
            b = make_float4(p[4], p[5], p[6], p[7]);
        }
    }
    __device__ __forceinline__ void zero() { a = b = make_float4(0.0f, 0.0f, 0.0f, 0.0f); }
    __device__ __forceinline__ void get(float *x) const {
        x[0] = a.x; x[1] = a.y; x[2] = a.z; x[3] = a.w;
        x[4] = b.x; x[5] = b.y; x[6] = b.z; x[7] = b.w;
    }
};
template <> struct Raw8<__nv_bfloat16> {
    uint32_t w[4];
    template <bool VEC> __device__ __forceinline__ void load(const __nv_bfloat16 *p) {
        if (VEC) {
            const uint4 v = *(const uint4 *)p;
            w[0] = v.x; w[1] = v.y; w[2] = v.z; w[3] = v.w;
        } else {
            const uint16_t *h = (const uint16_t *)p;
#pragma unroll
            for (int e = 0; e < 4; e++) w[e] = h[2 * e] | (uint32_t)h[2 * e + 1] << 16;
        }
    }
    __device__ __forceinline__ void zero() { w[0] = w[1] = w[2] = w[3] = 0; }
    __device__ __forceinline__ void get(float *x) const {
#pragma unroll
        for (int e = 0; e < 4; e++) {
            x[2 * e] = __uint_as_float(w[e] << 16);
            x[2 * e + 1] = __uint_as_float(w[e] & 0xffff0000u);
        }
    }
};
template <bool VEC> __device__ __forceinline__ void store8(float *p, const float *x, float f) {
    if (VEC) {
        ((float4 *)p)[0] = make_float4(x[0] * f, x[1] * f, x[2] * f, x[3] * f);
        ((float4 *)p)[1] = make_float4(x[4] * f, x[5] * f, x[6] * f, x[7] * f);
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = x[e] * f;
    }
}
template <bool VEC> __device__ __forceinline__ void store8(__nv_bfloat16 *p, const float *x, float f) {
    if (VEC) {
        __nv_bfloat162 h[4];
#pragma unroll
        for (int e = 0; e < 4; e++) h[e] = __floats2bfloat162_rn(x[2 * e] * f, x[2 * e + 1] * f);
        *(uint4 *)p = *(const uint4 *)h;
    } else {
#pragma unroll
        for (int e = 0; e < 8; e++) p[e] = __float2bfloat16_rn(x[e] * f);
    }
}

struct QkvArgs {
    l3m_qkv a;
    Kv4Dev c;
    int store, mx;
    int q_groups, k_groups, groups;       // a token's row groups (one warp's rows at a time): queries, keys, all
    int chunks, per_chunk;                // warps per token and the groups each takes
};

__device__ __forceinline__ double finite(double x) { return x != x ? 0.0 : isinf(x) ? copysign((double)FLT_MAX, x) : x; }
// A mean square, eps included, whose square root 32 bits have: sums of squares lose nothing above and do not overflow below.
__device__ __forceinline__ bool sound(float mean) { return mean > 0x1p-100f && mean < 0x1p100f; }

// What a lane stores of its row: the codes of its 8 values and its block's scale bits.
struct Held { unsigned codes, scale; };

// Two values as e2m1, rounded to nearest (ties to even), at most 6: the first in the low nibble.
__device__ __forceinline__ unsigned e2m1_codes(float lo, float hi) {
    uint32_t d;
    asm("{ .reg .b8 c, z;\n .reg .b16 w;\n mov.b16 w, 0;\n mov.b16 {z, z}, w;\n cvt.rn.satfinite.e2m1x2.f32 c, %2, %1;\n mov.b32 %0, {c, z, z, z}; }" : "=r"(d) : "f"(lo), "f"(hi));
    return d;
}
// Codes of -0 made 0.
__device__ __forceinline__ unsigned no_minus_zero(unsigned w) {
    const unsigned m = w & 0x77777777u, some = (m | m >> 1 | m >> 2) & 0x11111111u;
    return m | (w & some << 3);
}

// A row (a head of a token) is held by LPR lanes, 8 contiguous dims each, so 4 lanes hold a block; a group of 32 / LPR rows
// of one kind is a warp's work at a time. A warp takes a run of one token's groups (queries, then keys, then
// values): position, rotation and slot are read once, and the next group's rows are under way while one is worked on.
//
// Codes and scales have to be those of exact arithmetic, but a value next to a border between two codes may land
// on either side of it in 32 bits. So u (the normed, rotated value before the row's factor, which
// q4_0's codes do not depend on) is computed in 32 bits with a bound on its error, each decision with its
// distance from the border, and where the distance is within the bound the row is redone in 64 bits (about 1% of the rows).
enum { kQuery, kKey, kValue };

// Where a token's rows go: its tile of head 0 (null: nowhere) and its row there.
struct Place {
    uint8_t *tile;
    int tr;
};

// One lane's share of a row of head h: t of block j.
template <int KIND> __device__ __forceinline__ void put_row(const QkvArgs &p, const Place &to, int h, int lane, const Held &held) {
    const int j = lane >> 2, t = lane & 3, ng = p.c.ng;
    uint8_t *at = to.tile + (size_t)h * p.c.tiles * p.c.tile_bytes;
    if (KIND == kKey) {
        *(uint32_t *)(at + to.tr * 16 * ng + (t * ng + j) * 4) = held.codes;
    } else {
        uint16_t *v = (uint16_t *)(at + 256 * ng + to.tr * 16 * ng);
        v[2 * t * ng + j] = (uint16_t)held.codes;
        v[(2 * t + 1) * ng + j] = (uint16_t)(held.codes >> 16);
    }
    if (t == 0) {
        uint8_t *s = at + (KIND == kKey ? p.c.k_scales() : p.c.v_scales()) + (to.tr * ng + j) * p.c.sb;
        if (p.mx) *s = (uint8_t)held.scale;
        else *(uint16_t *)s = (uint16_t)held.scale;
    }
}

// Group g by the definition, in 64 bits: for rows whose 32-bit values lie too near a border, or whose squares leave 32 bits' range.
template <typename T, int LPR, int ROPE, int KIND>
__device__ __noinline__ void exact_rows(const QkvArgs &p, int tok, Place to, const float *turn, int g) {
    const l3m_qkv &a = p.a;
    const int wl = threadIdx.x & 31, lane = wl & (LPR - 1), d0 = lane * 8, h = g * (32 / LPR) + wl / LPR, D = a.head_dim;
    const int rot = KIND != kValue && ROPE ? a.rot_dim : 0, half = rot / 2;
    const bool live = h < (KIND == kQuery ? a.n_heads : a.n_kv_heads), mine = live && d0 < D;
    const T *src = (const T *)(KIND == kQuery ? a.q : KIND == kKey ? a.k : a.v) + (size_t)tok * (KIND == kQuery ? a.q_ld : KIND == kKey ? a.k_ld : a.v_ld) + (size_t)h * D;
    const float *w = KIND == kQuery ? a.q_norm : KIND == kKey ? a.k_norm : nullptr;
    T *out = KIND == kValue ? nullptr : (T *)(KIND == kQuery ? a.q_out : a.k_out);
    double u[8], ss = 0.0, f = 1.0;
#pragma unroll 1
    for (int e = 0; e < 8; e++) {
        const int d = d0 + e;
        double x = mine ? (double)to_f32(src[d]) : 0.0;
        if (w) ss += x * x;
        if (mine && w) x *= (double)w[d];
        if (mine && d < rot) {
            const int md = ROPE == 1 ? d ^ 1 : d < half ? d + half : d - half, i = ROPE == 1 ? d >> 1 : d < half ? d : d - half;
            const bool second = ROPE == 1 ? (d & 1) != 0 : d >= half;
            double m = (double)to_f32(src[md]);
            if (w) m *= (double)w[md];
            const double c = (double)turn[2 * i], s = (double)turn[2 * i + 1];
            x = second ? m * s + x * c : x * c - m * s;
        }
        u[e] = x;
    }
    for (int o = LPR / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
    if (w) f = 1.0 / sqrt(ss / D + (double)a.eps);
    __syncwarp();                                                        // in place: every lane has read its row
    if (KIND != kValue && out && mine) {
        float x[8];
#pragma unroll
        for (int e = 0; e < 8; e++) x[e] = (float)(u[e] * f);
        store8<false>(out + (size_t)tok * (KIND == kQuery ? a.q_out_ld : a.k_out_ld) + (size_t)h * D + d0, x, 1.0f);
    }
    if (KIND == kQuery || !to.tile) return;
    f = finite(f);
    double top = 0.0;
    int at = 0;
#pragma unroll
    for (int e = 0; e < 8; e++) {
        u[e] = finite(u[e]);
        if (fabs(u[e]) > fabs(top)) {
            top = u[e];
            at = e;
        }
    }
    at += (lane & 3) * 8;
    for (int o = 1; o < 4; o <<= 1) {                                   // the first of equals over the block's 4 lanes
        const double ot = __shfl_xor_sync(0xffffffffu, top, o);
        const int oa = __shfl_xor_sync(0xffffffffu, at, o);
        if (fabs(ot) > fabs(top) || (fabs(ot) == fabs(top) && oa < at)) {
            top = ot;
            at = oa;
        }
    }
    Held held = {0, 0};
    const double mag = fabs(top);
    if (!p.mx) {
        // As in quantise(), a candidate and the sign of its fma; within the rounding of the definition's own quotient, that quotient
        const double d = top / -8.0, inv = mag > 0.0 ? 1.0 / d : 0.0;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const double b = rint(fma(u[e], inv, 8.5)), r = fma(fma(b, 0.125, -1.0625), mag, top < 0.0 ? -u[e] : u[e]);
            int code = (int)b - (r <= 0.0 ? 0 : 1);
            if (fabs(r) <= 1e-14 * mag) code = (int)floor(u[e] / d + 8.5);
            held.codes |= (unsigned)min(max(code, 0), 15) << (4 * e);
        }
        held.scale = __half_as_ushort(__float2half_rn(fminf(fmaxf((float)(d * f), -65504.0f), 65504.0f)));
        if (mag == 0.0) held = {0x88888888u, 0};
    } else {
        const double m = mag * f;
        const int e8 = m > 0.0 ? min(max(ilogb(m) + 125, 0), 254) : 0;
        const double inv = ldexp(1.0, 127 - e8);
#pragma unroll
        for (int e = 0; e < 8; e++) {
            const double y = u[e] * f, v = fabs(y) * inv;
            const unsigned code = (v > 0.25) + (v > 0.75) + (v > 1.25) + (v > 1.75) + (v > 2.5) + (v > 3.5) + (v > 5.0);
            held.codes |= (code | (y < 0.0 && code ? 8u : 0u)) << (4 * e);
        }
        held.scale = (unsigned)e8;
    }
    if (live && lane < 4 * p.c.ng) put_row<KIND>(p, to, h, lane, held);
}

template <typename T, int LPR, int ROPE, bool VEC>
struct RowWorker {
    static constexpr int RPW = 32 / LPR;
    static constexpr bool FEW = sizeof(T) == 2;                              // 8 significant bits a value
    const QkvArgs &p;
    float *mate_buf;
    int wl, lane, sub, d0, half, tok;
    bool in, partial;
    int shift, mate_lane;
    float cs[8], sn[8];                   // cos and sin of this lane's dims, sin with the sign of the mate's term
    float turn_max;                       // the largest of them in magnitude: tables may carry a factor
    const float *turn;
    Place to;

    __device__ __forceinline__ RowWorker(const QkvArgs &args, float *buf) : p(args), mate_buf(buf) {
        wl = threadIdx.x & 31;
        lane = wl & (LPR - 1);
        sub = wl / LPR;
        d0 = lane * 8;
        half = ROPE ? p.a.rot_dim / 2 : 0;
        in = d0 < p.a.head_dim;
        partial = ROPE && p.a.rot_dim < p.a.head_dim;
        shift = ROPE == 2 && (half & 7) == 0 ? half >> 3 : 0;                 // halves: the mate's lane is this far away; 0: through shared memory
        mate_lane = (wl & ~(LPR - 1)) + (d0 < half ? lane + shift : d0 < 2 * half ? lane - shift : lane);
    }
    __device__ __forceinline__ void rotation(int pos) {
        turn = ROPE ? p.a.rope_table + (size_t)pos * half * 2 : nullptr;
        if (ROPE) {
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const int d = d0 + e;
                cs[e] = 1.0f;
                sn[e] = 0.0f;
                if (d < 2 * half) {
                    const int i = ROPE == 1 ? d >> 1 : d < half ? d : d - half;
                    const float2 t = *(const float2 *)(turn + 2 * i);
                    cs[e] = t.x;
                    sn[e] = (ROPE == 1 ? e & 1 : d >= half) ? t.y : -t.y;
                }
            }
            turn_max = 0.0f;
            if (p.store) {
#pragma unroll
                for (int e = 0; e < 8; e++) turn_max = fmaxf(turn_max, fmaxf(fabsf(cs[e]), fabsf(sn[e])));
            }
        }
    }

    // Groups [g0, g1) of a kind, 64 at most. Returns which of them are left for exact_rows(): nothing of those is written.
    template <int KIND> __device__ __forceinline__ unsigned long long rows(int g0, int g1) {
        const l3m_qkv &a = p.a;
        const int heads = KIND == kQuery ? a.n_heads : a.n_kv_heads, D = a.head_dim, step = RPW * D;
        int h = g0 * RPW + sub;
        const T *src = (const T *)(KIND == kQuery ? a.q : KIND == kKey ? a.k : a.v) + (size_t)tok * (KIND == kQuery ? a.q_ld : KIND == kKey ? a.k_ld : a.v_ld) + (size_t)h * D + d0;
        T *out = KIND == kValue ? nullptr : (T *)(KIND == kQuery ? a.q_out : a.k_out);
        if (out) out += (size_t)tok * (KIND == kQuery ? a.q_out_ld : a.k_out_ld) + (size_t)h * D + d0;
        const float *w = KIND == kQuery ? a.q_norm : KIND == kKey ? a.k_norm : nullptr;
        float wt[8];
        if (KIND != kValue && w) {
#pragma unroll
            for (int e = 0; e < 8; e++) wt[e] = in ? w[d0 + e] : 0.0f;
        }
        const float inv_d = __fdividef(1.0f, (float)D);
        unsigned long long left = 0;
        Raw8<T> next;
        next.zero();
        if (h < heads && in) next.template load<VEC>(src);
        for (int g = g0; g < g1; g++, h += RPW) {
            const bool live = h < heads;
            float u[8];
            next.get(u);
            src += step;
            if (g + 1 < g1 && h + RPW < heads && in) next.template load<VEC>(src);
            float f = 1.0f, size = 0.0f;                                     // size: the largest |a| + |b| behind a value, times the largest |cos| or |sin|
            bool near = false;
            if (KIND != kValue && w) {
                float ss = 0.0f;
#pragma unroll
                for (int e = 0; e < 8; e++) ss = fmaf(u[e], u[e], ss);
#pragma unroll
                for (int o = LPR / 2; o; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                const float mean = fmaf(ss, inv_d, a.eps);
                near = !sound(mean);
                f = rsqrtf(mean);
#pragma unroll
                for (int e = 0; e < 8; e++) u[e] *= wt[e];
            }
            if (KIND != kValue && ROPE) {
                float m[8];
                if (ROPE == 1) {
#pragma unroll
                    for (int e = 0; e < 8; e++) m[e] = u[e ^ 1];
                } else if (shift) {
#pragma unroll
                    for (int e = 0; e < 8; e++) m[e] = __shfl_sync(0xffffffffu, u[e], mate_lane);
                } else {
                    float *row = mate_buf + (threadIdx.x - lane) * 8;
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 8; e++) row[d0 + e] = u[e];
                    __syncwarp();
#pragma unroll
                    for (int e = 0; e < 8; e++) {
                        const int d = d0 + e;
                        m[e] = d < half ? row[d + half] : d < 2 * half ? row[d - half] : 0.0f;
                    }
                }
                if (partial) {                                               // dims behind rot_dim: no mate, whatever it holds
#pragma unroll
                    for (int e = 0; e < 8; e++) m[e] = d0 + e < a.rot_dim ? m[e] : 0.0f;
                }
#pragma unroll
                for (int e = 0; e < 8; e++) {
                    if (KIND == kKey) size = fmaxf(size, fabsf(u[e]) + fabsf(m[e]));
                    u[e] = fmaf(m[e], sn[e], u[e] * cs[e]);
                }
                if (KIND == kKey) size *= turn_max;
            }
            Held held = {0, 0};
            if (KIND != kQuery && to.tile) {
                bool close;
                held = quantise<KIND>(u, size, f, w, &close);
                near |= close;
            }
            if ((KIND != kValue || to.tile) && __any_sync(0xffffffffu, near && live)) {
                left |= 1ull << (g - g0);
                if (KIND != kValue && out) out += step;
                continue;
            }
            if (KIND != kValue && out) {
                __syncwarp();                                                // in place: every lane has read its row
                if (live && in) store8<VEC>(out, u, f);
                out += step;
            }
            if (KIND != kQuery && to.tile && live && lane < 4 * p.c.ng) put_row<KIND>(p, to, h, lane, held);
        }
        return left;
    }

    // A row's codes and scales; *close: some decision lies within the error's bound of its border. Each code is that of the value moved down
    // by the bound and that of the value moved up: where they agree they are right. Values of 8 bits that no
    // arithmetic has touched lie on a border or 2^-9 from it: a smaller move makes ties go as they should.
    template <int KIND> __device__ __forceinline__ Held quantise(const float *u, float size, float f, const float *w, bool *close) const {
        // The block's extremes; zero keeps a sum of zeros, anything not finite spoils it.
        float hi = u[0], lo = u[0], zero = 0.0f;
#pragma unroll
        for (int e = 0; e < 8; e++) {
            hi = fmaxf(hi, u[e]);
            lo = fminf(lo, u[e]);
            zero = fmaf(u[e], 0.0f, zero);
        }
#pragma unroll
        for (int o = 1; o < 4; o <<= 1) {
            hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
            lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
            if (KIND == kKey && ROPE) size = fmaxf(size, __shfl_xor_sync(0xffffffffu, size, o));
        }
        const float mag = fmaxf(hi, -lo);
        // An upper bound on the error of u: three roundings of (|a| + |b|) max(|cos|, |sin|) at 2^-24 (the weights, a product, the sum); one of u (the
        // weight) without a rotation.
        const bool exact = KIND == kValue || (!w && !ROPE);
        const float err = exact ? 0.0f : ROPE ? size * 0x1p-22f : mag * 0x1p-23f;
        bool again = !(zero == 0.0f) || (mag < 0x1p-100f && (mag > 0.0f || err > 0.0f)) || mag > 0x1p120f;
        Held held = {0, 0};
        if (!p.mx) {
            float top = hi >= -lo ? hi : lo;
            bool even = mag > 0.0f && fabsf(hi + lo) <= 2.0f * err;          // opposite signs of one size: the sign of the first decides
            if (exact && __any_sync(0xffffffffu, even)) {
                int first = 1 << 20;
#pragma unroll
                for (int e = 7; e >= 0; e--) first = fabsf(u[e]) == mag ? (lane & 3) * 16 + 2 * e + (u[e] < 0.0f) : first;
                first = min(first, __shfl_xor_sync(0xffffffffu, first, 1));
                first = min(first, __shfl_xor_sync(0xffffffffu, first, 2));
                top = even ? (first & 1 ? -mag : mag) : top;
                even = false;
            }
            again |= even;
            // code = the integer part of t = u / d + 8.5, 15 at most; rounded down into the low bits of t + 3 * 2^22
            const float inv = __fdividef(-8.0f, top), per = __fdividef(16.5f * err, mag), tau = exact && FEW ? 0x1p-12f : per + 0x1p-18f;
            unsigned down = 0, up = 0;
#pragma unroll
            for (int e = 0; e < 8; e++) {
                const float t = fmaf(u[e], inv, 8.5f);
                up += __float_as_uint(__fadd_rd(fminf(t + tau, 15.5f), 12582912.0f)) << (4 * e);
                if (!(exact && FEW)) down += __float_as_uint(__fadd_rd(fminf(t - tau, 15.5f), 12582912.0f)) << (4 * e);
            }
            constexpr unsigned kBase = 0x4b400000u * 0x11111111u;            // the sum of the numbers' other bits
            held.codes = up - kBase;
            if (!(exact && FEW)) again |= up != down;
            const float s = top * -0.125f * f;
            if (exact) {
                held.scale = __half_as_ushort(__float2half_rn(fminf(fmaxf(s, -65504.0f), 65504.0f)));
            } else {
                const float rel = 0x1p-20f + __fdividef(2.0f * err, mag);
                const unsigned short s0 = __half_as_ushort(__float2half_rn(fminf(fmaxf(s * (1.0f - rel), -65504.0f), 65504.0f)));
                const unsigned short s1 = __half_as_ushort(__float2half_rn(fminf(fmaxf(s * (1.0f + rel), -65504.0f), 65504.0f)));
                held.scale = s0;
                again |= s0 != s1;
            }
            if (mag == 0.0f) {
                held = {0x88888888u, 0};
                again = !(zero == 0.0f) || err > 0.0f;
            }
        } else {
            const float m = mag * f, rel = exact ? 0.0f : 0x1p-20f + __fdividef(2.0f * err, mag);
            const unsigned e0 = __float_as_uint(m * (1.0f - rel)) >> 23, e1 = __float_as_uint(m * (1.0f + rel)) >> 23;
            again |= mag > 0.0f && (e0 != e1 || e0 < 20u || e0 > 250u || f > 0x1p17f);   // far from either end, fi below is a normal number
            const float inv = mag > 0.0f ? __uint_as_float((256u - e0) << 23) : 0.0f;   // 2^(127 - e8), e8 = e0 - 2
            const float fi = f * inv, tau = exact ? 0.0f : (3.0f * err + mag * 0x1p-20f) * fi;
            // Rounded to nearest; ties go down because the number has been moved towards zero.
            unsigned down = 0, up = 0;
#pragma unroll
            for (int e = 0; e < 8; e += 2) {
                const float a = u[e] * fi, b = u[e + 1] * fi;
                const float ta = exact ? fabsf(a) * 0x1p-18f : tau, tb = exact ? fabsf(b) * 0x1p-18f : tau;
                const float da = a < 0.0f ? a + ta : a - ta, db = b < 0.0f ? b + tb : b - tb;
                down |= e2m1_codes(da, db) << (4 * e);
                if (!(exact && FEW)) up |= e2m1_codes(a < 0.0f ? a - tau : a + tau, b < 0.0f ? b - tau : b + tau) << (4 * e);
            }
            held.codes = no_minus_zero(down);
            if (!(exact && FEW)) again |= held.codes != no_minus_zero(up);
            held.scale = mag > 0.0f ? e0 - 2 : 0;
            if (mag == 0.0f) again = !(zero == 0.0f) || err > 0.0f;
        }
        *close = again;
        return held;
    }
};

// LPR lanes a row, 8 values a lane, so that a row is one access wide and its sums are shuffles; queries first, then keys, then
// values, the next rows' loads under way. Bound: bytes under way. A warp has one group of rows ahead of it, 512 bytes of bf16 at 128 dims, so the 24
// warps an SM that 80 registers allow have 12 KB, which at 0.8 us of latency is 2.3 TB/s; instructions (norm, rotation, bounds and two roundings of
// each value to codes) take 2.4 issue slots of 4. 8191 tokens of 32 + 8 + 8 heads of 128, bf16 to mxfp4: 76 us for 170 MB, 2.2 TB/s.
// 3 CTAs an SM of 80 registers; with fewer registers the bounds spill.
template <typename T, int LPR, int ROPE, bool VEC>
__global__ void __launch_bounds__(kQkvThreads, 3) qkv_kernel(const __grid_constant__ QkvArgs p) {
    const l3m_qkv &a = p.a;
    __shared__ float mate_buf[ROPE == 2 ? kQkvThreads * 8 : 1];
    RowWorker<T, LPR, ROPE, VEC> w(p, mate_buf);
    asm volatile("griddepcontrol.wait;" ::: "memory");                      // what ran before on the stream is done and visible
    const long long items = (long long)a.n_tokens * p.chunks;
    for (long long item = blockIdx.x * (kQkvThreads / 32) + (threadIdx.x >> 5); item < items; item += (long long)gridDim.x * (kQkvThreads / 32)) {
        const int tok = (int)(item / p.chunks), g0 = (int)(item - (long long)tok * p.chunks) * p.per_chunk, g1 = min(g0 + p.per_chunk, p.groups);
        const int pos = a.pos[tok];
        if (pos < 0) continue;
        if (ROPE && pos >= a.n_pos) {
            if (a.status && w.wl == 0) atomicOr((int *)a.status, L3M_KV4_BAD_POS);
            continue;
        }
        w.tok = tok;
        w.to.tile = nullptr;
        w.to.tr = 0;
        if (p.store) {
            const int slot = a.slot[tok];
            if (slot >= p.c.n_pages * p.c.page) {
                if (a.status && w.wl == 0) atomicOr((int *)a.status, L3M_KV4_BAD_PAGE);
            } else if (slot >= 0) {
                const int page = slot / p.c.page, off = slot - page * p.c.page;
                w.to.tile = p.c.data + p.c.tile_at(page, 0, off / kKvTile);
                w.to.tr = off % kKvTile;
            }
        }
        if (g0 < p.q_groups + p.k_groups) w.rotation(pos);
        for (int g = g0; g < min(g1, p.q_groups); g += 64)
            for (unsigned long long left = w.template rows<kQuery>(g, min(g + 64, min(g1, p.q_groups))); left; left &= left - 1) exact_rows<T, LPR, ROPE, kQuery>(p, tok, w.to, w.turn, g + __ffsll(left) - 1);
        const int k0 = p.q_groups, v0 = p.q_groups + p.k_groups;
        for (int g = max(g0 - k0, 0); g < min(g1, v0) - k0; g += 64)
            for (unsigned long long left = w.template rows<kKey>(g, min(g + 64, min(g1, v0) - k0)); left; left &= left - 1) exact_rows<T, LPR, ROPE, kKey>(p, tok, w.to, w.turn, g + __ffsll(left) - 1);
        for (int g = max(g0 - v0, 0); g < g1 - v0 && w.to.tile; g += 64)
            for (unsigned long long left = w.template rows<kValue>(g, min(g + 64, g1 - v0)); left; left &= left - 1) exact_rows<T, LPR, ROPE, kValue>(p, tok, w.to, nullptr, g + __ffsll(left) - 1);
    }
}

// ---- load

struct LoadArgs {
    Kv4Dev c;
    int mx, n, parts, vec, warps;         // warps per row
    unsigned per_part;                    // 2^32 / parts, rounded up: i / parts = i * per_part >> 32 for the small i here
    void *k, *v;
    const int32_t *slots;
};

__device__ __forceinline__ float code_value(unsigned nib, int mx) {
    if (!mx) return (float)(int)nib - 8.0f;
    const float m = (float)((0xC8643210u >> (4 * (nib & 7))) & 15) * 0.5f;
    return nib & 8 ? -m : m;
}
__device__ __forceinline__ float scale_value(const uint8_t *p, int mx) {
    return mx ? (*p ? __uint_as_float((uint32_t)*p << 23) : __uint_as_float(0x00400000u)) : __half2float(*(const __half *)p);
}

// One warp, or several, per row: the lanes go over its keys' and values' pieces of 8. 8191 rows of 8 heads of 128 to bf16: 20 us,
// 43 MB, bound by its short reads: 4 or 8 bytes of codes and a scale a lane.
template <typename T>
__global__ void __launch_bounds__(256) load_kernel(const __grid_constant__ LoadArgs p) {
    const int lane = threadIdx.x & 31, per = p.c.n_kv * p.parts, ng = p.c.ng;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    const long long w0 = blockIdx.x * 8LL + (threadIdx.x >> 5), row = w0 / p.warps;
    if (row < p.n) {
        const int slot = p.slots[row];
        if (slot < 0 || slot >= p.c.n_pages * p.c.page) return;
        const int page = slot / p.c.page, off = slot - page * p.c.page, tr = off % kKvTile;
        const uint8_t *tile0 = p.c.data + p.c.tile_at(page, 0, off / kKvTile);
        for (int i = (int)(w0 - row * p.warps) * 32 + lane; i < 2 * per; i += 32 * p.warps) {
            const int is_v = i >= per, x = is_v ? i - per : i, head = p.parts == 1 ? x : (int)__umulhi((unsigned)x, p.per_part), c = x - head * p.parts, j = c >> 2, t = c & 3;
            T *out = (T *)(is_v ? p.v : p.k);
            if (!out) continue;
            const uint8_t *tile = tile0 + (size_t)head * p.c.tiles * p.c.tile_bytes;
            const uint8_t *codes = tile + (is_v ? 256 * ng : 0) + tr * 16 * ng;
            uint32_t w;
            if (is_v) w = ((const uint16_t *)codes)[2 * t * ng + j] | (uint32_t)((const uint16_t *)codes)[(2 * t + 1) * ng + j] << 16;
            else w = ((const uint32_t *)codes)[t * ng + j];
            const float s = scale_value(tile + (is_v ? p.c.v_scales() : p.c.k_scales()) + (tr * ng + j) * p.c.sb, p.mx);
            float x8[8];
#pragma unroll
            for (int e = 0; e < 8; e++) x8[e] = code_value(w >> (4 * e) & 15, p.mx);
            T *to = out + ((size_t)row * p.c.n_kv + head) * p.c.dim + c * 8;
            if (p.vec) store8<true>(to, x8, s);
            else store8<false>(to, x8, s);
        }
    }
}

// Launches with the grid allowed up while what precedes it on the stream drains: the kernels here wait for it themselves.
template <typename... P, typename... A>
cudaError_t launch_early(void (*kernel)(P...), int grid, int block, size_t smem, cudaStream_t s, const A &...args) {
    cudaLaunchAttribute early;
    early.id = cudaLaunchAttributeProgrammaticStreamSerialization;
    early.val.programmaticStreamSerializationAllowed = 1;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(grid);
    cfg.blockDim = dim3(block);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = s;
    cfg.attrs = &early;
    cfg.numAttrs = 1;
    return cudaLaunchKernelEx(&cfg, kernel, args...);
}

int sm_count() {
    int dev = 0, sms = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || cudaDeviceGetAttribute(&sms, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || sms <= 0) return 148;
    return sms;
}

}  // namespace

extern "C" {

L3M_API size_t l3m_kv4_page_bytes(int dtype, int n_kv_heads, int head_dim, int page) {
    l3m_kv4 c = {nullptr, dtype, 0, page, n_kv_heads, head_dim};
    if (kv4_shape_error(&c)) return 0;
    const Kv4Dev d = kv4_dev(&c);
    return (size_t)d.tile_bytes * d.tiles * d.n_kv;
}

L3M_API int l3m_kv4_plan_dev(const l3m_kv4_plan *a, void *stream) {
    const char *me = "l3m_kv4_plan_dev";
    if (!a) return refuse(me, "arguments are required");
    if (a->n_req < 0 || a->n_req > kPlanMaxReq) return refuse(me, "n_req must be 0 to 16384");
    if (a->page < kKvTile || a->page > 4096 || a->page % kKvTile) return refuse(me, "page must be a multiple of 16 from 16 to 4096");
    if (a->max_tokens > 1 << 30) return refuse(me, "max_tokens must be at most 2^30");
    if (a->max_blocks < 0 || a->max_tokens < 0 || a->n_pages < 0 || (int64_t)a->n_pages * a->page > 0x7fffffff)
        return refuse(me, "max_blocks, max_tokens and n_pages must not be negative, n_pages * page below 2^31");
    if (!a->n_free || !a->n_free_out || !a->q_start || (a->n_pages && !a->free_pages) || (a->max_tokens && (!a->slot || !a->pos)) ||
        (a->n_req && (!a->kv_len || !a->new_len || !a->kv_total || (a->max_blocks && !a->tables))))
        return refuse(me, "a pointer is missing");
    if (a->n_free == a->n_free_out || (a->n_req && (a->kv_total == a->kv_len || a->kv_total == a->new_len)))
        return refuse(me, "n_free_out must not be n_free, nor kv_total kv_len or new_len");
    if (((uintptr_t)a->kv_len | (uintptr_t)a->new_len | (uintptr_t)a->tables | (uintptr_t)a->free_pages | (uintptr_t)a->n_free | (uintptr_t)a->n_free_out |
         (uintptr_t)a->q_start | (uintptr_t)a->kv_total | (uintptr_t)a->slot | (uintptr_t)a->pos | (uintptr_t)a->status) & 3)
        return refuse(me, "a pointer is not aligned to its type");
    PlanArgs p = {*a};
    // The limit is the function's, not the call's: always the same, so that no other host thread's call lowers it before this one's launch.
    const size_t smem = plan_smem(a->n_req);
    const cudaError_t e = cudaFuncSetAttribute(plan_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, (int)plan_smem(kPlanMaxReq));
    if (e != cudaSuccess) return l3m_error_cuda(e, me);
    const int threads = a->n_req <= 128 && a->max_tokens <= 2048 ? 128 : kPlanThreads;
    const int grid = std::max(1, std::min(sm_count(), (a->max_tokens + threads - 1) / threads));
    return launched(launch_early(plan_kernel, grid, threads, smem, (cudaStream_t)stream, p), me);
}

L3M_API int l3m_qkv_rope_dev(const l3m_kv4 *cache, const l3m_qkv *a, void *stream) {
    const char *me = "l3m_qkv_rope_dev";
    if (!a) return refuse(me, "arguments are required");
    if (a->dtype != L3M_DT_F32 && a->dtype != L3M_DT_BF16) return refuse(me, "dtype must be f32 or bf16");
    if (a->n_tokens < 0 || a->n_heads < 0 || a->n_kv_heads < 0 || a->n_heads > 65535 || a->n_kv_heads > 65535) return refuse(me, "bad token or head counts");
    if (a->head_dim < 8 || a->head_dim > 256 || a->head_dim % 8) return refuse(me, "head_dim must be a multiple of 8 from 8 to 256");
    if (a->rope < 0 || a->rope > 2) return refuse(me, "rope must be 0, 1 or 2");
    if (a->rope && (a->rot_dim < 0 || a->rot_dim % 2 || a->rot_dim > a->head_dim || a->n_pos < 0 || (a->rot_dim && a->n_pos && !a->rope_table)))
        return refuse(me, "the rotation needs an even rot_dim up to head_dim and a table of n_pos rows");
    if (!(a->eps >= 0.0f) || std::isinf(a->eps)) return refuse(me, "eps must be finite and not negative");
    if (cache) {
        if (const char *why = kv4_error(cache)) return refuse(me, why);
        if (cache->n_kv_heads != a->n_kv_heads || cache->head_dim != a->head_dim) return refuse(me, "the cache has another n_kv_heads or head_dim");
        if (a->n_kv_heads && a->n_tokens && (!a->k || !a->v || !a->slot)) return refuse(me, "a cache needs k, v and slot");
    }
    if (!a->n_tokens || !(a->n_heads + a->n_kv_heads)) return 0;
    if (!a->pos) return refuse(me, "pos is required");
    if (a->n_heads && (!a->q || !a->q_out)) return refuse(me, "q and q_out are required");
    if (!cache && a->k_out && !a->k) return refuse(me, "k_out needs k");
    const int64_t qw = (int64_t)a->n_heads * a->head_dim, kw = (int64_t)a->n_kv_heads * a->head_dim;
    const bool with_k = a->n_kv_heads && a->k && (cache || a->k_out), with_v = cache && a->n_kv_heads;
    if ((a->n_heads && (a->q_ld < qw || a->q_out_ld < qw)) || (with_k && (a->k_ld < kw || (a->k_out && a->k_out_ld < kw))) || (with_v && a->v_ld < kw))
        return refuse(me, "a token stride is smaller than its heads");
    const uintptr_t mask = a->dtype == L3M_DT_F32 ? 3 : 1;
    if ((((uintptr_t)a->q | (uintptr_t)a->k | (uintptr_t)a->v | (uintptr_t)a->q_out | (uintptr_t)a->k_out) & mask) ||
        (((uintptr_t)a->q_norm | (uintptr_t)a->k_norm | (uintptr_t)a->rope_table | (uintptr_t)a->pos | (uintptr_t)a->slot | (uintptr_t)a->status) & 3))
        return refuse(me, "a pointer is not aligned to its type");
    if (!a->n_heads && !with_k && !with_v) return 0;
    if (a->rope && ((uintptr_t)a->rope_table & 7)) return refuse(me, "rope_table must be 8-byte aligned");
    // In place a row may take only its own place: with another stride it would take rows that other warps still read.
    if (a->n_tokens > 1 && ((a->n_heads && a->q_out == a->q && a->q_out_ld != a->q_ld) || (with_k && a->k_out == a->k && a->k_out_ld != a->k_ld)))
        return refuse(me, "in place, a result needs its input's token stride");
    QkvArgs p = {*a, {}, with_v, cache && cache->dtype == L3M_DT_MXFP4, 0, 0, 0, 1, 1};
    if (cache) p.c = kv4_dev(cache);
    // 16-byte accesses where every row of every tensor starts on 16 bytes.
    const int per16 = a->dtype == L3M_DT_F32 ? 4 : 8;
    uintptr_t at = 0;
    int64_t ld = 0;
    if (a->n_heads) at |= (uintptr_t)a->q | (uintptr_t)a->q_out, ld |= a->q_ld | a->q_out_ld;
    if (with_k) at |= (uintptr_t)a->k, ld |= a->k_ld;
    if (with_k && a->k_out) at |= (uintptr_t)a->k_out, ld |= a->k_out_ld;
    if (with_v) at |= (uintptr_t)a->v, ld |= a->v_ld;
    const bool vec = !(at & 15) && ld % per16 == 0;
    const int rope = a->rope && a->rot_dim ? a->rope : 0;
    const int ng = (a->head_dim + kKvBlock - 1) / kKvBlock, lpr = ng == 1 ? 4 : ng == 2 ? 8 : ng <= 4 ? 16 : 32;
    const int rpw = 32 / lpr;
    p.q_groups = (a->n_heads + rpw - 1) / rpw;
    p.k_groups = with_k ? (a->n_kv_heads + rpw - 1) / rpw : 0;
    p.groups = p.q_groups + p.k_groups + (with_v ? (a->n_kv_heads + rpw - 1) / rpw : 0);
    // One warp per token takes all its rows when there are tokens enough to fill the GPU; else its rows are shared out. (Shared out
    // further, to 96 or 192 warps an SM, 8191 tokens took 99 and 112 us with their read-back in place of 95, and 4000 tokens of 6 + 6 heads of 48
    // 12.5 in place of 9.3: the rotation and the slot are read again for each part.)
    const int sms = sm_count();
    const long long want = (24LL * sms + a->n_tokens - 1) / a->n_tokens;
    p.chunks = (int)std::min<long long>(std::max(1LL, want), p.groups);
    p.per_chunk = (p.groups + p.chunks - 1) / p.chunks;
    p.chunks = (p.groups + p.per_chunk - 1) / p.per_chunk;
    const long long warps = (long long)a->n_tokens * p.chunks;
    const int grid = (int)std::min<long long>(1 << 20, (warps + kQkvThreads / 32 - 1) / (kQkvThreads / 32));
    const cudaStream_t s = (cudaStream_t)stream;
    auto go = [&](auto t, auto r) {
        typedef decltype(t) T;
        constexpr int R = decltype(r)::value;
        auto run = [&](auto v) {
            constexpr bool V = decltype(v)::value;
            if (lpr == 4) return launch_early(qkv_kernel<T, 4, R, V>, grid, kQkvThreads, 0, s, p);
            if (lpr == 8) return launch_early(qkv_kernel<T, 8, R, V>, grid, kQkvThreads, 0, s, p);
            if (lpr == 16) return launch_early(qkv_kernel<T, 16, R, V>, grid, kQkvThreads, 0, s, p);
            return launch_early(qkv_kernel<T, 32, R, V>, grid, kQkvThreads, 0, s, p);
        };
        return vec ? run(std::true_type{}) : run(std::false_type{});
    };
    auto by_rope = [&](auto t) {
        if (rope == 0) return go(t, std::integral_constant<int, 0>{});
        if (rope == 1) return go(t, std::integral_constant<int, 1>{});
        return go(t, std::integral_constant<int, 2>{});
    };
    return launched(a->dtype == L3M_DT_F32 ? by_rope(float{}) : by_rope(__nv_bfloat16{}), me);
}

L3M_API int l3m_kv4_load_dev(const l3m_kv4 *cache, int dtype, void *k, void *v, const int32_t *slots, int n, void *stream) {
    const char *me = "l3m_kv4_load_dev";
    if (const char *why = kv4_error(cache)) return refuse(me, why);
    if (dtype != L3M_DT_F32 && dtype != L3M_DT_BF16) return refuse(me, "dtype must be f32 or bf16");
    if (n < 0) return refuse(me, "n must not be negative");
    if (n == 0 || (!k && !v)) return 0;
    if (!slots) return refuse(me, "slots are required");
    if (((uintptr_t)k | (uintptr_t)v) & (dtype == L3M_DT_F32 ? 3 : 1) || (uintptr_t)slots & 3) return refuse(me, "a pointer is not aligned to its type");
    const int parts = cache->head_dim / 8, turns = (2 * cache->n_kv_heads * parts + 31) / 32;
    const int warps = (int)std::min<long long>(turns, std::max(1LL, (32LL * sm_count() + n - 1) / n));   // a row's turns shared out where rows are few
    const LoadArgs p = {kv4_dev(cache), cache->dtype == L3M_DT_MXFP4, n, parts, !(((uintptr_t)k | (uintptr_t)v) & 15), warps, (unsigned)(0xffffffffu / parts + 1), k, v, slots};
    const int grid = (int)(((long long)n * warps + 7) / 8);
    const cudaStream_t s = (cudaStream_t)stream;
    return launched(dtype == L3M_DT_F32 ? launch_early(load_kernel<float>, grid, 256, 0, s, p) : launch_early(load_kernel<__nv_bfloat16>, grid, 256, 0, s, p), me);
}

}  // extern "C"
