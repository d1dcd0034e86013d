// Kernels of the 8-bit paged key/value cache (include/bzb_ext.h, bzb_kv8_*): appending with the q/k
// norms and the rotation in the same pass, reading back, and attention of few rows (a step of each
// sequence, a few guessed tokens); attention of many rows is in kv8_tile.cu.
#include "kv8_dev.cuh"

#include <algorithm>
#include <climits>
#include <cmath>
#include <cstdlib>
#include <cstring>
#include <stdexcept>
#include <string>

namespace bzb {
namespace {

using namespace kv8;

// ---- append and read ----
//
// Append: x' = x rsqrt(mean x^2 + eps) w, pairs (x'_j, x'_{j + hd/2}) turned by (cos, sin), then for keys and values
// of a block 2^e from its largest magnitude and the bytes. Read: bytes times 2^e.
//
// A CTA takes one block of 16 positions of a sequence and a few heads of q, k or v: a warp holds 16 rows of
// a head of 64, or 8 of one of 128 (two warps share a block, and its maximum through shared memory). A lane
// holds, of each of four consecutive rows, the four elements from 4c and the four from hd/2 + 4c, c its
// column of hd/8: the two members of four rotated pairs, so the rotation needs no exchange and each
// (cos, sin) is read by one lane, and of the values whole 4 x 4 patches, stored as 16 bytes. All rows' loads are
// issued before the first is used; what an append needs of the page (its scale, earlier bytes) is
// on the way while the norm and the rotation run. No other CTA touches the block: no atomics, and the
// same bytes whatever the launch's shape.
//
// Bound by loads and the arithmetic between them, not by DRAM: 16384 rows of 32 + 2 x 8 heads of 128 in bf16 are
// appended in 105 us (363 MB, 3.5 TB/s), 14 of them the (cos, sin) loads, which every head repeats (from L1
// and L2), and 12 the keys' 64-bit arithmetic; at 80 registers 212 to 466 bytes a thread are spilled. Reading 16 x 700 to
// 4096 positions of 8 heads of 128 takes 48 us (236 MB, 4.9 TB/s). A batch of 64 single rows: 5.9 us. With a lane on one row the first took 246 us; with 8 warps
// a CTA it takes 8 us more, with 5 CTAs an SM (fewer spills) 6 more, with one launch for q and one for the cache 10 more.
constexpr int kRowWarps = 4;
template <int HD>
struct RowMap {
    static constexpr int LPR = HD / 8;              // lanes of a row
    static constexpr int WPB = HD / 64;             // warps of a block
    static constexpr int HEADS = kRowWarps / WPB;   // heads of a CTA
};

// four consecutive elements as loaded: what is in flight takes half the registers for 16-bit types
template <int TYPE>
struct Raw4 {
    uint2 u;
    __device__ float4 value() const {
        if constexpr (TYPE == BZB_F16) {
            const float2 a = __half22float2(*reinterpret_cast<const half2 *>(&u.x)), b = __half22float2(*reinterpret_cast<const half2 *>(&u.y));
            return make_float4(a.x, a.y, b.x, b.y);
        } else {
            return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xffff0000u), __uint_as_float(u.y << 16),
                               __uint_as_float(u.y & 0xffff0000u));
        }
    }
};
template <>
struct Raw4<BZB_F32> {
    float4 u;
    __device__ float4 value() const { return u; }
};
template <int TYPE, bool VEC>
__device__ __forceinline__ Raw4<TYPE> raw4(const void * p, long long i) {
    Raw4<TYPE> r;
    if constexpr (TYPE == BZB_F32) {
        r.u = load4<VEC>(static_cast<const float *>(p) + i);
    } else {
        const uint16_t * h = static_cast<const uint16_t *>(p) + i;
        if constexpr (VEC) r.u = *reinterpret_cast<const uint2 *>(h);
        else r.u = make_uint2((uint32_t) h[0] | (uint32_t) h[1] << 16, (uint32_t) h[2] | (uint32_t) h[3] << 16);
    }
    return r;
}

struct AppendArgs {
    Kv kv;
    Rows q, k, v, q_out;
    const float * q_norm, * k_norm;
    const float2 * rope;
    float eps;
    int n_head, q_out_type;
    bool q_out_vec, norm_vec;
};

// Mean squares between these need no second look: the products of elements that matter are normal numbers. Below, every
// element is less than 2^-36 and grows to 2^60 at most (2^-149 to 2^-53); above, none exceeds 2^128, which becomes 2^58.
constexpr float kTinySquares = 0x1p-80f, kHugeSquares = 0x1p120f, kSmallLift = 0x1p96f, kLargeDrop = 0x1p-70f;

// the f32 next to x towards zero, its last bit set where it is not x: rounded once more to fewer bits, it goes
// the way x would
__device__ __forceinline__ float to_odd(double x) {
    const float f = __double2float_rz(x);
    return (double) f == x ? f : __int_as_float(__float_as_int(f) | 1);
}
// a row's norm and rotation in 64 bits, for the lanes of RowMap
template <int HD>
__device__ __forceinline__ void turn_exactly(float4 & lo, float4 & hi, bool norm, float4 wl, float4 wh, float eps, bool turn, float4 t0,
                                             float4 t1) {
    double x[4] = { lo.x, lo.y, lo.z, lo.w }, y[4] = { hi.x, hi.y, hi.z, hi.w };
    if (norm) {
        const float u[4] = { wl.x, wl.y, wl.z, wl.w }, v[4] = { wh.x, wh.y, wh.z, wh.w };
        double ss = 0.0;
#pragma unroll
        for (int j = 0; j < 4; j++) ss = fma(x[j], x[j], fma(y[j], y[j], ss));
#pragma unroll
        for (int o = HD / 16; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
        const double r = rsqrt(ss * (1.0 / HD) + (double) eps);
#pragma unroll
        for (int j = 0; j < 4; j++) x[j] *= r * u[j], y[j] *= r * v[j];
    }
    const float c[4] = { t0.x, t0.z, t1.x, t1.z }, s[4] = { t0.y, t0.w, t1.y, t1.w };
    float p[4], q[4];
#pragma unroll
    for (int j = 0; j < 4; j++) {
        // (not a turn by nothing: 0 times an infinite partner is NaN)
        p[j] = to_odd(turn ? fma(x[j], (double) c[j], -(y[j] * s[j])) : x[j]);
        q[j] = to_odd(turn ? fma(x[j], (double) s[j], y[j] * c[j]) : y[j]);
    }
    lo = make_float4(p[0], p[1], p[2], p[3]);
    hi = make_float4(q[0], q[1], q[2], q[3]);
}

// FULL: all 16 positions of the block are new
template <int HD, int TYPE, bool VEC, bool FULL>
__device__ __forceinline__ void append_block(const AppendArgs & a, const Seq & s, int first, int blk, float * tops) {
    using R = RowMap<HD>;
    const Kv & kv = a.kv;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane % R::LPR;
    const int r0 = warp % R::WPB * (16 / R::WPB) + lane / R::LPR * 4;  // the lane's first row of the block
    const int p0 = blk << 4;
    const int nq = a.n_head, nkv = kv.n_kv;
    const int any = (int) blockIdx.x * R::HEADS + warp / R::WPB;
    const int kind = any < nq ? 0 : any < nq + nkv ? 1 : any < nq + 2 * nkv ? 2 : 3;
    const int head = kind == 0 ? any : kind == 1 ? any - nq : any - nq - nkv;
    const Rows src = kind == 0 ? a.q : kind == 1 ? a.k : a.v;
    const int live_lo = FULL ? 0 : max(first - p0, 0), live_hi = FULL ? 16 : min(16, s.len - p0);  // the block's new rows
    bool live[4];
#pragma unroll
    for (int i = 0; i < 4; i++) live[i] = kind < 3 && (FULL || (r0 + i >= live_lo && r0 + i < live_hi));
    const long long row = s.row0 + p0 + r0 - first;  // packed row of the lane's first position

    Raw4<TYPE> lo_raw[4] = {}, hi_raw[4] = {};
    long long at = row * src.row + head * src.head + 4 * c;
#pragma unroll
    for (int i = 0; i < 4; i++, at += src.row) {
        if (!live[i]) continue;
        lo_raw[i] = raw4<TYPE, VEC>(src.p, at);
        hi_raw[i] = raw4<TYPE, VEC>(src.p, at + HD / 2);
    }
    const float * w = kind == 0 ? a.q_norm : kind == 1 ? a.k_norm : nullptr;
    float4 wl = make_float4(0.0f, 0.0f, 0.0f, 0.0f), wh = wl;
    if (w) {
        wl = a.norm_vec ? load4<true>(w + 4 * c) : load4<false>(w + 4 * c);
        wh = a.norm_vec ? load4<true>(w + HD / 2 + 4 * c) : load4<false>(w + HD / 2 + 4 * c);
    }
    // row i's (cos, sin) of pairs 4c, 4c + 1 and of 4c + 2, 4c + 3
    auto turn_of = [&](int i, float4 & t0, float4 & t1) {
        t0 = t1 = make_float4(1.0f, 0.0f, 1.0f, 0.0f);
        if (!live[i] || !a.rope) return;
        const float4 * t = reinterpret_cast<const float4 *>(a.rope + (size_t) (p0 + r0 + i) * (HD / 2) + 4 * c);
        t0 = t[0];
        t1 = t[1];
    };
    const bool cached = kind == 1 || kind == 2, older = !FULL && cached && p0 < first;  // older: the block holds earlier positions
    const int pg = cached ? page_of(kv, s.slot, blk) : -1;
    uint8_t * dst = pg < 0 ? nullptr : block_ptr(kv, pg, blk, kind - 1, head, HD);
    float * sp = pg < 0 ? nullptr : scale_ptr(kv, pg, blk, kind - 1, head);
    float was = 1.0f;
    uint32_t old[8];  // keys: a row's words c and c + hd/8, row after row; values: the patch of quad c, then of c + hd/8
#pragma unroll
    for (int i = 0; i < 8; i++) old[i] = 0;
    if (older && pg >= 0) {
        was = *sp;
        if (p0 + r0 < first) {
            if (kind == 1) {
#pragma unroll
                for (int i = 0; i < 4; i++) {
                    const uint32_t * row = reinterpret_cast<const uint32_t *>(dst + (r0 + i) * HD);
                    old[2 * i] = row[c];
                    old[2 * i + 1] = row[c + HD / 8];
                }
            } else {
                const uint4 * pl = reinterpret_cast<const uint4 *>(dst + c * 64 + r0 * 4), x = pl[0], y = pl[HD / 8 * 4];
                old[0] = x.x, old[1] = x.y, old[2] = x.z, old[3] = x.w, old[4] = y.x, old[5] = y.y, old[6] = y.z, old[7] = y.w;
            }
        }
    }
    float4 lo[4], hi[4];
    if (kind == 0) {
        // (the table's loads of all rows are on the way while the norms are summed)
        float4 turn[4][2];
#pragma unroll
        for (int i = 0; i < 4; i++) turn_of(i, turn[i][0], turn[i][1]);
        long long to = row * a.q_out.row + head * a.q_out.head + 4 * c;
#pragma unroll
        for (int i = 0; i < 4; i++, to += a.q_out.row) {
            if (!FULL && !__any_sync(0xffffffffu, live[i])) continue;
            float4 x = lo_raw[i].value(), y = hi_raw[i].value();
            if (w) {
                auto mean_sq = [&] {
                    float2 sq = __fmul2_rn(make_float2(x.x, x.y), make_float2(x.x, x.y));
                    sq = __ffma2_rn(make_float2(x.z, x.w), make_float2(x.z, x.w), sq);
                    sq = __ffma2_rn(make_float2(y.x, y.y), make_float2(y.x, y.y), sq);
                    sq = __ffma2_rn(make_float2(y.z, y.w), make_float2(y.z, y.w), sq);
                    float ss = sq.x + sq.y;
#pragma unroll
                    for (int o = R::LPR / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xffffffffu, ss, o);
                    return ss * (1.0f / HD);
                };
                float eps = a.eps, ms = mean_sq();
                // Squares outside f32's range, above or (where eps does not outweigh them) below: once more with the row
                // times a power of two, which the norm takes out again. (f16's squares stay inside: 2^-48 to 2^32.)
                const bool out = TYPE != BZB_F16 && !(ms + eps > kTinySquares && ms < kHugeSquares);
                if (TYPE != BZB_F16 && __builtin_expect(__any_sync(0xffffffffu, out), 0)) {
                    if (out) {
                        const float f = ms < 1.0f ? kSmallLift : kLargeDrop;
                        x.x *= f, x.y *= f, x.z *= f, x.w *= f, y.x *= f, y.y *= f, y.z *= f, y.w *= f;
                        eps = eps * f * f;
                    }
                    ms = mean_sq();
                }
                const float r = rsqrtf(ms + eps);
                auto scale = [&](float4 & v, const float4 & w) {
                    const float2 p = __fmul2_rn(__fmul2_rn(make_float2(v.x, v.y), make_float2(r, r)), make_float2(w.x, w.y));
                    const float2 q = __fmul2_rn(__fmul2_rn(make_float2(v.z, v.w), make_float2(r, r)), make_float2(w.z, w.w));
                    v = make_float4(p.x, p.y, q.x, q.y);
                };
                scale(x, wl);
                scale(y, wh);
            }
            const float4 t0 = turn[i][0], t1 = turn[i][1];
            if (!live[i]) continue;
            float4 u = x, v = y;
            if (a.rope) {
                u = make_float4(x.x * t0.x - y.x * t0.y, x.y * t0.z - y.y * t0.w, x.z * t1.x - y.z * t1.y, x.w * t1.z - y.w * t1.w);
                v = make_float4(x.x * t0.y + y.x * t0.x, x.y * t0.w + y.y * t0.z, x.z * t1.y + y.z * t1.x, x.w * t1.w + y.w * t1.z);
            }
            store4(a.q_out_type, a.q_out_vec, a.q_out.p, to, u);
            store4(a.q_out_type, a.q_out_vec, a.q_out.p, to + HD / 2, v);
        }
    } else {
        const bool exact = kind == 1 && (w || a.rope);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            lo[i] = lo_raw[i].value();
            hi[i] = hi_raw[i].value();
            // Keys in 64 bits, then to odd f32: every cached byte is the correctly rounded one. (In f32, which took
            // 10 % less time, three of a million fell on the other side of a tie.)
            if (exact && (FULL || __any_sync(0xffffffffu, live[i]))) {
                float4 t0, t1;
                turn_of(i, t0, t1);
                turn_exactly<HD>(lo[i], hi[i], w != nullptr, wl, wh, a.eps, a.rope != nullptr, t0, t1);
            }
            // (a row that is not there has norm zero, which without eps is no number)
            if (!live[i]) lo[i] = hi[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        }
    }

    // the block's largest finite magnitude; what is not finite becomes NaN
    float top = 0.0f;
    if (cached) {
        // (a maximum that keeps NaNs tells whether any value needs a second look)
        auto larger = [](float m, float x) {
            float r;
            asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(m), "f"(fabsf(x)));
            return r;
        };
#pragma unroll
        for (int i = 0; i < 4; i++) {
            top = larger(larger(larger(larger(top, lo[i].x), lo[i].y), lo[i].z), lo[i].w);
            top = larger(larger(larger(larger(top, hi[i].x), hi[i].y), hi[i].z), hi[i].w);
        }
        if (!(top < INFINITY)) {
            top = 0.0f;
            auto finite = [&](float & x) {
                const float m = fabsf(x);
                if (m < INFINITY) top = fmaxf(top, m);
                else x = __int_as_float(0x7fffffff);
            };
#pragma unroll
            for (int i = 0; i < 4; i++) {
                finite(lo[i].x), finite(lo[i].y), finite(lo[i].z), finite(lo[i].w);
                finite(hi[i].x), finite(hi[i].y), finite(hi[i].z), finite(hi[i].w);
            }
        }
        __syncwarp();
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    }
    if (R::WPB > 1) {
        if (lane == 0) tops[warp] = top;
        __syncthreads();  // (also: both warps of a block have read its old scale before one writes the new)
        top = fmaxf(top, tops[warp ^ 1]);
    } else {
        __syncwarp();
    }
    if (pg < 0) return;
    int e = block_exponent(top);
    float keep = 1.0f;  // factor of the earlier values' bytes
    if (older) {
        const int e_old = min(kExpMax, max(kExpMin, exponent_of(was)));
        e = max(e, e_old);
        keep = pow2f(e_old - e);
    }
    const float inv = pow2f(-e);
    auto kept = [&](uint32_t w) {
        const float4 f = e4m3x4_to_f4(w);
        return to_e4m3x4(f.x * keep, f.y * keep, f.z * keep, f.w * keep);
    };
    if (kind == 1) {
#pragma unroll
        for (int i = 0; i < 4; i++) {
            uint32_t * row = reinterpret_cast<uint32_t *>(dst + (r0 + i) * HD);
            uint32_t wl = to_e4m3x4(lo[i].x * inv, lo[i].y * inv, lo[i].z * inv, lo[i].w * inv);
            uint32_t wh = to_e4m3x4(hi[i].x * inv, hi[i].y * inv, hi[i].z * inv, hi[i].w * inv);
            if (r0 + i < live_lo) wl = kept(old[2 * i]), wh = kept(old[2 * i + 1]);
            row[c] = wl;
            row[c + HD / 8] = wh;
        }
    } else {
        // patch (quad c or c + hd/8, the lane's four rows): word j holds element j of the four positions
        const int n_old = min(4, max(0, live_lo - r0));
        const uint32_t m = n_old == 4 ? 0xffffffffu : (1u << (8 * n_old)) - 1;
        auto word = [&](float v0, float v1, float v2, float v3, uint32_t o) {
            const uint32_t n = to_e4m3x4(v0 * inv, v1 * inv, v2 * inv, v3 * inv);
            return m ? (kept(o) & m) | (n & ~m) : n;
        };
        uint4 * pl = reinterpret_cast<uint4 *>(dst + c * 64 + r0 * 4);
        pl[0] = make_uint4(word(lo[0].x, lo[1].x, lo[2].x, lo[3].x, old[0]), word(lo[0].y, lo[1].y, lo[2].y, lo[3].y, old[1]),
                           word(lo[0].z, lo[1].z, lo[2].z, lo[3].z, old[2]), word(lo[0].w, lo[1].w, lo[2].w, lo[3].w, old[3]));
        pl[HD / 8 * 4] = make_uint4(word(hi[0].x, hi[1].x, hi[2].x, hi[3].x, old[4]), word(hi[0].y, hi[1].y, hi[2].y, hi[3].y, old[5]),
                                    word(hi[0].z, hi[1].z, hi[2].z, hi[3].z, old[6]), word(hi[0].w, hi[1].w, hi[2].w, hi[3].w, old[7]));
    }
    if (lane == 0 && warp % R::WPB == 0) *sp = pow2f(e);
}

template <int HD, int TYPE, bool VEC>
__global__ void __launch_bounds__(32 * kRowWarps, 6) kv8_append_kernel(const AppendArgs a) {
    __shared__ float tops[kRowWarps];
    start_after_previous();
    const Seq s = load_seq(a.kv, (int) blockIdx.z);
    if (s.slot < 0) return;
    const int first = s.len - s.n;  // position of the sequence's first row (negative: padding rows)
    const int blk = (max(first, 0) >> 4) + (int) blockIdx.y, p0 = blk << 4;
    if (p0 >= s.len || s.n == 0) return;  // (the whole CTA, as above)
    if (p0 >= first && p0 + 16 <= s.len) append_block<HD, TYPE, VEC, true>(a, s, first, blk, tops);
    else append_block<HD, TYPE, VEC, false>(a, s, first, blk, tops);
}

struct ReadArgs {
    Kv kv;
    Rows k, v;
    bool vec;
};

template <int HD, int TYPE>
__global__ void __launch_bounds__(32 * kRowWarps) kv8_read_kernel(const ReadArgs a) {
    using R = RowMap<HD>;
    const Kv & kv = a.kv;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, c = lane % R::LPR;
    const int r0 = warp % R::WPB * (16 / R::WPB) + lane / R::LPR * 4;
    start_after_previous();
    const Seq s = load_seq(kv, (int) blockIdx.z);
    if (s.slot < 0 || s.n == 0) return;
    // blocks count from the first row's position; `first` may be negative (padding rows, read as zeros)
    const int first = s.len - s.n, blk = (first >> 4) + (int) blockIdx.y, p0 = blk << 4;
    const int any = (int) blockIdx.x * R::HEADS + warp / R::WPB;
    if (p0 >= s.len || any >= 2 * kv.n_kv) return;
    const int plane = any >= kv.n_kv, head = any - plane * kv.n_kv;
    float4 lo[4], hi[4];
#pragma unroll
    for (int i = 0; i < 4; i++) lo[i] = hi[i] = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    if (blk >= 0) {
        const int pg = max(page_of(kv, s.slot, blk), 0);
        const uint8_t * src = block_ptr(kv, pg, blk, plane, head, HD);
        const float scale = *scale_ptr(kv, pg, blk, plane, head);
        uint32_t w[8];
        if (plane == 0) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const uint32_t * row = reinterpret_cast<const uint32_t *>(src + (r0 + i) * HD);
                w[2 * i] = row[c];
                w[2 * i + 1] = row[c + HD / 8];
            }
#pragma unroll
            for (int i = 0; i < 4; i++) lo[i] = e4m3x4_to_f4(w[2 * i]), hi[i] = e4m3x4_to_f4(w[2 * i + 1]);
        } else {
            const uint4 * pl = reinterpret_cast<const uint4 *>(src + c * 64 + r0 * 4);
            const uint4 x = pl[0], y = pl[HD / 8 * 4];
            auto patch = [&](float4 (&o)[4], uint4 w) {
                const float4 e0 = e4m3x4_to_f4(w.x), e1 = e4m3x4_to_f4(w.y), e2 = e4m3x4_to_f4(w.z), e3 = e4m3x4_to_f4(w.w);
                o[0] = make_float4(e0.x, e1.x, e2.x, e3.x);
                o[1] = make_float4(e0.y, e1.y, e2.y, e3.y);
                o[2] = make_float4(e0.z, e1.z, e2.z, e3.z);
                o[3] = make_float4(e0.w, e1.w, e2.w, e3.w);
            };
            patch(lo, x);
            patch(hi, y);
        }
#pragma unroll
        for (int i = 0; i < 4; i++) {
            lo[i] = make_float4(lo[i].x * scale, lo[i].y * scale, lo[i].z * scale, lo[i].w * scale);
            hi[i] = make_float4(hi[i].x * scale, hi[i].y * scale, hi[i].z * scale, hi[i].w * scale);
        }
    }
    const Rows dst = plane ? a.v : a.k;
    long long at = (long long) (s.row0 + p0 + r0 - first) * dst.row + head * dst.head + 4 * c;
#pragma unroll
    for (int i = 0; i < 4; i++, at += dst.row) {
        const int pos = p0 + r0 + i;
        if (pos < first || pos >= s.len) continue;
        store4(TYPE, a.vec, dst.p, at, lo[i]);
        store4(TYPE, a.vec, dst.p, at + HD / 2, hi[i]);
    }
}

__device__ __forceinline__ void mma16816(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
    uint32_t y;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}
// 16 elements of a query row from element i as f16 pairs: f16 rows as they are, bf16 rows times f (and
// their largest magnitude into amax)
__device__ __forceinline__ void load_q16(const AttnArgs & a, long long i, float f, uint32_t (&o)[8], float * amax) {
    float x[16];
    if (a.type == BZB_F16) {
        const half * h = static_cast<const half *>(a.q.p) + i;
        if (a.q_vec) {
            const uint4 u = *reinterpret_cast<const uint4 *>(h), v = *reinterpret_cast<const uint4 *>(h + 8);
            o[0] = u.x, o[1] = u.y, o[2] = u.z, o[3] = u.w, o[4] = v.x, o[5] = v.y, o[6] = v.z, o[7] = v.w;
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) {
                const half2 p = __halves2half2(h[2 * j], h[2 * j + 1]);
                o[j] = *reinterpret_cast<const uint32_t *>(&p);
            }
        }
        return;
    }
    const __nv_bfloat16 * h = static_cast<const __nv_bfloat16 *>(a.q.p) + i;
    if (a.q_vec) {
        const uint4 u = *reinterpret_cast<const uint4 *>(h), v = *reinterpret_cast<const uint4 *>(h + 8);
        const uint32_t w[8] = { u.x, u.y, u.z, u.w, v.x, v.y, v.z, v.w };
#pragma unroll
        for (int j = 0; j < 8; j++) x[2 * j] = __uint_as_float(w[j] << 16), x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    } else {
#pragma unroll
        for (int j = 0; j < 16; j++) x[j] = __bfloat162float(h[j]);
    }
    if (amax) {
#pragma unroll
        for (int j = 0; j < 16; j++) *amax = fmaxf(*amax, fabsf(x[j]));
    }
#pragma unroll
    for (int j = 0; j < 8; j++) o[j] = pack_half(x[2 * j] * f, x[2 * j + 1] * f);
}

// Few query rows (a step of each sequence, a few guessed tokens, short prompts): o = sum_j w_j v_j / sum_j w_j 2^-e_j,
// w_j = 2^(s_j + e_j - M), s_j = scale log2(e) q k_j, 2^e_j the values' scale, M the running maximum of
// s_j + e_j. One CTA per (sequence, kv head, 8 rows, range of the cache); the rows of a kv head are (token, head of the
// group) pairs, so a block read once serves the group. Four warps share out the range's blocks, two at a time,
// each with a ring of its own, and join their results at the end.
//
// Calls with more than 8 rows have more CTAs, which read the same blocks from L2 at about the same time: against a CTA
// with one ring for all rows, a warp for each 8, which waits on all its warps twice for each pair of blocks, that takes
// 20 against 21 us (16 sequences of 2000, 16 rows), 23 against 34 (64 of 1000, 16 rows), 40 against 49 (32 rows).
//
// The matrix products are m16n8k16 with the cache as the 16-row operand: S^T = K Q^T (16 positions x 8
// rows) and O^T = V^T W^T (16 of head_dim x 8 rows): no half of a tile is empty when a group has at
// most 8 rows. A lane's 16 bytes of a key row are the four k-steps' values of head_dim for it (the queries are
// read in the same order, and any order of the sum's terms will do), and the value patches are stored in operand
// order: no transposition but the 8x8 one of the weights. The blocks are copied as they lie in memory
// (cp.async), AHEAD pairs in advance: a pair's keys as soon as the scores are done with the pair that had
// their place, its values after the second product.
//
// Bound by DRAM with long contexts (8 sequences of 32000 positions, 8 kv heads of 128, 4 rows: 532 MB in 93 us,
// 5.7 TB/s; loads into registers instead of rings: 133). Ragged steps (64 sequences of 90 to 2030 positions, 8 kv heads
// of 64, 4 rows: 70 MB in 23 us, 3.0 TB/s) are bound by latency: 5 us from the sequence through its page to the data,
// then the longest contexts; 17 us remain without the arithmetic. One sequence of 218 positions: 4.3 us, a launch.
constexpr int kSmallWarps = 4, kSmallRows = 8;
constexpr int kTable = 128;  // blocks that a warp looks up at a time
constexpr int kShortRange = kSmallWarps * kTable;  // blocks of a range that needs one look-up

// CTAs that an SM holds, by their registers (96 and 128 a thread)
constexpr int small_ctas(int hd) { return (hd == 64 ? 20 : 16) / kSmallWarps; }

template <int HD>
struct SmallTile {
    static constexpr int KS = HD / 64, VS = HD / 32, MT = HD / 16, PL = HD + 4;
    static constexpr int PIECES = 2 * KS + VS;            // 512-byte pieces of a block
    static constexpr int AHEAD = HD == 64 ? 2 : 1;        // pairs of blocks that a warp's ring holds
    static constexpr int RING = kSmallWarps * AHEAD * 2 * PIECES * 512, MERGE = kSmallWarps * kSmallRows * PL * 4;
    static constexpr int BYTES = RING > MERGE ? RING : MERGE;
};

__device__ __forceinline__ void copy16(uint32_t dst, const void * src, bool there) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(there ? 16 : 0) : "memory");
}
__device__ __forceinline__ uint4 lds16(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}

// LONG: ranges of more than kShortRange blocks, looked up part by part. (A form of its own, for the registers that the
// outer loop keeps: with it, 64 sequences of 90 to 2030 positions take 24.9 us instead of 23.2. Ranges of any
// length keep the workspace small: with short ones only, 512 sequences bounded by 131072 positions needed 277 MB.)
template <int HD, bool LONG>
__global__ void __launch_bounds__(32 * kSmallWarps, small_ctas(HD)) kv8_attn_small_kernel(const AttnArgs a) {
    using T = SmallTile<HD>;
    extern __shared__ __align__(16) uint8_t ring[];
    __shared__ float sm_ml[kSmallWarps][kSmallRows][2];
    // the warps' next blocks: the head's keys (its values lie one plane on), the scales of both
    __shared__ const uint8_t * block_at[kSmallWarps * kTable];
    __shared__ float2 scales[kSmallWarps * kTable];
    const Kv & kv = a.kv;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, g = lane >> 2, t = lane & 3;
    // (heads fastest: neighbouring CTAs read neighbouring bytes of the same pages)
    unsigned id = blockIdx.x;
    const int h = (int) (id % (unsigned) kv.n_kv);
    id /= (unsigned) kv.n_kv;
    const int chunk = (int) (id % (unsigned) a.chunks);
    id /= (unsigned) a.chunks;
    const int tile = (int) (id % (unsigned) a.row_tiles), b = (int) (id / (unsigned) a.row_tiles);
    start_after_previous();
    const Seq s = load_seq(kv, b);
    if (s.slot < 0) return;
    const int row0 = tile * kSmallRows;
    const Span span = span_of(a, s, row0, kSmallRows);
    const int first = span.first, rows = span.rows, my_chunks = span.chunks;
    if (row0 >= rows || chunk >= my_chunks) return;
    // the keys that all rows see: [full_lo, full_hi)
    const int last_row = min(rows, row0 + kSmallRows) - 1;
    const int full_hi = keys_end(a, s, first + row0 / a.group);
    const int full_lo = a.window > 0 ? max(0, first + last_row / a.group - a.window + 1) : 0;
    const int c_lo = span.blk_lo + chunk * a.chunk_blocks, c_hi = min(span.blk_hi, c_lo + a.chunk_blocks);

    // this warp's blocks: base, base + kSmallWarps, ..., looked up by itself, n at a time
    int base = c_lo + warp, n = 0;
    const int mine0 = warp * kTable;
    const int kpos = (g >> 1) * 4 + (g & 1);  // the lane's key rows: kpos and kpos + 2 (see the patches' position order)
    const long long v_at = (long long) kv.n_kv * kv.page_tokens * HD;
    const uint32_t slots = (uint32_t) __cvta_generic_to_shared(ring) + warp * (T::AHEAD * 2 * T::PIECES * 512);
    // where the lane's 16 bytes of 512 go: rows of 128 bytes have their halves swapped in every second row,
    // which keeps the reading lanes on different banks
    const int k_to = HD == 64 ? 16 * lane : (lane >> 3) * 128 + (((lane & 7) ^ ((lane >> 3 & 1) << 2)) << 4);
    const int k_from = kpos * HD + 16 * t;
    // keys, or values, of blocks i and i + 1 into the ring; a block past the last is zeros
    auto fetch = [&](int i, bool values) {
        constexpr int PK = 2 * T::KS;
        const uint32_t slot = slots + i / 2 % T::AHEAD * 2 * (T::PIECES * 512);
#pragma unroll
        for (int x = 0; x < 2 * (PK > T::VS ? PK : T::VS); x++) {
            const int per = values ? T::VS : PK, k2 = x / per, k = x % per;
            if (k2 > 1) continue;
            const bool there = i + k2 < n;
            const uint8_t * p = block_at[mine0 + (there ? i + k2 : 0)] + 16 * lane + 512 * k;
            if (values) copy16(slot + (k2 * T::PIECES + PK + k) * 512 + 16 * lane, p + v_at, there);
            else copy16(slot + (k2 * T::PIECES + k) * 512 + k_to, p, there);
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    auto look_up = [&] {
        n = max(0, (c_hi - base + kSmallWarps - 1) / kSmallWarps);
        if (LONG) n = min(n, kTable);
        // (the first blocks' copies do not wait for their scales)
        float2 sc0 = make_float2(0.0f, 0.0f);
        if (lane < n) {
            const int blk = base + lane * kSmallWarps, pg = max(page_of(kv, s.slot, blk), 0);
            block_at[mine0 + lane] = block_ptr(kv, pg, blk, 0, h, HD);
            sc0 = make_float2(*scale_ptr(kv, pg, blk, 0, h), *scale_ptr(kv, pg, blk, 1, h));
        }
        __syncwarp();
        if (n > 0) {
#pragma unroll
            for (int i = 0; i < T::AHEAD; i++) {
                // (the first 32 blocks are in the table by now)
                fetch(2 * i, false);
                fetch(2 * i, true);
            }
        }
        if (lane < n) scales[mine0 + lane] = sc0;
        for (int i = lane + 32; i < n; i += 32) {
            const int blk = base + i * kSmallWarps, pg = max(page_of(kv, s.slot, blk), 0);
            block_at[mine0 + i] = block_ptr(kv, pg, blk, 0, h, HD);
            scales[mine0 + i] = make_float2(*scale_ptr(kv, pg, blk, 0, h), *scale_ptr(kv, pg, blk, 1, h));
        }
        __syncwarp();
    };
    look_up();

    // queries as the 8-column operand: lane (g, t) holds the warp's row g, elements 64 k + 16 t ..+15
    uint32_t qf[T::KS][8];
    float coef[2];      // the score's factor for the lane's two columns (rows 2 t, 2 t + 1)
    int lim_hi[2], lim_lo[2];
    const int r = row0 + g;
    float row_unit = 1.0f;
    if (r < rows) {
        const long long at = (long long) (s.row0 + r / a.group) * a.q.row + (h * a.group + r % a.group) * a.q.head + 16 * t;
        float amax = 0.0f;
#pragma unroll
        for (int k = 0; k < T::KS; k++) load_q16(a, at + 64 * k, 1.0f, qf[k], &amax);
        // bf16 may lie outside f16: the row is brought up to [2^14, 2^15) by a power of two (which the scores'
        // factor takes back); elements keep all their bits down to 2^-31 of the largest, and some down to 2^-38
        if (a.type == BZB_BF16) {
            const unsigned quad = 0xfu << (lane & 28);
            amax = fmaxf(amax, __shfl_xor_sync(quad, amax, 1));
            amax = fmaxf(amax, __shfl_xor_sync(quad, amax, 2));
            const int e = row_exponent(amax);
            row_unit = pow2f(e);
#pragma unroll
            for (int k = 0; k < T::KS; k++) load_q16(a, at + 64 * k, pow2f(-e), qf[k], nullptr);
        }
    } else {
#pragma unroll
        for (int k = 0; k < T::KS; k++)
#pragma unroll
            for (int j = 0; j < 8; j++) qf[k][j] = 0;
    }
#pragma unroll
    for (int i = 0; i < 2; i++) {
        const int rr = row0 + 2 * t + i, pos = first + rr / a.group;
        coef[i] = a.scale2 * __shfl_sync(0xffffffffu, row_unit, (2 * t + i) * 4);
        lim_hi[i] = rr < rows ? keys_end(a, s, pos) : 0;
        lim_lo[i] = a.window > 0 ? pos - a.window + 1 : 0;
    }

    float o[T::MT][4] = {}, m[2], l[2] = {};
    m[0] = m[1] = -INFINITY;

  for (;;) {  // once, or for each part of a long range
    for (int i = 0; i < n; i += 2) {
        asm volatile("cp.async.wait_group %0;" ::"n"(2 * T::AHEAD - 1) : "memory");  // the keys
        __syncwarp();
        const uint32_t pair = slots + i / 2 % T::AHEAD * 2 * (T::PIECES * 512);
        float x[2][4];  // columns 2t, 2t+1 at key kpos, then at key kpos + 2
        uint32_t seen[2][2];  // (positions x rows) the rows that see each position, as f16 ones
        bool whole[2];
        float inv_vs[2];
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) {
            const uint32_t slot = pair + k2 * (T::PIECES * 512) + k_from;
            float sc[4] = {}, sd[4] = {};  // (two sums: half as long a chain of MMAs)
#pragma unroll
            for (int k = 0; k < T::KS; k++) {
                const int at = HD == 64 ? 0 : 64 * (k ^ (g & 1));
                const uint4 u0 = lds16(slot + at), u1 = lds16(slot + 2 * HD + at);
                const uint32_t w0[4] = { u0.x, u0.y, u0.z, u0.w }, w1[4] = { u1.x, u1.y, u1.z, u1.w };
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const uint32_t a0 = e4m3x2_to_h2((uint16_t) w0[j]), a2 = e4m3x2_to_h2((uint16_t) (w0[j] >> 16));
                    const uint32_t a1 = e4m3x2_to_h2((uint16_t) w1[j]), a3 = e4m3x2_to_h2((uint16_t) (w1[j] >> 16));
                    mma16816(j & 1 ? sd : sc, a0, a1, a2, a3, qf[k][2 * j], qf[k][2 * j + 1]);
                }
            }
            const bool there = i + k2 < n;
            const float2 kvs = scales[mine0 + (there ? i + k2 : 0)];
            const float ks = kvs.x, vs = kvs.y;
            const int key0 = (base + (i + k2) * kSmallWarps) << 4;
            const float ev = (float) exponent_of(vs);
            inv_vs[k2] = pow2f(-exponent_of(vs));
            whole[k2] = there && key0 >= full_lo && key0 + 16 <= full_hi;
            const float c0 = coef[0] * ks, c1 = coef[1] * ks;
#pragma unroll
            for (int j = 0; j < 4; j++) x[k2][j] = fmaf(sc[j] + sd[j], j & 1 ? c1 : c0, ev);
            if (!whole[k2]) {
                uint32_t one[4];
#pragma unroll
                for (int j = 0; j < 4; j++) {
                    const int key = key0 + kpos + (j >> 1) * 2;
                    const bool in = there && key >= lim_lo[j & 1] && key < lim_hi[j & 1];
                    if (!in) x[k2][j] = -INFINITY;
                    one[j] = in ? 0x3c00u : 0u;
                }
                seen[k2][0] = one[0] | (one[1] << 16);
                seen[k2][1] = one[2] | (one[3] << 16);
            }
        }
        // (also past the end, where it copies zeros: the waits count groups)
        __syncwarp();
        fetch(i + 2 * T::AHEAD, false);
        uint32_t wb[2][2];
        bool moved = false;
        float corr[2];
#pragma unroll
        for (int i2 = 0; i2 < 2; i2++) {
            float mx = fmaxf(fmaxf(x[0][i2], x[0][i2 + 2]), fmaxf(x[1][i2], x[1][i2 + 2]));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 4));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 8));
            mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, 16));
            const float to = fmaxf(m[i2], mx), ref = to == -INFINITY ? 0.0f : to;
            corr[i2] = exp2_approx(m[i2] - ref);
            moved |= to != m[i2];
            m[i2] = to;
            float sum = 0.0f;
#pragma unroll
            for (int k2 = 0; k2 < 2; k2++) {
                x[k2][i2] = exp2_approx(x[k2][i2] - ref);
                x[k2][i2 + 2] = exp2_approx(x[k2][i2 + 2] - ref);
                sum = fmaf(x[k2][i2] + x[k2][i2 + 2], inv_vs[k2], sum);
            }
            l[i2] = fmaf(l[i2], corr[i2], sum);
        }
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) {
            wb[k2][0] = transpose8x8(pack_half(x[k2][0], x[k2][1]));
            wb[k2][1] = transpose8x8(pack_half(x[k2][2], x[k2][3]));
        }
        if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int j = 0; j < T::MT; j++)
#pragma unroll
                for (int i2 = 0; i2 < 4; i2++) o[j][i2] *= corr[i2 & 1];
        }
        asm volatile("cp.async.wait_group %0;" ::"n"(2 * T::AHEAD - 1) : "memory");  // the values
        __syncwarp();
#pragma unroll
        for (int k2 = 0; k2 < 2; k2++) {
            const uint32_t slot = pair + k2 * (T::PIECES * 512) + 16 * lane;
            uint4 vw[T::VS];
#pragma unroll
            for (int j = 0; j < T::VS; j++) vw[j] = lds16(slot + (2 * T::KS + j) * 512);
            if (!whole[k2]) {
                // a NaN at a position that some row does not see must not reach that row (0 x NaN):
                // NaNs are taken out of the product and given to the rows that see them
                uint32_t bad = 0;
#pragma unroll
                for (int j = 0; j < T::VS; j++) bad |= nan_bytes(vw[j].x) | nan_bytes(vw[j].y) | nan_bytes(vw[j].z) | nan_bytes(vw[j].w);
                if (__any_sync(0xffffffffu, bad != 0)) {
                    uint32_t sb0, sb1;
                    sb0 = transpose8x8(seen[k2][0]), sb1 = transpose8x8(seen[k2][1]);
#pragma unroll
                    for (int j = 0; j < T::VS; j++) {
                        uint32_t w[4] = { vw[j].x, vw[j].y, vw[j].z, vw[j].w };
#pragma unroll
                        for (int half_ = 0; half_ < 2; half_++) {
                            uint32_t f[4];  // f16 ones at NaNs
#pragma unroll
                            for (int i2 = 0; i2 < 2; i2++) {
                                const uint32_t nb = nan_bytes(w[2 * half_ + i2]);
                                f[i2] = ((nb & 1u) ? 0x3c00u : 0u) | ((nb & 0x100u) ? 0x3c000000u : 0u);
                                f[2 + i2] = ((nb & 0x10000u) ? 0x3c00u : 0u) | ((nb & 0x1000000u) ? 0x3c000000u : 0u);
                                w[2 * half_ + i2] &= ~nb;
                            }
                            float hit[4] = {};
                            mma16816(hit, f[0], f[1], f[2], f[3], sb0, sb1);
#pragma unroll
                            for (int i2 = 0; i2 < 4; i2++)
                                if (hit[i2] > 0.0f) o[2 * j + half_][i2] = __int_as_float(0x7fffffff);
                        }
                        vw[j] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < T::VS; j++) {
                const uint32_t w[4] = { vw[j].x, vw[j].y, vw[j].z, vw[j].w };
#pragma unroll
                for (int half_ = 0; half_ < 2; half_++) {
                    const uint32_t a0 = e4m3x2_to_h2((uint16_t) w[2 * half_]), a2 = e4m3x2_to_h2((uint16_t) (w[2 * half_] >> 16));
                    const uint32_t a1 = e4m3x2_to_h2((uint16_t) w[2 * half_ + 1]), a3 = e4m3x2_to_h2((uint16_t) (w[2 * half_ + 1] >> 16));
                    mma16816(o[2 * j + half_], a0, a1, a2, a3, wb[k2][0], wb[k2][1]);
                }
            }
        }
        __syncwarp();
        fetch(i + 2 * T::AHEAD, true);
    }
    asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (!LONG) break;
    base += kTable * kSmallWarps;
    if (base >= c_hi) break;
    // the next of the range's blocks (the copies of zeros behind the last have landed, and no lane looks back)
    __syncwarp();
    look_up();
  }
    __syncthreads();  // the rings become the warps' outputs
    float (*sm_o)[8][HD + 4] = reinterpret_cast<float (*)[8][HD + 4]>(ring);

    // the warps' states to shared memory: [row][element]; element of (mt, half, g): 32 (mt/2) + 4 g + 2 (mt%2) + half
#pragma unroll
    for (int i = 0; i < 2; i++) {
        float x = l[i];
        x += __shfl_xor_sync(0xffffffffu, x, 4);
        x += __shfl_xor_sync(0xffffffffu, x, 8);
        x += __shfl_xor_sync(0xffffffffu, x, 16);
        if (g == 0) sm_ml[warp][2 * t + i][0] = m[i], sm_ml[warp][2 * t + i][1] = x;
    }
#pragma unroll
    for (int j = 0; j < T::VS; j++)
#pragma unroll
        for (int i = 0; i < 2; i++)
            *reinterpret_cast<float4 *>(&sm_o[warp][2 * t + i][32 * j + 4 * g]) =
                make_float4(o[2 * j][i], o[2 * j][2 + i], o[2 * j + 1][i], o[2 * j + 1][2 + i]);
    __syncthreads();
    const int live = min(kSmallRows, rows - row0);
    const size_t unit = ((size_t) b * a.row_tiles + tile) * kv.n_kv + h;
    float * part = a.part ? a.part + unit * a.chunks * (kSmallRows * T::PL) : nullptr;
    auto finish = [&](int r, int d, float4 x, float mm, float ll) {
        const float inv = ll > 0.0f ? 1.0f / ll : (ll == 0.0f ? 0.0f : ll);  // (NaN stays NaN)
        const int rr = row0 + r, tok = s.row0 + rr / a.group, qh = h * a.group + rr % a.group;
        store4(a.type, a.out_vec, a.out.p, (long long) tok * a.out.row + qh * a.out.head + d,
               make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
        if (a.lse && d == 0) a.lse[(size_t) tok * a.n_head + qh] = ll == 0.0f ? -INFINITY : kLn2 * (mm + log2f(ll));
    };
    for (int i = threadIdx.x; i < live * (HD / 4); i += 32 * kSmallWarps) {
        const int r = i / (HD / 4), d = i % (HD / 4) * 4;
        float mm = -INFINITY, ll = 0.0f;
        float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int w = 0; w < kSmallWarps; w++) mm = fmaxf(mm, sm_ml[w][r][0]);
        const float ref = mm == -INFINITY ? 0.0f : mm;
#pragma unroll
        for (int w = 0; w < kSmallWarps; w++) {
            const float f = exp2_approx(sm_ml[w][r][0] - ref);
            const float4 y = *reinterpret_cast<const float4 *>(&sm_o[w][r][d]);
            ll = fmaf(sm_ml[w][r][1], f, ll);
            x.x = fmaf(y.x, f, x.x), x.y = fmaf(y.y, f, x.y), x.z = fmaf(y.z, f, x.z), x.w = fmaf(y.w, f, x.w);
        }
        if (my_chunks == 1) {
            finish(r, d, x, mm, ll);
        } else {
            float * pp = part + ((size_t) chunk * kSmallRows + r) * T::PL;
            *reinterpret_cast<float4 *>(pp + d) = x;
            if (d == 0) *reinterpret_cast<float2 *>(pp + HD) = make_float2(mm, ll);
        }
    }
}

// Joins the ranges' results of the rows that have several, in the ranges' order: one warp a row, its loads
// of all ranges under way together. (A launch of its own: joined by the last range's CTA to finish, one
// row after another behind a fence and an atomic, 64 units of 40 rows and 6 ranges took 12 us.)
template <int HD>
__global__ void __launch_bounds__(256) kv8_attn_join_kernel(const AttnArgs a, int tile_rows) {
    start_after_previous();
    constexpr int PL = HD + 4, E = HD / 32;
    const Kv & kv = a.kv;
    const int lane = threadIdx.x & 31;
    const unsigned id = blockIdx.x * 8 + (threadIdx.x >> 5), r = id % (unsigned) tile_rows, unit = id / (unsigned) tile_rows;
    const int h = (int) (unit % (unsigned) kv.n_kv), bt = (int) (unit / (unsigned) kv.n_kv);
    const int tile = bt % a.row_tiles, b = bt / a.row_tiles;
    if (b >= kv.n_seq) return;
    const Seq s = load_seq(kv, b);
    if (s.slot < 0) return;
    const Span span = span_of(a, s, tile * tile_rows, tile_rows);
    const int row = tile * tile_rows + (int) r;
    if (row >= span.rows || span.chunks == 1) return;
    const float * part = a.part + ((size_t) unit * a.chunks * tile_rows + r) * PL;
    const size_t step = (size_t) tile_rows * PL;
    float m = -INFINITY, l = 0.0f, o[E] = {};
    for (int c0 = 0; c0 < span.chunks; c0 += 32) {
        const int n = min(32, span.chunks - c0);
        const float2 ml = lane < n ? *reinterpret_cast<const float2 *>(part + (c0 + lane) * step + HD) : make_float2(-INFINITY, 0.0f);
        float top = ml.x;
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
        top = fmaxf(top, m);
        const float ref = top == -INFINITY ? 0.0f : top, f = exp2_approx(ml.x - ref), keep = exp2_approx(m - ref);
        m = top;
        l *= keep;
#pragma unroll
        for (int e = 0; e < E; e++) o[e] *= keep;
        for (int c = 0; c < n; c += 8) {
            float v[8][E];
#pragma unroll
            for (int k = 0; k < 8; k++)
#pragma unroll
                for (int e = 0; e < E; e++) v[k][e] = c + k < n ? part[(c0 + c + k) * step + lane * E + e] : 0.0f;
#pragma unroll
            for (int k = 0; k < 8; k++) {
                const float w = __shfl_sync(0xffffffffu, f, (c + k) & 31), lc = __shfl_sync(0xffffffffu, ml.y, (c + k) & 31);
                if (c + k < n) {
                    l = fmaf(lc, w, l);
#pragma unroll
                    for (int e = 0; e < E; e++) o[e] = fmaf(v[k][e], w, o[e]);
                }
            }
        }
    }
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);  // (NaN stays NaN)
    const int tok = s.row0 + row / a.group, qh = h * a.group + row % a.group;
    uint16_t * out = static_cast<uint16_t *>(a.out.p) + (long long) tok * a.out.row + qh * a.out.head + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2) {
        const uint32_t x = a.type == BZB_F16 ? pack_half(o[e] * inv, o[e + 1] * inv) : pack_bf16(o[e] * inv, o[e + 1] * inv);
        if (a.out_vec) {
            *reinterpret_cast<uint32_t *>(out + e) = x;
        } else {
            out[e] = (uint16_t) x;
            out[e + 1] = (uint16_t) (x >> 16);
        }
    }
    if (a.lse && lane == 0) a.lse[(size_t) tok * a.n_head + qh] = l == 0.0f ? -INFINITY : kLn2 * (m + log2f(l));
}

// ---- host side ----

void fail(const std::string & what) { throw std::runtime_error(what); }

Kv view(const bzb_kv8_cache & c, const bzb_kv8_batch & b) {
    if (!c.pages || !c.scales || !c.page_table) fail("null pages, scales or page_table");
    if (c.head_dim != 64 && c.head_dim != 128) fail("head_dim must be 64 or 128");
    if (c.page_tokens < 16 || c.page_tokens > 256 || (c.page_tokens & (c.page_tokens - 1)))
        fail("page_tokens must be 16, 32, 64, 128 or 256");
    if (c.n_kv < 1 || c.n_kv > 4096) fail("n_kv must be 1 to 4096");
    if (c.n_pages < 1 || c.n_slots < 1 || c.max_pages < 1) fail("n_pages, n_slots and max_pages must be positive");
    if ((long long) c.max_pages * c.page_tokens > INT_MAX / 2) fail("max_pages x page_tokens is too large");
    const long long page = 2ll * c.n_kv * c.page_tokens * c.head_dim;
    if (c.page_stride < page || c.page_stride % 16) fail("page_stride must be a multiple of 16 and hold a page");
    if (c.scale_stride < 2ll * c.n_kv * (c.page_tokens / 16)) fail("scale_stride must hold a page's scales");
    if ((uintptr_t) c.pages % 16) fail("pages must be 16-byte aligned");
    if ((uintptr_t) c.scales % 4 || (uintptr_t) c.page_table % 4 || (uintptr_t) c.status % 4)
        fail("scales, page_table and status must be 4-byte aligned");
    if (b.n_seq < 0 || b.n_tok < 0 || b.max_new < 0 || b.max_len < 0) fail("negative batch size");
    if (b.n_seq > 0 && (!b.q_start || !b.kv_len)) fail("null q_start or kv_len");
    if (!b.slots && b.n_seq > c.n_slots) fail("more sequences than page table rows and no slots");
    if (b.max_len > (long long) c.max_pages * c.page_tokens) fail("max_len is more than a page table row holds");
    if (b.max_new > (1 << 24) || b.n_seq > (1 << 24)) fail("max_new and n_seq must be at most 2^24");
    Kv kv;
    kv.pages = static_cast<uint8_t *>(c.pages);
    kv.scales = c.scales;
    kv.table = c.page_table;
    kv.status = c.status;
    kv.page_stride = c.page_stride;
    kv.scale_stride = c.scale_stride;
    kv.n_pages = c.n_pages;
    kv.n_slots = c.n_slots;
    kv.max_pages = c.max_pages;
    kv.page_tokens = c.page_tokens;
    kv.page_shift = __builtin_ctz((unsigned) c.page_tokens);
    kv.n_kv = c.n_kv;
    kv.q_start = b.q_start;
    kv.kv_len = b.kv_len;
    kv.slots = b.slots;
    kv.n_seq = b.n_seq;
    kv.n_tok = b.n_tok;
    kv.max_new = b.max_new;
    kv.max_len = b.max_len;
    return kv;
}

// checks a row tensor and says whether groups of `n` elements of it are aligned to their size
bool check_rows(const bzb_kv8_rows & r, const char * name, int heads, int hd, bool f32_allowed, int n, int n_tok) {
    const std::string nm(name);
    if (r.type != BZB_F16 && r.type != BZB_BF16 && !(f32_allowed && r.type == BZB_F32))
        fail(nm + (f32_allowed ? ": type must be f32, f16 or bf16" : ": type must be f16 or bf16"));
    if (r.n_head != heads) fail(nm + ": must have " + std::to_string(heads) + " heads");
    if (n_tok > 0 && !r.data) fail(nm + ": null data");
    if (r.row_stride < 0 || r.head_stride < 0 || (heads > 1 && r.head_stride < hd) || r.row_stride > (1ll << 40) ||
        r.head_stride > (1ll << 40))
        fail(nm + ": strides must be non-negative and heads may not overlap");
    const int size = r.type == BZB_F32 ? 4 : 2;
    if ((uintptr_t) r.data % size) fail(nm + ": data is not aligned to its type");
    return (uintptr_t) r.data % (size * n) == 0 && r.row_stride % n == 0 && r.head_stride % n == 0;
}
// of an output: no two rows may share elements
void check_distinct(const bzb_kv8_rows & r, const char * name, int hd, int n_tok) {
    const long long span = (r.n_head - 1) * r.head_stride + hd;
    const bool by_row = r.row_stride >= span, by_head = r.row_stride >= hd && r.head_stride >= (n_tok - 1) * r.row_stride + hd;
    if (n_tok > 1 && !by_row && !by_head) fail(std::string(name) + ": rows overlap");
}

// append and read: (heads, blocks of 16 positions that max_new rows can touch, sequences)
dim3 row_grid(const Kv & kv, int heads, int per_cta) {
    const int blocks = (kv.max_new + 30) / 16;
    if (blocks > 65535 || kv.n_seq > 65535) fail("at most 65535 sequences and 2^20 - 31 rows of each in one call");
    return dim3((heads + per_cta - 1) / per_cta, blocks, kv.n_seq);
}

template <int HD, int TYPE>
void run_append(const AppendArgs & a, bool vec, cudaStream_t s) {
    const dim3 grid = row_grid(a.kv, a.n_head + 2 * a.kv.n_kv, RowMap<HD>::HEADS);
    launch_chained(vec ? kv8_append_kernel<HD, TYPE, true> : kv8_append_kernel<HD, TYPE, false>, grid, 32 * kRowWarps, 0, s, a);
}

template <int HD, int TYPE>
void run_read(const ReadArgs & a, cudaStream_t s) {
    const dim3 grid = row_grid(a.kv, 2 * a.kv.n_kv, RowMap<HD>::HEADS);
    launch_chained(kv8_read_kernel<HD, TYPE>, grid, 32 * kRowWarps, 0, s, a);
}

// How the rows and the cache of a call are cut up: by which kernel, in tiles of how many rows and ranges of how many
// blocks. Costs are in the time that a CTA of the few-row kernel takes for a block of 16 positions (0.15 us with
// head_dim 64, 0.18 us with 128, the SM's other CTAs beside it).
struct Plan {
    bool tile = false;      // kv8_tile.cu's kernel
    int rows = kSmallRows;  // rows of a CTA
    int row_tiles = 1, chunks = 1, chunk_blocks = 1;
    double cost = 0;
};
Plan cut(const bzb_kv8_cache & c, const bzb_kv8_batch & b, int n_head, int causal, int window, bool tile) {
    Plan p;
    p.tile = tile;
    if (tile) p.rows = kTileRows;
    const int group = n_head / c.n_kv;
    const long long rows = (long long) b.max_new * group;
    // (the kernels number them in an int, up to a tile past the last)
    if (rows > 1 << 30) fail("max_new x heads per kv head is too large (2^30 at most)");
    p.row_tiles = (int) std::max<long long>(1, (rows + p.rows - 1) / p.rows);
    // blocks that one CTA's rows look at: its tokens' windows, at any offset within a block
    long long keys = b.max_len;
    if (causal && window > 0) keys = std::min<long long>(keys, (long long) window + (p.rows + group - 1) / group + 1 + 15);
    const int blocks = (int) std::max<long long>(1, (keys + 15) / 16 + (window > 0 ? 1 : 0));
    if ((double) b.n_seq * c.n_kv * p.row_tiles > INT_MAX) {  // (more CTAs than a launch takes)
        p.cost = HUGE_VAL;
        return p;
    }
    const long long units = std::max<long long>(1, (long long) b.n_seq * c.n_kv * p.row_tiles);
    // What a CTA's start and end cost; the join's launch and each MB of its input, written and read back.
    const double start = tile ? 43 : 32, launch = 24, mb = tile ? 3.4 : 0;
    // (the many-row kernel's block: one tile of 128 rows, or two whose waits overlap)
    const double block = !tile ? 1 : rows <= 128 ? 1.7 : 2.1;
    const long long slots = tile ? 148 : 148ll * small_ctas(c.head_dim);
    for (long long n = 1; n <= blocks; n++) {
        int size = (int) ((blocks + n - 1) / n);
        if (tile) size = (size + 7) / 8 * 8;  // whole stages
        // whole waves of the CTAs that the SMs hold: the last range to end is what counts
        const double waves = (double) ((units * n + slots - 1) / slots);
        const double cost = waves * (block * size + start) + (n > 1 ? launch + mb * units * n * p.rows * (c.head_dim + 4) * 4e-6 : 0);
        if (p.cost == 0 || cost < p.cost) p.cost = cost, p.chunk_blocks = size;
        if (tile ? units * (n + 1) > slots || size <= 16 : units * n >= 6 * slots || size <= 8) break;
    }
    p.chunks = (blocks + p.chunk_blocks - 1) / p.chunk_blocks;
    // without ranges the last wave's CTAs run faster by themselves: half of what it lacks is no loss
    const double waves = (double) units / slots;
    if (p.chunks == 1 && !tile && waves > 1) p.cost *= (waves + std::ceil(waves)) / 2 / std::ceil(waves);
    return p;
}
// The kernel by the lower cost. Measured with 4 rows a token and kv head, 8 kv heads of 64, few | many rows' kernel in us,
// the choice starred: one sequence of 216 positions, 64 rows *5.6 | 10.9; 64 of 1012, 48 rows *58 | 80 and 96 rows
// 109 | *80; 16 of 2008, 32 rows *27 | 34 and 64 rows 46 | *34; 30 prompts of 16, 64 rows *12.7 | 18.2, of
// 64, 256 rows 47 | *21. Over 216 such calls the choice cost more than 10 % in five, 34 % at most. One row tile always
// goes to the few rows' kernel. (BZB_KV8_ATTENTION=few or many takes one of them for every call.)
Plan plan_of(const bzb_kv8_cache & c, const bzb_kv8_batch & b, int n_head, int causal, int window) {
    const Plan few = cut(c, b, n_head, causal, window, false), many = cut(c, b, n_head, causal, window, true);
    const char * e = std::getenv("BZB_KV8_ATTENTION");
    const bool tile = e && !std::strcmp(e, "few") ? false : e && !std::strcmp(e, "many") ? true : many.cost < few.cost;
    const Plan & p = tile ? many : few;
    if ((double) b.n_seq * c.n_kv * p.row_tiles * p.chunks > INT_MAX) fail("the batch is too large for one call");
    return p;
}

long long workspace_of(const bzb_kv8_cache & c, const bzb_kv8_batch & b, const Plan & p) {
    if (p.chunks == 1) return 0;
    return (long long) b.n_seq * p.row_tiles * c.n_kv * p.chunks * p.rows * (c.head_dim + 4) * 4;
}

template <int HD, bool LONG>
void run_small(const AttnArgs & a, cudaStream_t s) {
    const long long grid = (long long) a.kv.n_seq * a.row_tiles * a.chunks * a.kv.n_kv;
    constexpr int bytes = SmallTile<HD>::BYTES;
    static std::atomic<uint64_t> ready{ 0 };
    allow_shared_memory(kv8_attn_small_kernel<HD, LONG>, bytes, ready);
    launch_chained(kv8_attn_small_kernel<HD, LONG>, dim3((unsigned) grid), 32 * kSmallWarps, bytes, s, a);
}

// Checks them and gives the window that counts: none where no context fills it, so that positions less a window stay
// far inside an int.
int check_attention(const bzb_kv8_cache & c, const bzb_kv8_batch & b, int n_head, int causal, int window) {
    if (n_head < 1 || n_head % c.n_kv) fail("the query heads must be a multiple of n_kv");
    if (n_head > (1 << 16)) fail("too many query heads");
    if (window < 0) fail("window must not be negative");
    if (window > 0 && !causal) fail("a window needs causal attention");
    return window < b.max_len ? window : 0;
}

}  // namespace

namespace {
std::atomic<long long> debug_polls{ -1 };
}
void kv8_debug_polls(long long polls) { debug_polls.store(polls, std::memory_order_relaxed); }

void kv8_append(const bzb_kv8_cache & c, const bzb_kv8_batch & b, const bzb_kv8_rows * q, const bzb_kv8_rows & k,
                const bzb_kv8_rows & v, const bzb_kv8_rows * q_out, const float * q_norm, const float * k_norm, float eps,
                const float * rope, int rope_len, cudaStream_t s) {
    AppendArgs a;
    a.kv = view(c, b);
    if (!q != !q_out) fail("q and q_out come together");
    if (k.type != v.type || (q && q->type != k.type)) fail("q, k and v must be of one type");
    bool vec = check_rows(k, "k", c.n_kv, c.head_dim, true, 4, b.n_tok);
    vec &= check_rows(v, "v", c.n_kv, c.head_dim, true, 4, b.n_tok);
    a.n_head = 0;
    a.q = a.q_out = Rows{ nullptr, 0, 0 };
    a.q_out_type = BZB_F16;
    a.q_out_vec = false;
    if (q) {
        a.n_head = q->n_head;
        if (q->n_head < 1 || q->n_head > (1 << 16)) fail("q: between 1 and 65536 heads");
        vec &= check_rows(*q, "q", q->n_head, c.head_dim, true, 4, b.n_tok);
        a.q_out_vec = check_rows(*q_out, "q_out", q->n_head, c.head_dim, false, 4, b.n_tok);
        check_distinct(*q_out, "q_out", c.head_dim, b.n_tok);
        a.q = Rows{ q->data, q->row_stride, q->head_stride };
        a.q_out = Rows{ q_out->data, q_out->row_stride, q_out->head_stride };
        a.q_out_type = q_out->type;
    }
    if (!(eps >= 0.0f)) fail("eps must not be negative");
    if ((uintptr_t) q_norm % 4 || (uintptr_t) k_norm % 4) fail("q_norm and k_norm must be 4-byte aligned");
    if ((uintptr_t) rope % 16) fail("rope must be 16-byte aligned");
    if (rope && rope_len < b.max_len) fail("rope has fewer positions than max_len");
    if (b.n_seq == 0 || b.n_tok == 0 || b.max_new == 0 || b.max_len == 0) return;
    a.k = Rows{ k.data, k.row_stride, k.head_stride };
    a.v = Rows{ v.data, v.row_stride, v.head_stride };
    a.q_norm = q_norm;
    a.k_norm = k_norm;
    a.rope = reinterpret_cast<const float2 *>(rope);
    a.norm_vec = (uintptr_t) q_norm % 16 == 0 && (uintptr_t) k_norm % 16 == 0;
    a.eps = eps;
    if (c.head_dim == 64) {
        if (k.type == BZB_F32) run_append<64, BZB_F32>(a, vec, s);
        else if (k.type == BZB_F16) run_append<64, BZB_F16>(a, vec, s);
        else run_append<64, BZB_BF16>(a, vec, s);
    } else {
        if (k.type == BZB_F32) run_append<128, BZB_F32>(a, vec, s);
        else if (k.type == BZB_F16) run_append<128, BZB_F16>(a, vec, s);
        else run_append<128, BZB_BF16>(a, vec, s);
    }
}

void kv8_read(const bzb_kv8_cache & c, const bzb_kv8_batch & b, const bzb_kv8_rows & k_out, const bzb_kv8_rows & v_out,
              cudaStream_t s) {
    ReadArgs a;
    a.kv = view(c, b);
    a.vec = check_rows(k_out, "k_out", c.n_kv, c.head_dim, true, 4, b.n_tok);
    a.vec &= check_rows(v_out, "v_out", c.n_kv, c.head_dim, true, 4, b.n_tok);
    check_distinct(k_out, "k_out", c.head_dim, b.n_tok);
    check_distinct(v_out, "v_out", c.head_dim, b.n_tok);
    if (k_out.type != v_out.type) fail("k_out and v_out must be of one type");
    if (b.n_seq == 0 || b.n_tok == 0 || b.max_new == 0) return;
    a.k = Rows{ k_out.data, k_out.row_stride, k_out.head_stride };
    a.v = Rows{ v_out.data, v_out.row_stride, v_out.head_stride };
    if (c.head_dim == 64) {
        if (k_out.type == BZB_F32) run_read<64, BZB_F32>(a, s);
        else if (k_out.type == BZB_F16) run_read<64, BZB_F16>(a, s);
        else run_read<64, BZB_BF16>(a, s);
    } else {
        if (k_out.type == BZB_F32) run_read<128, BZB_F32>(a, s);
        else if (k_out.type == BZB_F16) run_read<128, BZB_F16>(a, s);
        else run_read<128, BZB_BF16>(a, s);
    }
}

long long kv8_attention_workspace(const bzb_kv8_cache & c, const bzb_kv8_batch & b, int n_head, int causal, int window) {
    view(c, b);
    window = check_attention(c, b, n_head, causal, window);
    if (b.n_seq == 0 || b.n_tok == 0 || b.max_new == 0) return 0;
    return workspace_of(c, b, plan_of(c, b, n_head, causal, window));
}

void kv8_attention(const bzb_kv8_cache & c, const bzb_kv8_batch & b, const bzb_kv8_rows & q, const bzb_kv8_rows & out,
                   float * lse, float scale, int causal, int window, void * workspace, long long workspace_bytes,
                   cudaStream_t s) {
    AttnArgs a;
    a.kv = view(c, b);
    if (q.n_head != out.n_head) fail("q and out must have the same heads");
    window = check_attention(c, b, q.n_head, causal, window);
    if (!std::isfinite(scale * kLog2e)) fail("scale must be finite");
    if (q.type != out.type) fail("q and out must be of one type");
    a.q_vec = check_rows(q, "q", q.n_head, c.head_dim, false, 8, b.n_tok);
    a.out_vec = check_rows(out, "out", q.n_head, c.head_dim, false, 8, b.n_tok);
    check_distinct(out, "out", c.head_dim, b.n_tok);
    if ((uintptr_t) lse % 4) fail("lse is misaligned");
    const bool empty = b.n_seq == 0 || b.n_tok == 0 || b.max_new == 0;
    const Plan p = empty ? Plan() : plan_of(c, b, q.n_head, causal, window);
    const long long need = workspace_of(c, b, p);
    if (need > 0 && (!workspace || workspace_bytes < need))
        fail("workspace of " + std::to_string(need) + " bytes needed, " + std::to_string(workspace ? workspace_bytes : 0) + " given");
    if (need > 0 && (uintptr_t) workspace % 16) fail("workspace must be 16-byte aligned");
    if (empty) return;
    a.q = Rows{ q.data, q.row_stride, q.head_stride };
    a.out = Rows{ out.data, out.row_stride, out.head_stride };
    a.lse = lse;
    a.scale2 = scale * kLog2e;
    a.n_head = q.n_head;
    a.group = q.n_head / c.n_kv;
    a.causal = causal != 0;
    a.window = window;
    a.type = q.type;
    a.row_tiles = p.row_tiles;
    a.chunks = p.chunks;
    a.chunk_blocks = p.chunk_blocks;
    a.part = static_cast<float *>(workspace);
    a.polls = debug_polls.load(std::memory_order_relaxed);
    if (p.tile) {
        launch_attn_tile(a, c.head_dim, s);
    } else if (c.head_dim == 64) {
        if (p.chunk_blocks > kShortRange) run_small<64, true>(a, s);
        else run_small<64, false>(a, s);
    } else {
        if (p.chunk_blocks > kShortRange) run_small<128, true>(a, s);
        else run_small<128, false>(a, s);
    }
    if (p.chunks > 1) {
        const long long warps = (long long) b.n_seq * p.row_tiles * c.n_kv * p.rows;
        if (warps > (long long) INT_MAX) fail("the batch is too large for one call");
        launch_chained(c.head_dim == 64 ? kv8_attn_join_kernel<64> : kv8_attn_join_kernel<128>, dim3((unsigned) ((warps + 7) / 8)), 256, 0, s, a,
                       p.rows);
    }
}

}  // namespace bzb
