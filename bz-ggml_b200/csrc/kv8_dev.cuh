// Device side shared by the kernels of the 8-bit paged key/value cache (kv8.cu, kv8_tile.cu).
//
// Numbers. A cached value is an e4m3 byte times its block's scale 2^e (16 positions of one head). e4m3
// converts to f16 exactly, so the attention kernels multiply the bytes as f16 and bring the scales in
// where they are one number for a whole block: 2^e of the keys multiplies the scores, 2^e of the
// values goes into the exponent of the weights (see attention below). A power of two costs e4m3 no
// precision, since its relative spacing is the same at every magnitude, and lets an append
// rescale a block's earlier values without rounding them again (except below the smallest normal).
#pragma once

#include "kv8.h"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>
#include <cstdint>
#include <stdexcept>
#include <string>
#include <utility>

namespace bzb {
namespace kv8 {


constexpr int kExpMin = -24, kExpMax = 40;
constexpr float kLog2e = 1.4426950408889634f, kLn2 = 0.6931471805599453f;

// what every kernel needs of the cache and the batch
struct Kv {
    uint8_t * pages;
    float * scales;
    const int * table;
    int * status;
    long long page_stride, scale_stride;
    int n_pages, n_slots, max_pages, page_tokens, page_shift, n_kv;
    const int * q_start, * kv_len, * slots;
    int n_seq, n_tok, max_new, max_len;
};

struct Rows {
    void * p;
    long long row, head;  // strides in elements
};

struct Seq {
    int row0, n, len, slot;  // first packed row, rows, cached positions, page table row (-1: skip the sequence)
};

__device__ __forceinline__ void complain(const Kv & kv, int what) {
    if (kv.status) atomicOr(kv.status, what);
}

__device__ __forceinline__ Seq load_seq(const Kv & kv, int b) {
    Seq s;
    s.row0 = kv.q_start[b];
    const int end = kv.q_start[b + 1];
    s.n = end - s.row0;
    s.len = kv.kv_len[b];
    s.slot = kv.slots ? kv.slots[b] : b;
    // (end and row0 are compared before their difference is used: it may overflow)
    if (s.row0 < 0 || end < s.row0 || end > kv.n_tok || s.n > kv.max_new || s.len < 0 || s.len > kv.max_len || s.slot < 0 ||
        s.slot >= kv.n_slots) {
        complain(kv, BZB_KV8_OUT_OF_RANGE);
        s.slot = -1;
    }
    return s;
}

// the page of block `blk` (16 positions) of a sequence, or -1
__device__ __forceinline__ int page_of(const Kv & kv, int slot, int blk) {
    const int pg = kv.table[(size_t) slot * kv.max_pages + (blk >> (kv.page_shift - 4))];
    if ((unsigned) pg >= (unsigned) kv.n_pages) {
        complain(kv, BZB_KV8_OUT_OF_RANGE);
        return -1;
    }
    return pg;
}
__device__ __forceinline__ uint8_t * block_ptr(const Kv & kv, int pg, int blk, int plane, int head, int hd) {
    const int at = (blk << 4) & (kv.page_tokens - 1);
    return kv.pages + pg * kv.page_stride + ((size_t) (plane * kv.n_kv + head) * kv.page_tokens + at) * hd;
}
__device__ __forceinline__ float * scale_ptr(const Kv & kv, int pg, int blk, int plane, int head) {
    const int per = kv.page_tokens >> 4;
    return kv.scales + pg * kv.scale_stride + (plane * kv.n_kv + head) * per + (blk & (per - 1));
}

__device__ __forceinline__ float pow2f(int e) { return __int_as_float((e + 127) << 23); }
__device__ __forceinline__ int exponent_of(float pow2) { return (__float_as_int(pow2) >> 23) - 127; }
// e such that a bf16 row of largest magnitude x, times 2^-e, fills f16 from the top: [2^14, 2^15)
__device__ __forceinline__ int row_exponent(float x) {
    return x < INFINITY && x > 0.0f ? max(-125, (__float_as_int(x) >> 23) - 127 - 14) : 0;
}
// smallest e with 448 2^e >= x (448 = 1.75 2^8), clamped; x >= 0 and finite
__device__ __forceinline__ int block_exponent(float x) {
    const int bits = __float_as_int(x);
    const int e = (bits >> 23) - 127 - 8 + ((bits & 0x7fffff) > 0x600000);
    return max(kExpMin, min(kExpMax, e));  // (subnormals and zero have exponent field 0: clamped)
}

// four floats -> four e4m3 bytes, nearest with ties to even; NaN stays NaN
__device__ __forceinline__ uint32_t to_e4m3x4(float a, float b, float c, float d) {
    uint16_t lo, hi;
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(lo) : "f"(b), "f"(a));
    asm("cvt.rn.satfinite.e4m3x2.f32 %0, %1, %2;" : "=h"(hi) : "f"(d), "f"(c));
    return (uint32_t) lo | ((uint32_t) hi << 16);
}
__device__ __forceinline__ uint32_t e4m3x2_to_h2(uint16_t v) {
    uint32_t r;
    asm("cvt.rn.f16x2.e4m3x2 %0, %1;" : "=r"(r) : "h"(v));
    return r;
}
__device__ __forceinline__ float4 e4m3x4_to_f4(uint32_t w) {
    const uint32_t lo = e4m3x2_to_h2((uint16_t) w), hi = e4m3x2_to_h2((uint16_t) (w >> 16));
    const float2 a = __half22float2(*reinterpret_cast<const half2 *>(&lo));
    const float2 b = __half22float2(*reinterpret_cast<const half2 *>(&hi));
    return make_float4(a.x, a.y, b.x, b.y);
}

// ---- four consecutive elements of a row; VEC: they are aligned to their size ----
template <bool VEC>
__device__ __forceinline__ float4 load4(const float * f) {
    if constexpr (VEC) return *reinterpret_cast<const float4 *>(f);
    return make_float4(f[0], f[1], f[2], f[3]);
}
__device__ __forceinline__ uint32_t pack_half(float a, float b) {
    const half2 h = __floats2half2_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ uint32_t pack_bf16(float a, float b) {
    const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
    return *reinterpret_cast<const uint32_t *>(&h);
}
__device__ __forceinline__ void store4(int type, bool vec, void * p, long long i, float4 x) {
    if (type == BZB_F32) {
        float * f = static_cast<float *>(p) + i;
        if (vec) *reinterpret_cast<float4 *>(f) = x;
        else f[0] = x.x, f[1] = x.y, f[2] = x.z, f[3] = x.w;
    } else {
        const uint2 u = type == BZB_F16 ? make_uint2(pack_half(x.x, x.y), pack_half(x.z, x.w))
                                        : make_uint2(pack_bf16(x.x, x.y), pack_bf16(x.z, x.w));
        uint16_t * h = static_cast<uint16_t *>(p) + i;
        if (vec) *reinterpret_cast<uint2 *>(h) = u;
        else {
            h[0] = (uint16_t) u.x, h[1] = (uint16_t) (u.x >> 16);
            h[2] = (uint16_t) u.y, h[3] = (uint16_t) (u.y >> 16);
        }
    }
}

// ---- attention ----
//
// For a row with scores s_j (in powers of two: scale log2(e) q.k_j) and values 2^{e_j} v_j, the weights
// are kept relative to M = max_j (s_j + e_j):
//   w_j = 2^(s_j + e_j - M) <= 1,  O = sum_j w_j v_j,  l = sum_j w_j 2^-e_j,  out = O / l,
//   log-sum-exp = ln 2 (M + log2 l),
// so the f16 weights of the second product carry the values' block scales, and the sum undoes them
// in f32 (|e| <= 40: no weight that matters underflows). M, l and O are f32 and updated
// block by block. The weights are f16 because the cached bytes are exact in it and one product then takes both:
// 2^-11 of each weight, which leaves the result 10 to 35 % further from 64 bits than f32 weights would (f16 rows, 2.3e-4 to 2.7e-4
// against 2.1e-4, most of it the result's own rounding). l sums them before they are rounded.
struct AttnArgs {
    Kv kv;
    Rows q, out;
    float * lse;
    float scale2;  // scale log2(e)
    int n_head, group, causal, window;
    int type;      // of q and out
    bool q_vec, out_vec;
    int row_tiles, chunks, chunk_blocks;  // chunk_blocks: blocks of 16 positions in a range
    long long polls;  // of a wait in the many rows' kernel before it gives up (negative: the default)
    float * part;  // ranges' results, when there are several: [unit][range][row][head_dim, maximum, sum, 0, 0]
};

// one past the last key of the row at position pos; none for a padding row (zero or less)
__device__ __forceinline__ int keys_end(const AttnArgs & a, const Seq & s, int pos) {
    return a.causal ? pos + 1 : pos < 0 ? 0 : s.len;
}

// The blocks of the cache that a tile's rows look at, and the ranges they are cut into.
struct Span {
    int first, rows;             // position of the sequence's first row (negative: padding); its (token, head) rows
    int blk_lo, blk_hi, chunks;  // blocks of 16 keys [blk_lo, blk_hi) of any row; ranges, at least one
};
__device__ __forceinline__ Span span_of(const AttnArgs & a, const Seq & s, int row0, int tile_rows) {
    Span p;
    p.first = s.len - s.n;
    p.rows = s.n * a.group;
    const int pos_lo = p.first + row0 / a.group, pos_hi = p.first + min(p.rows - 1, row0 + tile_rows - 1) / a.group;
    const int key_hi = max(0, a.causal ? pos_hi + 1 : s.len), key_lo = a.window > 0 ? max(0, pos_lo - a.window + 1) : 0;
    p.blk_lo = key_lo >> 4;
    p.blk_hi = (key_hi + 15) >> 4;
    p.chunks = max(1, (p.blk_hi - p.blk_lo + a.chunk_blocks - 1) / a.chunk_blocks);
    return p;
}


// (2^-22 relative, below f16's rounding by far; less than 2^-126 becomes zero, beside a largest weight of about one)
__device__ __forceinline__ float exp2_approx(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
// bytes of w that are e4m3 NaN (0x7f or 0xff) become 0xff, the others 0
__device__ __forceinline__ uint32_t nan_bytes(uint32_t w) { return __vcmpeq4(w & 0x7f7f7f7fu, 0x7f7f7f7fu); }


// a kernel's shared-memory limit, set once for each device (`ready`: one bit per device that has it)
template <typename K>
void allow_shared_memory(K kernel, int bytes, std::atomic<uint64_t> & ready) {
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    const uint64_t bit = 1ull << (dev & 63);
    if (e == cudaSuccess && (ready.load(std::memory_order_acquire) & bit) && dev < 64) return;
    if (e == cudaSuccess) e = cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
    if (e != cudaSuccess) throw std::runtime_error(std::string("shared memory: ") + cudaGetErrorString(e));
    ready.fetch_or(bit, std::memory_order_release);
}

// Launches with programmatic dependent launch: the kernel's CTAs may take their places while the kernel before it in
// the stream still runs, and begin each with start_after_previous(), before which they touch no memory.
template <typename... P, typename... A>
void launch_chained(void (*kernel)(P...), dim3 grid, int threads, int shared, cudaStream_t s, A &&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = shared;
    cfg.stream = s;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    const cudaError_t e = cudaLaunchKernelEx(&cfg, kernel, std::forward<A>(args)...);
    if (e != cudaSuccess) throw std::runtime_error(std::string("launch: ") + cudaGetErrorString(e));
}
// Lets the next kernel's CTAs be placed, then waits until the kernels before this one are done and their writes visible.
// What they may have written -- which for a caller's buffers is everything -- is read with ordinary loads:
// the compiler is free to move non-coherent ones (__ldg) ahead of this wait.
__device__ __forceinline__ void start_after_previous() {
    asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
    asm volatile("griddepcontrol.wait;" ::: "memory");
}

// the attention of many rows (kv8_tile.cu): rows of a kv head in tiles of kTileRows
constexpr int kTileRows = 256;
void launch_attn_tile(AttnArgs a, int head_dim, cudaStream_t s);

}  // namespace kv8
}  // namespace bzb
