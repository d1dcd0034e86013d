// Attention of many rows over the 8-bit paged cache on the tensor cores (tcgen05): prompts, and whatever
// else has more rows to a kv head than the few-row kernel of kv8.cu is made for.
//
// One CTA takes up to 256 rows of one kv head -- (token, head of the group) pairs, so the group shares
// the cache's tiles -- as two M = 128 tiles, and walks its keys 128 at a time:
//   producers (4 warps)  bytes of 128 keys and values from global memory to registers, one tile ahead;
//                        converted to f16 into shared memory in the MMAs' swizzled layout (two stages),
//                        the blocks' scales beside them;
//   MMA (1 thread)       S_i = Q_i K^T into tensor memory, O_i += W_i V with the weights W_i read from
//                        tensor memory;
//   softmax (4 warps a tile, one row a thread)  S_i from tensor memory, the running maximum and sum,
//                        the weights back to tensor memory as f16.
// While one tile's rows are in the softmax, the other's products run. The exponentials bound it: 16 a
// clock and SM against 4096 multiply-adds, so for head_dim 64 a tile of 128 x 128 scores costs 1024 clocks there
// and 512 in the MMAs; no key is converted more than once for 256 rows.
// O is rescaled only when a row's maximum has grown by more than 2^8 since the last time (the
// weights then stay below 2^8, which f16 holds as precisely), so that the tile of outputs in
// tensor memory is seldom read back.
#include "kv8_dev.cuh"
#include "tc_ptx.cuh"

#include <climits>
#include <stdexcept>
#include <string>

namespace bzb {
namespace kv8 {
namespace {

using namespace tc;

constexpr int kKeys = 128;                 // keys of a tile
constexpr int kProducers = 4, kSoftmax = 8;
constexpr int kMmaWarp = kSoftmax + kProducers;
constexpr int kTileThreads = 32 * (kMmaWarp + 1);
constexpr float kSlack = 8.0f;             // how far (powers of two) weights may exceed 1 before O is rescaled

template <int HD>
struct Smem {
    static constexpr int kHalf = kKeys * 128;          // 128 rows x 64 f16, 128-byte swizzle
    static constexpr int kQ = 128 * HD * 2, kK = kKeys * HD * 2, kV = kKeys * HD * 2;
    static constexpr int oQ = 0, oK = 2 * kQ, oV = oK + 2 * kK, oEnd = oV + 2 * kV;
    static constexpr size_t kBytes = 1024 + oEnd;
    // tensor memory columns: scores of the two tiles, outputs; the weights of head_dim 64 have
    // columns of their own, those of head_dim 128 lie over the scores they came from
    static constexpr int cO = 2 * kKeys, cW = HD == 64 ? cO + 2 * HD : 0;
    static constexpr int kWStride = HD == 64 ? kKeys / 2 : kKeys;
    static constexpr bool kOver = HD != 64;
};

struct Shared {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], s_full[2], w_full[2], o_full[2], pv_done[2], drain;
    uint64_t c_full[4], n_full[4];  // scale[] and nan_v[] of a tile (rings of four: see the producers)
    uint32_t tmem;
    int err;
    int last;
    int nan_v[4][kProducers];   // a producer warp found NaN values in this tile (only where it looked)
    float scale[4][8][4];       // per block of 16 keys: scale of the keys, exponent of the values' scale, 2^-it
    float unit[2][128];         // power of two taken out of each query row
};

__device__ __forceinline__ void ld32(uint32_t addr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
          "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]),
          "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]),
          "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(addr));
}
__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[16]) { tmem_st16(addr, r); }

// a whole warp's bounded wait: all lanes succeed, or all take it as failed
__device__ __forceinline__ bool warp_wait(uint64_t * bar, uint32_t parity, int * err) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, err));
}

// The part of the cache and the rows that a CTA works on.
struct Work {
    int h, tile, chunk, b, my_chunks;
    Seq s;
    int first, rows, row0;       // the sequence's first row's position, its (token, head) rows, this tile's first
    int full_lo, full_hi;        // keys that every row of the tile sees
    int blk0, n_tiles, blk_hi;   // first block, tiles of 128 keys, blocks that exist
};

__device__ __forceinline__ bool find_work(const AttnArgs & a, Work & w) {
    const Kv & kv = a.kv;
    long long id = blockIdx.x;
    w.h = (int) (id % kv.n_kv);
    id /= kv.n_kv;
    w.chunk = (int) (id % a.chunks);
    id /= a.chunks;
    // the last tiles of causal sequences have the most keys: they start first
    w.b = (int) (id % kv.n_seq);
    w.tile = a.row_tiles - 1 - (int) (id / kv.n_seq);
    w.s = load_seq(kv, w.b);
    if (w.s.slot < 0) return false;
    w.rows = w.s.n * a.group;
    w.row0 = w.tile * kTileRows;
    if (w.row0 >= w.rows) return false;
    w.first = w.s.len - w.s.n;
    const int pos_lo = w.first + w.row0 / a.group, pos_hi = w.first + min(w.rows - 1, w.row0 + kTileRows - 1) / a.group;
    const int key_hi = max(0, a.causal ? pos_hi + 1 : w.s.len), key_lo = a.window > 0 ? max(0, pos_lo - a.window + 1) : 0;
    w.full_hi = a.causal ? pos_lo + 1 : w.s.len;
    w.full_lo = a.window > 0 ? max(0, pos_hi - a.window + 1) : 0;
    const int lo = key_lo >> 4;
    w.blk_hi = (key_hi + 15) >> 4;
    w.my_chunks = max(1, (w.blk_hi - lo + a.chunk_blocks - 1) / a.chunk_blocks);
    if (w.chunk >= w.my_chunks) return false;
    w.blk0 = lo + w.chunk * a.chunk_blocks;
    w.blk_hi = min(w.blk_hi, w.blk0 + a.chunk_blocks);
    w.n_tiles = max(0, (w.blk_hi - w.blk0 + 7) / 8);
    return true;
}

// 8 consecutive query elements as f16 pairs times f (f16 rows: unchanged)
__device__ __forceinline__ uint4 load_q8(const AttnArgs & a, long long i, float (&x)[8]) {
    const uint16_t * p = static_cast<const uint16_t *>(a.q.p) + i;
    uint4 u;
    if (a.q_vec) {
        u = *reinterpret_cast<const uint4 *>(p);
    } else {
        uint32_t w[4];
#pragma unroll
        for (int j = 0; j < 4; j++) w[j] = (uint32_t) p[2 * j] | ((uint32_t) p[2 * j + 1] << 16);
        u = make_uint4(w[0], w[1], w[2], w[3]);
    }
    if (a.type == BZB_BF16) {
        const uint32_t w[4] = { u.x, u.y, u.z, u.w };
#pragma unroll
        for (int j = 0; j < 4; j++) x[2 * j] = __uint_as_float(w[j] << 16), x[2 * j + 1] = __uint_as_float(w[j] & 0xffff0000u);
    }
    return u;
}

// a softmax warp's 32 query rows into the swizzled tile; rows that do not exist become zero
template <int HD>
__device__ __forceinline__ void load_queries(const AttnArgs & a, const Work & w, Shared & sh, uint8_t * sq, int tile, int quarter, int lane) {
    constexpr int LPR = HD / 8, RPP = 32 / LPR;  // lanes of a row, rows of a pass
    const int c = lane % LPR;
    for (int p = 0; p < LPR; p++) {
        const int r = quarter * 32 + p * RPP + lane / LPR, rr = w.row0 + tile * 128 + r;
        uint4 u = make_uint4(0, 0, 0, 0);
        float unit = 1.0f;
        float x[8] = {};
        if (rr < w.rows)
            u = load_q8(a, (long long) (w.s.row0 + rr / a.group) * a.q.row + (w.h * a.group + rr % a.group) * a.q.head + 8 * c, x);
        if (a.type == BZB_BF16) {
            // bf16 may lie outside f16: the row is brought to about [1, 2) by a power of two
            float amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 8; j++) amax = fmaxf(amax, fabsf(x[j]));
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            const int e = amax < INFINITY && amax > 0.0f ? min(126, max(-125, (__float_as_int(amax) >> 23) - 127)) : 0;
            unit = pow2f(e);
            const float f = pow2f(-e);
            u = make_uint4(pack_half(x[0] * f, x[1] * f), pack_half(x[2] * f, x[3] * f), pack_half(x[4] * f, x[5] * f),
                           pack_half(x[6] * f, x[7] * f));
        }
        *reinterpret_cast<uint4 *>(sq + (c / 8) * Smem<HD>::kHalf + r * 128 + (((c % 8) ^ (r & 7)) << 4)) = u;
        if (c == 0) sh.unit[tile][r] = unit;
    }
}

// ---- producers: tile after tile of keys and values, bytes to swizzled f16 ----
template <int HD>
struct Producer {
    static constexpr int NK = HD / 16;  // 16-byte pieces of keys a thread takes of a tile (128 threads)
    static constexpr int NV = HD / 32;  // 32-byte pieces (two patches) of values
    uint4 k[NK], v[NV][2];
    const AttnArgs & a;
    const Work & w;
    int tid, lane;

    // (page of each block, one block per lane 0..7; -1 past the last)
    __device__ int pages(int j) const {
        const int blk = w.blk0 + 8 * j + (lane & 7);
        if (j >= w.n_tiles || blk >= w.blk_hi) return -1;
        return max(page_of(a.kv, w.s.slot, blk), 0);
    }
    // row of the tile and 16-byte piece of the row: lanes of a store phase fall on different banks
    __device__ static void key_piece(int i, int & row, int & c) {
        if (HD == 64) {
            row = i >> 2, c = i & 3;
        } else {
            c = (i & 3) | ((i >> 3) & 1) << 2;
            row = ((i >> 2) & 1) | (i >> 4) << 1;
        }
    }
    // block of the tile, group of 4 elements, pair of position groups
    __device__ static void value_piece(int i, int & kb, int & q, int & u) {
        u = i & 1;
        q = (i >> 3) & (HD / 4 - 1);
        kb = ((i >> 1) & 3) | (i / (HD / 4 * 8)) << 2;
    }
    __device__ void load_k(int j, int pg) {
#pragma unroll
        for (int i = 0; i < NK; i++) {
            int row, c;
            key_piece(i * 128 + tid, row, c);
            const int p = __shfl_sync(0xffffffffu, pg, row >> 4);
            k[i] = make_uint4(0, 0, 0, 0);
            if (p >= 0) {
                const uint8_t * src = block_ptr(a.kv, p, w.blk0 + 8 * j + (row >> 4), 0, w.h, HD) + (row & 15) * HD + 16 * c;
                k[i] = __ldg(reinterpret_cast<const uint4 *>(src));
            }
        }
    }
    __device__ void load_v(int j, int pg) {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            int kb, q, u;
            value_piece(i * 128 + tid, kb, q, u);
            const int p = __shfl_sync(0xffffffffu, pg, kb);
            v[i][0] = v[i][1] = make_uint4(0, 0, 0, 0);
            if (p >= 0) {
                const uint4 * src = reinterpret_cast<const uint4 *>(block_ptr(a.kv, p, w.blk0 + 8 * j + kb, 1, w.h, HD) + q * 64 + u * 32);
                v[i][0] = __ldg(src);
                v[i][1] = __ldg(src + 1);
            }
        }
    }
    __device__ void store_k(uint8_t * dst) const {
#pragma unroll
        for (int i = 0; i < NK; i++) {
            int row, c;
            key_piece(i * 128 + tid, row, c);
            const uint32_t x[4] = { k[i].x, k[i].y, k[i].z, k[i].w };
            uint32_t y[8];
#pragma unroll
            for (int m = 0; m < 4; m++) y[2 * m] = e4m3x2_to_h2((uint16_t) x[m]), y[2 * m + 1] = e4m3x2_to_h2((uint16_t) (x[m] >> 16));
            uint8_t * r = dst + (c >> 2) * Smem<HD>::kHalf + row * 128;
            const int c0 = (c & 3) * 2;
            *reinterpret_cast<uint4 *>(r + ((c0 ^ (row & 7)) << 4)) = make_uint4(y[0], y[1], y[2], y[3]);
            *reinterpret_cast<uint4 *>(r + (((c0 + 1) ^ (row & 7)) << 4)) = make_uint4(y[4], y[5], y[6], y[7]);
        }
    }
    // NaNs of a tile that some row does not see in whole are stored as zero; says whether there were any
    __device__ bool clear_nan() {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < NV; i++)
#pragma unroll
            for (int m = 0; m < 2; m++) {
                uint4 & x = v[i][m];
                const uint4 n = make_uint4(nan_bytes(x.x), nan_bytes(x.y), nan_bytes(x.z), nan_bytes(x.w));
                any |= n.x | n.y | n.z | n.w;
                x = make_uint4(x.x & ~n.x, x.y & ~n.y, x.z & ~n.z, x.w & ~n.w);
            }
        return any != 0;
    }
    __device__ void store_v(uint8_t * dst) const {
#pragma unroll
        for (int i = 0; i < NV; i++) {
            int kb, q, u;
            value_piece(i * 128 + tid, kb, q, u);
            const uint32_t x[4] = { v[i][0].x, v[i][0].y, v[i][0].z, v[i][0].w }, y[4] = { v[i][1].x, v[i][1].y, v[i][1].z, v[i][1].w };
            const int chunk = (kb & 3) * 2 + u;
#pragma unroll
            for (int m = 0; m < 4; m++) {
                const int d = 4 * q + m;
                *reinterpret_cast<uint4 *>(dst + (kb >> 2) * (HD * 128) + d * 128 + ((chunk ^ (d & 7)) << 4)) =
                    make_uint4(e4m3x2_to_h2((uint16_t) x[m]), e4m3x2_to_h2((uint16_t) (x[m] >> 16)),
                               e4m3x2_to_h2((uint16_t) y[m]), e4m3x2_to_h2((uint16_t) (y[m] >> 16)));
            }
        }
    }
};

template <int HD>
__global__ void __launch_bounds__(kTileThreads, 1) kv8_attn_tile_kernel(const AttnArgs a) {
    using M = Smem<HD>;
    extern __shared__ uint8_t raw[];
    __shared__ Shared sh;
    Work w;
    if (!find_work(a, w)) return;  // (the whole CTA)
    uint8_t * base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles = w.rows - w.row0 > 128 ? 2 : 1;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.k_full[i], kProducers);
            mbar_init(&sh.v_full[i], kProducers);
            mbar_init(&sh.k_empty[i], 1);
            mbar_init(&sh.v_empty[i], 1);
            mbar_init(&sh.s_full[i], 1);
            mbar_init(&sh.w_full[i], 4);
            mbar_init(&sh.o_full[i], 1);
            mbar_init(&sh.pv_done[i], 1);
        }
        for (int i = 0; i < 4; i++) {
            mbar_init(&sh.c_full[i], 1);
            mbar_init(&sh.n_full[i], kProducers);
        }
        mbar_init(&sh.drain, 1);
        sh.err = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) tmem_alloc(&sh.tmem, 512);
    if (warp < 4 * tiles) {
        load_queries<HD>(a, w, sh, base + M::oQ + (warp >> 2) * M::kQ, warp >> 2, warp & 3, lane);
        fence_proxy_async();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const int n = w.n_tiles;
    int * err = &sh.err;
    constexpr int PL = HD + 4;
    const size_t unit = ((size_t) w.b * a.row_tiles + w.tile) * a.kv.n_kv + w.h;
    float * part = w.my_chunks > 1 ? a.part + unit * a.chunks * ((size_t) kTileRows * PL) : nullptr;

    auto finish = [&](int r, int d, float4 x, float inv) {
        const int rr = w.row0 + r;
        store4(a.type, a.out_vec, a.out.p,
               (long long) (w.s.row0 + rr / a.group) * a.out.row + (w.h * a.group + rr % a.group) * a.out.head + d,
               make_float4(x.x * inv, x.y * inv, x.z * inv, x.w * inv));
    };
    auto inverse = [](float l) { return l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l); };  // (NaN stays NaN)
    auto put_lse = [&](int r, float m, float l) {
        const int rr = w.row0 + r;
        if (a.lse)
            a.lse[(size_t) (w.s.row0 + rr / a.group) * a.n_head + w.h * a.group + rr % a.group] = l == 0.0f ? -INFINITY : kLn2 * (m + log2f(l));
    };

    if (warp < kSoftmax) {
        const int i = warp >> 2, r = threadIdx.x & 127, rr = w.row0 + 128 * i + r;
        if (i < tiles) {
            const uint32_t lanes = (uint32_t) (warp & 3) << 21;  // tensor memory lanes 32 (warp % 4) ..
            const uint32_t ts = tmem + lanes + i * kKeys, tw = tmem + lanes + M::cW + i * M::kWStride, to = tmem + lanes + M::cO + i * HD;
            const bool real = rr < w.rows;
            const int pos = w.first + rr / a.group;
            const int hi = !real ? INT_MAX : a.causal ? pos + 1 : w.s.len, lo = real && a.window > 0 ? pos - a.window + 1 : INT_MIN;
            const int warp_hi = __reduce_min_sync(0xffffffffu, hi), warp_lo = __reduce_max_sync(0xffffffffu, lo);
            const float coef = a.scale2 * sh.unit[i][r];
            float m = -INFINITY, l = 0.0f;
            uint32_t nan_d[HD / 32] = {};
            bool ok = true;
            for (int j = 0; j < n; j++) {
                const int key0 = (w.blk0 + 8 * j) << 4;
                ok = warp_wait(&sh.c_full[j & 3], (j >> 2) & 1, err) && warp_wait(&sh.s_full[i], j & 1, err);
                if (!ok) break;
                tc_fence_after();
                const bool whole = key0 >= warp_lo && key0 + kKeys <= warp_hi;
                float top = -INFINITY;
#pragma unroll 1
                for (int c = 0; c < 4; c++) {
                    uint32_t x[32];
                    ld32(ts + 32 * c, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int g = 0; g < 2; g++) {
                        const float ks = sh.scale[j & 3][2 * c + g][0] * coef, ev = sh.scale[j & 3][2 * c + g][1];
#pragma unroll
                        for (int t = 0; t < 16; t++) {
                            float s = fmaf(__uint_as_float(x[16 * g + t]), ks, ev);
                            if (!whole) {
                                const int key = key0 + 32 * c + 16 * g + t;
                                if (key < lo || key >= hi) s = -INFINITY;
                            }
                            top = fmaxf(top, s);
                        }
                    }
                }
                // (the first maximum is taken as it is; -inf while a row has seen no key)
                const bool grow = top > m + kSlack || (m == -INFINITY && top > m);
                if (__any_sync(0xffffffffu, grow)) {
                    const float f = grow ? exp2_approx(m - top) : 1.0f;
                    if (grow) m = top;
                    l *= f;
                    if (j > 0) {
#pragma unroll 1
                        for (int c = 0; c < HD / 16; c++) {
                            float y[16];
                            tmem_ld16(to + 16 * c, y);
                            tmem_wait_ld();
                            uint32_t z[16];
#pragma unroll
                            for (int t = 0; t < 16; t++) z[t] = __float_as_uint(y[t] * f);
                            st16(to + 16 * c, z);
                        }
                    }
                }
                const float ref = m == -INFINITY ? 0.0f : m;
#pragma unroll 1
                for (int c = 0; c < 4; c++) {
                    uint32_t x[32], p[16];
                    ld32(ts + 32 * c, x);
                    tmem_wait_ld();
#pragma unroll
                    for (int g = 0; g < 2; g++) {
                        const float ks = sh.scale[j & 3][2 * c + g][0] * coef, ev = sh.scale[j & 3][2 * c + g][1] - ref;
                        const float inv = sh.scale[j & 3][2 * c + g][2];
                        float sum = 0.0f;
#pragma unroll
                        for (int t = 0; t < 16; t += 2) {
                            float s0 = fmaf(__uint_as_float(x[16 * g + t]), ks, ev), s1 = fmaf(__uint_as_float(x[16 * g + t + 1]), ks, ev);
                            if (!whole) {
                                const int key = key0 + 32 * c + 16 * g + t;
                                if (key < lo || key >= hi) s0 = -INFINITY;
                                if (key + 1 < lo || key + 1 >= hi) s1 = -INFINITY;
                            }
                            s0 = exp2_approx(s0), s1 = exp2_approx(s1);
                            sum += s0 + s1;
                            p[8 * g + t / 2] = pack_half(s0, s1);
                        }
                        l = fmaf(sum, inv, l);
                    }
                    st16(tw + 16 * c, p);
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) mbar_arrive(&sh.w_full[i]);
                // NaN values in a tile that some row of the CTA does not see in whole: the producers left them
                // out; the rows that see one get it at the end
                if (key0 < w.full_lo || key0 + kKeys > w.full_hi) {
                    ok = warp_wait(&sh.n_full[j & 3], (j >> 2) & 1, err);
                    if (!ok) break;
                    bool any = false;
                    for (int q = 0; q < kProducers; q++) any |= sh.nan_v[j & 3][q] != 0;
                    if (any && real)
                        for (int key = max(lo, key0); key < min(hi, key0 + kKeys) && (key >> 4) < w.blk_hi; key++) {
                            const int pg = max(page_of(a.kv, w.s.slot, key >> 4), 0);
                            const uint8_t * src = block_ptr(a.kv, pg, key >> 4, 1, w.h, HD) + ((key >> 2) & 3) * 16 + (key & 3);
#pragma unroll
                            for (int d32 = 0; d32 < HD / 32; d32++)
#pragma unroll 1
                                for (int d = 0; d < 32; d++)
                                    if ((src[(8 * d32 + d / 4) * 64 + (d & 3) * 4] & 0x7f) == 0x7f) nan_d[d32] |= 1u << d;
                        }
                    __syncwarp();
                }
            }
            if (ok && n > 0) ok = warp_wait(&sh.o_full[i], 0, err);
            if (ok) {
                tc_fence_after();
                const float inv = inverse(l);
                float * pp = part ? part + ((size_t) w.chunk * kTileRows + 128 * i + r) * PL : nullptr;
#pragma unroll
                for (int c = 0; c < HD / 16; c++) {
                    float y[16];
                    if (n > 0) {
                        tmem_ld16(to + 16 * c, y);
                        tmem_wait_ld();
                    }
#pragma unroll
                    for (int t = 0; t < 16; t++) {
                        if (n == 0) y[t] = 0.0f;
                        if (nan_d[c / 2] >> (16 * (c & 1) + t) & 1) y[t] = __int_as_float(0x7fffffff);
                    }
                    if (real) {
#pragma unroll
                        for (int t = 0; t < 16; t += 4) {
                            const float4 x = make_float4(y[t], y[t + 1], y[t + 2], y[t + 3]);
                            if (part) *reinterpret_cast<float4 *>(pp + 16 * c + t) = x;
                            else finish(128 * i + r, 16 * c + t, x, inv);
                        }
                    }
                    __syncwarp();
                }
                if (real) {
                    if (part) *reinterpret_cast<float2 *>(pp + HD) = make_float2(m, l);
                    else put_lse(128 * i + r, m, l);
                }
            }
            tc_fence_before();
        }
    } else if (warp < kMmaWarp) {
        Producer<HD> p = { {}, {}, a, w, (int) threadIdx.x - 32 * kSoftmax, lane };
        const int pw = warp - kSoftmax;
        int pg = p.pages(0), next = p.pages(1);
        if (n > 0) p.load_k(0, pg), p.load_v(0, pg);
        for (int j = 0; j < n; j++) {
            const int st = j & 1, key0 = (w.blk0 + 8 * j) << 4;
            if (!warp_wait(&sh.k_empty[st], ((j >> 1) & 1) ^ 1, err)) break;
            p.store_k(base + M::oK + st * M::kK);
            if (pw == 0 && lane < 8) {
                const bool there = pg >= 0;
                const int blk = w.blk0 + 8 * j + lane;
                const float vs = there ? __ldg(scale_ptr(a.kv, pg, blk, 1, w.h)) : 1.0f;
                sh.scale[j & 3][lane][0] = there ? __ldg(scale_ptr(a.kv, pg, blk, 0, w.h)) : 0.0f;
                sh.scale[j & 3][lane][1] = (float) exponent_of(vs);
                sh.scale[j & 3][lane][2] = 1.0f / vs;
            }
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) {
                mbar_arrive(&sh.k_full[st]);
                // scale[] and nan_v[] are rings of four: tile j + 4 is stored when the products of tile j + 2
                // are done, which every softmax warp's weights of tile j + 1 come before
                if (pw == 0) mbar_arrive(&sh.c_full[j & 3]);
            }
            if (j + 1 < n) p.load_k(j + 1, next);
            if (!warp_wait(&sh.v_empty[st], ((j >> 1) & 1) ^ 1, err)) break;
            bool bad = false;
            if (key0 < w.full_lo || key0 + kKeys > w.full_hi) bad = p.clear_nan();
            bad = __any_sync(0xffffffffu, bad);
            if (lane == 0) sh.nan_v[j & 3][pw] = bad;
            p.store_v(base + M::oV + st * M::kV);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.v_full[st]), mbar_arrive(&sh.n_full[j & 3]);
            if (j + 1 < n) p.load_v(j + 1, next);
            pg = next;
            next = p.pages(j + 2);
        }
    } else if (lane == 0 && n > 0) {
        constexpr uint32_t idesc_s = (1u << 4) | ((uint32_t) (kKeys >> 3) << 17) | (8u << 24);
        constexpr uint32_t idesc_o = (1u << 4) | ((uint32_t) (HD >> 3) << 17) | (8u << 24);
        const uint32_t q0 = smem_u32(base + M::oQ), k0 = smem_u32(base + M::oK), v0 = smem_u32(base + M::oV);
        auto scores = [&](int i, int j) {
#pragma unroll
            for (int kk = 0; kk < HD / 16; kk++) {
                const uint32_t at = (kk / 4) * M::kHalf + (kk % 4) * 32;
                umma_f16(tmem + i * kKeys, sw128_desc(q0 + i * M::kQ + at), sw128_desc(k0 + (j & 1) * M::kK + at), idesc_s, kk > 0);
            }
            umma_commit(&sh.s_full[i]);
        };
        bool ok = mbar_wait(&sh.k_full[0], 0, err);
        tc_fence_after();
        if (ok) {
            for (int i = 0; i < tiles; i++) scores(i, 0);
            umma_commit(&sh.k_empty[0]);
        }
        for (int j = 0; ok && j < n; j++) {
            for (int i = 0; ok && i < tiles; i++) {
                ok = mbar_wait(&sh.w_full[i], j & 1, err);
                if (ok && i == 0) ok = mbar_wait(&sh.v_full[j & 1], (j >> 1) & 1, err);
                if (!ok) break;
                tc_fence_after();
#pragma unroll
                for (int kk = 0; kk < kKeys / 16; kk++)
                    umma_f16_tmem_a(tmem + M::cO + i * HD, tmem + M::cW + i * M::kWStride + kk * 8,
                                    sw128_desc(v0 + (j & 1) * M::kV + (kk / 4) * (HD * 128) + (kk % 4) * 32), idesc_o, j > 0 || kk > 0);
                if (j + 1 == n) {
                    umma_commit(&sh.o_full[i]);
                } else {
                    if (i == 0) ok = mbar_wait(&sh.k_full[(j + 1) & 1], ((j + 1) >> 1) & 1, err);
                    if (ok && M::kOver) {
                        // the next scores overwrite the weights: MMAs of different accumulators have no
                        // guaranteed order, so the product that reads them is waited for (the other tile's
                        // softmax covers it)
                        umma_commit(&sh.pv_done[i]);
                        ok = mbar_wait(&sh.pv_done[i], j & 1, err);
                    }
                    if (!ok) break;
                    tc_fence_after();
                    scores(i, j + 1);
                }
            }
            if (!ok) break;
            umma_commit(&sh.v_empty[j & 1]);
            if (j + 1 < n) umma_commit(&sh.k_empty[(j + 1) & 1]);
        }
        if (!ok) {
            // what was issued lands before shared and tensor memory are given up
            umma_commit(&sh.drain);
            mbar_drain(&sh.drain, 0, err);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
    if (threadIdx.x == 0 && sh.err && a.kv.status) atomicExch(a.kv.status, 2);
    if (w.my_chunks == 1) return;

    // the last range of these rows to finish joins them all, in the ranges' order
    __threadfence();
    __syncthreads();
    if (threadIdx.x == 0) {
        sh.last = atomicAdd(a.counters + unit, 1) == w.my_chunks - 1;
        if (sh.last) a.counters[unit] = 0;
    }
    __syncthreads();
    if (!sh.last) return;
    __threadfence();
    const int live = min(kTileRows, w.rows - w.row0);
    for (int x = threadIdx.x; x < live * (HD / 4); x += kTileThreads) {
        const int r = x / (HD / 4), d = x % (HD / 4) * 4;
        float m = -INFINITY, l = 0.0f;
        float4 o = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        for (int c = 0; c < w.my_chunks; c++) {
            const float * pp = part + ((size_t) c * kTileRows + r) * PL;
            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(pp + HD));
            const float4 y = __ldcg(reinterpret_cast<const float4 *>(pp + d));
            const float mx = fmaxf(m, ml.x), ref = mx == -INFINITY ? 0.0f : mx;
            const float f = exp2_approx(m - ref), fc = exp2_approx(ml.x - ref);
            m = mx;
            l = l * f + ml.y * fc;
            o = make_float4(o.x * f + y.x * fc, o.y * f + y.y * fc, o.z * f + y.z * fc, o.w * f + y.w * fc);
        }
        finish(r, d, o, inverse(l));
        if (d == 0) put_lse(r, m, l);
    }
}

template <int HD>
void launch(const AttnArgs & a, cudaStream_t s) {
    const long long grid = (long long) a.kv.n_seq * a.row_tiles * a.chunks * a.kv.n_kv;
    if (grid > INT_MAX) throw std::runtime_error("the batch is too large for one call");
    // (set on every call: the attribute belongs to the current device)
    cudaError_t e = cudaFuncSetAttribute(kv8_attn_tile_kernel<HD>, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) Smem<HD>::kBytes);
    if (e == cudaSuccess) {
        kv8_attn_tile_kernel<HD><<<(unsigned) grid, kTileThreads, Smem<HD>::kBytes, s>>>(a);
        e = cudaGetLastError();
    }
    if (e != cudaSuccess) throw std::runtime_error(std::string("launch: ") + cudaGetErrorString(e));
}

}  // namespace

void launch_attn_tile(const AttnArgs & a, int head_dim, cudaStream_t s) {
    if (head_dim == 64) launch<64>(a, s);
    else launch<128>(a, s);
}

}  // namespace kv8
}  // namespace bzb
