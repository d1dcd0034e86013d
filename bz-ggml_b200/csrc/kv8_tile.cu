// Attention of many rows over the 8-bit paged cache on the tensor cores (tcgen05): prompts, and whatever
// else the few-row kernel of kv8.cu would need more time for (its formulas; the rule stands there).
//
// One CTA takes up to 256 rows of one kv head -- (token, head of the group) pairs, so the group shares
// the cache's tiles -- as two M = 128 tiles, and walks its keys 128 at a time:
//   producers (4 warps)  bytes of 128 keys and values from global memory to registers, one tile ahead;
//                        converted to f16 into shared memory in the MMAs' swizzled layout (two stages),
//                        the blocks' scales beside them;
//   MMA (4 warps)        S_i = Q_i K^T into tensor memory, O_i += W_i V with the weights W_i read from
//                        tensor memory, in steps of 64 keys: two buffers of scores a tile fit beside the
//                        outputs, so the scores of the next step are there when a softmax ends. Each of the
//                        four chains has a warp of its own, so that one's waits are under another's MMAs;
//   softmax (4 warps a tile, one row a thread)  S_i from tensor memory, the running maximum and sum,
//                        the weights back to tensor memory as f16. The exponentials bound it: 16 a
// clock and SM against 4096 multiply-adds, so for head_dim 64 a tile of 128 x 128 scores costs 1024 clocks there
// and 512 in the MMAs; no key is converted more than once for 256 rows.
// O is rescaled only when a row's maximum has grown by more than 2^8 since the last time (the
// weights then stay below 2^8, which f16 holds as precisely), so that the tile of outputs in
// tensor memory is seldom read back.
//
// 8192 rows behind 4100 positions, 32 query and 8 kv heads of 128: 1.19 to 1.23 ms, 900 to 920 TFLOP/s, tensor pipes 43 % active;
// 1.26 ms where every stage has blocks 2^30 apart (see stage_scale).
// What bounds it is one softmax's chain (scores from tensor memory, maximum, 64 exponentials, weights back): about 2200
// clocks for a step of 64 keys of both tiles, whose MMAs take 1280 and exponentials 1024. It was 2.36 ms with one
// warp issuing both tiles' MMAs and 128-key steps, 1.42 with a warp for each chain, 64-key steps and two buffers of
// scores, 1.25 with the scales of a whole stage put beside it by the producers, 1.20 with the second tile half a
// step late. Two CTAs an SM with 128 rows each: 2.16 ms (twice the conversions); a quarter to a half of the exponentials as a
// polynomial on the FMA units: 1.15 to 1.23 against 1.16, prompts slower. 24 packed prompts of 17 to 301 tokens, 8 kv heads
// of 64: 50 us (49 without the check of the stages' spread), about 9 us of set-up, first loads and output in each of four waves of CTAs.
#include "kv8_dev.cuh"
#include "tc_ptx.cuh"

#include <climits>
#include <stdexcept>
#include <string>

namespace bzb {
namespace kv8 {
namespace {

using namespace tc;

constexpr int kKeys = 128, kStep = 64;     // keys of a stage in shared memory; of a step of the softmax
constexpr int kProducers = 4, kSoftmax = 8;  // warps
constexpr int kMmaWarp = kSoftmax + kProducers;
constexpr int kTileThreads = 32 * (kMmaWarp + 4);
// registers a thread: at launch, and after the softmax warps have taken what the others give back
constexpr int kLaunchRegs = 128, kSoftmaxRegs = 152, kOtherRegs = 104;
static_assert(32 * kSoftmax * kSoftmaxRegs + (kTileThreads - 32 * kSoftmax) * kOtherRegs <= kTileThreads * kLaunchRegs,
              "the warps' registers must fit those of the launch");
constexpr float kSlack = 8.0f;             // how far (powers of two) weights may exceed 1 before O is rescaled

template <int HD>
struct Smem {
    static constexpr int kHalf = kKeys * 128;          // 128 rows x 64 f16, 128-byte swizzle
    static constexpr int kQ = 128 * HD * 2, kK = kKeys * HD * 2, kV = kKeys * HD * 2;
    static constexpr int oQ = 0, oK = 2 * kQ, oV = oK + 2 * kK, oEnd = oV + 2 * kV;
    static constexpr size_t kBytes = 1024 + oEnd;
    // tensor memory columns: two buffers of scores for each tile, then the tiles' outputs. A step's weights
    // (f16, 32 columns) lie over its scores
    static constexpr int cO = 4 * kStep;
};

struct Shared {
    uint64_t k_full[2], k_empty[2], v_full[2], v_empty[2], q_full[2], o_full[2], lead, drain[4];
    uint64_t s_full[2][2], w_full[2][2], pv_done[2][2];  // [tile][step & 1]
    uint64_t n_full[4];  // nan_v[] of a stage (a ring of four, as scale[]: see the producers)
    uint32_t tmem;
    int err;
    int nan_v[4][kProducers];   // a producer warp found NaN values in this tile (only where it looked)
    float4 scale[4];            // of a stage: the keys' scale, the values' exponent, 2^-it; not 0: each block's in block[]
    float4 block[4][8];         // of a stage whose blocks' scales lie far apart: the same three of each
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
// two f32 operations an instruction
__device__ __forceinline__ float2 pair(uint32_t a, uint32_t b) { return make_float2(__uint_as_float(a), __uint_as_float(b)); }
__device__ __forceinline__ float2 fma2(float2 a, float b, float c) { return __ffma2_rn(a, make_float2(b, b), make_float2(c, c)); }
__device__ __forceinline__ float2 add2(float2 a, float2 b) { return __fadd2_rn(a, b); }
// scores of 64 keys from key0: those outside [lo, hi) become -inf
__device__ __forceinline__ void mask(float2 (&s)[32], int key0, int lo, int hi) {
#pragma unroll
    for (int t = 0; t < 32; t++) {
        const int key = key0 + 2 * t;
        if (key < lo || key >= hi) s[t].x = -INFINITY;
        if (key + 1 < lo || key + 1 >= hi) s[t].y = -INFINITY;
    }
}

__device__ __forceinline__ void st16(uint32_t addr, const uint32_t (&r)[16]) { tmem_st16(addr, r); }

// one lane of a converged warp, the same one every time
__device__ __forceinline__ bool elect_one() {
    uint32_t p;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(p));
    return p != 0;
}

// a whole warp's bounded wait: all lanes succeed, or all take it as failed
__device__ __forceinline__ bool warp_wait(uint64_t * bar, uint32_t parity, int * err, long long polls) {
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, err, polls));
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
    unsigned id = blockIdx.x;
    w.h = (int) (id % (unsigned) kv.n_kv);
    id /= (unsigned) kv.n_kv;
    w.chunk = (int) (id % (unsigned) a.chunks);
    id /= (unsigned) a.chunks;
    // the last tiles of causal sequences have the most keys: they start first
    w.b = (int) (id % (unsigned) kv.n_seq);
    w.tile = a.row_tiles - 1 - (int) (id / (unsigned) kv.n_seq);
    w.s = load_seq(kv, w.b);
    if (w.s.slot < 0) return false;
    w.row0 = w.tile * kTileRows;
    const Span p = span_of(a, w.s, w.row0, kTileRows);
    w.rows = p.rows;
    if (w.row0 >= w.rows || w.chunk >= p.chunks) return false;
    w.first = p.first;
    w.my_chunks = p.chunks;
    const int pos_lo = w.first + w.row0 / a.group, pos_hi = w.first + min(w.rows - 1, w.row0 + kTileRows - 1) / a.group;
    w.full_hi = keys_end(a, w.s, pos_lo);
    w.full_lo = a.window > 0 ? max(0, pos_hi - a.window + 1) : 0;
    w.blk0 = p.blk_lo + w.chunk * a.chunk_blocks;
    w.blk_hi = min(p.blk_hi, w.blk0 + a.chunk_blocks);
    w.n_tiles = max(0, (w.blk_hi - w.blk0 + 7) / 8);
    return true;
}

// 8 consecutive query elements, as they are
__device__ __forceinline__ uint4 load_q8(const AttnArgs & a, long long i) {
    const uint16_t * p = static_cast<const uint16_t *>(a.q.p) + i;
    if (a.q_vec) return *reinterpret_cast<const uint4 *>(p);
    uint32_t w[4];
#pragma unroll
    for (int j = 0; j < 4; j++) w[j] = (uint32_t) p[2 * j] | ((uint32_t) p[2 * j + 1] << 16);
    return make_uint4(w[0], w[1], w[2], w[3]);
}

// a softmax warp's 32 query rows into the swizzled tile; rows that do not exist become zero
template <int HD>
__device__ __forceinline__ void load_queries(const AttnArgs & a, const Work & w, Shared & sh, uint8_t * sq, int tile, int quarter, int lane) {
    constexpr int LPR = HD / 8, RPP = 32 / LPR;  // lanes of a row, rows of a pass
    const int c = lane % LPR;
    uint4 u[LPR];
    // (all of them under way before the first is used)
#pragma unroll
    for (int p = 0; p < LPR; p++) {
        const int rr = w.row0 + tile * 128 + quarter * 32 + p * RPP + lane / LPR;
        u[p] = make_uint4(0, 0, 0, 0);
        if (rr < w.rows)
            u[p] = load_q8(a, (long long) (w.s.row0 + rr / a.group) * a.q.row + (w.h * a.group + rr % a.group) * a.q.head + 8 * c);
    }
#pragma unroll
    for (int p = 0; p < LPR; p++) {
        const int r = quarter * 32 + p * RPP + lane / LPR;
        float unit = 1.0f;
        if (a.scale2 < 0.0f) u[p] = make_uint4(u[p].x ^ 0x80008000u, u[p].y ^ 0x80008000u, u[p].z ^ 0x80008000u, u[p].w ^ 0x80008000u);
        if (a.type == BZB_BF16) {
            // bf16 may lie outside f16: the row is brought up to [2^14, 2^15) by a power of two
            const uint32_t v[4] = { u[p].x, u[p].y, u[p].z, u[p].w };
            float x[8], amax = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; j++) x[2 * j] = __uint_as_float(v[j] << 16), x[2 * j + 1] = __uint_as_float(v[j] & 0xffff0000u);
#pragma unroll
            for (int j = 0; j < 8; j += 2) amax = fmaxf(fmaxf(amax, fabsf(x[j])), fabsf(x[j + 1]));
#pragma unroll
            for (int o = LPR / 2; o > 0; o >>= 1) amax = fmaxf(amax, __shfl_xor_sync(0xffffffffu, amax, o));
            const int e = row_exponent(amax);
            unit = pow2f(e);
            const float f = pow2f(-e);
            u[p] = make_uint4(pack_half(x[0] * f, x[1] * f), pack_half(x[2] * f, x[3] * f), pack_half(x[4] * f, x[5] * f),
                              pack_half(x[6] * f, x[7] * f));
        }
        *reinterpret_cast<uint4 *>(sq + (c / 8) * Smem<HD>::kHalf + r * 128 + (((c % 8) ^ (r & 7)) << 4)) = u[p];
        if (c == 0) sh.unit[tile][r] = unit;
    }
}

// ---- producers: tile after tile, bytes in registers to swizzled f16 ----
//
// A thread's pieces of a tile lie at the same place of
// successive blocks, so their addresses differ by the blocks' alone.
__device__ __forceinline__ const uint8_t * shfl_ptr(const uint8_t * p, int lane) {
    return reinterpret_cast<const uint8_t *>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(p), lane));
}

// block b (0..7) of tile j, one block per lane (lane & 7): its page, or -1 past the last
__device__ __forceinline__ int tile_page(const AttnArgs & a, const Work & w, int j, int lane) {
    const int blk = w.blk0 + 8 * j + (lane & 7);
    return j < w.n_tiles && blk < w.blk_hi ? max(page_of(a.kv, w.s.slot, blk), 0) : -1;
}

// The blocks' scales are brought to that of the stage, 2^(E - kLift), E the largest exponent, by multiplying the f16
// values with 2^(e - E + kLift). One factor then serves 128 keys in the softmax. Exact while the exponents lie within
// kSpread of each other: 448 becomes 57344 at most, and the last bit of a subnormal byte, 2^-9, no less than f16's last,
// 2^-24. Stages with a wider spread -- a loud block, which may be one that no row of the tile sees -- keep their values as
// they are, and the softmax applies each block's scales for itself.
constexpr int kLift = 7, kSpread = 22;
struct StageScale {
    int top;         // E - kLift
    bool apart;      // a wider spread than kSpread
    uint32_t mine;   // lane & 7's block: its factor twice, as f16 (one where they are apart)
};
__device__ __forceinline__ StageScale stage_scale(float scale, bool there) {
    const int e = there ? exponent_of(scale) : -1000;
    const int top = __reduce_max_sync(0xffffffffu, e), low = __reduce_min_sync(0xffffffffu, there ? e : 1000);
    const int d = max(e - top, -kSpread) + kLift;  // f16: 2^d has exponent field d + 15; 2^-15 is subnormal
    const uint32_t h = d >= -14 ? (uint32_t) (d + 15) << 10 : 1u << (d + 24);
    const bool apart = top - low > kSpread;
    return { top - kLift, apart, apart ? 0x3c003c00u : h | h << 16 };
}
__device__ __forceinline__ uint32_t scaled(uint16_t e4m3x2, uint32_t f) {
    const uint32_t h = e4m3x2_to_h2(e4m3x2);
    const half2 r = __hmul2(*reinterpret_cast<const half2 *>(&h), *reinterpret_cast<const half2 *>(&f));
    return *reinterpret_cast<const uint32_t *>(&r);
}

template <int HD>
struct Keys {
    static constexpr int N = HD / 16;  // 16-byte pieces of a tile for each of 128 threads
    uint4 x[N];
    int in_block, dst, first, step;    // bytes into a block; bytes into the tile; block of piece 0, blocks between pieces

    __device__ explicit Keys(int tid) {
        // row of the block and 16 bytes of the row, so that the lanes of a store fall on different banks
        const int row = HD == 64 ? tid >> 2 : ((tid >> 2) & 1) | (tid >> 4) << 1;
        const int c = HD == 64 ? tid & 3 : (tid & 3) | ((tid >> 3) & 1) << 2;
        in_block = (row & 15) * HD + 16 * c;
        first = row >> 4;
        step = HD == 64 ? 2 : 1;
        dst = (c >> 2) * Smem<HD>::kHalf + row * 128 + ((((c & 3) * 2) ^ (row & 7)) << 4);
    }
    __device__ void load(const uint8_t * block) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint8_t * p = shfl_ptr(block, first + step * i);
            x[i] = make_uint4(0, 0, 0, 0);
            if (p) x[i] = *reinterpret_cast<const uint4 *>(p + in_block);
        }
    }
    __device__ void store(uint8_t * tile, uint32_t factor) const {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t f = __shfl_sync(0xffffffffu, factor, first + step * i);
            const uint32_t v[4] = { x[i].x, x[i].y, x[i].z, x[i].w };
            uint32_t y[8];
#pragma unroll
            for (int m = 0; m < 4; m++) y[2 * m] = scaled((uint16_t) v[m], f), y[2 * m + 1] = scaled((uint16_t) (v[m] >> 16), f);
            uint8_t * at = tile + dst + i * step * 16 * 128;
            *reinterpret_cast<uint4 *>(at) = make_uint4(y[0], y[1], y[2], y[3]);
            // (the second half is the next 16-byte chunk before the swizzle: chunk number ^ 1)
            *reinterpret_cast<uint4 *>(tile + ((dst + i * step * 16 * 128) ^ 16)) = make_uint4(y[4], y[5], y[6], y[7]);
        }
    }
};

template <int HD>
struct Values {
    static constexpr int N = HD / 32;  // 32-byte pieces (two patches: 4 elements x 8 positions) for each of 128 threads
    uint4 x[N][2];
    int in_block, first, tid;

    __device__ explicit Values(int t) : tid(t) {
        in_block = ((t >> 3) & 15) * 64 + (t & 1) * 32;
        first = (t >> 1) & 3;
    }
    // piece i: blocks first + 4 (i of the tile's halves), element quads of the low or high half
    static __device__ constexpr int half_of(int i) { return HD == 64 ? i : i >> 1; }
    static __device__ constexpr int quads_of(int i) { return HD == 64 ? 0 : (i & 1) * 16; }
    __device__ void load(const uint8_t * block) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint8_t * p = shfl_ptr(block, first + 4 * half_of(i));
            x[i][0] = x[i][1] = make_uint4(0, 0, 0, 0);
            if (p) {
                const uint4 * src = reinterpret_cast<const uint4 *>(p + in_block + quads_of(i) * 64);
                x[i][0] = src[0];
                x[i][1] = src[1];
            }
        }
    }
    // NaNs become zero; says whether there were any
    __device__ bool clear_nan() {
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < N; i++)
#pragma unroll
            for (int m = 0; m < 2; m++) {
                uint4 & v = x[i][m];
                const uint4 n = make_uint4(nan_bytes(v.x), nan_bytes(v.y), nan_bytes(v.z), nan_bytes(v.w));
                any |= n.x | n.y | n.z | n.w;
                v = make_uint4(v.x & ~n.x, v.y & ~n.y, v.z & ~n.z, v.w & ~n.w);
            }
        return any != 0;
    }
    __device__ void store(uint8_t * tile, uint32_t factor) const {
        const int q = (tid >> 3) & 15, chunk = first * 2 + (tid & 1);
        uint8_t * row = tile + q * 4 * 128;
        int at[4];
#pragma unroll
        for (int m = 0; m < 4; m++) at[m] = m * 128 + ((chunk ^ ((4 * q + m) & 7)) << 4);
#pragma unroll
        for (int i = 0; i < N; i++) {
            const uint32_t f = __shfl_sync(0xffffffffu, factor, first + 4 * half_of(i));
            const uint32_t v[4] = { x[i][0].x, x[i][0].y, x[i][0].z, x[i][0].w }, y[4] = { x[i][1].x, x[i][1].y, x[i][1].z, x[i][1].w };
#pragma unroll
            for (int m = 0; m < 4; m++)
                *reinterpret_cast<uint4 *>(row + half_of(i) * (HD * 128) + quads_of(i) * 512 + at[m]) =
                    make_uint4(scaled((uint16_t) v[m], f), scaled((uint16_t) (v[m] >> 16), f), scaled((uint16_t) y[m], f),
                               scaled((uint16_t) (y[m] >> 16), f));
        }
    }
};

template <int HD>
__global__ void __launch_bounds__(kTileThreads, 1) kv8_attn_tile_kernel(const AttnArgs a) {
    using M = Smem<HD>;
    extern __shared__ uint8_t raw[];
    __shared__ Shared sh;
    start_after_previous();
    Work w;
    if (!find_work(a, w)) return;  // (the whole CTA)
    uint8_t * base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tiles = w.rows - w.row0 > 128 ? 2 : 1;
    if (threadIdx.x == 0) {
        for (int i = 0; i < 2; i++) {
            mbar_init(&sh.k_full[i], kProducers);
            mbar_init(&sh.v_full[i], kProducers);
            mbar_init(&sh.k_empty[i], tiles);
            mbar_init(&sh.v_empty[i], tiles);
            mbar_init(&sh.q_full[i], 4);
            mbar_init(&sh.o_full[i], 1);
            for (int b = 0; b < 2; b++) {
                mbar_init(&sh.s_full[i][b], 2);
                mbar_init(&sh.w_full[i][b], 4);
                mbar_init(&sh.pv_done[i][b], 1);
            }
        }
        for (int i = 0; i < 4; i++) {
            mbar_init(&sh.n_full[i], kProducers);
            mbar_init(&sh.drain[i], 1);
        }
        mbar_init(&sh.lead, 4);
        sh.err = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) tmem_alloc(&sh.tmem, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = sh.tmem;
    const int n = w.n_tiles, steps = max(0, (w.blk_hi - w.blk0 + 3) / 4);
    int * err = &sh.err;
    constexpr int PL = HD + 4;
    const size_t unit = ((size_t) w.b * a.row_tiles + w.tile) * a.kv.n_kv + w.h;
    float * part = w.my_chunks > 1 ? a.part + unit * a.chunks * ((size_t) kTileRows * PL) : nullptr;

    auto inverse = [](float l) { return l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l); };  // (NaN stays NaN)
    auto put_lse = [&](int r, float m, float l) {
        const int rr = w.row0 + r;
        if (a.lse)
            a.lse[(size_t) (w.s.row0 + rr / a.group) * a.n_head + w.h * a.group + rr % a.group] = l == 0.0f ? -INFINITY : kLn2 * (m + log2f(l));
    };

    if (warp < kSoftmax) {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kSoftmaxRegs));
        const int i = warp >> 2, r = threadIdx.x & 127, rr = w.row0 + 128 * i + r;
        if (i < tiles) {
            uint8_t * sq = base + M::oQ + i * M::kQ;
            load_queries<HD>(a, w, sh, sq, i, warp & 3, lane);
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.q_full[i]);
            const uint32_t lanes = (uint32_t) (warp & 3) << 21;  // tensor memory lanes 32 (warp % 4) ..
            const uint32_t ts = tmem + lanes + i * 2 * kStep, to = tmem + lanes + M::cO + i * HD;
            const bool real = rr < w.rows;
            const int pos = w.first + rr / a.group;
            const int hi = real ? keys_end(a, w.s, pos) : INT_MAX, lo = real && a.window > 0 ? pos - a.window + 1 : INT_MIN;
            const int warp_hi = __reduce_min_sync(0xffffffffu, hi), warp_lo = __reduce_max_sync(0xffffffffu, lo);
            // (a negative scale's sign is in the queries; never zero, nor with a key scale of 2^-31, which times -inf
            // would be NaN: 1e-30 moves scores by 1e-8 at most)
            const float row_coef = fmaxf(fabsf(a.scale2) * sh.unit[i][r], 1e-30f);
            float m = -INFINITY, l = 0.0f;
            uint32_t nan_d[HD / 32] = {};
            bool ok = true;
            float4 c = make_float4(0.0f, 0.0f, 0.0f, 0.0f);  // the stage's scale[], the keys' times the row's factor
            for (int u = 0; u < steps; u++) {
                const int j = u >> 1, key0 = (w.blk0 << 4) + kStep * u;
                ok = warp_wait(&sh.s_full[i][u & 1], j & 1, err, a.polls);
                if (!ok) break;
                if (!(u & 1)) {
                    c = sh.scale[j & 3];
                    c.x *= row_coef;
                }
                tc_fence_after();
                const bool whole = key0 >= warp_lo && key0 + kStep <= warp_hi;
                const uint32_t at = ts + (u & 1) * kStep;
                uint32_t x[2][32];
                ld32(at, x[0]);
                ld32(at + 32, x[1]);
                tmem_wait_ld();
                float2 s[32];
#pragma unroll
                for (int t = 0; t < 32; t++) s[t] = pair(x[t / 16][2 * (t % 16)], x[t / 16][2 * (t % 16) + 1]);
                if (!whole) mask(s, key0, lo, hi);
                float z[4] = { c.z, c.z, c.z, c.z };  // 2^-exponent of the values of the step's blocks
                if (__builtin_expect(c.w != 0.0f, 0)) {
                    const float4 * block = &sh.block[j & 3][4 * (u & 1)];
#pragma unroll
                    for (int b = 0; b < 4; b++) {
                        const float4 f = block[b];
#pragma unroll
                        for (int t = 0; t < 8; t++) s[8 * b + t] = fma2(s[8 * b + t], f.x * row_coef, f.y);
                        z[b] = f.z;
                    }
                    c.x = 1.0f;
                    c.y = 0.0f;
                }
                float tops[4] = { -INFINITY, -INFINITY, -INFINITY, -INFINITY };
#pragma unroll
                for (int t = 0; t < 32; t++) tops[t & 3] = fmaxf(fmaxf(tops[t & 3], s[t].x), s[t].y);
                const float top = fmaf(fmaxf(fmaxf(tops[0], tops[1]), fmaxf(tops[2], tops[3])), c.x, c.y);
                // (the first maximum is taken as it is; -inf while a row has seen no key)
                const bool grow = top > m + kSlack;
                if (__any_sync(0xffffffffu, grow)) {
                    const float f = grow ? exp2_approx(m - top) : 1.0f;
                    if (grow) m = top;
                    l *= f;
                    if (u > 0) {
                        // the last product into these outputs must be in before they are scaled
                        ok = warp_wait(&sh.pv_done[i][(u - 1) & 1], ((u - 1) >> 1) & 1, err, a.polls);
                        if (!ok) break;
                        tc_fence_after();
#pragma unroll 1
                        for (int d = 0; d < HD; d += 16) {
                            float y[16];
                            tmem_ld16(to + d, y);
                            tmem_wait_ld();
                            uint32_t z[16];
#pragma unroll
                            for (int t = 0; t < 16; t++) z[t] = __float_as_uint(y[t] * f);
                            st16(to + d, z);
                        }
                    }
                }
                const float ref = c.y - (m == -INFINITY ? 0.0f : m);
#pragma unroll
                for (int g = 0; g < 2; g++) {
                    float2 sum[2] = { { 0.0f, 0.0f }, { 0.0f, 0.0f } };  // a block's
                    uint32_t p[16];
#pragma unroll
                    for (int t = 0; t < 16; t++) {
                        const float2 v = fma2(s[16 * g + t], c.x, ref);
                        const float2 e = make_float2(exp2_approx(v.x), exp2_approx(v.y));
                        sum[t >> 3] = add2(sum[t >> 3], e);
                        p[t] = pack_half(e.x, e.y);
                    }
                    st16(at + 16 * g, p);
                    l = fmaf(sum[0].x + sum[0].y, z[2 * g], fmaf(sum[1].x + sum[1].y, z[2 * g + 1], l));
                }
                tmem_wait_st();
                tc_fence_before();
                __syncwarp();
                if (lane == 0) {
                    mbar_arrive(&sh.w_full[i][u & 1]);
                    if (u == 0 && i == 0) mbar_arrive(&sh.lead);
                }
                // NaN values in a stage that some row of the CTA does not see in whole: the producers left them
                // out; the rows that see one get it at the end
                const int stage0 = (w.blk0 + 8 * j) << 4;
                if (stage0 < w.full_lo || stage0 + kKeys > w.full_hi) {
                    ok = warp_wait(&sh.n_full[j & 3], (j >> 2) & 1, err, a.polls);
                    if (!ok) break;
                    bool any = false;
                    for (int q = 0; q < kProducers; q++) any |= sh.nan_v[j & 3][q] != 0;
                    if (any && real)
                        for (int key = max(lo, key0); key < min(hi, key0 + kStep) && (key >> 4) < w.blk_hi; key++) {
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
            if (ok && n > 0) ok = warp_wait(&sh.o_full[i], 0, err, a.polls);
            if (ok) {
                tc_fence_after();
                // rows go out through this tile's query buffer, whose products are done, so that a warp writes whole
                // rows; its 32 rows are its own. f16 rows fit at once, f32 partials half a row at a time
                const float inv = inverse(l);
                uint8_t * mine = sq + (warp & 3) * (32 * HD * 2);
                const int me = 128 * i + (warp & 3) * 32, live = min(32, w.rows - w.row0 - me);
                const auto pull = [&](int d, float (&y)[16]) {
                    if (n > 0) {
                        tmem_ld16(to + d, y);
                        tmem_wait_ld();
                    }
#pragma unroll
                    for (int t = 0; t < 16; t++) {
                        if (n == 0) y[t] = 0.0f;
                        if (nan_d[d / 32] >> (d % 32 + t) & 1) y[t] = __int_as_float(0x7fffffff);
                    }
                };
                constexpr int C = HD / 8;  // 16-byte chunks of a row in the buffer
                if (part) {
                    float * pp = part + ((size_t) w.chunk * kTileRows + me) * PL;
#pragma unroll
                    for (int half_ = 0; half_ < 2; half_++) {
#pragma unroll
                        for (int d = 0; d < HD / 2; d += 16) {
                            float y[16];
                            pull(half_ * (HD / 2) + d, y);
#pragma unroll
                            for (int t = 0; t < 16; t += 4)
                                *reinterpret_cast<float4 *>(mine + lane * (HD * 2) + (((d + t) / 4 ^ (lane & 7)) << 4)) = make_float4(y[t], y[t + 1], y[t + 2], y[t + 3]);
                        }
                        __syncwarp();
                        for (int x = lane; x < live * C; x += 32) {
                            const int row = x / C, c = x % C;
                            *reinterpret_cast<float4 *>(pp + row * PL + half_ * (HD / 2) + c * 4) =
                                *reinterpret_cast<const float4 *>(mine + row * (HD * 2) + ((c ^ (row & 7)) << 4));
                        }
                        __syncwarp();
                    }
                    if (real) *reinterpret_cast<float2 *>(pp + lane * PL + HD) = make_float2(m, l);
                } else {
#pragma unroll
                    for (int d = 0; d < HD; d += 16) {
                        float y[16];
                        pull(d, y);
                        uint32_t z[8];
#pragma unroll
                        for (int t = 0; t < 8; t++)
                            z[t] = a.type == BZB_F16 ? pack_half(y[2 * t] * inv, y[2 * t + 1] * inv) : pack_bf16(y[2 * t] * inv, y[2 * t + 1] * inv);
#pragma unroll
                        for (int t = 0; t < 2; t++)
                            *reinterpret_cast<uint4 *>(mine + lane * (HD * 2) + ((d / 8 + t ^ (lane & 7)) << 4)) =
                                make_uint4(z[4 * t], z[4 * t + 1], z[4 * t + 2], z[4 * t + 3]);
                    }
                    __syncwarp();
                    for (int x = lane; x < live * C; x += 32) {
                        const int row = x / C, c = x % C, rr = w.row0 + me + row;
                        const uint4 v = *reinterpret_cast<const uint4 *>(mine + row * (HD * 2) + ((c ^ (row & 7)) << 4));
                        uint16_t * to_row = static_cast<uint16_t *>(a.out.p) + (long long) (w.s.row0 + rr / a.group) * a.out.row +
                                            (w.h * a.group + rr % a.group) * a.out.head + c * 8;
                        if (a.out_vec) {
                            *reinterpret_cast<uint4 *>(to_row) = v;
                        } else {
                            const uint32_t e[4] = { v.x, v.y, v.z, v.w };
#pragma unroll
                            for (int t = 0; t < 4; t++) to_row[2 * t] = (uint16_t) e[t], to_row[2 * t + 1] = (uint16_t) (e[t] >> 16);
                        }
                    }
                    if (real) put_lse(me + lane, m, l);
                }
            }
            tc_fence_before();
        }
    } else if (warp < kMmaWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
        const int pw = warp - kSoftmax, tid = (int) threadIdx.x - 32 * kSoftmax;
        Keys<HD> k(tid);
        Values<HD> v(tid);
        auto block = [&](int pg, int j, int plane) -> const uint8_t * {
            return pg < 0 ? nullptr : block_ptr(a.kv, pg, w.blk0 + 8 * j + (lane & 7), plane, w.h, HD);
        };
        int pg = tile_page(a, w, 0, lane), next = tile_page(a, w, 1, lane);
        float ks = 0.0f, vs = 0.0f;
        auto load_scales = [&](int j) {
            if (pg < 0) return;
            ks = *scale_ptr(a.kv, pg, w.blk0 + 8 * j + (lane & 7), 0, w.h);
            vs = *scale_ptr(a.kv, pg, w.blk0 + 8 * j + (lane & 7), 1, w.h);
        };
        k.load(block(pg, 0, 0));
        v.load(block(pg, 0, 1));
        load_scales(0);
        for (int j = 0; j < n; j++) {
            const int st = j & 1, key0 = (w.blk0 + 8 * j) << 4;
            const StageScale sk = stage_scale(ks, pg >= 0), sv = stage_scale(vs, pg >= 0);
            if (!warp_wait(&sh.k_empty[st], ((j >> 1) & 1) ^ 1, err, a.polls)) break;
            k.store(base + M::oK + st * M::kK, sk.mine);
            const bool apart = sk.apart || sv.apart;
            if (pw == 0 && lane == 0) sh.scale[j & 3] = make_float4(pow2f(sk.top), (float) sv.top, pow2f(-sv.top), apart ? 1.0f : 0.0f);
            if (pw == 0 && lane < 8 && apart) {
                // (blocks that are not there: any finite numbers, their keys are masked)
                const int ev = !sv.apart ? sv.top : pg < 0 ? 0 : exponent_of(vs);
                sh.block[j & 3][lane] = make_float4(!sk.apart ? pow2f(sk.top) : pg < 0 ? 1.0f : ks, (float) ev, pow2f(-ev), 0.0f);
            }
            fence_proxy_async();
            __syncwarp();
            // (scale[], block[] and nan_v[] are rings of four: those of stage j + 4 are stored when the products of stage
            // j + 2 have been issued, which every softmax warp's weights of stage j + 1 come before)
            if (lane == 0) mbar_arrive(&sh.k_full[st]);
            pg = next;
            next = tile_page(a, w, j + 2, lane);
            k.load(block(pg, j + 1, 0));
            load_scales(j + 1);
            bool bad = false;
            if (key0 < w.full_lo || key0 + kKeys > w.full_hi) bad = v.clear_nan();
            bad = __any_sync(0xffffffffu, bad);
            if (!warp_wait(&sh.v_empty[st], ((j >> 1) & 1) ^ 1, err, a.polls)) break;
            v.store(base + M::oV + st * M::kV, sv.mine);
            if (lane == 0) sh.nan_v[j & 3][pw] = bad;
            fence_proxy_async();
            __syncwarp();
            if (lane == 0) mbar_arrive(&sh.v_full[st]), mbar_arrive(&sh.n_full[j & 3]);
            v.load(block(pg, j + 1, 1));
        }
    } else {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kOtherRegs));
    }
    const int mma = warp - kMmaWarp, mt = mma & 1;
    if (mma >= 0 && mt < tiles && n > 0) {
        // (offsets are added to the descriptors' 16-byte address field, which no tile here carries out of)
        const uint32_t sc = tmem + mt * 2 * kStep;
        // a producer waits for step u's stage to be free. (The last two stages' are not signalled: an arrival that
        // nothing waits for could come when the CTA has left and its shared memory is another's)
        const auto freed = [&](int u) { return (u >> 1) + 2 < n; };
        bool ok = true;
        if (mma < 2) {
            constexpr uint32_t idesc = (1u << 4) | ((uint32_t) (kStep >> 3) << 17) | (8u << 24);
            const uint64_t q = sw128_desc(smem_u32(base + M::oQ + mt * M::kQ)), k0 = sw128_desc(smem_u32(base + M::oK));
            for (int u = 0; u < steps; u++) {
                const int st = (u >> 1) & 1;
                // the buffer's last weights have been read (MMAs of different accumulators have no guaranteed
                // order, so that product is waited for; the other buffer's scores keep the softmax busy)
                if (u >= 2) ok = warp_wait(&sh.pv_done[mt][u & 1], ((u - 2) >> 1) & 1, err, a.polls);
                else if (u == 0 && mt == 0) ok = warp_wait(&sh.q_full[0], 0, err, a.polls);
                // the second tile starts when the first has done its first step: the two softmaxes then take the
                // exponential units in turn instead of both at once and both not at all. (A barrier that completes
                // once: this wait may come any time after)
                else if (u == 0) ok = warp_wait(&sh.q_full[1], 0, err, a.polls) && warp_wait(&sh.lead, 0, err, a.polls);
                if (ok && !(u & 1)) ok = warp_wait(&sh.k_full[st], (u >> 2) & 1, err, a.polls);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t k = k0 + ((st * M::kK + (u & 1) * kStep * 128) >> 4);
#pragma unroll
                    for (int kk = 0; kk < HD / 16; kk++) {
                        const uint32_t at = ((kk / 4) * M::kHalf + (kk % 4) * 32) >> 4;
                        umma_f16(sc + (u & 1) * kStep, q + at, k + at, idesc, kk > 0);
                    }
                    umma_commit(&sh.s_full[mt][u & 1]);
                    // (and this thread's own arrival, which hands on what the wait for the keys made visible: the
                    // stage's scales)
                    mbar_arrive(&sh.s_full[mt][u & 1]);
                    if ((u & 1) && freed(u)) umma_commit(&sh.k_empty[st]);
                }
                __syncwarp();
            }
        } else {
            constexpr uint32_t idesc = (1u << 4) | ((uint32_t) (HD >> 3) << 17) | (8u << 24);
            const uint64_t v0 = sw128_desc(smem_u32(base + M::oV));
            for (int u = 0; u < steps; u++) {
                const int st = (u >> 1) & 1;
                if (!(u & 1)) ok = warp_wait(&sh.v_full[st], (u >> 2) & 1, err, a.polls);
                if (ok) ok = warp_wait(&sh.w_full[mt][u & 1], (u >> 1) & 1, err, a.polls);
                if (!ok) break;
                tc_fence_after();
                if (elect_one()) {
                    const uint64_t v = v0 + ((st * M::kV + (u & 1) * HD * 128) >> 4);
#pragma unroll
                    for (int kk = 0; kk < kStep / 16; kk++)
                        umma_f16_tmem_a(tmem + M::cO + mt * HD, sc + (u & 1) * kStep + kk * 8, v + (kk * 32 >> 4), idesc, u > 0 || kk > 0);
                    umma_commit(u + 1 == steps ? &sh.o_full[mt] : &sh.pv_done[mt][u & 1]);
                    if ((u & 1) && freed(u)) umma_commit(&sh.v_empty[st]);
                }
                __syncwarp();
            }
        }
        if (!ok) {
            // what was issued lands before shared and tensor memory are given up
            if (elect_one()) umma_commit(&sh.drain[mma]);
            __syncwarp();
            mbar_drain(&sh.drain[mma], 0, err);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    if (warp == kMmaWarp) tmem_dealloc(tmem, 512);
    if (threadIdx.x == 0 && sh.err) complain(a.kv, BZB_KV8_TIMED_OUT);
}

template <int HD>
void launch(const AttnArgs & a, cudaStream_t s) {
    const long long grid = (long long) a.kv.n_seq * a.row_tiles * a.chunks * a.kv.n_kv;
    static std::atomic<uint64_t> ready{ 0 };
    if (!ready.load(std::memory_order_acquire)) {
        // the register split adds up only for the launch it was made for: a build that gives the kernel
        // another count must not reach the GPU, where it would wait for registers that never come free
        cudaFuncAttributes at;
        if (cudaFuncGetAttributes(&at, kv8_attn_tile_kernel<HD>) != cudaSuccess || at.numRegs != kLaunchRegs)
            throw std::runtime_error("kv8_attn_tile_kernel: built with another register count than its split needs");
    }
    allow_shared_memory(kv8_attn_tile_kernel<HD>, (int) Smem<HD>::kBytes, ready);
    launch_chained(kv8_attn_tile_kernel<HD>, dim3((unsigned) grid), kTileThreads, (int) Smem<HD>::kBytes, s, a);
}

}  // namespace

void launch_attn_tile(AttnArgs a, int head_dim, cudaStream_t s) {
    if (a.polls < 0) a.polls = kSpinLimit;
    if (head_dim == 64) launch<64>(a, s);
    else launch<128>(a, s);
}

}  // namespace kv8
}  // namespace bzb
