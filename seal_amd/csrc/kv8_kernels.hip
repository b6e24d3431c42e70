// A key / value cache in 8 bits: e4m3 codes with one power-of-two scale for every (slot, head, block of `block` tokens), the write into it and
// the attention that reads it (include/sealnn.h: sealnn_kv8_append, sealnn_kv8_attend).
//
// Layout, made for the matrix instructions of the attention:
//   K  [slots][heads][T][dh]              a token's row; T a multiple of 64
//   V  [slots][heads][T / 64][dh][64]     per tile of 64 tokens the dims as rows; the tokens of a row in the order (g, j, r), token = 16 j + 4 g + r
//   scales [slots][heads][T / block] fp32, each 2^e, -64 <= e <= 120
// A power of two costs e4m3 no precision (it is a floating type), makes every rounding of the write exact arithmetic, and lets a block
// whose scale has to grow be re-encoded by an exponent shift.
#include "nn_common.h"

#include <algorithm>

enum { E_MIN = -64 };

static __device__ __forceinline__ float pow2i(int e) { return as_f32((uint32_t)(e + 127) << 23); }
static __device__ __forceinline__ int exponent_of(float pow2) { return (int)(as_u32(pow2) >> 23) - 127; }
// the smallest e >= E_MIN with amax <= 448 * 2^e (448 = 0.875 * 2^9; amax = m * 2^x, 0.5 <= m < 1); amax finite
static __device__ __forceinline__ int exponent_for(float amax)
{
    int x;
    const float m = frexpf(amax, &x);
    return amax > 0.f ? max(x - (m <= 0.875f ? 9 : 8), (int)E_MIN) : (int)E_MIN;
}
// Four numbers, already divided by the scale, as e4m3 codes: to nearest, ties to even; NaN stays.  A block's scale holds its finite values (the instruction alone does
// then); with `wild` there may be infinities, which become +-448.
static __device__ __forceinline__ float sat(float y) { return y != y ? y : fminf(fmaxf(y, -448.f), 448.f); }
static __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d, bool wild = false)
{
    if (wild) { a = sat(a); b = sat(b); c = sat(c); d = sat(d); }
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(a, b, 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(c, d, w, true);
}
// four codes times 2^shift (shift <= 0), re-encoded
static __device__ __forceinline__ uint32_t shift4(uint32_t w, float f)
{
    const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
    return encode4(lo[0] * f, lo[1] * f, hi[0] * f, hi[1] * f);
}

struct AppendArgs {
    const void *src[2];              // new K, V
    uint64_t slot_stride[2], token_stride[2], head_stride[2];
    uint8_t *codes[2];
    float *scale[2];
    const int32_t *lengths, *counts;
    uint32_t n, slots, heads, T, block, dh;
};

// Sixteen consecutive dims of a new token
template <typename T_>
static __device__ __forceinline__ void load16(const T_ *p, bool vec, float v[16])
{
    if (vec) {
        if constexpr (std::is_same<T_, float>::value) {
#pragma unroll
            for (int i = 0; i < 4; i++) {
                const f32x4 a = ((const f32x4 *)p)[i];
#pragma unroll
                for (int j = 0; j < 4; j++) v[4 * i + j] = a[j];
            }
        } else {
#pragma unroll
            for (int i = 0; i < 2; i++) {
                const u32x4 a = ((const u32x4 *)p)[i];
#pragma unroll
                for (int j = 0; j < 4; j++) { v[8 * i + 2 * j] = as_f32(a[j] << 16); v[8 * i + 2 * j + 1] = as_f32(a[j] & 0xffff0000u); }
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < 16; i++) v[i] = load1(p + i);
    }
}

static __device__ __forceinline__ float larger(float m, float v) { return fmaxf(m, fabsf(v)); }                      // (NaN is left out)
static __device__ __forceinline__ float larger_finite(float m, float v) { return fabsf(v) < __builtin_huge_valf() ? fmaxf(m, fabsf(v)) : m; }
static __device__ __forceinline__ float wave_largest(float m)
{
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    return m;
}

// One new token (a decode step): a wave per (slot, head), a lane per dim (two for 128).  The codes of the block before it are only touched where its scale has to grow.
// 300 slots x 16 heads fp32: 7.2 us, a launch (3.5 to 4) and what the layout of V costs: a dim's new byte is a write of 32 bytes to memory of its own (10.3 MB written for 0.6 MB of
// codes, by the counters), behind two round trips (the length, then the scale).
template <typename T_, int DH>
__global__ __launch_bounds__(256) void k_kv8_append_one(AppendArgs a)
{
    enum { N = DH / 64 };
    const uint32_t lane = threadIdx.x & 63, sh = blockIdx.x * 4 + (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6));
    if (sh >= a.slots * a.heads) return;
    const uint32_t slot = sh / a.heads, head = sh % a.heads, blk = a.block;
    float x[2][N], m[2];
#pragma unroll
    for (int w = 0; w < 2; w++) {
        const T_ *src = (const T_ *)a.src[w] + slot * a.slot_stride[w] + head * a.head_stride[w];
        m[w] = 0.f;
#pragma unroll
        for (int i = 0; i < N; i++) x[w][i] = load1(src + 64 * i + lane);
    }
    const int32_t len = a.lengths[slot];
    if (len < 0 || len >= (int32_t)a.T || (a.counts && a.counts[slot] <= 0)) return;
    const uint32_t t = (uint32_t)len % 64, held = (uint32_t)len % blk;                // place in the tile; tokens that the block holds
    const uint64_t tile = (uint32_t)len / 64;
    float *scale[2] = {a.scale[0] + (uint64_t)sh * (a.T / blk) + (uint32_t)len / blk, a.scale[1] + (uint64_t)sh * (a.T / blk) + (uint32_t)len / blk};
    int e_old[2], e[2];
    if (held) { e_old[0] = exponent_of(*scale[0]); e_old[1] = exponent_of(*scale[1]); }
#pragma unroll
    for (int w = 0; w < 2; w++) {
#pragma unroll
        for (int i = 0; i < N; i++) m[w] = larger_finite(m[w], x[w][i]);
        e[w] = exponent_for(wave_largest(m[w]));
        if (held) e[w] = max(e[w], e_old[w]);
    }
    uint8_t *k = a.codes[0] + ((uint64_t)sh * a.T + tile * 64) * DH, *v = a.codes[1] + ((uint64_t)sh * a.T + tile * 64) * DH;
    if (held && e[0] > e_old[0]) {
        const float f = pow2i(max(e_old[0] - e[0], -126));
        for (uint32_t u = lane; u < held * (DH / 16); u += 64) {
            u32x4 *p = (u32x4 *)(k + (uint64_t)(t - held) * DH + 16 * u);
            u32x4 w = *p;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = shift4(w[i], f);
            *p = w;
        }
    }
    if (held && e[1] > e_old[1]) {
        const float f = pow2i(max(e_old[1] - e[1], -126));
        for (uint32_t u = lane; u < DH * 4; u += 64) {           // 16 bytes: dim u / 4, tokens 16 j + 4 (u % 4) + r
            u32x4 *p = (u32x4 *)(v + 16 * u);
            u32x4 w = *p;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {
                uint32_t mask = 0;
#pragma unroll
                for (uint32_t r = 0; r < 4; r++) { const uint32_t s = 16 * j + 4 * (u % 4) + r; if (s >= t - held && s < t) mask |= 0xffu << (8 * r); }
                w[j] = (w[j] & ~mask) | (shift4(w[j], f) & mask);
            }
            *p = w;
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");   // (the new token's bytes below go on top of these words)
        __builtin_amdgcn_s_waitcnt(0);
    }
    if (lane < 2) *(lane ? scale[1] : scale[0]) = pow2i(lane ? e[1] : e[0]);
    const uint32_t at = ((t >> 2) & 3) * 16 + (t >> 4) * 4 + (t & 3);
    const float f0 = pow2i(-e[0]), f1 = pow2i(-e[1]);
#pragma unroll
    for (int i = 0; i < N; i++) {
        const uint32_t w = encode4(x[0][i] * f0, x[1][i] * f1, 0.f, 0.f, true);
        k[(uint64_t)t * DH + 64 * i + lane] = (uint8_t)w;
        v[(uint64_t)(64 * i + lane) * 64 + at] = (uint8_t)(w >> 8);
    }
}

// Many new tokens: a workgroup of 256 threads per (slot, head, 64-token tile).  Nobody else writes the tile, so bytes that the call does not touch are carried over by
// reading them.  K and V together -- what limits the call is how many loads a CU has on their way --, held from the search for the blocks' largest
// magnitudes to the codes.  K: a thread has sixteen dims of a token, 16 bytes of its row.  V: four dims of four tokens -- the four tokens' codes of a
// dim are a word of its row, turned round in LDS (swizzled: 64 lanes, 64 banks).  24 slots x 16 heads x 1000 tokens bf16: 26.7 us, 4.1 TB/s read and written (a large copy: 4.65);
// 36 with each load behind a condition of its own, which the compiler waits for one by one.
template <typename T_, int DH>
__global__ __launch_bounds__(256) void k_kv8_append(AppendArgs a, uint32_t vec)
{
    enum { N = DH / 64, PITCH = 20 };                            // words of a row of V in LDS
    __shared__ uint32_t s_max[2][4];
    __shared__ uint32_t s_tile[DH * PITCH];
    // (the heads of a tile next to each other: their values are neighbours in memory)
    const uint32_t head = blockIdx.x % a.heads, slot = blockIdx.y, tid = threadIdx.x;
    const int64_t len = a.lengths[slot];
    const int64_t cnt = a.counts ? min((int64_t)a.counts[slot], (int64_t)a.n) : (int64_t)a.n;
    if (len < 0 || len >= (int64_t)a.T || cnt <= 0) return;
    const int64_t tile = len / 64 + blockIdx.x / a.heads, base = tile * 64;
    const int64_t lo = max(len, base), hi = min(min(len + cnt, (int64_t)a.T), base + 64);
    if (lo >= hi) return;
    const uint32_t l0 = (uint32_t)(lo - base), l1 = (uint32_t)(hi - base);           // new tokens of the tile
    const uint32_t blk = a.block, t_own = tid / 4, tq = tid / 16;
    const uint64_t sh = (uint64_t)slot * a.heads + head;
    float x[2][N][4][4];                                         // K: [half][run of four dims][dim] of token t_own; V: [half][token 4 tq + r][dim]
    {
        // every load first, then what is done with the values (a thread without a token of the call reads the first one's)
        typedef typename std::conditional<std::is_same<T_, float>::value, f32x4, u32x2>::type Raw;
        const T_ *p[2][4];
        Raw raw[2][N][4];
#pragma unroll
        for (int w = 0; w < 2; w++)
#pragma unroll
            for (uint32_t r = 0; r < 4; r++) {
                const uint32_t t = w ? 4 * tq + r : t_own;
                p[w][r] = (const T_ *)a.src[w] + slot * a.slot_stride[w] + head * a.head_stride[w] + (w ? tid % 16 * 4 : tid % 4 * 16 + 4 * r) +
                          (uint64_t)(base + (t >= l0 && t < l1 ? t : l0) - len) * a.token_stride[w];
            }
        if (vec) {
#pragma unroll
            for (int w = 0; w < 2; w++)
#pragma unroll
                for (int i = 0; i < N; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) raw[w][i][r] = *(const Raw *)(p[w][r] + 64 * i);
        } else {
#pragma unroll
            for (int w = 0; w < 2; w++)
#pragma unroll
                for (int i = 0; i < N; i++)
#pragma unroll
                    for (int r = 0; r < 4; r++) {
                        const T_ *q = p[w][r] + 64 * i;
                        if constexpr (std::is_same<T_, float>::value) raw[w][i][r] = f32x4{q[0], q[1], q[2], q[3]};
                        else { const uint16_t *h = (const uint16_t *)q; raw[w][i][r] = u32x2{(uint32_t)h[0] | ((uint32_t)h[1] << 16), (uint32_t)h[2] | ((uint32_t)h[3] << 16)}; }
                    }
        }
#pragma unroll
        for (int w = 0; w < 2; w++)
#pragma unroll
            for (uint32_t r = 0; r < 4; r++) {
                const uint32_t t = w ? 4 * tq + r : t_own;
                const bool live = t >= l0 && t < l1;
#pragma unroll
                for (int i = 0; i < N; i++)
#pragma unroll
                    for (int d = 0; d < 4; d++) {
                        if constexpr (std::is_same<T_, float>::value) x[w][i][r][d] = live ? raw[w][i][r][d] : 0.f;
                        else x[w][i][r][d] = live ? as_f32(d & 1 ? raw[w][i][r][d / 2] & 0xffff0000u : raw[w][i][r][d / 2] << 16) : 0.f;
                    }
            }
    }
    // the blocks of this tile that the call touches; the first of them may have had tokens before
    const uint32_t b0 = l0 / blk, b1 = (l1 - 1) / blk;
    const bool held = l0 % blk != 0;
    float *scale[2];
    int e_old[2] = {0, 0};
#pragma unroll
    for (int w = 0; w < 2; w++) {
        scale[w] = a.scale[w] + sh * (a.T / blk) + (uint64_t)base / blk;
        if (held) e_old[w] = exponent_of(scale[w][b0]);
    }
    if (tid < 8) s_max[tid / 4][tid % 4] = 0;
    float m[2];
    bool wild[2];
#pragma unroll
    for (int w = 0; w < 2; w++) {
        m[w] = 0.f;
#pragma unroll
        for (int i = 0; i < 16 * N; i++) m[w] = larger(m[w], x[w][i / 16][i / 4 % 4][i % 4]);
        m[w] = wave_largest(m[w]);                               // (a wave has sixteen tokens: of one block)
        wild[w] = !(m[w] < __builtin_huge_valf());               // infinities do not count
        if (wild[w]) {
            m[w] = 0.f;
#pragma unroll
            for (int i = 0; i < 16 * N; i++) m[w] = larger_finite(m[w], x[w][i / 16][i / 4 % 4][i % 4]);
            m[w] = wave_largest(m[w]);
        }
    }
    __syncthreads();
    if ((tid & 63) == 0) { atomicMax(&s_max[0][t_own / blk], as_u32(m[0])); atomicMax(&s_max[1][t_own / blk], as_u32(m[1])); }     // (magnitudes order as their bits)
    __syncthreads();
    auto exp_of = [&](int w, uint32_t b) { const int e = exponent_for(as_f32(s_max[w][b])); return held && b == b0 ? max(e, e_old[w]) : e; };
    float f[2], shift[2];
    bool grow[2];
#pragma unroll
    for (int w = 0; w < 2; w++) {
        const int e = exp_of(w, b0);
        grow[w] = held && e > e_old[w];
        shift[w] = grow[w] ? pow2i(max(e_old[w] - e, -126)) : 1.f;
        f[w] = pow2i(-exp_of(w, t_own / blk));                   // (4 tq and t_own are of the same sixteen tokens)
        if (tid >= b0 && tid <= b1) scale[w][tid] = pow2i(exp_of(w, tid));           // (every thread has read the old scale: two barriers ago)
    }
    uint8_t *k = a.codes[0] + (sh * a.T + (uint64_t)base) * DH, *v = a.codes[1] + (sh * a.T + (uint64_t)base) * DH;
    if (t_own >= l0 && t_own < l1) {
#pragma unroll
        for (int i = 0; i < N; i++) {
            u32x4 c;
#pragma unroll
            for (int r = 0; r < 4; r++) c[r] = encode4(x[0][i][r][0] * f[0], x[0][i][r][1] * f[0], x[0][i][r][2] * f[0], x[0][i][r][3] * f[0], wild[0]);
            *(u32x4 *)(k + (uint64_t)t_own * DH + 64 * i + tid % 4 * 16) = c;
        }
    }
    if (grow[0])
        for (uint32_t u = tid; u < (l0 - b0 * blk) * (DH / 16); u += 256) {
            u32x4 *p = (u32x4 *)(k + (uint64_t)(b0 * blk) * DH + 16 * u);
            u32x4 c = *p;
#pragma unroll
            for (int i = 0; i < 4; i++) c[i] = shift4(c[i], shift[0]);
            *p = c;
        }
    // V: row d, word 4 g + j (tokens 16 j + 4 g .. + 3, tq = 4 j + g) stands at word (4 g + j + d / 16) % 16
    const uint32_t col = 4 * (tq & 3) + (tq >> 2);
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
        for (int d = 0; d < 4; d++) {
            const uint32_t row = 64 * i + tid % 16 * 4 + d;
            s_tile[row * PITCH + ((col + row / 16) & 15)] = encode4(x[1][i][0][d] * f[1], x[1][i][1][d] * f[1], x[1][i][2][d] * f[1], x[1][i][3][d] * f[1], wild[1]);
        }
    __syncthreads();
    const bool whole = l0 == 0 && l1 == 64;
    for (uint32_t u = tid; u < DH * 4; u += 256) {
        const uint32_t d = u / 4, g = u % 4;
        u32x4 *p = (u32x4 *)(v + 16 * u);
        u32x4 fresh, c;
#pragma unroll
        for (uint32_t j = 0; j < 4; j++) fresh[j] = s_tile[d * PITCH + ((4 * g + j + d / 16) & 15)];
        c = fresh;
        if (!whole) {
            c = *p;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {                   // word j: tokens 16 j + 4 g .. + 3
                const uint32_t t0 = 16 * j + 4 * g;
                uint32_t m_new = 0, m_old = 0;
#pragma unroll
                for (uint32_t r = 0; r < 4; r++) {
                    if (t0 + r >= l0 && t0 + r < l1) m_new |= 0xffu << (8 * r);
                    if (t0 + r >= b0 * blk && t0 + r < l0) m_old |= 0xffu << (8 * r);
                }
                const uint32_t again = grow[1] ? shift4(c[j], shift[1]) : c[j];
                c[j] = (c[j] & ~(m_new | m_old)) | (again & m_old) | (fresh[j] & m_new);
            }
        }
        *p = c;
    }
}

// ---------------------------------------------------------------------------------------------------------------------------------
// Attention of single positions: every slot's `beams` x (q_heads / heads) query vectors of a cached head over the slot's first `length` tokens
// that `keep` leaves.  A wave takes tiles of 64 tokens with the online softmax (running maximum m, sum l, output o):
//   S^T [64 tokens x 16 queries] = K (A) q^T (B)       4 x dh / 32 matrix instructions a plane; K's bytes become bf16 exactly
//   p = exp2(S - m),  o^T [dh x 16 queries] += V^T (A) p^T (B)
// Both operands come from memory straight into the registers that the instruction reads: the contraction index of a matrix instruction may be
// permuted as long as both operands agree, so lane (g, t) takes 16 consecutive bytes of token t of K (dims 16 g .. of a 64-dim half), and the
// S values that a lane holds (tokens 16 j + 4 g + r of its query) are, unmoved, the B operand of the second product -- V's tiles are laid out
// for that.  q and p are fp32 numbers and enter as three bf16 planes each (exact); for bf16 queries q is one plane and p two
// (what they leave of p is cut off: up to 2^-15 of it, about 2^-17 on average, always towards zero while the sum l takes p whole; the store's own half step is 2^-8).
// A block's scale is a factor of S's rows (K) or of p (V).
// Bytes behind `length` or masked may be anything: S is selected, p is 0 there and V's bytes are cleared.
// Measured: 32 slots x 8 heads of 4001 .. 8192 tokens, dh 128, bf16 80 us, 5.0 TB/s (memory); 1 slot x 16 heads of 32001 tokens bf16 in 32 parts 18.3 us, 3.6 TB/s, the join
// 3 of them; 40 slots x 16 heads x 15 beams of 500 .. 1024 tokens fp32 20.6 us, 3.3 TB/s (640 workgroups of unequal length on 256 CUs; the vector units issue in a third
// of the cycles, the matrix units in a tenth); 20 x 16 heads x 15
// beams of 12 .. 30 tokens 5.0 us, a launch and one tile's round trips.
// ---------------------------------------------------------------------------------------------------------------------------------
struct AttendArgs {
    const void *q;
    uint64_t q_row, q_head;          // strides in elements
    const uint8_t *k, *v;
    const float *k_scale, *v_scale;
    const int32_t *lengths;
    const uint8_t *keep;             // [slots][keep_stride] or null
    uint64_t keep_stride;
    void *out;
    float *part;                     // [slots][heads][beams * share][splits][dh + 4] when splits > 1
    uint32_t slots, heads, share, beams, T, block, splits, qtiles, items, vec;
    float scale2;                    // scale * log2(e)
};

template <typename T_> struct QP;
template <> struct QP<float> { enum { Q = 3, P = 3 }; };
template <> struct QP<bf16> { enum { Q = 1, P = 2 }; };

static __device__ __forceinline__ bf16x8 bytes8(uint32_t a, uint32_t b)
{
    u32x4 o;
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, false));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(a, 1.0f, true));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, false));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(b, 1.0f, true));
    return __builtin_bit_cast(bf16x8, o);
}

// what a wave needs of a tile of 64 tokens, as it lies in memory: K's rows with scales and mask bytes, V's rows
template <int DH> struct TileK {
    u32x4 k[4][DH / 64];
    float ks[4], vs[4];
    uint32_t keep[4];
};
template <int DH>
static __device__ __forceinline__ void load_k(const AttendArgs &a, const uint8_t *kb, const float *ksc, const float *vsc, const uint8_t *keep, uint32_t t, uint32_t subtiles,
                                              uint32_t c, uint32_t g, TileK<DH> &x)
{
    const uint32_t base = t * 64;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (j < (int)subtiles) {                                 // (a short tile: its last sixteens are not read)
#pragma unroll
            for (int h = 0; h < DH / 64; h++) x.k[j][h] = *(const u32x4 *)(kb + (uint64_t)(base + 16 * j + c) * DH + 64 * h + 16 * g);
        } else {
#pragma unroll
            for (int h = 0; h < DH / 64; h++) x.k[j][h] = u32x4{0, 0, 0, 0};
        }
        const uint32_t b = (base + 16 * j) / a.block;
        x.ks[j] = ksc[b];
        x.vs[j] = vsc[b];
        x.keep[j] = keep ? *(const uint32_t *)(keep + base + 16 * j + 4 * g) : 0x01010101u;
    }
}
template <int DH>
static __device__ __forceinline__ void load_v(const uint8_t *vb, uint32_t t, uint32_t c, uint32_t g, u32x4 v[DH / 16])
{
#pragma unroll
    for (int d = 0; d < DH / 16; d++) v[d] = *(const u32x4 *)(vb + (uint64_t)t * 64 * DH + (16 * d + c) * 64 + 16 * g);
}

// WAVES > 1: a workgroup per (slot, head, 16 queries, part of the tokens), its waves take the tiles in turn and are joined in LDS.  WAVES == 1 (one tile is all there is): four
// waves of a workgroup with an item each.
template <typename T_, int DH, int WAVES>
__global__ __launch_bounds__(256, DH == 64 ? 3 : 2) void k_kv8_attend(AttendArgs a)
{
    enum { HALVES = DH / 64, DT = DH / 16, NQ = QP<T_>::Q, NP = QP<T_>::P };
    const float NINF = -__builtin_huge_valf();
    __shared__ float s_m[WAVES][16], s_l[WAVES][16];
    __shared__ f32x4 s_o[WAVES][WAVES > 1 ? DT : 1][64];
    // (the wave's number as a scalar: what follows from it -- slot, lengths, scales, base addresses -- stays out of the vector registers)
    const uint32_t lane = threadIdx.x & 63, w4 = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), wave = WAVES > 1 ? w4 : 0, c = lane & 15, g = lane >> 4;
    const uint32_t id = WAVES > 1 ? blockIdx.x : blockIdx.x * 4 + w4;
    if (id >= a.items * a.splits) return;
    const uint32_t item = id / a.splits, split = id % a.splits;
    const uint32_t qt = item % a.qtiles, sh = item / a.qtiles, slot = sh / a.heads, head = sh % a.heads;
    const int32_t raw = a.lengths[slot];
    const uint32_t len = raw < 0 ? 0 : min((uint32_t)raw, a.T), tiles = (len + 63) / 64;
    const uint32_t t_begin = (uint32_t)((uint64_t)tiles * split / a.splits), t_end = (uint32_t)((uint64_t)tiles * (split + 1) / a.splits);
    const uint8_t *kb = a.k + (uint64_t)sh * a.T * DH, *vb = a.v + (uint64_t)sh * a.T * DH;
    const float *ksc = a.k_scale + (uint64_t)sh * (a.T / a.block), *vsc = a.v_scale + (uint64_t)sh * (a.T / a.block);
    const uint8_t *keep = a.keep ? a.keep + slot * a.keep_stride : nullptr;
    uint32_t t = t_begin + wave;
    TileK<DH> x;
    u32x4 v[DT];
    if (t < t_end) { load_k<DH>(a, kb, ksc, vsc, keep, t, min(4u, (len - 64 * t + 15) / 16), c, g, x); load_v<DH>(vb, t, c, g, v); }
    const uint32_t queries = a.beams * a.share, qi = qt * 16 + c;
    const bool live = qi < queries;
    const uint64_t row = (uint64_t)slot * a.beams + (live ? qi / a.share : 0);
    const uint32_t hq = head * a.share + (live ? qi % a.share : 0);
    bf16x8 q[HALVES][2][NQ];
    {
        const T_ *p = (const T_ *)a.q + row * a.q_row + (uint64_t)hq * a.q_head + 16 * g;
#pragma unroll
        for (int h = 0; h < HALVES; h++) {
            float y[16];
            if (live) load16(p + 64 * h, a.vec, y);
#pragma unroll
            for (int i = 0; i < 16; i++) y[i] = live ? y[i] : 0.f;
#pragma unroll
            for (int s = 0; s < 2; s++) {
                Planes pl;
                split8(y + 8 * s, pl);
#pragma unroll
                for (int n = 0; n < NQ; n++) q[h][s][n] = pl.p[n];
            }
        }
    }
    float m = NINF, l = 0.f;
    f32x4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    while (t < t_end) {
        // the next tile's K is in flight while this one is worked on, its V while the next scores are
        const uint32_t base = t * 64;
        TileK<DH> y;
        t += WAVES;
        if (WAVES > 1 && t < t_end) load_k<DH>(a, kb, ksc, vsc, keep, t, 4, c, g, y);
        uint32_t ok = 0;                                         // bit 4 j + r: token 16 j + 4 g + r counts
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (base + 16 * j + 4 * g + r < len && ((x.keep[j] >> (8 * r)) & 0xffu)) ok |= 1u << (4 * j + r);
        f32x4 s[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            s[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < HALVES; h++)
#pragma unroll
                for (int i = 0; i < 2; i++) {
                    const bf16x8 A = bytes8(x.k[j][h][2 * i], x.k[j][h][2 * i + 1]);
#pragma unroll
                    for (int n = 0; n < NQ; n++) s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, q[h][i][n], s[j], 0, 0, 0);
                }
        }
        float mx = m;
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const float f = x.ks[j] * a.scale2;
#pragma unroll
            for (int r = 0; r < 4; r++) {
                s[j][r] = (ok >> (4 * j + r)) & 1 ? s[j][r] * f : NINF;
                mx = fmaxf(mx, s[j][r]);
            }
        }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float mu = mx == NINF ? 0.f : mx;                  // (nothing seen yet: every p below is exp2(-inf) = 0)
        if (__any(mx != m)) {
            const float alpha = __builtin_amdgcn_exp2f(m - mu);
            l *= alpha;
#pragma unroll
            for (int d = 0; d < DT; d++) o[d] *= alpha;
        }
        m = mx;
        float pv[16];
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float p = __builtin_amdgcn_exp2f(s[j][r] - mu);
                l += p;
                pv[4 * j + r] = (ok >> (4 * j + r)) & 1 ? p * x.vs[j] : 0.f;      // (a block behind the length may have any scale)
            }
        if (__any(ok != 0xffffu)) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t b = ok >> (4 * j);
                const uint32_t mask = (b & 1 ? 0xffu : 0u) | (b & 2 ? 0xff00u : 0u) | (b & 4 ? 0xff0000u : 0u) | (b & 8 ? 0xff000000u : 0u);
#pragma unroll
                for (int d = 0; d < DT; d++) v[d][j] &= mask;
            }
        }
#pragma unroll
        for (int i = 0; i < 2; i++) {
            Planes pl;
            split8(pv + 8 * i, pl);
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const bf16x8 A = bytes8(v[d][2 * i], v[d][2 * i + 1]);
#pragma unroll
                for (int n = 0; n < NP; n++) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, pl.p[n], o[d], 0, 0, 0);
            }
        }
        if (WAVES > 1 && t < t_end) { load_v<DH>(vb, t, c, g, v); x = y; }
    }
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (WAVES > 1) {
        if (g == 0) { s_m[wave][c] = m; s_l[wave][c] = l; }
#pragma unroll
        for (int d = 0; d < DT; d++) s_o[wave][d][lane] = o[d];
        __syncthreads();
        float mm = NINF;
#pragma unroll
        for (int w = 0; w < WAVES; w++) mm = fmaxf(mm, s_m[w][c]);
        const float mu = mm == NINF ? 0.f : mm;
        l = 0.f;
        float f[WAVES];
#pragma unroll
        for (int w = 0; w < WAVES; w++) { f[w] = __builtin_amdgcn_exp2f(s_m[w][c] - mu); l += f[w] * s_l[w][c]; }
        m = mm;
#pragma unroll
        for (int d = 0; d < DT; d += WAVES) {                    // (DT is a multiple of the waves: each joins its share of the dims)
            f32x4 v = f[0] * s_o[0][d + wave][lane];
#pragma unroll
            for (int w = 1; w < WAVES; w++) v += f[w] * s_o[w][d + wave][lane];
            o[d / WAVES] = v;
        }
    }
    if (!live) return;
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);    // (nothing left: zeros; NaN stays)
    float *part = nullptr;
    T_ *out = (T_ *)a.out + (row * a.heads * a.share + hq) * DH;
    if (a.splits > 1) {
        part = a.part + (((uint64_t)sh * queries + qi) * a.splits + split) * (DH + 4);
        if (wave == 0 && g == 0) { part[DH] = m; part[DH + 1] = l; }
    }
#pragma unroll
    for (int d = 0; d < DT / (WAVES > 1 ? WAVES : 1); d++) {
        const uint32_t dim = 16 * (d * (WAVES > 1 ? WAVES : 1) + wave) + 4 * g;
        if (part) *(f32x4 *)(part + dim) = o[d];
        else {
#pragma unroll
            for (int r = 0; r < 4; r++) store1(out + dim + r, o[d][r] * inv);
        }
    }
}

// One query on a cache of one tile (a decode step over the short history of each of many rows): the matrix instructions would compute sixteen, and the registers of their
// operands keep waves away that this case needs -- 300 rows x 16 heads of 1 .. 17 tokens are one wave each: 7.8 us, a launch and 26 MB read (by the counters),
// three times what the tokens hold: the first sixteen tokens of V lie in every 16 bytes of its tile, so all 4 KB of it are read.  Plain
// multiply-adds on the same loads: lane (g, c) has dims 16 g .. of token c of each sixteen, then tokens 4 g .. of dim c.
template <typename T_, int DH>
__global__ __launch_bounds__(256) void k_kv8_attend_one(AttendArgs a)
{
    enum { HALVES = DH / 64, DT = DH / 16 };
    const float NINF = -__builtin_huge_valf();
    __shared__ __attribute__((aligned(16))) float s_p[4][64];
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), c = lane & 15, g = lane >> 4;
    const uint32_t sh = blockIdx.x * 4 + wave;
    if (sh >= a.items) return;
    const uint32_t slot = sh / a.heads, head = sh % a.heads;
    const uint8_t *kb = a.k + (uint64_t)sh * 64 * DH, *vb = a.v + (uint64_t)sh * 64 * DH;
    const float *ksc = a.k_scale + (uint64_t)sh * (64 / a.block), *vsc = a.v_scale + (uint64_t)sh * (64 / a.block);
    const uint8_t *keep = a.keep ? a.keep + slot * a.keep_stride : nullptr;
    u32x4 v[DT];
    load_v<DH>(vb, 0, c, g, v);
    float q[16 * HALVES];
#pragma unroll
    for (int h = 0; h < HALVES; h++) load16((const T_ *)a.q + slot * a.q_row + (uint64_t)head * a.q_head + 64 * h + 16 * g, a.vec, q + 16 * h);
    const int32_t raw = a.lengths[slot];
    const uint32_t len = raw < 0 ? 0 : min((uint32_t)raw, 64u);
    u32x4 k[4][HALVES];
    float s[4], m = NINF;
#pragma unroll
    for (int j = 0; j < 4; j++)
        if (16 * j < (int)len) {
#pragma unroll
            for (int h = 0; h < HALVES; h++) k[j][h] = *(const u32x4 *)(kb + (16 * j + c) * DH + 64 * h + 16 * g);
        }
#pragma unroll
    for (int j = 0; j < 4; j++) {
        s[j] = NINF;
        if (16 * j >= (int)len) continue;
        float acc = 0.f;
#pragma unroll
        for (int h = 0; h < HALVES; h++)
#pragma unroll
            for (int w = 0; w < 4; w++) {
                const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)k[j][h][w], false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)k[j][h][w], true);
                const float *x = q + 16 * h + 4 * w;
                acc = fmaf(lo[0], x[0], acc); acc = fmaf(lo[1], x[1], acc); acc = fmaf(hi[0], x[2], acc); acc = fmaf(hi[1], x[3], acc);
            }
        acc += __shfl_xor(acc, 16);
        acc += __shfl_xor(acc, 32);
        const uint32_t t = 16 * j + c;
        if (t < len && (!keep || keep[t])) s[j] = acc * (ksc[16 * j / a.block] * a.scale2);
        m = fmaxf(m, s[j]);
    }
    for (int o = 8; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float mu = m == NINF ? 0.f : m;
    float l = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        const float p = __builtin_amdgcn_exp2f(s[j] - mu);
        l += p;
        if (g == 0) s_p[wave][16 * j + c] = s[j] == NINF ? 0.f : p * vsc[16 * j / a.block];       // (a block behind the length may have any scale)
    }
    for (int o = 8; o > 0; o >>= 1) l += __shfl_xor(l, o);
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");       // (the wave's own: its LDS operations stay in order)
    float o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = 0.f;
#pragma unroll
    for (int j = 0; j < 4; j++) {
        if (16 * j >= (int)len) continue;
        const f32x4 p = *(const f32x4 *)&s_p[wave][16 * j + 4 * g];
        // (bytes of tokens that do not count may be NaN)
        uint32_t mask = 0xffffffffu;
        const int left = (int)len - (16 * j + 4 * (int)g);
        if (left < 4) mask = left <= 0 ? 0u : mask >> (8 * (4 - left));
        if (keep) {
            const uint32_t kp = *(const uint32_t *)(keep + 16 * j + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; r++) if (!((kp >> (8 * r)) & 0xffu)) mask &= ~(0xffu << (8 * r));
        }
#pragma unroll
        for (int d = 0; d < DT; d++) {
            const uint32_t w = v[d][j] & mask;
            const auto lo = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, false), hi = __builtin_amdgcn_cvt_pk_f32_fp8((int)w, true);
            o[d] = fmaf(lo[0], p[0], o[d]); o[d] = fmaf(lo[1], p[1], o[d]); o[d] = fmaf(hi[0], p[2], o[d]); o[d] = fmaf(hi[1], p[3], o[d]);
        }
    }
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    T_ *out = (T_ *)a.out + (uint64_t)sh * DH;
#pragma unroll
    for (int d = 0; d < DT; d++) {
        o[d] += __shfl_xor(o[d], 16);
        o[d] += __shfl_xor(o[d], 32);
        if ((d & 3) == (int)g) store1(out + 16 * d + c, o[d] * inv);
    }
}

// the parts of one (query row, query head) joined: a workgroup, whose waves take the parts in turn
template <typename T_, int DH>
__global__ __launch_bounds__(256) void k_kv8_join(AttendArgs a)
{
    enum { H = DH / 64 };
    const float NINF = -__builtin_huge_valf();
    __shared__ float s_l[4], s_v[4][DH];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint64_t id = blockIdx.x;
    const uint32_t queries = a.beams * a.share, qi = (uint32_t)(id % queries), sh = (uint32_t)(id / queries), slot = sh / a.heads, head = sh % a.heads;
    const float *part = a.part + id * a.splits * (DH + 4);
    float m = NINF;
    for (uint32_t s = lane; s < a.splits; s += 64) m = fmaxf(m, part[s * (uint64_t)(DH + 4) + DH]);
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float mu = m == NINF ? 0.f : m;
    float l = 0.f, v[H];
#pragma unroll
    for (int h = 0; h < H; h++) v[h] = 0.f;
#pragma unroll 4
    for (uint32_t s = wave; s < a.splits; s += 4) {
        const float *p = part + s * (uint64_t)(DH + 4);
        const float f = __builtin_amdgcn_exp2f(p[DH] - mu);
        l += f * p[DH + 1];
#pragma unroll
        for (int h = 0; h < H; h++) v[h] += f * p[64 * h + lane];
    }
    if (lane == 0) s_l[wave] = l;
#pragma unroll
    for (int h = 0; h < H; h++) s_v[wave][64 * h + lane] = v[h];
    __syncthreads();
    l = s_l[0] + s_l[1] + s_l[2] + s_l[3];
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    const uint64_t row = (uint64_t)slot * a.beams + qi / a.share;
    T_ *out = (T_ *)a.out + (row * a.heads * a.share + head * a.share + qi % a.share) * DH;
    if (threadIdx.x < DH) store1(out + threadIdx.x, (s_v[0][threadIdx.x] + s_v[1][threadIdx.x] + s_v[2][threadIdx.x] + s_v[3][threadIdx.x]) * inv);
}

// ---- C ABI ----
static int check_cache(const char *who, uint32_t T, uint32_t block, uint32_t dh, const void *k, const void *v, const void *ks, const void *vs)
{
    if (dh != 64 && dh != 128) { fmi_set_error("%s: head_dim %u must be 64 or 128", who, dh); return FMI_ERR_UNSUPPORTED; }
    if (block != 16 && block != 32 && block != 64) { fmi_set_error("%s: block of %u tokens must be 16, 32 or 64", who, block); return FMI_ERR_UNSUPPORTED; }
    if (!T || T % 64 || T > (1u << 30)) { fmi_set_error("%s: %u tokens must be a multiple of 64", who, T); return FMI_ERR_UNSUPPORTED; }
    if (!k || !v || !ks || !vs || ((uintptr_t)k & 15) || ((uintptr_t)v & 15) || ((uintptr_t)ks & 3) || ((uintptr_t)vs & 3)) {
        fmi_set_error("%s: the cache must be given, its codes aligned to 16 bytes", who);
        return FMI_ERR_ARG;
    }
    return FMI_OK;
}

template <typename T_>
static int kv8_append(void *stream, const void *k_new, const void *v_new, const uint64_t *strides, uint32_t n, const int32_t *lengths, const int32_t *counts,
                      void *k, void *v, float *k_scale, float *v_scale, uint32_t slots, uint32_t heads, uint32_t T, uint32_t block, uint32_t dh)
{
    const int rc = check_cache("sealnn_kv8_append", T, block, dh, k, v, k_scale, v_scale);
    if (rc) return rc;
    if (!slots || !heads || !n) return FMI_OK;
    if (!k_new || !v_new || !strides || !lengths || ((uintptr_t)k_new & (sizeof(T_) - 1)) || ((uintptr_t)v_new & (sizeof(T_) - 1))) {
        fmi_set_error("sealnn_kv8_append: the new tokens, their strides and the lengths must be given");
        return FMI_ERR_ARG;
    }
    if (slots > 65535u || (uint64_t)slots * heads > 0x7fffffffu || ((uint64_t)std::min(n, T) / 64 + 2) * heads > 0x7fffffffu) {
        fmi_set_error("sealnn_kv8_append: %u slots (up to 65535) x %u heads x %u tokens are too many", slots, heads, n);
        return FMI_ERR_UNSUPPORTED;
    }
    AppendArgs a;
    a.src[0] = k_new; a.src[1] = v_new;
    uint64_t odd = (uintptr_t)k_new | (uintptr_t)v_new;
    for (int i = 0; i < 2; i++) {
        a.slot_stride[i] = strides[3 * i]; a.token_stride[i] = strides[3 * i + 1]; a.head_stride[i] = strides[3 * i + 2];
        odd |= (strides[3 * i] | strides[3 * i + 1] | strides[3 * i + 2]) * sizeof(T_);
    }
    a.codes[0] = (uint8_t *)k; a.codes[1] = (uint8_t *)v;
    a.scale[0] = k_scale; a.scale[1] = v_scale;
    a.lengths = lengths; a.counts = counts;
    a.n = std::min(n, T); a.slots = slots; a.heads = heads; a.T = T; a.block = block; a.dh = dh;
    const uint32_t vec = (odd & (4 * sizeof(T_) - 1)) == 0;
    const hipStream_t st = (hipStream_t)stream;
    if (n == 1) {
        const dim3 grid((slots * heads + 3) / 4);
        if (dh == 64) hipLaunchKernelGGL((k_kv8_append_one<T_, 64>), grid, dim3(256), 0, st, a);
        else hipLaunchKernelGGL((k_kv8_append_one<T_, 128>), grid, dim3(256), 0, st, a);
    } else {
        const dim3 grid(((a.n + 62) / 64 + 1) * heads, slots);
        if (dh == 64) hipLaunchKernelGGL((k_kv8_append<T_, 64>), grid, dim3(256), 0, st, a, vec);
        else hipLaunchKernelGGL((k_kv8_append<T_, 128>), grid, dim3(256), 0, st, a, vec);
    }
    NNCHK();
    return FMI_OK;
}

template <typename T_, int DH>
static void launch_attend(hipStream_t st, const AttendArgs &a)
{
    if (a.T == 64 && a.beams * a.share == 1) hipLaunchKernelGGL((k_kv8_attend_one<T_, DH>), dim3((a.items + 3) / 4), dim3(256), 0, st, a);
    else if (a.T == 64) hipLaunchKernelGGL((k_kv8_attend<T_, DH, 1>), dim3((a.items + 3) / 4), dim3(256), 0, st, a);
    else hipLaunchKernelGGL((k_kv8_attend<T_, DH, 4>), dim3(a.items * a.splits), dim3(256), 0, st, a);
    if (a.splits > 1) hipLaunchKernelGGL((k_kv8_join<T_, DH>), dim3(a.slots * a.heads * a.beams * a.share), dim3(256), 0, st, a);
}

template <typename T_>
static int kv8_attend(void *stream, const void *q, uint64_t q_row_stride, uint64_t q_head_stride, const void *k, const void *v, const float *k_scale,
                      const float *v_scale, const int32_t *lengths, const uint8_t *keep, uint64_t keep_stride, uint32_t slots, uint32_t beams, uint32_t heads,
                      uint32_t share, uint32_t T, uint32_t block, uint32_t dh, float scale, uint32_t splits, void *work, uint64_t work_bytes, void *out)
{
    const int rc = check_cache("sealnn_kv8_attend", T, block, dh, k, v, k_scale, v_scale);
    if (rc) return rc;
    if (!slots || !heads || !beams || !share) return FMI_OK;
    if (!q || !out || !lengths || ((uintptr_t)q & (sizeof(T_) - 1)) || (keep && (((uintptr_t)keep | keep_stride) & 3))) {
        fmi_set_error("sealnn_kv8_attend: q, out and lengths must be given, the mask's rows aligned to 4 bytes");
        return FMI_ERR_ARG;
    }
    if (splits < 1 || splits > T / 64) { fmi_set_error("sealnn_kv8_attend: %u parts of %u tiles", splits, T / 64); return FMI_ERR_ARG; }
    AttendArgs a;
    a.q = q; a.q_row = q_row_stride; a.q_head = q_head_stride;
    a.k = (const uint8_t *)k; a.v = (const uint8_t *)v; a.k_scale = k_scale; a.v_scale = v_scale;
    a.lengths = lengths; a.keep = keep; a.keep_stride = keep_stride;
    a.out = out; a.part = (float *)work;
    a.slots = slots; a.heads = heads; a.share = share; a.beams = beams; a.T = T; a.block = block; a.splits = splits;
    const uint64_t queries = (uint64_t)beams * share, qtiles = (queries + 15) / 16, items = (uint64_t)slots * heads * qtiles;
    if (queries > (1u << 20) || items * splits > 0x7fffffffull || (uint64_t)slots * heads * queries > 0x7fffffffull) {
        fmi_set_error("sealnn_kv8_attend: %u slots x %u heads x %llu queries are too many", slots, heads, (unsigned long long)queries);
        return FMI_ERR_UNSUPPORTED;
    }
    a.qtiles = (uint32_t)qtiles;
    a.items = (uint32_t)items;
    a.vec = (((uintptr_t)q | q_row_stride * sizeof(T_) | q_head_stride * sizeof(T_)) & 15) == 0;
    a.scale2 = scale * 1.4426950408889634f;
    if (splits > 1 && (!work || ((uintptr_t)work & 15) || work_bytes < (uint64_t)slots * heads * queries * splits * (dh + 4) * sizeof(float))) {
        fmi_set_error("sealnn_kv8_attend: the workspace must hold %llu bytes", (unsigned long long)((uint64_t)slots * heads * queries * splits * (dh + 4) * sizeof(float)));
        return FMI_ERR_CAPACITY;
    }
    if (dh == 64) launch_attend<T_, 64>((hipStream_t)stream, a);
    else launch_attend<T_, 128>((hipStream_t)stream, a);
    NNCHK();
    return FMI_OK;
}

extern "C" int sealnn_kv8_append(void *stream, const float *k_new, const float *v_new, const uint64_t *strides, uint32_t n, const int32_t *lengths,
                                 const int32_t *counts, void *k, void *v, float *k_scale, float *v_scale, uint32_t slots, uint32_t heads, uint32_t T,
                                 uint32_t block, uint32_t dh)
{ return kv8_append<float>(stream, k_new, v_new, strides, n, lengths, counts, k, v, k_scale, v_scale, slots, heads, T, block, dh); }
extern "C" int sealnn_kv8_append_bf16(void *stream, const void *k_new, const void *v_new, const uint64_t *strides, uint32_t n, const int32_t *lengths,
                                      const int32_t *counts, void *k, void *v, float *k_scale, float *v_scale, uint32_t slots, uint32_t heads, uint32_t T,
                                      uint32_t block, uint32_t dh)
{ return kv8_append<bf16>(stream, k_new, v_new, strides, n, lengths, counts, k, v, k_scale, v_scale, slots, heads, T, block, dh); }
extern "C" int sealnn_kv8_attend(void *stream, const float *q, uint64_t q_row_stride, uint64_t q_head_stride, const void *k, const void *v,
                                 const float *k_scale, const float *v_scale, const int32_t *lengths, const uint8_t *keep, uint64_t keep_stride,
                                 uint32_t slots, uint32_t beams, uint32_t heads, uint32_t share, uint32_t T, uint32_t block, uint32_t dh, float scale,
                                 uint32_t splits, void *work, uint64_t work_bytes, float *out)
{ return kv8_attend<float>(stream, q, q_row_stride, q_head_stride, k, v, k_scale, v_scale, lengths, keep, keep_stride, slots, beams, heads, share, T, block, dh, scale, splits, work, work_bytes, out); }
extern "C" int sealnn_kv8_attend_bf16(void *stream, const void *q, uint64_t q_row_stride, uint64_t q_head_stride, const void *k, const void *v,
                                      const float *k_scale, const float *v_scale, const int32_t *lengths, const uint8_t *keep, uint64_t keep_stride,
                                      uint32_t slots, uint32_t beams, uint32_t heads, uint32_t share, uint32_t T, uint32_t block, uint32_t dh, float scale,
                                      uint32_t splits, void *work, uint64_t work_bytes, void *out)
{ return kv8_attend<bf16>(stream, q, q_row_stride, q_head_stride, k, v, k_scale, v_scale, lengths, keep, keep_stride, slots, beams, heads, share, T, block, dh, scale, splits, work, work_bytes, out); }
