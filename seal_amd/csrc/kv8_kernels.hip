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
// four numbers, already divided by the scale, as e4m3 codes: to nearest, ties to even; infinities become +-448, NaN stays
static __device__ __forceinline__ float sat(float y) { return y != y ? y : fminf(fmaxf(y, -448.f), 448.f); }
static __device__ __forceinline__ uint32_t encode4(float a, float b, float c, float d)
{
    int w = __builtin_amdgcn_cvt_pk_fp8_f32(sat(a), sat(b), 0, false);
    return (uint32_t)__builtin_amdgcn_cvt_pk_fp8_f32(sat(c), sat(d), w, true);
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

// One workgroup of NTHR threads per (slot, head, 64-token tile, K or V).  Nobody else writes the tile, so bytes that the call does not
// touch are carried over by reading them.  First the largest magnitude of the new tokens of each block, then the codes.
template <typename T_, int NTHR>
__global__ __launch_bounds__(NTHR) void k_kv8_append(AppendArgs a, uint32_t vec)
{
    __shared__ uint32_t s_max[4];
    __shared__ __attribute__((aligned(16))) uint8_t s_tile[128 * 80];     // V: [dh][64 tokens + padding]
    const uint32_t which = blockIdx.z, slot = blockIdx.y / a.heads, head = blockIdx.y % a.heads, tid = threadIdx.x;
    const int64_t len = a.lengths[slot];
    const int64_t cnt = a.counts ? min((int64_t)a.counts[slot], (int64_t)a.n) : (int64_t)a.n;
    if (len < 0 || len >= (int64_t)a.T || cnt <= 0) return;
    const int64_t tile = len / 64 + blockIdx.x, base = tile * 64;
    const int64_t lo = max(len, base), hi = min(min(len + cnt, (int64_t)a.T), base + 64);
    if (lo >= hi) return;
    const uint32_t l0 = (uint32_t)(lo - base), l1 = (uint32_t)(hi - base);           // new tokens of the tile
    const uint32_t dh = a.dh, chunks = dh / 16, blk = a.block;
    const uint64_t sh = (uint64_t)slot * a.heads + head;
    const T_ *src = (const T_ *)a.src[which] + slot * a.slot_stride[which] + head * a.head_stride[which];
    float *scale = a.scale[which] + sh * (a.T / blk) + (uint64_t)base / blk;
    if (tid < 4) s_max[tid] = 0;
    __syncthreads();
    for (uint32_t u = tid; u < (l1 - l0) * chunks; u += NTHR) {
        const uint32_t t = l0 + u / chunks, c = u % chunks;
        float v[16], m = 0.f;
        load16(src + (uint64_t)(base + t - len) * a.token_stride[which] + 16 * c, vec, v);
#pragma unroll
        for (int i = 0; i < 16; i++) m = fabsf(v[i]) < __builtin_huge_valf() ? fmaxf(m, fabsf(v[i])) : m;
        atomicMax(&s_max[t / blk], as_u32(m));                   // (magnitudes order as their bits: the same whatever the order)
    }
    __syncthreads();
    // the blocks of this tile that the call touches, their old and new exponents
    const uint32_t b0 = l0 / blk, b1 = (l1 - 1) / blk;
    const bool held = l0 % blk != 0;                             // the first touched block had tokens before
    int e_new[4], e_old = 0;
#pragma unroll
    for (uint32_t b = 0; b < 4; b++) e_new[b] = (b >= b0 && b <= b1) ? exponent_for(as_f32(s_max[b])) : 0;
    if (held) {
        e_old = exponent_of(scale[b0]);
        e_new[0] = b0 == 0 ? max(e_new[0], e_old) : e_new[0]; e_new[1] = b0 == 1 ? max(e_new[1], e_old) : e_new[1];
        e_new[2] = b0 == 2 ? max(e_new[2], e_old) : e_new[2]; e_new[3] = b0 == 3 ? max(e_new[3], e_old) : e_new[3];
    }
    auto exp_of = [&](uint32_t b) { return b == 0 ? e_new[0] : b == 1 ? e_new[1] : b == 2 ? e_new[2] : e_new[3]; };
    const int e_held = exp_of(b0);
    const bool grow = held && e_held > e_old;
    const float shift = grow ? pow2i(max(e_old - e_held, -126)) : 1.f;
    __syncthreads();                                             // (every thread has read the old scale)
    if (tid < 4 && tid >= b0 && tid <= b1) scale[tid] = pow2i(exp_of(tid));
    if (which == 0) {
        uint8_t *codes = a.codes[0] + (sh * a.T + (uint64_t)base) * dh;
        for (uint32_t u = tid; u < (l1 - l0) * chunks; u += NTHR) {
            const uint32_t t = l0 + u / chunks, c = u % chunks;
            float v[16];
            load16(src + (uint64_t)(base + t - len) * a.token_stride[which] + 16 * c, vec, v);
            const float f = pow2i(-exp_of(t / blk));
            u32x4 w;
#pragma unroll
            for (int i = 0; i < 4; i++) w[i] = encode4(v[4 * i] * f, v[4 * i + 1] * f, v[4 * i + 2] * f, v[4 * i + 3] * f);
            *(u32x4 *)(codes + (uint64_t)t * dh + 16 * c) = w;
        }
        if (grow)
            for (uint32_t u = tid; u < (l0 - b0 * blk) * chunks; u += NTHR) {
                u32x4 *p = (u32x4 *)(codes + (uint64_t)(b0 * blk + u / chunks) * dh + 16 * (u % chunks));
                u32x4 w = *p;
#pragma unroll
                for (int i = 0; i < 4; i++) w[i] = shift4(w[i], shift);
                *p = w;
            }
        return;
    }
    // V: the codes of the new tokens transposed through LDS, then merged into the tile's rows
    for (uint32_t u = tid; u < (l1 - l0) * chunks; u += NTHR) {
        const uint32_t t = l0 + u / chunks, c = u % chunks;
        float v[16];
        load16(src + (uint64_t)(base + t - len) * a.token_stride[which] + 16 * c, vec, v);
        const float f = pow2i(-exp_of(t / blk));
        const uint32_t at = ((t >> 2) & 3) * 16 + (t >> 4) * 4 + (t & 3);
#pragma unroll
        for (int i = 0; i < 4; i++) {
            const uint32_t w = encode4(v[4 * i] * f, v[4 * i + 1] * f, v[4 * i + 2] * f, v[4 * i + 3] * f);
#pragma unroll
            for (int j = 0; j < 4; j++) s_tile[(16 * c + 4 * i + j) * 80 + at] = (uint8_t)(w >> (8 * j));
        }
    }
    __syncthreads();
    uint8_t *codes = a.codes[1] + (sh * a.T + (uint64_t)base) * dh;
    const bool whole = l0 == 0 && l1 == 64;
    for (uint32_t u = tid; u < dh * 4; u += NTHR) {
        const uint32_t d = u / 4, g = u % 4;
        u32x4 *p = (u32x4 *)(codes + (uint64_t)d * 64 + g * 16);
        const u32x4 fresh = *(const u32x4 *)(s_tile + d * 80 + g * 16);
        u32x4 w = fresh;
        if (!whole) {
            w = *p;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) {                   // word j: tokens 16 j + 4 g .. + 3
                const uint32_t t0 = 16 * j + 4 * g;
                uint32_t m_new = 0, m_old = 0;
#pragma unroll
                for (uint32_t r = 0; r < 4; r++) {
                    if (t0 + r >= l0 && t0 + r < l1) m_new |= 0xffu << (8 * r);
                    if (t0 + r >= b0 * blk && t0 + r < l0) m_old |= 0xffu << (8 * r);
                }
                const uint32_t again = grow ? shift4(w[j], shift) : w[j];
                w[j] = (w[j] & ~(m_new | m_old)) | (again & m_old) | (fresh[j] & m_new);
            }
        }
        *p = w;
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
// for that.  q and p are fp32 numbers and enter as three bf16 planes each (exact); for bf16 queries q is one plane and p two (2^-17 relative:
// the rounding of p stays far below the output's own).  A block's scale is a factor of S's rows (K) or of p (V).
// Bytes behind `length` or masked may be anything: S is selected, p is 0 there and V's bytes are cleared.
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
    float *part;                     // [items][splits][16][dh + 2] when splits > 1
    uint32_t slots, heads, share, beams, T, block, splits, qtiles;
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

template <typename T_, int DH, int WAVES>
__global__ __launch_bounds__(64 * WAVES) void k_kv8_attend(AttendArgs a)
{
    enum { HALVES = DH / 64, DT = DH / 16, NQ = QP<T_>::Q, NP = QP<T_>::P };
    const float NINF = -__builtin_huge_valf();
    __shared__ float s_m[WAVES][16], s_l[WAVES][16];
    __shared__ f32x4 s_o[WAVES > 1 ? WAVES : 1][DT][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, c = lane & 15, g = lane >> 4;
    const uint32_t item = blockIdx.x / a.splits, split = blockIdx.x % a.splits;
    const uint32_t qt = item % a.qtiles, sh = item / a.qtiles, slot = sh / a.heads, head = sh % a.heads;
    const int32_t raw = a.lengths[slot];
    const uint32_t len = raw < 0 ? 0 : min((uint32_t)raw, a.T), tiles = (len + 63) / 64;
    const uint32_t t_begin = (uint32_t)((uint64_t)tiles * split / a.splits), t_end = (uint32_t)((uint64_t)tiles * (split + 1) / a.splits);
    const uint32_t queries = a.beams * a.share, qi = qt * 16 + c;
    const bool live = qi < queries;
    const uint64_t row = (uint64_t)slot * a.beams + (live ? qi / a.share : 0);
    const uint32_t hq = head * a.share + (live ? qi % a.share : 0);
    bf16x8 q[HALVES][2][NQ];
    {
        const T_ *p = (const T_ *)a.q + row * a.q_row + (uint64_t)hq * a.q_head;
#pragma unroll
        for (int h = 0; h < HALVES; h++)
#pragma unroll
            for (int s = 0; s < 2; s++) {
                float x[8];
#pragma unroll
                for (int i = 0; i < 8; i++) x[i] = live ? load1(p + 64 * h + 16 * g + 8 * s + i) : 0.f;
                Planes pl;
                split8(x, pl);
#pragma unroll
                for (int n = 0; n < NQ; n++) q[h][s][n] = pl.p[n];
            }
    }
    float m = NINF, l = 0.f;
    f32x4 o[DT];
#pragma unroll
    for (int d = 0; d < DT; d++) o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
    const uint8_t *kb = a.k + (uint64_t)sh * a.T * DH, *vb = a.v + (uint64_t)sh * a.T * DH;
    const float *ksc = a.k_scale + (uint64_t)sh * (a.T / a.block), *vsc = a.v_scale + (uint64_t)sh * (a.T / a.block);
    for (uint32_t t = t_begin + wave; t < t_end; t += WAVES) {
        const uint32_t base = t * 64;
        u32x4 kw[4][HALVES], vw[DT];
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int h = 0; h < HALVES; h++) kw[j][h] = *(const u32x4 *)(kb + (uint64_t)(base + 16 * j + c) * DH + 64 * h + 16 * g);
#pragma unroll
        for (int d = 0; d < DT; d++) vw[d] = *(const u32x4 *)(vb + (uint64_t)base * DH + (16 * d + c) * 64 + 16 * g);
        float ks[4], vs[4];
        uint32_t ok = 0;                                         // bit 4 j + r: token 16 j + 4 g + r counts
#pragma unroll
        for (int j = 0; j < 4; j++) {
            const uint32_t b = (base + 16 * j) / a.block;
            ks[j] = ksc[b] * a.scale2;
            vs[j] = vsc[b];
            uint32_t kp = 0x01010101u;
            if (a.keep) kp = *(const uint32_t *)(a.keep + slot * a.keep_stride + base + 16 * j + 4 * g);
#pragma unroll
            for (int r = 0; r < 4; r++)
                if (base + 16 * j + 4 * g + r < len && ((kp >> (8 * r)) & 0xffu)) ok |= 1u << (4 * j + r);
        }
        f32x4 s[4];
#pragma unroll
        for (int j = 0; j < 4; j++) {
            s[j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int h = 0; h < HALVES; h++)
#pragma unroll
                for (int x = 0; x < 2; x++) {
                    const bf16x8 A = bytes8(kw[j][h][2 * x], kw[j][h][2 * x + 1]);
#pragma unroll
                    for (int n = 0; n < NQ; n++) s[j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, q[h][x][n], s[j], 0, 0, 0);
                }
        }
        float mx = m;
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                s[j][r] = (ok >> (4 * j + r)) & 1 ? s[j][r] * ks[j] : NINF;
                mx = fmaxf(mx, s[j][r]);
            }
        mx = fmaxf(mx, __shfl_xor(mx, 16));
        mx = fmaxf(mx, __shfl_xor(mx, 32));
        const float mu = mx == NINF ? 0.f : mx;                  // (nothing seen yet: every p below is exp2(-inf) = 0)
        const float alpha = __builtin_amdgcn_exp2f(m - mu);
        m = mx;
        l *= alpha;
#pragma unroll
        for (int d = 0; d < DT; d++) o[d] *= alpha;
        float pv[16];
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int r = 0; r < 4; r++) {
                const float p = __builtin_amdgcn_exp2f(s[j][r] - mu);
                l += p;
                pv[4 * j + r] = (ok >> (4 * j + r)) & 1 ? p * vs[j] : 0.f;      // (a block behind the length may have any scale)
            }
        if (__any(ok != 0xffffu)) {
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t b = ok >> (4 * j);
                const uint32_t mask = (b & 1 ? 0xffu : 0u) | (b & 2 ? 0xff00u : 0u) | (b & 4 ? 0xff0000u : 0u) | (b & 8 ? 0xff000000u : 0u);
#pragma unroll
                for (int d = 0; d < DT; d++) vw[d][j] &= mask;
            }
        }
#pragma unroll
        for (int x = 0; x < 2; x++) {
            Planes pl;
            split8(pv + 8 * x, pl);
#pragma unroll
            for (int d = 0; d < DT; d++) {
                const bf16x8 A = bytes8(vw[d][2 * x], vw[d][2 * x + 1]);
#pragma unroll
                for (int n = 0; n < NP; n++) o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(A, pl.p[n], o[d], 0, 0, 0);
            }
        }
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
        for (uint32_t d = wave; d < DT; d += WAVES) {
            f32x4 v = f[0] * s_o[0][d][lane];
#pragma unroll
            for (int w = 1; w < WAVES; w++) v += f[w] * s_o[w][d][lane];
            s_o[0][d][lane] = v;                                 // (this wave's d alone)
        }
    }
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);    // (nothing left: zeros; NaN stays)
    if (a.splits == 1) {
        if (!live) return;
        T_ *out = (T_ *)a.out + (row * a.heads * a.share + hq) * DH;
#pragma unroll
        for (int d = 0; d < DT; d++) {
            if (WAVES > 1 && d % WAVES != wave) continue;
            const f32x4 v = WAVES > 1 ? s_o[0][d][lane] : o[d];
#pragma unroll
            for (int r = 0; r < 4; r++) store1(out + 16 * d + 4 * g + r, v[r] * inv);
        }
        return;
    }
    float *part = a.part + (((uint64_t)item * a.splits + split) * 16 + c) * (DH + 4);
    if (wave == 0 && g == 0) { part[DH] = m; part[DH + 1] = l; }
#pragma unroll
    for (int d = 0; d < DT; d++) {
        if (WAVES > 1 && d % WAVES != wave) continue;
        *(f32x4 *)(part + 16 * d + 4 * g) = WAVES > 1 ? s_o[0][d][lane] : o[d];
    }
}

// the parts of one (query row, query head) joined: one wave each
template <typename T_, int DH>
__global__ __launch_bounds__(256) void k_kv8_join(AttendArgs a)
{
    const float NINF = -__builtin_huge_valf();
    const uint32_t lane = threadIdx.x & 63;
    const uint64_t id = (uint64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const uint32_t queries = a.beams * a.share;
    if (id >= (uint64_t)a.slots * a.heads * queries) return;
    const uint32_t qi = (uint32_t)(id % queries), sh = (uint32_t)(id / queries), slot = sh / a.heads, head = sh % a.heads;
    const float *part = a.part + (((uint64_t)sh * a.qtiles + qi / 16) * a.splits * 16 + qi % 16) * (DH + 4);
    const uint64_t step = (uint64_t)16 * (DH + 4);
    float m = NINF;
    for (uint32_t s = lane; s < a.splits; s += 64) m = fmaxf(m, part[s * step + DH]);
    for (int o = 32; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor(m, o));
    const float mu = m == NINF ? 0.f : m;
    float l = 0.f, v[DH / 64];
#pragma unroll
    for (int h = 0; h < DH / 64; h++) v[h] = 0.f;
    for (uint32_t s = 0; s < a.splits; s++) {
        const float f = __builtin_amdgcn_exp2f(part[s * step + DH] - mu);
        l += f * part[s * step + DH + 1];
#pragma unroll
        for (int h = 0; h < DH / 64; h++) v[h] += f * part[s * step + 64 * h + lane];
    }
    const float inv = l > 0.f ? 1.f / l : (l == l ? 0.f : l);
    const uint64_t row = (uint64_t)slot * a.beams + qi / a.share;
    T_ *out = (T_ *)a.out + (row * a.heads * a.share + head * a.share + qi % a.share) * DH;
#pragma unroll
    for (int h = 0; h < DH / 64; h++) store1(out + 64 * h + lane, v[h] * inv);
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
    if ((uint64_t)slots * heads > 65535u) { fmi_set_error("sealnn_kv8_append: %u slots x %u heads are more than 65535", slots, heads); return FMI_ERR_UNSUPPORTED; }
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
    const uint32_t vec = (odd & 15) == 0;
    const dim3 grid((a.n + 62) / 64 + 1, slots * heads, 2);
    if (n == 1) hipLaunchKernelGGL((k_kv8_append<T_, 64>), grid, dim3(64), 0, (hipStream_t)stream, a, vec);
    else hipLaunchKernelGGL((k_kv8_append<T_, 256>), grid, dim3(256), 0, (hipStream_t)stream, a, vec);
    NNCHK();
    return FMI_OK;
}

template <typename T_, int DH>
static void launch_attend(hipStream_t st, const AttendArgs &a)
{
    const uint32_t grid = a.slots * a.heads * a.qtiles * a.splits;
    if (a.T == 64) hipLaunchKernelGGL((k_kv8_attend<T_, DH, 1>), dim3(grid), dim3(64), 0, st, a);
    else hipLaunchKernelGGL((k_kv8_attend<T_, DH, 4>), dim3(grid), dim3(256), 0, st, a);
    if (a.splits > 1) hipLaunchKernelGGL((k_kv8_join<T_, DH>), dim3((uint32_t)(((uint64_t)a.slots * a.heads * a.beams * a.share + 3) / 4)), dim3(256), 0, st, a);
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
    if (queries > (1u << 20) || items * splits > 0x7fffffffull || (uint64_t)slots * heads * queries > 0xfffffff0ull) {
        fmi_set_error("sealnn_kv8_attend: %u slots x %u heads x %llu queries are too many", slots, heads, (unsigned long long)queries);
        return FMI_ERR_UNSUPPORTED;
    }
    a.qtiles = (uint32_t)qtiles;
    a.scale2 = scale * 1.4426950408889634f;
    if (splits > 1 && (!work || ((uintptr_t)work & 15) || work_bytes < items * splits * 16 * (dh + 4) * sizeof(float))) {
        fmi_set_error("sealnn_kv8_attend: the workspace must hold %llu bytes", (unsigned long long)(items * splits * 16 * (dh + 4) * sizeof(float)));
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
