// y = x W^T + b with 4-bit weights (e2m1 codes, a bf16 scale for every `group` columns of a row): the products of a decode step of few
// rows, which are bound by reading W once (include/sealnn.h: sealnn_w4_linear).
//
// Layout: a wave reads one 16-row x 128-column tile of W as ONE 16-byte load per lane, 1 KB contiguous, and the bytes arrive where the
// matrix instruction wants them: lane (g, row) = (lane >> 4, lane & 15) holds in word s the eight codes of columns 32 s + 8 g .. + 7, the A
// fragment of v_mfma_f32_16x16x32_bf16 number s.  e2m1 -> bf16 is one instruction per two codes and exact; x enters as bf16 planes whose sum
// it is (three for fp32, one for bf16).  The 32 columns of one instruction lie in one group, so the scale is applied to the fp32
// accumulator: 4 multiply-adds per lane, group and tile.
#include "nn_common.h"

#include <algorithm>

template <typename T> struct XPlanes;
template <> struct XPlanes<float> { enum { N = 3 }; };
template <> struct XPlanes<bf16> { enum { N = 1 }; };

// columns k .. k + 7 of a row of x as bf16 planes; columns from K on are zero (`vec`: rows and pointer allow 16-byte loads)
template <typename T>
static __device__ __forceinline__ void load_x(const T *row, uint32_t k, uint32_t K, bool vec, bf16x8 out[XPlanes<T>::N])
{
    if constexpr (std::is_same<T, float>::value) {
        float v[8];
        if (vec && k + 8 <= K) {
            const f32x4 a = *(const f32x4 *)(row + k), b = *(const f32x4 *)(row + k + 4);
#pragma unroll
            for (int i = 0; i < 4; i++) { v[i] = a[i]; v[4 + i] = b[i]; }
        } else {
#pragma unroll
            for (int i = 0; i < 8; i++) v[i] = k + i < K ? row[k + i] : 0.f;
        }
        Planes p;
        split8(v, p);
#pragma unroll
        for (int i = 0; i < 3; i++) out[i] = p.p[i];
    } else {
        u32x4 w = {0, 0, 0, 0};
        const uint16_t *r = reinterpret_cast<const uint16_t *>(row) + k;
        if (vec && k + 8 <= K) w = *(const u32x4 *)r;
        else {
#pragma unroll
            for (int i = 0; i < 8; i++) if (k + i < K) w[i / 2] |= (uint32_t)r[i] << (16 * (i & 1));
        }
        out[0] = __builtin_bit_cast(bf16x8, w);
    }
}

// a lane's part of a 128-column chunk of a row of x: columns 32 s + 8 g .. + 7 for s = 0 .. 3.  A chunk that ends within the row is loaded whole before
// anything is made of it (one after the other, each behind its own condition, they cost a round trip to memory each).
template <typename T>
static __device__ __forceinline__ void load_chunk(const T *row, uint32_t c, uint32_t g, uint32_t K, bool vec, bf16x8 out[4][XPlanes<T>::N])
{
    const uint32_t k = 128 * c + 8 * g;
    if (vec && 128 * (c + 1) <= K) {
        if constexpr (std::is_same<T, float>::value) {
            f32x4 v[4][2];
#pragma unroll
            for (int s = 0; s < 4; s++) { v[s][0] = *(const f32x4 *)(row + k + 32 * s); v[s][1] = *(const f32x4 *)(row + k + 32 * s + 4); }
#pragma unroll
            for (int s = 0; s < 4; s++) {
                const float y[8] = {v[s][0][0], v[s][0][1], v[s][0][2], v[s][0][3], v[s][1][0], v[s][1][1], v[s][1][2], v[s][1][3]};
                Planes p;
                split8(y, p);
#pragma unroll
                for (int i = 0; i < 3; i++) out[s][i] = p.p[i];
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; s++) out[s][0] = __builtin_bit_cast(bf16x8, *(const u32x4 *)(row + k + 32 * s));
        }
    } else {
#pragma unroll
        for (int s = 0; s < 4; s++) load_x<T>(row, k + 32 * s, K, vec, out[s]);
    }
}

// eight e2m1 codes -> bf16 (exact)
static __device__ __forceinline__ bf16x8 codes8(uint32_t w)
{
    u32x4 o;
    o[0] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 0));
    o[1] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 1));
    o[2] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 2));
    o[3] = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, 1.0f, 3));
    return __builtin_bit_cast(bf16x8, o);
}

// acc += scales * d: the scales of four outputs, bf16
static __device__ __forceinline__ void add_scaled(f32x4 &acc, u32x2 sc, f32x4 d)
{
    const f32x4 f = {as_f32(sc[0] << 16), as_f32(sc[0] & 0xffff0000u), as_f32(sc[1] << 16), as_f32(sc[1] & 0xffff0000u)};
#pragma unroll
    for (int r = 0; r < 4; r++) acc[r] = fmaf(f[r], d[r], acc[r]);
}

// one output: bias, GELU, the only rounding to T
template <typename T>
static __device__ __forceinline__ void put(float v, const T *bias, uint32_t gelu, uint32_t row, uint32_t out, uint32_t N, T *y)
{
    if (out >= N) return;
    v += bias ? load1(bias + out) : 0.f;
    if (gelu) v = 0.5f * v * (1.f + erff(v * 0.70710678118654752f));
    store1(y + (uint64_t)row * N + out, v);
}

// More than 1024 columns: a workgroup of W waves has NT tiles of 16 outputs and 16 rows of x, the waves take the 128-column chunks in turn and their sums meet
// in LDS.  GS: matrix instructions per scale group (group / 32).  Rows of x beyond the last repeat it: what a matrix instruction makes of them is not stored.  1 x 1024 x 4096
// fp32 6.3 us, 64 workgroups each of whose waves has two chunks: latency; 300 x 1024 x 4096 32 (the library's fp32 product 34).
template <typename T, int NT, int GS, int W>
__global__ __launch_bounds__(64 * W) void k_w4_linear_long(const T *x, uint64_t x_stride, const uint32_t *codes, const uint16_t *scales, const T *bias,
                                                           uint32_t M, uint32_t N, uint32_t K, uint32_t vec, uint32_t gelu, T *y)
{
    enum { XP = XPlanes<T>::N, GROUPS = 4 / GS };
    __shared__ f32x4 s_sum[W][NT][64];
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), col = lane & 15, g = lane >> 4;
    const uint32_t tiles = (N + 15) / 16, chunks = (K + 127) / 128, tile0 = blockIdx.x * NT, row = blockIdx.y * 16 + col;
    const T *xr = x + (uint64_t)min(row, M - 1) * x_stride;
    f32x4 acc[NT];
#pragma unroll
    for (int n = 0; n < NT; n++) acc[n] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (uint32_t c = wave; c < chunks; c += W) {
        u32x4 w[NT];
        u32x2 sc[NT][GROUPS];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const uint64_t t = min(tile0 + n, tiles - 1);           // (a tile beyond the last reads the last and is not stored)
            w[n] = *(const u32x4 *)(codes + (t * chunks + c) * 256 + lane * 4);
#pragma unroll
            for (int q = 0; q < GROUPS; q++) sc[n][q] = *(const u32x2 *)(scales + ((t * chunks + c) * GROUPS + q) * 16 + 4 * g);
        }
        // (four tiles and the planes of a whole chunk of fp32 would cost waves: 64 x 5000 x 1800 15.5 us, 13.5 with a quarter of the chunk at a time)
        constexpr bool WHOLE = NT == 1 || XP == 1;
        bf16x8 b[WHOLE ? 4 : 1][XP];
        if constexpr (WHOLE) load_chunk<T>(xr, c, g, K, vec, b);
#pragma unroll
        for (int q = 0; q < GROUPS; q++) {
            f32x4 d[NT];
#pragma unroll
            for (int n = 0; n < NT; n++) d[n] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int s = q * GS; s < (q + 1) * GS; s++) {
                if constexpr (!WHOLE) load_x<T>(xr, 128 * c + 32 * s + 8 * g, K, vec, b[0]);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const bf16x8 a = codes8(w[n][s]);
#pragma unroll
                    for (int p = 0; p < XP; p++) d[n] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[WHOLE ? s : 0][p], d[n], 0, 0, 0);
                }
            }
#pragma unroll
            for (int n = 0; n < NT; n++) add_scaled(acc[n], sc[n][q], d[n]);
        }
    }
#pragma unroll
    for (int n = 0; n < NT; n++) s_sum[wave][n][lane] = acc[n];
    __syncthreads();
    if (wave >= NT) return;
    f32x4 v = s_sum[0][wave][lane];
#pragma unroll
    for (uint32_t o = 1; o < W; o++) v += s_sum[o][wave][lane];
    if (row >= M) return;
#pragma unroll
    for (uint32_t r = 0; r < 4; r++) put(v[r], bias, gelu, row, (tile0 + wave) * 16 + 4 * g + r, N, y);
}

// At most 1024 columns: `kw` of a workgroup's eight waves (1, 2, 4 or 8) have one 128-column chunk each, 8 / kw such teams NT tiles of 16 outputs x MT tiles of 16 rows of
// x.  A wave's chunk of x stays in its registers as planes (splitting fp32 into them costs more instructions than the products) while the workgroup goes
// from tiles to tiles, every gridDim.x * 8 / kw * NT; the next round's codes are on their way while it works on these.  The waves' sums of two rounds lie side by side in LDS:
// one barrier a round.  1 x 50265 x 1024 fp32 in 10.6 us, 2.6 TB/s of codes and scales; a launch and the first loads are 4 of them, its 1571 pairs of tiles
// are 3.07 rounds of 512 workgroups (the last of 35 alone), and the joining sums all 16 columns though one is stored.  Vector units issue in a quarter of the cycles.
// From 17 rows on fp32 decodes the codes again for every 16 rows: 64 x 50265 x 1024 33 us, 300 x 50265 x 1024 143.
template <typename T, int NT, int MT, int GS>
__global__ __launch_bounds__(512, 2) void k_w4_linear_many(const T *x, uint64_t x_stride, const uint32_t *codes, const uint16_t *scales, const T *bias,
                                                           uint32_t M, uint32_t N, uint32_t K, uint32_t kw, uint32_t vec, uint32_t gelu, T *y)
{
    enum { XP = XPlanes<T>::N, GROUPS = 4 / GS };
    __shared__ f32x4 s_sum[2][8][NT][MT][64];
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), col = lane & 15, g = lane >> 4;
    const uint32_t tiles = (N + 15) / 16, chunks = (K + 127) / 128, teams = 8 / kw, team = wave / kw, c = wave % kw, m0 = blockIdx.y * MT * 16;
    const uint32_t step = gridDim.x * teams * NT, first = blockIdx.x * teams * NT, mine = first + team * NT;
    const bool has = c < chunks;                                 // (kw waves, maybe fewer chunks)
    const uint32_t cc = has ? c : 0;
    u32x4 w[NT];
    u32x2 sc[NT][GROUPS];
    auto fetch = [&](uint32_t tile0) {
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const uint64_t t = min(tile0 + n, tiles - 1);           // (a tile beyond the last reads the last and is not stored)
            w[n] = *(const u32x4 *)(codes + (t * chunks + cc) * 256 + lane * 4);
#pragma unroll
            for (int q = 0; q < GROUPS; q++) sc[n][q] = *(const u32x2 *)(scales + ((t * chunks + cc) * GROUPS + q) * 16 + 4 * g);
        }
    };
    fetch(mine);
    bf16x8 b[MT][4][XP];
#pragma unroll
    for (int m = 0; m < MT; m++) load_chunk<T>(x + (uint64_t)min(m0 + 16 * m + col, M - 1) * x_stride, cc, g, K, vec, b[m]);
    uint32_t side = 0;
    for (uint32_t from = first; from < tiles; from += step, side ^= 1) {
        f32x4 acc[NT][MT];
        u32x4 now[NT];
        u32x2 scale[NT][GROUPS];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            now[n] = w[n];
#pragma unroll
            for (int q = 0; q < GROUPS; q++) scale[n][q] = sc[n][q];
#pragma unroll
            for (int m = 0; m < MT; m++) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
        }
        fetch(from + team * NT + step);
        if (has) {
#pragma unroll
            for (int q = 0; q < GROUPS; q++) {
                f32x4 d[NT][MT];
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int m = 0; m < MT; m++) d[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = q * GS; s < (q + 1) * GS; s++)
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const bf16x8 a = codes8(now[n][s]);
#pragma unroll
                        for (int p = 0; p < XP; p++)
#pragma unroll
                            for (int m = 0; m < MT; m++) d[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[m][s][p], d[n][m], 0, 0, 0);
                    }
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int m = 0; m < MT; m++) add_scaled(acc[n][m], scale[n][q], d[n][m]);
            }
        }
#pragma unroll
        for (int n = 0; n < NT; n++)
#pragma unroll
            for (int m = 0; m < MT; m++) s_sum[side][wave][n][m][lane] = acc[n][m];
        __syncthreads();
        // two neighbouring outputs of a row a thread and turn
        for (uint32_t i = threadIdx.x; i < teams * NT * MT * 128; i += 512) {
            const uint32_t half = i & 1, l = (i >> 1) & 63, tm = i >> 7, m = tm % MT, n = tm / MT % NT, t = tm / (MT * NT);
            f32x2 v = {0.f, 0.f};
            for (uint32_t o = 0; o < kw; o++) {
                const f32x4 *p = &s_sum[side][t * kw + o][n][m][l];
                v += ((const f32x2 *)p)[half];
            }
            const uint32_t row = m0 + 16 * m + (l & 15), out = (from + t * NT + n) * 16 + 4 * (l >> 4) + 2 * half;
            if (row >= M) continue;
#pragma unroll
            for (uint32_t r = 0; r < 2; r++) put(v[r], bias, gelu, row, out + r, N, y);
        }
    }
}

struct W4Call {
    const void *x, *codes, *scales, *bias;
    void *y;
    uint64_t x_stride;
    uint32_t M, N, K, group, vec, gelu, kw;
};
template <typename T, int NT, int W>
static void launch_long(hipStream_t st, const W4Call &c)
{
    const dim3 grid(((c.N + 15) / 16 + NT - 1) / NT, (c.M + 15) / 16), block(64 * W);
    auto go = [&](auto k) {
        hipLaunchKernelGGL(k, grid, block, 0, st, (const T *)c.x, c.x_stride, (const uint32_t *)c.codes, (const uint16_t *)c.scales, (const T *)c.bias, c.M, c.N, c.K, c.vec, c.gelu, (T *)c.y);
    };
    if (c.group == 32) go(k_w4_linear_long<T, NT, 1, W>);
    else if (c.group == 64) go(k_w4_linear_long<T, NT, 2, W>);
    else go(k_w4_linear_long<T, NT, 4, W>);
}

template <typename T, int NT, int MT>
static void launch_many(hipStream_t st, const W4Call &c)
{
    const uint32_t per = NT * (8 / c.kw), mb = (c.M + 16 * MT - 1) / (16 * MT), most = std::max(1u, 512 / mb);
    const dim3 grid(std::min(((c.N + 15) / 16 + per - 1) / per, most), mb), block(512);
    auto go = [&](auto k) {
        hipLaunchKernelGGL(k, grid, block, 0, st, (const T *)c.x, c.x_stride, (const uint32_t *)c.codes, (const uint16_t *)c.scales, (const T *)c.bias, c.M, c.N, c.K, c.kw, c.vec, c.gelu, (T *)c.y);
    };
    if (c.group == 32) go(k_w4_linear_many<T, NT, MT, 1>);
    else if (c.group == 64) go(k_w4_linear_many<T, NT, MT, 2>);
    else go(k_w4_linear_many<T, NT, MT, 4>);
}

template <typename T>
static int w4_linear(void *stream, const void *x, uint64_t x_stride, const void *codes, const void *scales, const void *bias, uint32_t M, uint32_t N, uint32_t K,
                     uint32_t group, uint32_t gelu, void *y)
{
    if (group != 32 && group != 64 && group != 128) { fmi_set_error("sealnn_w4_linear: group = %u must be 32, 64 or 128", group); return FMI_ERR_UNSUPPORTED; }
    if (!M || !N) return FMI_OK;
    if (!K || !x || !codes || !scales || !y || ((uintptr_t)codes & 15) || ((uintptr_t)scales & 7) || ((uintptr_t)x & (sizeof(T) - 1))) {
        fmi_set_error("sealnn_w4_linear: K = %u, operands must be given and aligned (codes to 16 bytes, scales to 8)", K);
        return FMI_ERR_ARG;
    }
    if (N > (1u << 26) || K > (1u << 26) || M > (1u << 19)) { fmi_set_error("sealnn_w4_linear: %u x %u x %u is too large", M, N, K); return FMI_ERR_UNSUPPORTED; }
    const uint32_t vec = ((uintptr_t)x & 15) == 0 && (x_stride * sizeof(T)) % 16 == 0;
    hipStream_t st = (hipStream_t)stream;
    const uint32_t tiles = (N + 15) / 16, chunks = (K + 127) / 128;
    const W4Call c = {x, codes, scales, bias, y, x_stride, M, N, K, group, vec, gelu, chunks > 4 ? 8u : chunks > 2 ? 4u : chunks};
    // Measured (us; M x N x K):
    //   x in registers against read again for each tile of outputs: 1 x 50265 x 1024 10.6 / 14.5, 64 x 50265 x 1024 fp32 33 / 63, 1 x 1024 x 1024 3.7 / 4.0.
    //   one tile a wave / two, where every CU has one anyway or not: 1 x 1024 x 1024 3.7 / 4.4, 4 x 4096 x 1024 3.9 / 4.2; 1 x 16384 x 1024 6.0 / 5.8,
    //   32 x 3000 x 1024 7.4 / 5.9, 64 x 50265 x 1024 36 / 33; four: 1 x 50265 x 1024 15.5.
    //   16 rows of x a wave / 32: fp32, whose planes take three times the registers, 64 x 50265 x 1024 33 / 37; bf16 27 / 24, 60 x 4096 x 1024 6.7 / 5.8, but 60 x 1024 x 1024 3.8 / 5.5.
    //   more than 1024 columns, one tile / four: 1 x 1024 x 4096 6.2 / 11.8, 4 x 4096 x 2048 5.0 / 7.4; 40 x 24000 x 2000 bf16 33 / 20, 64 x 12000 x 4096 fp32 95 / 38.
    //   (32 rows a wave there: 50 to 97.)
    const uint64_t tiles16 = (uint64_t)tiles * ((M + 15) / 16), tiles32 = (uint64_t)tiles * ((M + 31) / 32);
    auto rows16 = [&] { if (tiles16 > 256) launch_many<T, 2, 1>(st, c); else launch_many<T, 1, 1>(st, c); };
    if (chunks > 8) {
        if (tiles16 >= 1024) launch_long<T, 4, 8>(st, c);
        else launch_long<T, 1, 16>(st, c);
    } else if constexpr (std::is_same<T, bf16>::value) {
        if (M > 16 && tiles32 >= 512) launch_many<T, 2, 2>(st, c);
        else rows16();
    } else rows16();
    NNCHK();
    return FMI_OK;
}

extern "C" int sealnn_w4_linear(void *stream, const float *x, uint64_t x_stride, const void *codes, const void *scales, const float *bias, uint32_t M, uint32_t N,
                                uint32_t K, uint32_t group, uint32_t gelu, float *y)
{ return w4_linear<float>(stream, x, x_stride, codes, scales, bias, M, N, K, group, gelu, y); }
extern "C" int sealnn_w4_linear_bf16(void *stream, const void *x, uint64_t x_stride, const void *codes, const void *scales, const void *bias, uint32_t M, uint32_t N,
                                     uint32_t K, uint32_t group, uint32_t gelu, void *y)
{ return w4_linear<bf16>(stream, x, x_stride, codes, scales, bias, M, N, K, group, gelu, y); }
