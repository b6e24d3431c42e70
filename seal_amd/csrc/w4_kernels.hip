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

// A workgroup of eight waves: `kw` of them (1, 2, 4 or 8) take the 128-column chunks in turn, 8 / kw such teams have NT tiles of 16 outputs x MT tiles of 16 rows of x
// each; a team's sums meet in LDS.  GS: matrix instructions per scale group (group / 32).  The planes of x are made once for the NT tiles.  Rows of x
// beyond the last repeat it: what a matrix instruction makes of them is not stored.
template <typename T, int NT, int MT, int GS>
__global__ __launch_bounds__(512) void k_w4_linear(const T *x, uint64_t x_stride, const uint32_t *codes, const uint16_t *scales, const T *bias,
                                                   uint32_t M, uint32_t N, uint32_t K, uint32_t kw, uint32_t vec, uint32_t gelu, T *y)
{
    enum { XP = XPlanes<T>::N, GROUPS = 4 / GS };
    __shared__ f32x4 s_sum[8][NT][MT][64];
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), col = lane & 15, g = lane >> 4;
    const uint32_t tiles = (N + 15) / 16, chunks = (K + 127) / 128, team = wave / kw, part = wave % kw;
    const uint32_t tile0 = (blockIdx.x * (8 / kw) + team) * NT, m0 = blockIdx.y * MT * 16;
    f32x4 acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int m = 0; m < MT; m++) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    if (tile0 < tiles)
        for (uint32_t c = part; c < chunks; c += kw) {
            u32x4 w[NT];
            u32x2 sc[NT][GROUPS];
#pragma unroll
            for (int n = 0; n < NT; n++) {
                const uint64_t t = min(tile0 + n, tiles - 1);           // (a tile beyond the last reads the last and is not stored)
                w[n] = *(const u32x4 *)(codes + (t * chunks + c) * 256 + lane * 4);
#pragma unroll
                for (int q = 0; q < GROUPS; q++) sc[n][q] = *(const u32x2 *)(scales + ((t * chunks + c) * GROUPS + q) * 16 + 4 * g);
            }
#pragma unroll
            for (int q = 0; q < GROUPS; q++) {
                f32x4 d[NT][MT];
#pragma unroll
                for (int n = 0; n < NT; n++)
#pragma unroll
                    for (int m = 0; m < MT; m++) d[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int s = q * GS; s < (q + 1) * GS; s++) {
                    bf16x8 b[MT][XP];
#pragma unroll
                    for (int m = 0; m < MT; m++) load_x<T>(x + (uint64_t)min(m0 + 16 * m + col, M - 1) * x_stride, 128 * c + 32 * s + 8 * g, K, vec, b[m]);
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        const bf16x8 a = codes8(w[n][s]);
#pragma unroll
                        for (int p = 0; p < XP; p++)
#pragma unroll
                            for (int m = 0; m < MT; m++) d[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a, b[m][p], d[n][m], 0, 0, 0);
                    }
                }
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const f32x4 f = {as_f32(sc[n][q][0] << 16), as_f32(sc[n][q][0] & 0xffff0000u), as_f32(sc[n][q][1] << 16), as_f32(sc[n][q][1] & 0xffff0000u)};
#pragma unroll
                    for (int m = 0; m < MT; m++)
#pragma unroll
                        for (int r = 0; r < 4; r++) acc[n][m][r] = fmaf(f[r], d[n][m][r], acc[n][m][r]);
                }
            }
        }
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int m = 0; m < MT; m++) s_sum[wave][n][m][lane] = acc[n][m];
    __syncthreads();
    for (uint32_t i = part; i < NT * MT; i += kw) {
        const uint32_t n = i / MT, m = i % MT;
        f32x4 v = s_sum[team * kw][n][m][lane];
        for (uint32_t o = 1; o < kw; o++) v += s_sum[team * kw + o][n][m][lane];
        const uint32_t row = m0 + 16 * m + col, out = (tile0 + n) * 16 + 4 * g;
        if (row >= M) continue;
#pragma unroll
        for (int r = 0; r < 4; r++) {
            if (out + r >= N) continue;
            float t = v[r] + (bias ? load1(bias + out + r) : 0.f);
            if (gelu) t = 0.5f * t * (1.f + erff(t * 0.70710678118654752f));
            store1(y + (uint64_t)row * N + out + r, t);
        }
    }
}

struct W4Call {
    const void *x, *codes, *scales, *bias;
    void *y;
    uint64_t x_stride;
    uint32_t M, N, K, group, vec, gelu, kw;
};
template <typename T, int NT, int MT>
static void launch_w4(hipStream_t st, const W4Call &c)
{
    const uint32_t per = NT * (8 / c.kw);
    const dim3 grid(((c.N + 15) / 16 + per - 1) / per, (c.M + 16 * MT - 1) / (16 * MT)), block(512);
    auto go = [&](auto k) {
        hipLaunchKernelGGL(k, grid, block, 0, st, (const T *)c.x, c.x_stride, (const uint32_t *)c.codes, (const uint16_t *)c.scales, (const T *)c.bias, c.M, c.N, c.K, c.kw, c.vec, c.gelu, (T *)c.y);
    };
    if (c.group == 32) go(k_w4_linear<T, NT, MT, 1>);
    else if (c.group == 64) go(k_w4_linear<T, NT, MT, 2>);
    else go(k_w4_linear<T, NT, MT, 4>);
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
    if (N > (1u << 26) || K > (1u << 26) || M > (1u << 20)) { fmi_set_error("sealnn_w4_linear: %u x %u x %u is too large", M, N, K); return FMI_ERR_UNSUPPORTED; }
    const uint32_t vec = ((uintptr_t)x & 15) == 0 && (x_stride * sizeof(T)) % 16 == 0;
    hipStream_t st = (hipStream_t)stream;
    const uint32_t tiles = (N + 15) / 16, chunks = (K + 127) / 128, kw = chunks >= 8 ? 8 : chunks >= 4 ? 4 : chunks >= 2 ? 2 : 1;
    const W4Call c = {x, codes, scales, bias, y, x_stride, M, N, K, group, vec, gelu, kw};
    // Several tiles a wave share the planes of x, as long as that leaves a workgroup and a half or two for every CU (256 CUs).  us, one tile / several:
    // 1 x 50265 x 1024 17.8 / 14.5, 1 x 1024 x 1024 4.0 / 5.8, 1 x 50265 x 64 5.0 / 7.6; 64 x 50265 x 1024 fp32 102 / 63, 60 x 4096 x 1024 bf16 7.7 / 6.3, 60 x 1024 x 4096 11.2 / 12.6.
    // Two tiles of rows: four (64 rows of x at once) are 1.2 to 1.6 times slower, their registers leave one workgroup a CU.
    const uint64_t teams = 8 / kw;
    if (M <= 16) {
        if (tiles >= 512 * 4 * teams) launch_w4<T, 4, 1>(st, c);
        else launch_w4<T, 1, 1>(st, c);
    } else if ((uint64_t)tiles * ((M + 31) / 32) >= 256 * 2 * teams) launch_w4<T, 2, 2>(st, c);
    else launch_w4<T, 1, 2>(st, c);
    NNCHK();
    return FMI_OK;
}

extern "C" int sealnn_w4_linear(void *stream, const float *x, uint64_t x_stride, const void *codes, const void *scales, const float *bias, uint32_t M, uint32_t N,
                                uint32_t K, uint32_t group, uint32_t gelu, float *y)
{ return w4_linear<float>(stream, x, x_stride, codes, scales, bias, M, N, K, group, gelu, y); }
extern "C" int sealnn_w4_linear_bf16(void *stream, const void *x, uint64_t x_stride, const void *codes, const void *scales, const void *bias, uint32_t M, uint32_t N,
                                     uint32_t K, uint32_t group, uint32_t gelu, void *y)
{ return w4_linear<bf16>(stream, x, x_stride, codes, scales, bias, M, N, K, group, gelu, y); }
