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
static __device__ __forceinline__ void load_x(const T *row, uint32_t k, uint32_t K, bool live, bool vec, bf16x8 out[XPlanes<T>::N])
{
    if constexpr (std::is_same<T, float>::value) {
        float v[8];
#pragma unroll
        for (int i = 0; i < 8; i++) v[i] = 0.f;
        if (live && k < K) {
            if (vec && k + 8 <= K) {
                const f32x4 a = *(const f32x4 *)(row + k), b = *(const f32x4 *)(row + k + 4);
#pragma unroll
                for (int i = 0; i < 4; i++) { v[i] = a[i]; v[4 + i] = b[i]; }
            } else {
#pragma unroll
                for (int i = 0; i < 8; i++) if (k + i < K) v[i] = row[k + i];
            }
        }
        Planes p;
        split8(v, p);
#pragma unroll
        for (int i = 0; i < 3; i++) out[i] = p.p[i];
    } else {
        u32x4 w = {0, 0, 0, 0};
        if (live && k < K) {
            const uint16_t *r = reinterpret_cast<const uint16_t *>(row) + k;
            if (vec && k + 8 <= K) w = *(const u32x4 *)r;
            else {
#pragma unroll
                for (int i = 0; i < 8; i++) if (k + i < K) w[i / 2] |= (uint32_t)r[i] << (16 * (i & 1));
            }
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

// One workgroup: NT tiles of 16 outputs x MT tiles of 16 rows of x; its waves take the 128-column chunks in turn and their sums meet in LDS.
// GS: matrix instructions per scale group (group / 32).
template <typename T, int NT, int MT, int WAVES, int GS>
__global__ __launch_bounds__(64 * WAVES) void k_w4_linear(const T *x, uint64_t x_stride, const uint32_t *codes, const uint16_t *scales, const T *bias,
                                                          uint32_t M, uint32_t N, uint32_t K, uint32_t vec, uint32_t gelu, T *y)
{
    enum { XP = XPlanes<T>::N, GROUPS = 4 / GS };
    __shared__ f32x4 s_sum[WAVES][NT][MT][64];
    const uint32_t lane = threadIdx.x & 63, wave = threadIdx.x >> 6, col = lane & 15, g = lane >> 4;
    const uint32_t tiles = (N + 15) / 16, chunks = (K + 127) / 128;
    const uint32_t tile0 = blockIdx.x * NT, m0 = blockIdx.y * MT * 16;
    f32x4 acc[NT][MT];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int m = 0; m < MT; m++) acc[n][m] = f32x4{0.f, 0.f, 0.f, 0.f};
    for (uint32_t c = wave; c < chunks; c += WAVES) {
        u32x4 w[NT];
        u32x2 sc[NT][GROUPS];
#pragma unroll
        for (int n = 0; n < NT; n++) {
            const uint64_t t = min(tile0 + n, tiles - 1);               // (a tile beyond the last reads the last and is not stored)
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
                bf16x8 a[NT];
#pragma unroll
                for (int n = 0; n < NT; n++) a[n] = codes8(w[n][s]);
#pragma unroll
                for (int m = 0; m < MT; m++) {
                    const uint32_t row = m0 + 16 * m + col;
                    bf16x8 b[XP];
                    load_x<T>(x + (uint64_t)min(row, M - 1) * x_stride, 128 * c + 32 * s + 8 * g, K, row < M, vec, b);
#pragma unroll
                    for (int n = 0; n < NT; n++)
#pragma unroll
                        for (int p = 0; p < XP; p++) d[n][m] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(a[n], b[p], d[n][m], 0, 0, 0);
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
    for (uint32_t i = wave; i < NT * MT; i += WAVES) {
        const uint32_t n = i / MT, m = i % MT;
        f32x4 v = s_sum[0][n][m][lane];
#pragma unroll
        for (int o = 1; o < WAVES; o++) v += s_sum[o][n][m][lane];
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

template <typename T, int NT, int MT, int WAVES>
static void launch_w4(hipStream_t st, const void *x, uint64_t xs, const void *codes, const void *scales, const void *bias, uint32_t M, uint32_t N, uint32_t K,
                      uint32_t group, uint32_t vec, uint32_t gelu, void *y)
{
    const dim3 grid(((N + 15) / 16 + NT - 1) / NT, (M + 16 * MT - 1) / (16 * MT)), block(64 * WAVES);
    auto go = [&](auto k) { hipLaunchKernelGGL(k, grid, block, 0, st, (const T *)x, xs, (const uint32_t *)codes, (const uint16_t *)scales, (const T *)bias, M, N, K, vec, gelu, (T *)y); };
    if (group == 32) go(k_w4_linear<T, NT, MT, WAVES, 1>);
    else if (group == 64) go(k_w4_linear<T, NT, MT, WAVES, 2>);
    else go(k_w4_linear<T, NT, MT, WAVES, 4>);
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
    if (M <= 16) launch_w4<T, 2, 1, 4>(st, x, x_stride, codes, scales, bias, M, N, K, group, vec, gelu, y);
    else launch_w4<T, 2, 4, 4>(st, x, x_stride, codes, scales, bias, M, N, K, group, vec, gelu, y);
    NNCHK();
    return FMI_OK;
}

extern "C" int sealnn_w4_linear(void *stream, const float *x, uint64_t x_stride, const void *codes, const void *scales, const float *bias, uint32_t M, uint32_t N,
                                uint32_t K, uint32_t group, uint32_t gelu, float *y)
{ return w4_linear<float>(stream, x, x_stride, codes, scales, bias, M, N, K, group, gelu, y); }
extern "C" int sealnn_w4_linear_bf16(void *stream, const void *x, uint64_t x_stride, const void *codes, const void *scales, const void *bias, uint32_t M, uint32_t N,
                                     uint32_t K, uint32_t group, uint32_t gelu, void *y)
{ return w4_linear<bf16>(stream, x, x_stride, codes, scales, bias, M, N, K, group, gelu, y); }
