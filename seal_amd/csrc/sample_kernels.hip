// Drawing tokens from logits: temperature, top-k, top-p and min-p under an optional allowed-token bitmap, from given random numbers
// (include/sealnn.h: sealnn_sample_tokens).
//
// With the tokens ordered by (logit falling, index rising) every filter keeps a PREFIX: the first k; the smallest prefix with at least p of
// the mass of those; the tokens of at least min_p of the largest weight.  So the kernel never sorts: it finds the logit at which the prefix ends
// by counting (or weighing) buckets of logits and looking again inside the one bucket that the border falls into, and then draws in the order
// of the vocabulary from the tokens above it: the first token whose cumulative weight passes u * total.
//
// Weights are whole numbers, exp((x - max) / T) * 2^44 rounded, computed in 64-bit floats (the exponential to 2^-39 of itself: up to 21 units near the
// largest, less than the rounding's half unit below 2^-6 of it) and added in 64-bit integers: sums of up to 2^18 of them are exact, so neither the order of the atomics nor the shape of a reduction changes which
// token a random number falls on.  A weight below 2^-45 of the largest is 0.
#include "nn_common.h"

#include <algorithm>

enum { THREADS = 1024, WAVES = THREADS / 64, STRIPE = 4 * THREADS, BUCKETS = 2048, LIST = 2048, MAX_VOCAB = 1 << 18 };

struct SampleArgs {
    const void *logits;
    uint64_t row_stride;
    const uint32_t *bits;
    uint64_t bits_stride;
    const float *u, *temperature_v, *top_p_v, *min_p_v;
    const int32_t *top_k_v;
    uint32_t rows, vocab, draws;
    float temperature, top_p, min_p;
    int32_t top_k;
    int64_t *tokens;
    float *logprobs;
    char *work;                                                  // NULL: one kernel
};

// What the kernels of a split row hand on, per row: a record and four part sums for every 1024 tokens, the list's length and the list
enum { SEGMENT = 1024, MAX_SEGMENTS = MAX_VOCAB / SEGMENT, RUNGS = 7 };
struct Record { float max, z, rung[RUNGS], unused[7]; };         // the largest logit, the sum of exponentials against it; rungs: see k_sample_segments
static_assert(sizeof(Record) == 64, "a record is four 16-byte words");
static __host__ __device__ __forceinline__ uint64_t row_work(uint32_t vocab) { return (uint64_t)((vocab + SEGMENT - 1) / SEGMENT) * (sizeof(Record) + 32) + 64 + 8 * LIST; }
struct RowWork {
    Record *record;
    uint64_t *part, *list;
    uint32_t *count;
    __device__ __forceinline__ RowWork(const SampleArgs &a, uint32_t row)
    {
        const uint32_t n = (a.vocab + SEGMENT - 1) / SEGMENT;
        char *p = a.work + row * row_work(a.vocab);
        record = (Record *)p;
        part = (uint64_t *)(p + n * sizeof(Record));
        count = (uint32_t *)(part + 4 * n);
        list = (uint64_t *)((char *)count + 64);
    }
};

// monotone in x; +0 and -0 alike
static __device__ __forceinline__ uint32_t key_of(float x) { const uint32_t u = as_u32(x + 0.f); return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u); }
// NaN counts as -inf, +inf as the largest number (the larger of NaN and a number is the number)
static __device__ __forceinline__ float clean(float x) { return fminf(fmaxf(x, -__builtin_huge_valf()), 3.402823466e38f); }

struct Shared {
    uint64_t mass[BUCKETS];                              // a histogram, or the running weights of `order`
    uint64_t list[LIST];                                 // (key << 32 | ~index) of the tokens that matter: falling order = falling logit, equal ones by rising index
    uint64_t order[LIST];                                // those of them that a border falls between
    uint64_t part[MAX_VOCAB / 256];                      // weights of 256 consecutive tokens each
    float top[MAX_VOCAB / STRIPE / 4 * WAVES];           // the largest that may be drawn of a wave's tokens in four stripes
    uint64_t wave[WAVES];
    float wavef[2 * WAVES];
    double root[32];                                     // 2^(i / 32)
    uint32_t kmin, kmax, found, bucket, n, thr, lim;
    uint64_t before, total;
};

// exp((x - m) / T) * 2^44 as a 64-bit float (a whole number; 0 below 2^-45): 2^t = 2^floor * 2^(k / 32) * e^y, |y| <= ln 2 / 64, where the
// series ends at y^4 (what it leaves out is y^5 / 120 < 2^-39 relative: below half a unit for weights up to 2^-6 of the largest, up to 21 units above)
static __device__ __forceinline__ double weight(float x, double m, double inv_t_log2e, const double *root)
{
    const double t = fmax(((double)x - m) * inv_t_log2e, -64.0);
    const double r = t + 211106232532992.0;                                           // 1.5 * 2^47: the unit in the last place is 1 / 32
    const double f = t - (r - 211106232532992.0);
    const int k = __double2loint(r);                                                   // 32 t to nearest
    const double y = f * 0.69314718055994530942;
    const double e = 1.0 + y * (1.0 + y * (0.5 + y * (1.0 / 6 + y * (1.0 / 24))));
    const double p = __hiloint2double((1023 + 44 + (k >> 5)) << 20, 0);               // 2^(44 + floor(k / 32))
    return fma(root[k & 31] * e, p, 4503599627370496.0) - 4503599627370496.0;          // (+- 2^52: to the nearest whole number)
}

// DPP: the value of another lane of the wave without a trip through LDS (lanes that have none get `none`)
template <int CTRL, int ROWS> static __device__ __forceinline__ uint32_t dpp(uint32_t none, uint32_t v)
{ return (uint32_t)__builtin_amdgcn_update_dpp((int)none, (int)v, CTRL, ROWS, 0xf, false); }
template <int CTRL, int ROWS> static __device__ __forceinline__ uint64_t dpp_add(uint64_t v)
{ return v + (((uint64_t)dpp<CTRL, ROWS>(0, (uint32_t)(v >> 32)) << 32) | dpp<CTRL, ROWS>(0, (uint32_t)v)); }
// inclusive sums over the wave: within rows of 16 lanes, then the rows' last lanes onwards
static __device__ __forceinline__ uint64_t wave_scan(uint64_t v)
{
    v = dpp_add<0x111, 0xf>(v); v = dpp_add<0x112, 0xf>(v); v = dpp_add<0x114, 0xf>(v); v = dpp_add<0x118, 0xf>(v);
    v = dpp_add<0x142, 0xa>(v);
    return dpp_add<0x143, 0xc>(v);
}
static __device__ __forceinline__ uint64_t wave_total(uint64_t scanned)
{
    return ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(scanned >> 32), 63) << 32) | (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)scanned, 63);
}
// (NaN comes through: an instruction less a step than a maximum that drops it)
template <int CTRL, int ROWS> static __device__ __forceinline__ float dpp_max(float v)
{ return __builtin_elementwise_maximum(v, as_f32(dpp<CTRL, ROWS>(0xff800000u, as_u32(v)))); }
static __device__ __forceinline__ float wave_max(float v)
{
    v = dpp_max<0x111, 0xf>(v); v = dpp_max<0x112, 0xf>(v); v = dpp_max<0x114, 0xf>(v); v = dpp_max<0x118, 0xf>(v);
    v = dpp_max<0x142, 0xa>(v);
    v = dpp_max<0x143, 0xc>(v);
    return as_f32((uint32_t)__builtin_amdgcn_readlane((int)as_u32(v), 63));
}

// inclusive sums over the workgroup; `total` the whole sum
static __device__ __forceinline__ uint64_t block_scan(uint64_t v, Shared &s, uint32_t lane, uint32_t wave, uint64_t &total)
{
    v = wave_scan(v);
    __syncthreads();
    if (lane == 63) s.wave[wave] = v;
    __syncthreads();
    const uint64_t w = wave_scan(lane < WAVES ? s.wave[lane] : 0);
    total = wave_total(w);
    const uint64_t before = wave ? (((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(w >> 32), (int)(wave - 1)) << 32) |
                                    (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)w, (int)(wave - 1))) : 0;
    return v + before;
}

// The bucket (in order) at which the running sum of s.mass reaches what is asked for: s.bucket, s.before (the sum in front of it), s.total;
// s.found = 0 if it never does
template <typename REACHED>
static __device__ __forceinline__ void find_bucket(Shared &s, uint32_t tid, uint32_t lane, uint32_t wave, REACHED reached)
{
    static_assert(BUCKETS == 2 * THREADS, "two buckets a thread");
    const uint64_t a = s.mass[2 * tid], b = s.mass[2 * tid + 1];
    uint64_t total;
    const uint64_t incl = block_scan(a + b, s, lane, wave, total);
    if (tid == 0) { s.found = 0; s.total = total; }
    __syncthreads();
    const uint64_t f0 = incl - a - b, f1 = incl - b;
    if (!reached(f0, total) && reached(f1, total)) { s.found = 1; s.bucket = 2 * tid; s.before = f0; }
    else if (!reached(f1, total) && reached(incl, total)) { s.found = 1; s.bucket = 2 * tid + 1; s.before = f1; }
    __syncthreads();
}

// s.order[0 .. n) into falling order (zeros behind it)
static __device__ __forceinline__ void sort_order(Shared &s, uint32_t n, uint32_t tid)
{
    uint32_t size = 2;
    while (size < n) size <<= 1;
    for (uint32_t i = n + tid; i < size; i += THREADS) s.order[i] = 0;
    __syncthreads();
    for (uint32_t k = 2; k <= size; k <<= 1)
        for (uint32_t j = k >> 1; j > 0; j >>= 1) {
            if (tid < size / 2) {
                const uint32_t i = ((tid & ~(j - 1)) << 1) | (tid & (j - 1)), o = i | j;
                const uint64_t a = s.order[i], b = s.order[o];
                if ((a < b) == ((i & k) == 0)) { s.order[i] = b; s.order[o] = a; }
            }
            __syncthreads();
        }
}
// a value per lane of one wave into falling order
static __device__ __forceinline__ uint64_t sort_wave(uint64_t v, uint32_t lane)
{
#pragma unroll
    for (uint32_t k = 2; k <= 64; k <<= 1)
#pragma unroll
        for (uint32_t j = k >> 1; j > 0; j >>= 1) {
            const uint64_t o = __shfl_xor(v, (int)j);
            const bool larger = ((lane & k) == 0) == ((lane & j) == 0);                // this lane keeps the larger of the two
            v = (o > v) == larger ? o : v;
        }
    return v;
}

// A row of logits in stripes of 4096: thread t = 0 .. 1023 of stripe i has the four from 4096 i + 4 t
template <typename T, bool BITS>
struct Row {
    // Four logits as they lie in memory, without a branch: lanes that reach over the end of the row read its last four (a row of less than four its
    // first, again and again), and `unpack` moves them into place -- so that several stripes' loads are in flight at once
    typedef typename std::conditional<std::is_same<T, float>::value, f32x4, u32x2>::type Raw;
    const T *x;
    const uint32_t *bits;
    uint32_t V;
    __device__ __forceinline__ Row(const SampleArgs &a, uint32_t row)
        : x((const T *)a.logits + (uint64_t)row * a.row_stride), bits(BITS ? a.bits + (uint64_t)row * a.bits_stride : nullptr), V(a.vocab) {}
    __device__ __forceinline__ Raw load(uint32_t i, uint32_t t) const
    {
        const uint32_t at = min(i * STRIPE + 4 * t, V < 4 ? 0 : V - 4);
        if constexpr (std::is_same<T, float>::value) {
            if (V >= 4) { const f32x4_a4 w = *(const f32x4_a4 *)(x + at); return f32x4{w[0], w[1], w[2], w[3]}; }
            return f32x4{x[0], x[min(1u, V - 1)], x[min(2u, V - 1)], -__builtin_huge_valf()};
        } else {
            const uint16_t *h = (const uint16_t *)x;
            if (V >= 4) { const u16x4_a2 w = *(const u16x4_a2 *)(h + at); return __builtin_bit_cast(u32x2, w); }
            return u32x2{(uint32_t)h[0] | ((uint32_t)h[min(1u, V - 1)] << 16), (uint32_t)h[min(2u, V - 1)]};
        }
    }
    __device__ __forceinline__ uint32_t load_bits(uint32_t i, uint32_t t) const { return BITS ? bits[min(i * STRIPE + 4 * t, V - 1) >> 5] : 0; }
    // the logits as they are (-inf beyond the row); returns which of them may be drawn
    __device__ __forceinline__ uint32_t unpack(uint32_t i, uint32_t t, Raw w, uint32_t word, float v[4]) const
    {
        const float NINF = -__builtin_huge_valf();
        const uint32_t at = i * STRIPE + 4 * t;
#pragma unroll
        for (int e = 0; e < 4; e++) {
            if constexpr (std::is_same<T, float>::value) v[e] = w[e];
            else v[e] = as_f32(e & 1 ? w[e / 2] & 0xffff0000u : w[e / 2] << 16);
        }
        if ((i + 1) * STRIPE >= V) {
            if (V >= 4 && at + 4 > V) {
                const uint32_t skip = at + 4 - V;
                v[0] = skip == 1 ? v[1] : skip == 2 ? v[2] : skip == 3 ? v[3] : NINF;
                v[1] = skip == 1 ? v[2] : skip == 2 ? v[3] : NINF;
                v[2] = skip == 1 ? v[3] : NINF;
                v[3] = NINF;
            }
            if (V < 4) {
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) if (at + e >= V) v[e] = NINF;
            }
        }
        return BITS ? (word >> (at & 31)) & 15u : 15u;
    }
};

// A row's settings
struct Settings {
    float temperature, top_p, min_p;
    int32_t top_k;
    bool has_k, has_p;
    __device__ __forceinline__ Settings(const SampleArgs &a, uint32_t row)
    {
        temperature = a.temperature_v ? a.temperature_v[row] : a.temperature;
        top_k = a.top_k_v ? a.top_k_v[row] : a.top_k;
        top_p = a.top_p_v ? a.top_p_v[row] : a.top_p;
        min_p = a.min_p_v ? a.min_p_v[row] : a.min_p;
        min_p = min_p > 0.f ? fminf(min_p, 1.f) : 0.f;
        if (!(temperature > 0.f)) { temperature = 1.f; top_k = 1; }                   // greedy: the first of the largest
        has_k = top_k > 0 && (uint32_t)top_k < a.vocab;
        has_p = top_p < 1.f;
    }
    // a list of the largest tokens is made for a nucleus of all, and where the k largest fit it
    __device__ __forceinline__ bool lists() const { return has_k ? (uint32_t)top_k <= THREADS / 2 : has_p; }
};

// what is the same in every lane, out of the vector registers (a row's constants would fill a quarter of them)
static __device__ __forceinline__ float uniform(float v) { return as_f32((uint32_t)__builtin_amdgcn_readfirstlane((int)as_u32(v))); }
static __device__ __forceinline__ double uniform(double v)
{ return __hiloint2double(__builtin_amdgcn_readfirstlane(__double2hiint(v)), __builtin_amdgcn_readfirstlane(__double2loint(v))); }

// How a row's logits become weights and buckets; mz: the largest that may be drawn
struct Scale {
    double m, inv, floor_w;
    float mz, c, low;
    __device__ __forceinline__ Scale(const Settings &t, float mz_)
    {
        mz = uniform(mz_);
        m = uniform((double)mz);
        inv = uniform(1.4426950408889634074 / (double)t.temperature);
        // buckets of 1 / 64 of a temperature below the largest logit: they order as the logits do (a rounded difference and product are monotone)
        c = uniform(fminf(64.f / t.temperature, 1e30f));
        // a logit below `low` has no weight: less than min_p of the largest, or 2^-45
        floor_w = uniform(t.min_p > 0.f ? (double)t.min_p * 17592186044416.0 : 0.0);
        const float reach = mz - t.temperature * fminf(31.5f, t.min_p > 0.f ? 1e-3f - 0.69314718f * __builtin_amdgcn_logf(t.min_p) : 31.5f) * 1.00001f;
        low = uniform(fmaxf(reach, -3.402823466e38f));
    }
    __device__ __forceinline__ uint32_t bucket(float v) const { const float b = (mz - v) * c; return b < (float)(BUCKETS - 1) ? (uint32_t)b : (uint32_t)(BUCKETS - 1); }
};

// The first kernel of a split row, a wave for every 1024 tokens: their largest logit and sum of exponentials, and rungs -- of the lanes' own maxima (16 tokens that may
// be drawn) the largest, 2nd, 4th, 8th, 16th, 32nd and 56th.  The rungs of all waves tell a logit that at least so and so many tokens reach.  Latency: a row of 50265 is 13 workgroups, 4.5 us.
static __device__ __forceinline__ uint32_t rung_rank(uint32_t i) { return i < 6 ? 1u << i : 56u; }
template <typename T, bool BITS>
__global__ __launch_bounds__(256) void k_sample_segments(SampleArgs a)
{
    const float NINF = -__builtin_huge_valf(), L2E = 1.4426950408889634f;
    const uint32_t lane = threadIdx.x & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(threadIdx.x >> 6)), seg = blockIdx.x * 4 + wave, row = blockIdx.y;
    if (seg * SEGMENT >= a.vocab) return;
    const Row<T, BITS> x(a, row);
    RowWork out(a, row);
    typename Row<T, BITS>::Raw w[4];
    uint32_t b[4];
    float v[4][4], mx = NINF, mz = NINF;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) { w[j] = x.load(blockIdx.x, wave * 256 + j * 64 + lane); b[j] = x.load_bits(blockIdx.x, wave * 256 + j * 64 + lane); }
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
        const uint32_t ok = x.unpack(blockIdx.x, wave * 256 + j * 64 + lane, w[j], b[j], v[j]);
#pragma unroll
        for (int e = 0; e < 4; e++) {
            v[j][e] = clean(v[j][e]);
            mx = fmaxf(mx, v[j][e]);
            if (BITS) mz = fmaxf(mz, (ok >> e) & 1 ? v[j][e] : NINF);
        }
    }
    const float own = BITS ? mz : mx;
    mx = wave_max(mx);
    float z = 0.f;
    if (mx > NINF) {
#pragma unroll
        for (int j = 0; j < 4; j++)
#pragma unroll
            for (int e = 0; e < 4; e++) z += __builtin_amdgcn_exp2f((v[j][e] - mx) * L2E);
    }
    for (int o = 32; o > 0; o >>= 1) z += __shfl_xor(z, o);
    uint32_t above = 0, reach = 0;                               // lanes with a larger maximum, with one at least as large
#pragma unroll
    for (int l = 0; l < 64; l++) {
        const float o = as_f32((uint32_t)__builtin_amdgcn_readlane((int)as_u32(own), l));
        above += o > own;
        reach += o >= own;
    }
    Record &r = out.record[seg];
#pragma unroll
    for (uint32_t i = 0; i < RUNGS; i++) if (above < rung_rank(i) && rung_rank(i) <= reach) r.rung[i] = own;    // (equal lanes write the same)
    if (lane == 0) { r.max = mx; r.z = z; if (seg == 0) *out.count = 0; }
}

// The largest logit of a row and the largest that may be drawn, from its records (every thread below `segments` has read its own)
static __device__ __forceinline__ void row_maxima(const Record &r, float *shared, uint32_t lane, uint32_t wave, float &mx, float &mz)
{
    mx = wave_max(r.max);
    mz = wave_max(r.rung[0]);
    if (lane == 0 && wave < 4) { shared[wave] = mx; shared[4 + wave] = mz; }
    __syncthreads();
    mx = wave_max(shared[lane & 3]);
    mz = wave_max(shared[4 + (lane & 3)]);
}
static __device__ __forceinline__ Record no_record()
{
    Record r;
    r.max = -__builtin_huge_valf();
    r.z = 0.f;
#pragma unroll
    for (int i = 0; i < RUNGS; i++) r.rung[i] = -__builtin_huge_valf();
    return r;
}

// The second: the row's tokens in buckets as high as its rungs ask for go on its list, and the weights of every 256 tokens are added up (those of min_p where no other filter
// is on; not at all under a top_k, which weighs no more than its list).  A row of 50265: 13 workgroups, each of which goes over the row's rungs itself, a lane weighing 16 tokens one
// after the other: 8.8 us of latency.
template <typename T, bool BITS>
__global__ __launch_bounds__(256) void k_sample_lists(SampleArgs a)
{
    __shared__ uint32_t s_count[BUCKETS], s_wave[4], s_bucket;
    __shared__ float s_max[8];
    __shared__ double s_root[32];
    const float NINF = -__builtin_huge_valf(), LOWEST = -3.402823466e38f;
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = (uint32_t)__builtin_amdgcn_readfirstlane((int)(tid >> 6)), row = blockIdx.y, seg = blockIdx.x * 4 + wave;
    const uint32_t segments = (a.vocab + SEGMENT - 1) / SEGMENT;
    const Row<T, BITS> x(a, row);
    RowWork out(a, row);
    typename Row<T, BITS>::Raw w[4];
    uint32_t b[4];
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) { w[j] = x.load(blockIdx.x, wave * 256 + j * 64 + lane); b[j] = x.load_bits(blockIdx.x, wave * 256 + j * 64 + lane); }
    Record r = tid < segments ? out.record[tid] : no_record();
    const Settings t(a, row);
    if (tid < 32) s_root[tid] = exp2((double)tid / 32.0);
    float mx, mz;
    row_maxima(r, s_max, lane, wave, mx, mz);
    if (mz == NINF) return;
    const Scale sc(t, mz);
    uint32_t last = 0;                                           // tokens of this bucket and those before go on the list
    if (t.lists()) {
        const uint32_t want = t.has_k ? (uint32_t)t.top_k : min(900u, 32 * segments);
#pragma unroll
        for (uint32_t i = 0; i < BUCKETS / 256; i++) s_count[i * 256 + tid] = 0;
        if (tid == 0) s_bucket = BUCKETS - 1;                    // (not so many: all of them)
        __syncthreads();
#pragma unroll
        for (uint32_t i = 0; i < RUNGS; i++) if (r.rung[i] > NINF) atomicAdd(&s_count[sc.bucket(r.rung[i])], rung_rank(i) - (i ? rung_rank(i - 1) : 0));
        __syncthreads();
        uint32_t mine[8], sum = 0;
#pragma unroll
        for (uint32_t i = 0; i < 8; i++) { mine[i] = s_count[tid * 8 + i]; sum += mine[i]; }
        uint32_t incl = (uint32_t)wave_scan(sum);
        if (lane == 63) s_wave[wave] = incl;
        __syncthreads();
        for (uint32_t o = 0; o < wave; o++) incl += s_wave[o];
        uint32_t run = incl - sum;
        if (run < want && incl >= want) {
#pragma unroll
            for (uint32_t i = 0; i < 8; i++) { if (run < want && run + mine[i] >= want) s_bucket = tid * 8 + i; run += mine[i]; }
        }
        __syncthreads();
        last = s_bucket;
    }
    if (seg >= segments) return;
    uint64_t entry[16];
    uint32_t n = 0;
#pragma unroll
    for (uint32_t j = 0; j < 4; j++) {
        const uint32_t st = wave * 256 + j * 64 + lane, at = blockIdx.x * STRIPE + 4 * st;
        float v[4];
        const uint32_t ok = x.unpack(blockIdx.x, st, w[j], b[j], v);
        double mass = 0.0;                                       // (whole numbers below 2^53: exact)
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) {
            v[e] = clean(v[e]);
            const bool may = v[e] >= LOWEST && (!BITS || ((ok >> e) & 1));
            if (may && !t.has_k && (t.has_p || v[e] >= sc.low)) {
                const double we = weight(v[e], sc.m, sc.inv, s_root);
                if (t.has_p || we >= sc.floor_w) mass += we;
            }
            entry[4 * j + e] = may && t.lists() && sc.bucket(v[e]) <= last ? ((uint64_t)key_of(v[e]) << 32) | (uint32_t)~(at + e) : 0;
            n += entry[4 * j + e] != 0;
        }
        if (!t.has_k) {
            const uint64_t sum = wave_scan((uint64_t)mass);
            if (lane == 63) out.part[seg * 4 + j] = sum;
        }
    }
    if (!t.lists()) return;
    const uint32_t incl = (uint32_t)wave_scan(n), all = (uint32_t)__builtin_amdgcn_readlane((int)incl, 63);
    if (!all) return;
    uint32_t at = 0;
    if (lane == 0) at = __hip_atomic_fetch_add(out.count, all, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    at = (uint32_t)__builtin_amdgcn_readfirstlane((int)at) + incl - n;
#pragma unroll
    for (int i = 0; i < 16; i++)
        if (entry[i]) { if (at < LIST) out.list[at] = entry[i]; at++; }
}

// One workgroup per row.  The row is read for the maxima and the sum of exponentials, then once more: for a list of the largest tokens -- those that reach the k-th
// largest (top-k) or the 768th largest (a nucleus of all) of the threads' own maxima, or min_p of the largest weight -- and the weights where a nucleus needs
// their total.  Of the second reading a wave leaves out what its maxima show to be below.  Where the list holds what the filters leave, everything else
// happens on it; otherwise they read the row again.  SPLIT: the two kernels before this one have read the row already.
// Bound by instructions and waiting, not by memory: 512 rows of 131072 bf16 under min_p 55 us (2.4 TB/s; 83 with the weights taken four a lane in the second
// reading instead of from the list), 300 rows of 50265 fp32 under a bitmap, top-k and top-p 34 us (the 44 rows beyond one for every CU cost 10 of them), a nucleus
// of all 69 (its 50265 weights in 64 bits).  Vector units issue in 45 and 29 % of the cycles of the first two, about 31 instructions a token, and waves wait in 60 % of theirs.  All filters, the loops
// for values that are not finite and the re-reading paths are one body: 200 scalar registers are spilled into vector lanes (SPLIT: 87 to 99).  Eight waves a SIMD: a workgroup of 16 waves
// more to hide a row's latency behind, for 4 to 18 spilled vector registers.  SPLIT, one row of 50265: 12.4 us, 1024 threads and some twenty barriers over a list of about a thousand.
template <typename T, bool BITS, bool SPLIT>
__global__ __launch_bounds__(THREADS, SPLIT ? 4 : 8) void k_sample_tokens(SampleArgs a)
{
    __shared__ Shared s;
    const float NINF = -__builtin_huge_valf();
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x, V = a.vocab;
    const Row<T, BITS> x(a, row);
    typedef typename Row<T, BITS>::Raw Raw;
    const uint32_t stripes = (V + STRIPE - 1) / STRIPE;
    // Stripes of the row (a bit each), four of them in flight: f(the stripes, how many, indices of the first logits, four logits each, which may be drawn)
    static_assert(MAX_VOCAB <= 64 * STRIPE, "a bit for each stripe");
    auto stripe_pass = [&](uint64_t mask, auto f) {
        enum { FLY = 4 };
        while (mask) {
            uint32_t at[FLY], n = 0;
            Raw w[FLY];
            uint32_t b[FLY];
#pragma unroll
            for (uint32_t j = 0; j < FLY; j++) {
                at[j] = mask ? (uint32_t)__ffsll((unsigned long long)mask) - 1 : at[j ? j - 1 : 0];
                n += mask != 0;
                mask &= mask - 1;
                w[j] = x.load(at[j], tid);
                b[j] = x.load_bits(at[j], tid);
            }
            float v[FLY][4];
            uint32_t ok[FLY];
#pragma unroll
            for (uint32_t j = 0; j < FLY; j++) ok[j] = x.unpack(at[j], tid, w[j], b[j], v[j]);
            f(at, n, v, ok);
        }
    };
    const uint64_t every = stripes < 64 ? ((uint64_t)1 << stripes) - 1 : ~(uint64_t)0;
    // the wave's stripes, four by four, with a token that may be drawn of at least `from`
    const Settings set(a, row);
    const bool skips = !SPLIT && (set.has_k || (!set.has_p && set.min_p > 0.f));     // (a nucleus of all weighs every token, and without a filter every token stays)
    auto stripes_from = [&](float from) -> uint64_t { return !skips ? every : __ballot(lane < stripes && s.top[lane / 4 * WAVES + wave] >= from); };
    auto row_pass = [&](uint64_t mask, auto f) {                 // f(index of the first, four logits, which may be drawn)
        stripe_pass(mask, [&](const uint32_t *at, uint32_t n, float (*v)[4], const uint32_t *ok) {
#pragma unroll
            for (uint32_t j = 0; j < 4; j++) if (j < n) f(at[j] * STRIPE + 4 * tid, v[j], ok[j]);
        });
    };
    const float L2E = 1.4426950408889634f, LOWEST = -3.402823466e38f;
    if (tid < 32) s.root[tid] = exp2((double)tid / 32.0);
    // the largest logit, and the largest that may be drawn (fmaxf leaves NaN out)
    float mx = NINF, mz = NINF, own = NINF;                      // own: the thread's largest that may be drawn
    float z = 0.f;                                               // the sum of exponentials against `base` (fp32: it enters the log-probabilities only)
    double base;
    Record rec;
    uint64_t part = 0;
    uint32_t on_list = 0;
    if constexpr (SPLIT) {
        const uint32_t segments = (V + SEGMENT - 1) / SEGMENT;
        const RowWork in(a, row);
        rec = tid < segments ? in.record[tid] : no_record();
        part = tid < 4 * segments ? in.part[tid] : 0;
        on_list = *in.count;
        s.list[tid] = in.list[tid];                              // (all of it: its length is on its way, too)
        s.list[tid + THREADS] = in.list[tid + THREADS];
        row_maxima(rec, s.wavef, lane, wave, mx, mz);
        z = rec.z * __builtin_amdgcn_exp2f((rec.max - mx) * L2E);
        base = (double)mx;
    } else {
        // On the values as they are, 16 a thread and turn; NaN comes through a maximum, and with anything beyond +-1e30 it is for the careful loops below.  The sum of
        // exponentials is taken against `ref` in the exponent of 2, so that x log2(e) - ref is one instruction and rounds once.
        float ref = -1.5e30f;
        stripe_pass(every, [&](const uint32_t *at, uint32_t n, float (*v)[4], const uint32_t *ok) {
            float top = NINF;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++)
                if (j < n) {
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        mx = __builtin_elementwise_maximum(mx, v[j][e]);
                        if (BITS) top = __builtin_elementwise_maximum(top, as_f32((ok[j] >> e) & 1 ? as_u32(v[j][e]) : 0xff800000u));
                    }
                }
            const float to = fmaxf(mx, -1e30f) * L2E;
            z *= __builtin_amdgcn_exp2f(ref - to);
            ref = to;
#pragma unroll
            for (uint32_t j = 0; j < 4; j++)
                if (j < n) {
                    if (!BITS) {
#pragma unroll
                        for (int e = 0; e < 4; e++) top = __builtin_elementwise_maximum(top, v[j][e]);
                    }
#pragma unroll
                    for (int e = 0; e < 4; e++) z += __builtin_amdgcn_exp2f(fmaf(v[j][e], L2E, -to));
                }
            own = __builtin_elementwise_maximum(own, top);
            if (!skips) return;
            top = wave_max(top);
            if (lane == 0) s.top[at[0] / 4 * WAVES + wave] = top;
        });
        const bool wild = __any(!(mx <= 1e30f) || (mx < -1e30f && mx > NINF));
        mx = wave_max(mx);
        mz = wave_max(own);
        if (lane == 0) { s.wavef[wave] = wild ? __builtin_nanf("") : mx; s.wavef[WAVES + wave] = mz; }
        __syncthreads();
        mx = s.wavef[lane % WAVES];
        mz = wave_max(s.wavef[WAVES + lane % WAVES]);
        if (!__any(mx != mx)) {
            mx = wave_max(mx);
            const float to = mx * L2E;
            z *= __builtin_amdgcn_exp2f(ref - to);
            base = uniform((double)to / (double)L2E);
        } else {
            z = 0.f;
            mx = own = NINF;
            stripe_pass(every, [&](const uint32_t *at, uint32_t n, float (*v)[4], const uint32_t *ok) {
                float top = NINF;
#pragma unroll
                for (uint32_t j = 0; j < 4; j++)
                    if (j < n) {
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            const float c = clean(v[j][e]);
                            mx = fmaxf(mx, c);
                            if (!BITS || ((ok[j] >> e) & 1)) top = fmaxf(top, c);
                        }
                    }
                own = fmaxf(own, top);
                if (!skips) return;
                top = wave_max(top);
                if (lane == 0) s.top[at[0] / 4 * WAVES + wave] = top;
            });
            mx = wave_max(mx);
            mz = wave_max(own);
            __syncthreads();
            if (lane == 0) { s.wavef[wave] = mx; s.wavef[WAVES + wave] = mz; }
            __syncthreads();
            mx = wave_max(s.wavef[lane % WAVES]);
            mz = wave_max(s.wavef[WAVES + lane % WAVES]);
            base = (double)mx;
            row_pass(every, [&](uint32_t, const float *v, uint32_t) {
#pragma unroll
                for (int e = 0; e < 4; e++) z += __builtin_amdgcn_exp2f((clean(v[e]) - mx) * L2E);
            });
        }
    }
    if (mz == NINF) {                                            // nothing may be drawn
        for (uint32_t d = tid; d < a.draws; d += THREADS) { a.tokens[(uint64_t)row * a.draws + d] = -1; a.logprobs[(uint64_t)row * a.draws + d] = NINF; }
        return;
    }
    const Scale sc(set, mz);
    auto weigh = [&](float v) { return weight(v, sc.m, sc.inv, s.root); };
    auto one = [](float) { return 1.0; };
    auto bucket0 = [&](float v) { return sc.bucket(v); };
    auto value_of = [](uint64_t e) { const uint32_t k = (uint32_t)(e >> 32); return as_f32((k >> 31) ? k ^ 0x80000000u : ~k); };
    uint32_t thr = 0, lim = 0xffffffffu;                         // kept: key > thr, or key == thr and index <= lim
    auto kept = [&](float v, uint32_t idx) { const uint32_t k = key_of(v); return k > thr || (k == thr && idx <= lim); };
    // every token that may be drawn and is at least `from`: f(logit, index)
    auto row_from = [&](float from, auto f) {
        row_pass(stripes_from(from), [&](uint32_t at, float *v, uint32_t ok) {
            bool any = false;
#pragma unroll
            for (int e = 0; e < 4; e++) any |= v[e] >= from;
            if (any) {
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) if (v[e] >= from && (!BITS || ((ok >> e) & 1))) f(clean(v[e]), at + e);
            }
        });
    };
    auto clear_buckets = [&]() {
        __syncthreads();
        s.mass[tid] = s.mass[tid + THREADS] = 0;
        if (tid == 0) s.n = 0;
        __syncthreads();
    };
    uint32_t listed = 0;                                         // > 0: everything that is kept is among the list's first entries (in no order)
    auto list_pass = [&](auto f) { for (uint32_t i = tid; i < listed; i += THREADS) f(value_of(s.list[i]), ~(uint32_t)s.list[i]); };
    auto put_list = [&](float v, uint32_t idx) { const uint32_t at = atomicAdd(&s.n, 1u); if (at < LIST) s.list[at] = ((uint64_t)key_of(v) << 32) | (uint32_t)~idx; };
    auto put_order = [&](float v, uint32_t idx) { const uint32_t at = atomicAdd(&s.n, 1u); if (at < LIST) s.order[at] = ((uint64_t)key_of(v) << 32) | (uint32_t)~idx; };

    // The border inside s.order[0 .. n), all of it kept so far, behind a sum of `front`: thr and lim become the first token (in order) whose running sum
    // of `value` reaches what is asked for.  Up to 64 tokens one wave sorts in registers.
    auto border = [&](uint32_t n, uint64_t front, auto value, auto reached) {
        if (n <= 64) {
            if (wave == 0) {
                const uint64_t e = sort_wave(lane < n ? s.order[lane] : 0, lane);
                const uint64_t run = front + wave_scan(lane < n ? (uint64_t)value(value_of(e)) : 0);
                const uint64_t hit = __ballot(lane < n && reached(run));
                const uint32_t first = hit ? (uint32_t)__ffsll((unsigned long long)hit) - 1 : n - 1;
                if (lane == first) { s.thr = (uint32_t)(e >> 32); s.lim = ~(uint32_t)e; }
            }
        } else {
            sort_order(s, n, tid);
            const uint64_t w0 = 2 * tid < n ? (uint64_t)value(value_of(s.order[2 * tid])) : 0, w1 = 2 * tid + 1 < n ? (uint64_t)value(value_of(s.order[2 * tid + 1])) : 0;
            uint64_t sum;
            const uint64_t incl = front + block_scan(w0 + w1, s, lane, wave, sum);
            // (the running sums grow: one thread finds the first that reaches it, or the last entry stands)
            const bool r0 = reached(incl - w1), r1 = reached(incl), before = 2 * tid > 0 && reached(incl - w0 - w1);
            const uint32_t at = r0 ? 2 * tid : 2 * tid + 1;
            if (tid == 0) { s.thr = (uint32_t)(s.order[n - 1] >> 32); s.lim = ~(uint32_t)s.order[n - 1]; }
            __syncthreads();
            if ((r0 || r1) && !before && at < n) { s.thr = (uint32_t)(s.order[at] >> 32); s.lim = ~(uint32_t)s.order[at]; }
        }
        __syncthreads();
        thr = s.thr;
        lim = s.lim;
        __syncthreads();
    };
    // Shortens the prefix to where the running sum of `value` over the kept tokens reaches what is asked for (false: it never does; nothing changes): sums buckets,
    // then orders the one bucket that the border falls into.  `pass` goes over the list or the row.
    auto shorten = [&](auto pass, auto value, auto reached) -> bool {
        clear_buckets();
        pass([&](float v, uint32_t idx) {
            if (!kept(v, idx)) return;
            const uint64_t w = (uint64_t)value(v);
            if (w) atomicAdd((unsigned long long *)&s.mass[bucket0(v)], (unsigned long long)w);
        });
        __syncthreads();
        find_bucket(s, tid, lane, wave, [&](uint64_t f, uint64_t) { return reached(f); });
        if (!s.found) return false;
        const uint32_t B = s.bucket;
        uint64_t front = s.before;
        uint32_t lo = 0, hi = 0xffffffffu;                       // keys that the border lies between
        auto member = [&](float v, uint32_t idx) { const uint32_t k = key_of(v); return k >= lo && k <= hi && bucket0(v) == B && kept(v, idx); };
        for (;;) {
            __syncthreads();
            if (tid == 0) { s.n = 0; s.kmin = 0xffffffffu; s.kmax = 0; }
            __syncthreads();
            pass([&](float v, uint32_t idx) { if (member(v, idx)) put_order(v, idx); });
            __syncthreads();
            const uint32_t n = s.n;
            if (n <= LIST) {
                border(n, front, value, reached);
                return true;
            }
            // more than can be sorted (many equal logits): narrowed by key, level by level
            uint32_t kmin = 0xffffffffu, kmax = 0;
            pass([&](float v, uint32_t idx) { if (member(v, idx)) { kmin = min(kmin, key_of(v)); kmax = max(kmax, key_of(v)); } });
            for (int o = 32; o > 0; o >>= 1) { kmin = min(kmin, __shfl_xor(kmin, o)); kmax = max(kmax, __shfl_xor(kmax, o)); }
            if (lane == 0) { atomicMin(&s.kmin, kmin); atomicMax(&s.kmax, kmax); }
            __syncthreads();
            lo = s.kmin; hi = s.kmax;
            if (lo >= hi) break;
            const uint32_t width = 32 - __clz(hi - lo), shift = width > 11 ? width - 11 : 0;
            clear_buckets();
            pass([&](float v, uint32_t idx) {
                if (member(v, idx)) atomicAdd((unsigned long long *)&s.mass[(hi - key_of(v)) >> shift], (unsigned long long)(uint64_t)value(v));
            });
            __syncthreads();
            find_bucket(s, tid, lane, wave, [&](uint64_t f, uint64_t) { return reached(front + f); });
            if (!s.found) return true;                           // (cannot be: the bucket's members sum to what the level before saw)
            front += s.before;
            const uint32_t top = hi - (s.bucket << shift);
            lo = max(lo, shift ? top - ((1u << shift) - 1) : top);
            hi = top;
        }
        // more equal logits than can be sorted: how many of them stay (each adds w), and the index of the last of those
        const uint32_t old_lim = hi == thr ? lim : 0xffffffffu;
        thr = hi;
        const uint64_t w = (uint64_t)value(value_of((uint64_t)thr << 32));
        uint64_t stay = 0, step = (uint64_t)1 << 18;             // the largest number that does not reach it, plus one
        for (; step; step >>= 1) if (!reached(front + (stay + step) * w)) stay += step;
        stay++;
        __syncthreads();
        s.part[tid] = 0;
        __syncthreads();
        pass([&](float v, uint32_t idx) { if (key_of(v) == thr && idx <= old_lim) atomicAdd((unsigned long long *)&s.part[idx >> 8], 1ull); });
        __syncthreads();
        uint64_t sum;
        const uint64_t n = s.part[tid], incl = block_scan(n, s, lane, wave, sum);
        if (tid == 0) { s.found = 0xffffffffu; s.lim = old_lim; }
        __syncthreads();
        if (incl >= stay && incl - n < stay) { s.found = tid; s.before = incl - n; }
        __syncthreads();
        const uint32_t at = s.found;
        if (at != 0xffffffffu && wave == 0) {                   // those 256 logits again, in order
            float v[4];
            const uint32_t i = at / WAVES, t = (at % WAVES) * 64 + lane, idx = at * 256 + 4 * lane;
            uint32_t ok = x.unpack(i, t, x.load(i, t), x.load_bits(i, t), v), mine = 0;
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) { if (!(clean(v[e]) >= LOWEST) || key_of(clean(v[e])) != thr || idx + e > old_lim) ok &= ~(1u << e); mine += (ok >> e) & 1; }
            const uint32_t rank = (uint32_t)wave_scan(mine) - mine, want = (uint32_t)(stay - s.before);
            if (rank < want && rank + mine >= want) {
                uint32_t left = want - rank;
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) if (((ok >> e) & 1) && --left == 0) s.lim = min(old_lim, idx + e);
            }
        }
        __syncthreads();
        lim = s.lim;
        __syncthreads();
        return true;
    };
    auto row_all = [&](auto f) { row_from(LOWEST, f); };        // (a logit of -inf is never drawn)
    const bool has_k = set.has_k, has_p = set.has_p;
    const uint64_t k = (uint64_t)set.top_k;
    const double p = (double)fmaxf(set.top_p, 0.f);
    double own_mass = 0.0;                                       // (whole numbers below 2^53: exact)
    uint64_t total = 0;                                          // the weight that a nucleus is a part of
    if (SPLIT) {
        if (set.lists() && on_list <= LIST) listed = on_list;
        if (!has_k) block_scan(part, s, lane, wave, total);
        __syncthreads();
    } else if (set.lists()) {
        // the smallest of the `want` largest of the threads' maxima: at least `want` tokens reach it
        const uint64_t want = has_k ? k : 3 * THREADS / 4;
        clear_buckets();
        if (own > NINF) atomicAdd((unsigned long long *)&s.mass[bucket0(own)], 1ull);
        if (tid == 0) s.kmin = 0xffffffffu;
        __syncthreads();
        find_bucket(s, tid, lane, wave, [&](uint64_t f, uint64_t) { return f >= want; });
        const bool enough_of_them = s.found != 0;
        float from = LOWEST;
        if (enough_of_them) {
            if (own > NINF && bucket0(own) <= s.bucket) atomicMin(&s.kmin, key_of(own));
            __syncthreads();
            from = value_of((uint64_t)s.kmin << 32);
        }
        __syncthreads();
        if (has_k) row_from(from, put_list);
        else
            row_from(LOWEST, [&](float v, uint32_t idx) {
                own_mass += weigh(v);
                if (v >= from) put_list(v, idx);
            });
        __syncthreads();
        listed = s.n <= LIST ? s.n : 0;
        if (!has_k) { block_scan((uint64_t)own_mass, s, lane, wave, total); }
        __syncthreads();
    } else if (skips && !has_k) {                                // min_p alone: the tokens that it leaves, if they fit
        if (tid == 0) s.n = 0;
        __syncthreads();
        row_from(sc.low, put_list);
        __syncthreads();
        listed = s.n <= LIST ? s.n : 0;
        __syncthreads();
    }
    auto row_lse = [&]() {                                       // of the waves' sums in s.wavef
        double sum = 0.0;
        for (int w = 0; w < WAVES; w++) sum += (double)s.wavef[w];
        return base + log(sum);
    };
    auto put_z = [&]() {
        float sum = z;
        for (int o = 32; o > 0; o >>= 1) sum += __shfl_xor(sum, o);
        if (lane == 0) s.wavef[wave] = sum;
    };
    // floor(u * all), u as 63 bits
    auto target_of = [](float u, uint64_t all) -> uint64_t {
        const double uc = u > 0.f ? fmin((double)u, 1.0 - 1.0 / 16777216) : 0.0;
        const uint64_t u63 = (uint64_t)(uc * 9223372036854775808.0);
        return (__umul64hi(u63, all) << 1) | ((u63 * all) >> 63);
    };
    if (listed && listed <= 64) {
        // One wave does what is left, a token a lane: in falling order for the filters, then in the order of the vocabulary for the draws (300 rows of 50265 under
        // a bitmap with top-k 50 and top-p: 34 us, 39 with the general steps below)
        put_z();
        if (tid == 0) s.found = 0;
        __syncthreads();
        if (wave == 0) {
            const uint64_t e = sort_wave(lane < listed ? s.list[lane] : 0, lane);
            const float v = value_of(e);
            bool in = lane < listed && (!has_k || lane < k);
            const double w = in ? weigh(v) : 0.0;
            bool enough = true;
            if (has_p) {
                const uint64_t run = wave_scan((uint64_t)w), all = has_k ? wave_total(run) : total;
                const uint64_t hit = __ballot(in && run > 0 && (double)run >= p * (double)all);
                enough = hit != 0;
                in = in && lane < (uint32_t)__ffsll((unsigned long long)hit);
            }
            in = in && v >= sc.low && w >= sc.floor_w;
            if (enough) {
                if (lane == 0) s.found = 1;
                const uint64_t by_index = sort_wave((e << 32) | lane, lane);         // (the low half of an entry is ~index)
                const int from = (int)(by_index & 63);
                const uint32_t idx = ~(uint32_t)(by_index >> 32);
                const float x_at = __shfl(v, from);
                const uint64_t incl = wave_scan(__shfl(in ? (uint64_t)w : 0, from)), left = wave_total(incl);
                const double lse = row_lse();
                for (uint32_t d0 = 0; d0 < a.draws; d0 += 64) {  // a draw a lane; where each falls is the wave's question
                    const uint32_t many = min(a.draws - d0, 64u);
                    const uint64_t at = (uint64_t)row * a.draws + d0 + lane, mine = target_of(lane < many ? a.u[at] : 0.f, left);
                    int drawn = 0;
                    for (uint32_t j = 0; j < many; j++) {
                        const uint64_t target = ((uint64_t)(uint32_t)__builtin_amdgcn_readlane((int)(mine >> 32), (int)j) << 32) |
                                                (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)mine, (int)j);
                        const int first = __ffsll((unsigned long long)__ballot(incl > target)) - 1;
                        if (lane == j) drawn = first;
                    }
                    const uint32_t token = __shfl(idx, drawn);
                    const float x_drawn = __shfl(x_at, drawn);
                    if (lane < many) { a.tokens[at] = token; a.logprobs[at] = (float)((double)x_drawn - lse); }
                }
            }
        }
        if (has_k || !has_p) return;                             // (a nucleus of all may be larger than the list)
        __syncthreads();
        if (s.found) return;
        __syncthreads();
    }
    if (has_k) {
        auto reached = [&](uint64_t f) { return f >= k; };
        if (!listed) shorten(row_all, one, reached);
        else shorten(list_pass, one, reached);
    }
    if (has_p) {
        // (a prefix of mass f is long enough; an empty one never is)
        auto reached = [&](uint64_t f) { return f > 0 && (double)f >= p * (double)total; };
        if (has_k) {
            // the weight of the k largest
            own_mass = 0.0;
            auto add = [&](float v, uint32_t idx) { if (kept(v, idx)) own_mass += weigh(v); };
            if (listed) list_pass(add);
            else row_all(add);
            block_scan((uint64_t)own_mass, s, lane, wave, total);
        }
        bool done = false;
        if (listed > 64) done = shorten(list_pass, weigh, reached);
        if (!done) {                                             // the nucleus is larger than the list
            listed = 0;
            shorten(row_all, weigh, reached);
        }
    }
    // The weights of what is left, summed for every 256 tokens
    const double floor_w = sc.floor_w;
    const float low = sc.low;
    auto final_weight = [&](float v, uint32_t idx) -> uint64_t {
        if (!(v >= low) || !kept(v, idx)) return 0;
        const double w = weigh(v);
        return w >= floor_w ? (uint64_t)w : 0;
    };
    const uint32_t parts = stripes * WAVES;
    __syncthreads();
    s.part[tid] = SPLIT && !has_k && !has_p ? part : 0;
    __syncthreads();
    if (SPLIT && !has_k && !has_p) {}
    else if (listed) list_pass([&](float v, uint32_t idx) { const uint64_t w = final_weight(v, idx); if (w) atomicAdd((unsigned long long *)&s.part[idx >> 8], (unsigned long long)w); });
    else
        row_pass(stripes_from(low), [&](uint32_t at, float *v, uint32_t ok) {
            uint64_t w = 0;
            bool any = false;
#pragma unroll
            for (int e = 0; e < 4; e++) any |= v[e] >= low;
            if (any) {
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) if (!BITS || ((ok >> e) & 1)) w += final_weight(clean(v[e]), at + e);
            }
            if (__any(w != 0)) {
                const uint64_t sum = wave_scan(w);
                if (lane == 63) s.part[at >> 8] = sum;
            }
        });
    __syncthreads();
    uint64_t left;
    const uint64_t incl = block_scan(tid < parts ? s.part[tid] : 0, s, lane, wave, left);
    s.part[tid] = incl;
    put_z();
    __syncthreads();
    if (wave >= a.draws) return;
    const double lse = row_lse();
    for (uint32_t d = wave; d < a.draws; d += WAVES) {
        // floor(u * left), and the first 256 tokens whose running sum passes it
        const uint64_t target = target_of(a.u[(uint64_t)row * a.draws + d], left);
        uint32_t lo = 0, hi = parts - 1;
        while (lo < hi) { const uint32_t mid = (lo + hi) / 2; if (s.part[mid] > target) hi = mid; else lo = mid + 1; }
        const uint64_t rest = target - (lo ? s.part[lo - 1] : 0);
        float v[4];
        uint64_t w[4];
        const uint32_t i = lo / WAVES, t = (lo % WAVES) * 64 + lane, idx = lo * 256 + 4 * lane;
        const uint32_t ok = x.unpack(i, t, x.load(i, t), x.load_bits(i, t), v);
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) { v[e] = clean(v[e]); w[e] = !BITS || ((ok >> e) & 1) ? final_weight(v[e], idx + e) : 0; }
        const uint64_t mine = w[0] + w[1] + w[2] + w[3], sum = wave_scan(mine);
        if (sum > rest && sum - mine <= rest) {
            uint64_t run = sum - mine;
            bool done = false;
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                run += w[e];
                if (!done && run > rest) {
                    done = true;
                    a.tokens[(uint64_t)row * a.draws + d] = idx + e;
                    a.logprobs[(uint64_t)row * a.draws + d] = (float)((double)v[e] - lse);
                }
            }
        }
    }
}

template <typename T>
static int sample_tokens(void *stream, const SampleArgs &a, uint64_t work_bytes)
{
    if (!a.rows || !a.draws) return FMI_OK;
    if (!a.vocab || a.vocab > MAX_VOCAB) { fmi_set_error("sealnn_sample_tokens: a vocabulary of %u (1 .. %u)", a.vocab, (unsigned)MAX_VOCAB); return FMI_ERR_UNSUPPORTED; }
    if (!a.logits || !a.u || !a.tokens || !a.logprobs || ((uintptr_t)a.logits & (sizeof(T) - 1))) { fmi_set_error("sealnn_sample_tokens: null or misaligned argument"); return FMI_ERR_ARG; }
    if (a.work && (a.vocab < 4 || a.rows > 65535 || work_bytes < a.rows * row_work(a.vocab) || ((uintptr_t)a.work & 15))) {
        fmi_set_error("sealnn_sample_tokens: %u rows of %u in a workspace of %llu bytes (16-byte aligned; %llu for a row of at least 4, at most 65535 rows)", a.rows, a.vocab,
                      (unsigned long long)work_bytes, (unsigned long long)row_work(a.vocab));
        return FMI_ERR_ARG;
    }
    hipStream_t st = (hipStream_t)stream;
    auto go = [&](auto bits) {
        constexpr bool B = decltype(bits)::value;
        if (!a.work) { hipLaunchKernelGGL((k_sample_tokens<T, B, false>), dim3(a.rows), dim3(THREADS), 0, st, a); return; }
        const dim3 grid((a.vocab + STRIPE - 1) / STRIPE, a.rows);
        hipLaunchKernelGGL((k_sample_segments<T, B>), grid, dim3(256), 0, st, a);
        hipLaunchKernelGGL((k_sample_lists<T, B>), grid, dim3(256), 0, st, a);
        hipLaunchKernelGGL((k_sample_tokens<T, B, true>), dim3(a.rows), dim3(THREADS), 0, st, a);
    };
    if (a.bits) go(std::true_type());
    else go(std::false_type());
    NNCHK();
    return FMI_OK;
}

static SampleArgs sample_args(const void *logits, uint64_t row_stride, uint32_t rows, uint32_t vocab, const float *u, uint32_t draws, const uint32_t *bits,
                              uint64_t bits_stride, float temperature, int32_t top_k, float top_p, float min_p, const float *temperature_v,
                              const int32_t *top_k_v, const float *top_p_v, const float *min_p_v, int64_t *tokens, float *logprobs, void *work)
{
    SampleArgs a;
    a.logits = logits; a.row_stride = row_stride; a.bits = bits; a.bits_stride = bits_stride; a.u = u;
    a.temperature_v = temperature_v; a.top_p_v = top_p_v; a.min_p_v = min_p_v; a.top_k_v = top_k_v;
    a.rows = rows; a.vocab = vocab; a.draws = draws; a.temperature = temperature; a.top_p = top_p; a.min_p = min_p; a.top_k = top_k;
    a.tokens = tokens; a.logprobs = logprobs; a.work = (char *)work;
    return a;
}

extern "C" int sealnn_sample_tokens(void *stream, const float *logits, uint64_t row_stride, uint32_t rows, uint32_t vocab, const float *u, uint32_t draws,
                                    const uint32_t *bits, uint64_t bits_stride, float temperature, int32_t top_k, float top_p, float min_p,
                                    const float *temperature_v, const int32_t *top_k_v, const float *top_p_v, const float *min_p_v, int64_t *tokens, float *logprobs,
                                    void *work, uint64_t work_bytes)
{ return sample_tokens<float>(stream, sample_args(logits, row_stride, rows, vocab, u, draws, bits, bits_stride, temperature, top_k, top_p, min_p, temperature_v, top_k_v, top_p_v, min_p_v, tokens, logprobs, work), work_bytes); }
extern "C" int sealnn_sample_tokens_bf16(void *stream, const void *logits, uint64_t row_stride, uint32_t rows, uint32_t vocab, const float *u, uint32_t draws,
                                         const uint32_t *bits, uint64_t bits_stride, float temperature, int32_t top_k, float top_p, float min_p,
                                         const float *temperature_v, const int32_t *top_k_v, const float *top_p_v, const float *min_p_v, int64_t *tokens, float *logprobs,
                                         void *work, uint64_t work_bytes)
{ return sample_tokens<bf16>(stream, sample_args(logits, row_stride, rows, vocab, u, draws, bits, bits_stride, temperature, top_k, top_p, min_p, temperature_v, top_k_v, top_p_v, min_p_v, tokens, logprobs, work), work_bytes); }
