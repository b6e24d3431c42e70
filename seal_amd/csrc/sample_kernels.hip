// Drawing tokens from logits: temperature, top-k, top-p and min-p under an optional allowed-token bitmap, from given random numbers
// (include/sealnn.h: sealnn_sample_tokens).
//
// With the tokens ordered by (logit falling, index rising) every filter keeps a PREFIX: the first k; the smallest prefix with at least p of
// the mass of those; the tokens of at least min_p of the largest weight.  So the kernel never sorts: it finds the logit at which the prefix ends
// by counting (or weighing) buckets of logits and looking again inside the one bucket that the border falls into, and then draws in the order
// of the vocabulary from the tokens above it: the first token whose cumulative weight passes u * total.
//
// Weights are whole numbers, exp((x - max) / T) * 2^44 to nearest, computed in 64-bit floats and added in 64-bit integers: sums of up to 2^18 of
// them are exact, so neither the order of the atomics nor the shape of a reduction changes which token a random number falls on.
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
};

static __device__ __forceinline__ uint32_t key_of(float x) { const uint32_t u = as_u32(x); return u ^ ((u >> 31) ? 0xffffffffu : 0x80000000u); }
// NaN counts as -inf, +inf as the largest number, -0 as +0
static __device__ __forceinline__ float clean(float x) { return x != x ? -__builtin_huge_valf() : fminf(x, 3.402823466e38f) + 0.f; }

struct Shared {
    union {
        uint64_t mass[BUCKETS];                          // a histogram ...
        uint64_t run[LIST];                              // ... or the running weights of the list
    };
    uint64_t list[LIST];                                 // (key << 32 | ~index): tokens in falling order of logit, equal ones in rising order of index
    uint64_t part[MAX_VOCAB / STRIPE * WAVES];
    uint64_t wave[WAVES];
    float wavef[3 * WAVES];
    double root[32];                                     // 2^(i / 32)
    uint32_t kmin, kmax, found, bucket, n;
    uint64_t before, total;
};

// exp((x - m) / T) * 2^44 to nearest, as a 64-bit float (a whole number; 0 below 2^-45): 2^t = 2^floor * 2^(k / 32) * e^y, |y| <= ln 2 / 64, where the
// series ends at y^4 (y^5 / 120 < 2^-39 relative, below the step of any weight that is not near the largest)
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

template <typename V> static __device__ __forceinline__ V wave_scan(V v, uint32_t lane)
{
    for (uint32_t o = 1; o < 64; o <<= 1) { const V w = __shfl_up(v, o); if (lane >= o) v += w; }
    return v;
}

// inclusive sums over the workgroup
static __device__ __forceinline__ uint64_t block_scan(uint64_t v, Shared &s, uint32_t lane, uint32_t wave)
{
    v = wave_scan(v, lane);
    __syncthreads();
    if (lane == 63) s.wave[wave] = v;
    __syncthreads();
    uint64_t add = 0;
    for (uint32_t w = 0; w < wave; w++) add += s.wave[w];
    return v + add;
}

// The bucket (in order) at which the running sum of s.mass reaches what is asked for: s.bucket, s.before (the sum in front of it), s.total;
// s.found = 0 if it never does
template <typename REACHED>
static __device__ __forceinline__ void find_bucket(Shared &s, uint32_t tid, uint32_t lane, uint32_t wave, REACHED reached)
{
    static_assert(BUCKETS == 2 * THREADS, "two buckets a thread");
    const uint64_t a = s.mass[2 * tid], b = s.mass[2 * tid + 1];
    const uint64_t incl = block_scan(a + b, s, lane, wave);
    if (tid == 0) s.found = 0;
    if (tid == THREADS - 1) s.total = incl;
    __syncthreads();
    const uint64_t total = s.total, f0 = incl - a - b, f1 = incl - b;
    if (!reached(f0, total) && reached(f1, total)) { s.found = 1; s.bucket = 2 * tid; s.before = f0; }
    else if (!reached(f1, total) && reached(incl, total)) { s.found = 1; s.bucket = 2 * tid + 1; s.before = f1; }
    __syncthreads();
}

// s.list[0 .. n) into falling order (zeros behind it).  Up to 128 entries one wave does it alone.
static __device__ __forceinline__ void sort_list(Shared &s, uint32_t n, uint32_t tid)
{
    uint32_t size = 2;
    while (size < n) size <<= 1;
    for (uint32_t i = n + tid; i < size; i += THREADS) s.list[i] = 0;
    __syncthreads();
    const bool alone = size <= 128;
    if (!alone || tid < 64) {
        for (uint32_t k = 2; k <= size; k <<= 1)
            for (uint32_t j = k >> 1; j > 0; j >>= 1) {
                if (tid < size / 2) {
                    const uint32_t i = ((tid & ~(j - 1)) << 1) | (tid & (j - 1)), o = i | j;
                    const uint64_t a = s.list[i], b = s.list[o];
                    if ((a < b) == ((i & k) == 0)) { s.list[i] = b; s.list[o] = a; }
                }
                if (alone) __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
                else __syncthreads();
            }
    }
    __syncthreads();
}

// One workgroup per row.  The row is read for the maxima and the sum of exponentials, and then once or twice more (from the caches) for what
// the filters need; the work behind them is done on a list of the few tokens that matter, wherever there are few.
template <typename T>
__global__ __launch_bounds__(THREADS) void k_sample_tokens(SampleArgs a)
{
    __shared__ Shared s;
    const float NINF = -__builtin_huge_valf();
    const uint32_t tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, row = blockIdx.x, V = a.vocab;
    const T *x = (const T *)a.logits + (uint64_t)row * a.row_stride;
    const uint32_t *bits = a.bits ? a.bits + (uint64_t)row * a.bits_stride : nullptr;
    const uint32_t stripes = (V + STRIPE - 1) / STRIPE;
    // four logits of stripe i (-inf beyond the row) and which of them may be drawn
    auto fetch = [&](uint32_t i, uint32_t t, float v[4]) -> uint32_t {
        const uint32_t at = i * STRIPE + 4 * t;
        uint32_t ok = 0;
        if (at + 4 <= V) {
            if constexpr (std::is_same<T, float>::value) {
                const f32x4_a4 w = *(const f32x4_a4 *)(x + at);
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = w[e];
            } else {
                const u16x4_a2 w = *(const u16x4_a2 *)(x + at);
#pragma unroll
                for (int e = 0; e < 4; e++) v[e] = as_f32((uint32_t)w[e] << 16);
            }
            ok = 15;
        } else {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                v[e] = at + e < V ? load1(x + at + e) : NINF;
                ok |= at + e < V ? 1u << e : 0u;
            }
        }
        if (bits && at < V) ok &= bits[at >> 5] >> (at & 31);
#pragma unroll
        for (int e = 0; e < 4; e++) { v[e] = clean(v[e]); if (v[e] == NINF) ok &= ~(1u << e); }
        return ok & 15;
    };
    auto all = [&](auto f) {                                     // f(stripe, four logits, which may be drawn)
#pragma unroll 2
        for (uint32_t i = 0; i < stripes; i++) { float v[4]; const uint32_t ok = fetch(i, tid, v); f(i, v, ok); }
    };
    if (tid < 32) s.root[tid] = exp2((double)tid / 32.0);
    // the largest logit with the sum of exponentials (fp32: it enters the log-probabilities only), and the largest that may be drawn
    const float L2E = 1.4426950408889634f;
    float mx = NINF, z = 0.f, mz = NINF;
    all([&](uint32_t, const float *v, uint32_t ok) {
        const float m4 = fmaxf(fmaxf(fmaxf(v[0], v[1]), fmaxf(v[2], v[3])), mx);
        if (m4 > NINF) {
            float t = 0.f;
#pragma unroll
            for (int e = 0; e < 4; e++) t += __builtin_amdgcn_exp2f((v[e] - m4) * L2E);
            z = z * __builtin_amdgcn_exp2f((mx - m4) * L2E) + t;
            mx = m4;
        }
#pragma unroll
        for (int e = 0; e < 4; e++) mz = fmaxf(mz, (ok >> e) & 1 ? v[e] : NINF);
    });
    const float own_mz = mz;
    for (int o = 32; o > 0; o >>= 1) {
        const float om = __shfl_xor(mx, o), oz = __shfl_xor(z, o), nm = fmaxf(mx, om);
        z = nm > NINF ? z * __builtin_amdgcn_exp2f((mx - nm) * L2E) + oz * __builtin_amdgcn_exp2f((om - nm) * L2E) : 0.f;
        mx = nm;
        mz = fmaxf(mz, __shfl_xor(mz, o));
    }
    if (lane == 0) { s.wavef[wave] = mx; s.wavef[WAVES + wave] = mz; s.wavef[2 * WAVES + wave] = z; }
    __syncthreads();
    for (int w = 0; w < WAVES; w++) { mx = fmaxf(mx, s.wavef[w]); mz = fmaxf(mz, s.wavef[WAVES + w]); }
    if (mz == NINF) {                                            // nothing may be drawn
        for (uint32_t d = tid; d < a.draws; d += THREADS) { a.tokens[(uint64_t)row * a.draws + d] = -1; a.logprobs[(uint64_t)row * a.draws + d] = NINF; }
        return;
    }
    double zs = 0.0;
    for (int w = 0; w < WAVES; w++) zs += (double)(s.wavef[2 * WAVES + w] * __builtin_amdgcn_exp2f((s.wavef[w] - mx) * L2E));
    const double lse = (double)mx + log(zs);

    float temperature = a.temperature_v ? a.temperature_v[row] : a.temperature;
    int32_t top_k = a.top_k_v ? a.top_k_v[row] : a.top_k;
    const float top_p = a.top_p_v ? a.top_p_v[row] : a.top_p, min_p_ = a.min_p_v ? a.min_p_v[row] : a.min_p;
    if (!(temperature > 0.f)) { temperature = 1.f; top_k = 1; }                       // greedy: the first of the largest
    const double inv = 1.4426950408889634074 / (double)temperature, m = (double)mz;
    const double floor_w = min_p_ > 0.f ? (double)fminf(min_p_, 1.f) * 17592186044416.0 : 0.0;
    const float c = fminf(64.f / temperature, 1e30f);
    // buckets of 1 / 64 of a temperature below the largest logit: they order as the logits do (a rounded difference and product are monotone)
    auto bucket0 = [&](float v) { const float b = (mz - v) * c; return b < (float)(BUCKETS - 1) ? (uint32_t)b : (uint32_t)(BUCKETS - 1); };
    auto entry = [&](float v, uint32_t idx) { return ((uint64_t)key_of(v) << 32) | (uint32_t)~idx; };
    auto value_of = [](uint64_t e) { const uint32_t k = (uint32_t)(e >> 32); return as_f32((k >> 31) ? k ^ 0x80000000u : ~k); };
    uint32_t thr = 0, lim = 0xffffffffu;                         // kept: key > thr, or key == thr and index <= lim
    auto kept = [&](float v, uint32_t idx) { const uint32_t k = key_of(v); return k > thr || (k == thr && idx <= lim); };
    // Tokens that satisfy `want` (of those that may be drawn) into s.list, unordered; their number (those beyond LIST are counted, not stored)
    auto collect = [&](auto want) {
        __syncthreads();
        if (tid == 0) s.n = 0;
        __syncthreads();
        all([&](uint32_t i, const float *v, uint32_t ok) {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                const uint32_t idx = i * STRIPE + 4 * tid + e;
                if (((ok >> e) & 1) && want(v[e], idx)) { const uint32_t at = atomicAdd(&s.n, 1u); if (at < LIST) s.list[at] = entry(v[e], idx); }
            }
        });
        __syncthreads();
        return s.n;
    };
    auto clear_buckets = [&]() {
        __syncthreads();
        for (uint32_t b = tid; b < BUCKETS; b += THREADS) s.mass[b] = 0;
        __syncthreads();
    };
    // running weights (or counts) of the sorted list into s.run: thread t holds entries 2 t and 2 t + 1
    auto run_list = [&](uint32_t n, auto value) {
        static_assert(LIST == 2 * THREADS, "two entries a thread");
        const uint64_t w0 = 2 * tid < n ? (uint64_t)value(value_of(s.list[2 * tid])) : 0, w1 = 2 * tid + 1 < n ? (uint64_t)value(value_of(s.list[2 * tid + 1])) : 0;
        const uint64_t incl = block_scan(w0 + w1, s, lane, wave);
        s.run[2 * tid] = incl - w1;
        s.run[2 * tid + 1] = incl;
        __syncthreads();
    };
    // how many entries of the sorted list stand in front of the first whose running sum (plus `front`) reaches what is asked for, that one included
    auto first_reached = [&](uint32_t n, auto reached) {
        __syncthreads();
        if (tid == 0) s.n = n;
        __syncthreads();
        for (uint32_t i = tid; i < n; i += THREADS)
            if (reached(s.run[i]) && (i == 0 || !reached(s.run[i - 1]))) s.n = i + 1;
        __syncthreads();
        return s.n;
    };
    auto weigh = [&](float v) { return weight(v, m, inv, s.root); };
    auto one = [](float) { return 1.0; };

    // Shortens the prefix to where the running sum of `value` reaches what `reached`(sum, total) asks for: sums buckets, then orders the one bucket that the border
    // falls into (its tokens on the list; more than the list holds -- many equal logits -- are narrowed by key, level by level).
    auto shorten = [&](auto value, auto reached) {
        clear_buckets();
        all([&](uint32_t i, const float *v, uint32_t ok) {
#pragma unroll
            for (uint32_t e = 0; e < 4; e++)
                if (((ok >> e) & 1) && kept(v[e], i * STRIPE + 4 * tid + e)) {
                    const uint64_t w = (uint64_t)value(v[e]);
                    if (w) atomicAdd((unsigned long long *)&s.mass[bucket0(v[e])], (unsigned long long)w);
                }
        });
        __syncthreads();
        find_bucket(s, tid, lane, wave, reached);
        if (!s.found) return;
        const uint32_t B = s.bucket;
        uint64_t front = s.before;
        const uint64_t total = s.total;
        uint32_t lo = 0, hi = 0xffffffffu;                       // keys that the border lies between
        auto member = [&](float v, uint32_t idx) { const uint32_t k = key_of(v); return k >= lo && k <= hi && bucket0(v) == B && kept(v, idx); };
        for (;;) {
            const uint32_t n = collect(member);
            if (n <= LIST) {
                sort_list(s, n, tid);
                run_list(n, value);
                const uint32_t stay = first_reached(n, [&](uint64_t f) { return reached(front + f, total); });
                const uint64_t last = s.list[stay - 1];
                thr = (uint32_t)(last >> 32);
                lim = ~(uint32_t)last;
                __syncthreads();
                return;
            }
            if (tid == 0) { s.kmin = 0xffffffffu; s.kmax = 0; }
            __syncthreads();
            uint32_t kmin = 0xffffffffu, kmax = 0;
            all([&](uint32_t i, const float *v, uint32_t ok) {
#pragma unroll
                for (uint32_t e = 0; e < 4; e++)
                    if (((ok >> e) & 1) && member(v[e], i * STRIPE + 4 * tid + e)) { kmin = min(kmin, key_of(v[e])); kmax = max(kmax, key_of(v[e])); }
            });
            for (int o = 32; o > 0; o >>= 1) { kmin = min(kmin, __shfl_xor(kmin, o)); kmax = max(kmax, __shfl_xor(kmax, o)); }
            if (lane == 0) { atomicMin(&s.kmin, kmin); atomicMax(&s.kmax, kmax); }
            __syncthreads();
            lo = s.kmin; hi = s.kmax;
            if (lo >= hi) break;
            const uint32_t width = 32 - __clz(hi - lo), shift = width > 11 ? width - 11 : 0;
            clear_buckets();
            all([&](uint32_t i, const float *v, uint32_t ok) {
#pragma unroll
                for (uint32_t e = 0; e < 4; e++)
                    if (((ok >> e) & 1) && member(v[e], i * STRIPE + 4 * tid + e))
                        atomicAdd((unsigned long long *)&s.mass[(hi - key_of(v[e])) >> shift], (unsigned long long)(uint64_t)value(v[e]));
            });
            __syncthreads();
            find_bucket(s, tid, lane, wave, [&](uint64_t f, uint64_t) { return reached(front + f, total); });
            if (!s.found) return;                                // (cannot be: the bucket's members sum to what the level before saw)
            front += s.before;
            const uint32_t top = hi - (s.bucket << shift);
            lo = max(lo, shift ? top - ((1u << shift) - 1) : top);
            hi = top;
        }
        // more equal logits than the list holds: how many of them stay (each adds w), and the index of the last of those
        const uint32_t old_lim = hi == thr ? lim : 0xffffffffu;
        thr = hi;
        const uint64_t w = (uint64_t)value(value_of((uint64_t)thr << 32));
        uint64_t stay = 0, step = (uint64_t)1 << 18;             // the largest number that does not reach it, plus one
        for (; step; step >>= 1) if (!reached(front + (stay + step) * w, total)) stay += step;
        stay++;
        __syncthreads();
        all([&](uint32_t i, const float *v, uint32_t ok) {
            uint32_t n = 0;
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) n += ((ok >> e) & 1) && key_of(v[e]) == thr && i * STRIPE + 4 * tid + e <= old_lim;
            for (int o = 32; o > 0; o >>= 1) n += __shfl_xor(n, o);
            if (lane == 0) s.part[i * WAVES + wave] = n;
        });
        __syncthreads();
        const uint64_t n = tid < stripes * WAVES ? s.part[tid] : 0, incl = block_scan(n, s, lane, wave);
        if (tid == 0) s.found = 0xffffffffu;
        __syncthreads();
        if (incl >= stay && incl - n < stay) { s.found = tid; s.before = incl - n; }
        __syncthreads();
        const uint32_t at = s.found;
        if (at != 0xffffffffu && wave == 0) {                   // the wave's 256 logits again, in order
            float v[4];
            uint32_t ok = fetch(at / WAVES, (at % WAVES) * 64 + lane, v), mine = 0;
            const uint32_t idx = at / WAVES * STRIPE + 4 * ((at % WAVES) * 64 + lane);
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) { if (key_of(v[e]) != thr || idx + e > old_lim) ok &= ~(1u << e); mine += (ok >> e) & 1; }
            const uint32_t rank = wave_scan(mine, lane) - mine, want = (uint32_t)(stay - s.before);
            if (rank < want && rank + mine >= want) {
                uint32_t left = want - rank;
#pragma unroll
                for (uint32_t e = 0; e < 4; e++) if (((ok >> e) & 1) && --left == 0) s.bucket = idx + e;
            }
        }
        __syncthreads();
        lim = at != 0xffffffffu ? min(old_lim, s.bucket) : old_lim;
        __syncthreads();
    };
    // (a prefix of mass f is long enough; an empty one never is)
    const double p = (double)fmaxf(top_p, 0.f);
    auto enough = [&](uint64_t f, uint64_t total) { return f > 0 && (double)f >= p * (double)total; };
    uint32_t listed = 0;                                         // > 0: the kept tokens, and no others, are the first `listed` of the sorted list
    if (top_k > 0 && (uint32_t)top_k < V) {
        const uint64_t k = (uint64_t)top_k;
        // k of the threads' largest logits are at least as large as what bucket B holds: so are the k largest of the row
        uint32_t n = LIST + 1;
        if (k <= THREADS / 2) {
            clear_buckets();
            if (own_mz > NINF) atomicAdd((unsigned long long *)&s.mass[bucket0(own_mz)], 1ull);
            __syncthreads();
            find_bucket(s, tid, lane, wave, [&](uint64_t f, uint64_t) { return f >= k; });
            const uint32_t B = s.found ? s.bucket : BUCKETS - 1;
            n = collect([&](float v, uint32_t) { return bucket0(v) <= B; });
        }
        if (n <= LIST) {
            sort_list(s, n, tid);
            listed = min(n, (uint32_t)k);
        } else {
            shorten(one, [&](uint64_t f, uint64_t) { return f >= k; });
        }
    }
    if (top_p < 1.f) {
        if (listed) {
            run_list(listed, weigh);
            const uint64_t total = s.run[listed - 1];
            listed = first_reached(listed, [&](uint64_t f) { return enough(f, total); });
        } else {
            shorten(weigh, enough);
        }
    }
    // a draw's place in the running weights: floor(u * total)
    auto target_of = [&](uint32_t d, uint64_t total) {
        const float u = a.u[(uint64_t)row * a.draws + d];
        const double uc = u > 0.f ? fmin((double)u, 1.0 - 1.0 / 16777216) : 0.0;
        const uint64_t u63 = (uint64_t)(uc * 9223372036854775808.0);
        return (__umul64hi(u63, total) << 1) | ((u63 * total) >> 63);
    };
    auto put = [&](uint32_t d, uint32_t idx, float v) {
        a.tokens[(uint64_t)row * a.draws + d] = idx;
        a.logprobs[(uint64_t)row * a.draws + d] = (float)((double)v - lse);
    };
    auto floored = [&](float v) { const double w = weigh(v); return w >= floor_w ? w : 0.0; };
    if (listed) {
        // into the order of the vocabulary: (~index << 32 | key) falls as the index rises
        __syncthreads();
        for (uint32_t i = tid; i < listed; i += THREADS) s.list[i] = (s.list[i] << 32) | (s.list[i] >> 32);
        sort_list(s, listed, tid);
        for (uint32_t i = tid; i < listed; i += THREADS) s.list[i] = (s.list[i] << 32) | (s.list[i] >> 32);
        __syncthreads();
        run_list(listed, floored);
        const uint64_t total = s.run[listed - 1];
        for (uint32_t d = tid; d < a.draws; d += THREADS) {
            const uint64_t target = target_of(d, total);
            uint32_t lo = 0, hi = listed - 1;
            while (lo < hi) { const uint32_t mid = (lo + hi) / 2; if (s.run[mid] > target) hi = mid; else lo = mid + 1; }
            put(d, ~(uint32_t)s.list[lo], value_of(s.list[lo]));
        }
        return;
    }
    // the weights of what is left, summed for every 256 tokens (a logit below `reach` has none: less than min_p of the largest weight, or 2^-45)
    const float reach = mz - temperature * fminf(31.5f, floor_w > 0.0 ? 1e-3f - 0.69314718f * __builtin_amdgcn_logf(fminf(min_p_, 1.f)) : 31.5f) * 1.00001f;
    auto final_weight = [&](float v, uint32_t idx, uint32_t ok) -> uint64_t { return ok && !(v < reach) && kept(v, idx) ? (uint64_t)floored(v) : 0; };
    __syncthreads();
    all([&](uint32_t i, const float *v, uint32_t ok) {
        uint64_t w = 0;
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) w += final_weight(v[e], i * STRIPE + 4 * tid + e, (ok >> e) & 1);
        if (__any(w != 0))
            for (int o = 32; o > 0; o >>= 1) w += __shfl_xor(w, o);
        if (lane == 0) s.part[i * WAVES + wave] = w;
    });
    __syncthreads();
    const uint32_t parts = stripes * WAVES;
    const uint64_t incl = block_scan(tid < parts ? s.part[tid] : 0, s, lane, wave);
    if (tid < parts) s.part[tid] = incl;
    __syncthreads();
    const uint64_t total = s.part[parts - 1];
    for (uint32_t d = wave; d < a.draws; d += WAVES) {
        const uint64_t target = target_of(d, total);
        uint32_t lo = 0, hi = parts - 1;                         // the first part whose running sum passes the target
        while (lo < hi) { const uint32_t mid = (lo + hi) / 2; if (s.part[mid] > target) hi = mid; else lo = mid + 1; }
        const uint64_t rest = target - (lo ? s.part[lo - 1] : 0);
        float v[4];
        const uint32_t t = (lo % WAVES) * 64 + lane, ok = fetch(lo / WAVES, t, v), idx = lo / WAVES * STRIPE + 4 * t;
        uint64_t w[4], mine = 0;
#pragma unroll
        for (uint32_t e = 0; e < 4; e++) { w[e] = final_weight(v[e], idx + e, (ok >> e) & 1); mine += w[e]; }
        const uint64_t sum = wave_scan(mine, lane);
        if (sum > rest && sum - mine <= rest) {
            uint64_t run = sum - mine;
            bool done = false;
#pragma unroll
            for (uint32_t e = 0; e < 4; e++) {
                run += w[e];
                if (!done && run > rest) { done = true; put(d, idx + e, v[e]); }
            }
        }
    }
}

template <typename T>
static int sample_tokens(void *stream, const SampleArgs &a)
{
    if (!a.rows || !a.draws) return FMI_OK;
    if (!a.vocab || a.vocab > MAX_VOCAB) { fmi_set_error("sealnn_sample_tokens: a vocabulary of %u (1 .. %u)", a.vocab, (unsigned)MAX_VOCAB); return FMI_ERR_UNSUPPORTED; }
    if (!a.logits || !a.u || !a.tokens || !a.logprobs || ((uintptr_t)a.logits & (sizeof(T) - 1))) { fmi_set_error("sealnn_sample_tokens: null or misaligned argument"); return FMI_ERR_ARG; }
    hipLaunchKernelGGL(k_sample_tokens<T>, dim3(a.rows), dim3(THREADS), 0, (hipStream_t)stream, a);
    NNCHK();
    return FMI_OK;
}

static SampleArgs sample_args(const void *logits, uint64_t row_stride, uint32_t rows, uint32_t vocab, const float *u, uint32_t draws, const uint32_t *bits,
                              uint64_t bits_stride, float temperature, int32_t top_k, float top_p, float min_p, const float *temperature_v,
                              const int32_t *top_k_v, const float *top_p_v, const float *min_p_v, int64_t *tokens, float *logprobs)
{
    SampleArgs a;
    a.logits = logits; a.row_stride = row_stride; a.bits = bits; a.bits_stride = bits_stride; a.u = u;
    a.temperature_v = temperature_v; a.top_p_v = top_p_v; a.min_p_v = min_p_v; a.top_k_v = top_k_v;
    a.rows = rows; a.vocab = vocab; a.draws = draws; a.temperature = temperature; a.top_p = top_p; a.min_p = min_p; a.top_k = top_k;
    a.tokens = tokens; a.logprobs = logprobs;
    return a;
}

extern "C" int sealnn_sample_tokens(void *stream, const float *logits, uint64_t row_stride, uint32_t rows, uint32_t vocab, const float *u, uint32_t draws,
                                    const uint32_t *bits, uint64_t bits_stride, float temperature, int32_t top_k, float top_p, float min_p,
                                    const float *temperature_v, const int32_t *top_k_v, const float *top_p_v, const float *min_p_v, int64_t *tokens, float *logprobs)
{ return sample_tokens<float>(stream, sample_args(logits, row_stride, rows, vocab, u, draws, bits, bits_stride, temperature, top_k, top_p, min_p, temperature_v, top_k_v, top_p_v, min_p_v, tokens, logprobs)); }
extern "C" int sealnn_sample_tokens_bf16(void *stream, const void *logits, uint64_t row_stride, uint32_t rows, uint32_t vocab, const float *u, uint32_t draws,
                                         const uint32_t *bits, uint64_t bits_stride, float temperature, int32_t top_k, float top_p, float min_p,
                                         const float *temperature_v, const int32_t *top_k_v, const float *top_p_v, const float *min_p_v, int64_t *tokens, float *logprobs)
{ return sample_tokens<bf16>(stream, sample_args(logits, row_stride, rows, vocab, u, draws, bits, bits_stride, temperature, top_k, top_p, min_p, temperature_v, top_k_v, top_p_v, min_p_v, tokens, logprobs)); }
