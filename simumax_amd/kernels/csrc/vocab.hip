// Operators over the rows of a language model's logits, gfx950:
//   * log probabilities of given tokens, with each row's entropy and its top
//     alternatives, and the gradient of the logits;
//   * the divergence of a student from a teacher's top log probabilities,
//     and the gradient of the logits.
// Logits are bf16, fp16 or fp32, [rows, V] with any row strides; every sum,
// maximum and statistic is held in 32 bits or more.
//
// z = x / T, c = log2(e) / T. With m the largest x of a stretch and mc = m*c:
//   s = sum 2^(x*c - mc),  t = sum (x*c - mc) 2^(x*c - mc)
// so that  lse = m/T + ln s  and  H = ln s - ln 2 * t / s  (t <= 0: no
// cancellation). Stretches join by s = sum s_i f_i, t = sum (t_i + d_i s_i)
// f_i with d_i = (m_i - m) c and f_i = 2^d_i.
//
// Three launches, none of which synchronises with the host:
//   partials: one wave per 16-byte x 64 lanes x 8 stretch of a row, held in
//             registers: one read for the maximum and the sums;
//   join:     one workgroup per row: statistics, top alternatives, loss;
//   grad:     one wave per stretch again: p from the statistics, plus what
//             the given tokens or the teacher's entries add.
// No floating-point atomics: the same input gives the same bits.
#include <hip/hip_fp16.h>

#include "common.h"
#include "vocab.h"

#define BLOCK 256
#define WAVES (BLOCK / WAVE)
#define NVEC 8  // 16-byte vectors per lane and stretch

typedef unsigned int u32;
typedef unsigned long long u64;

// ---- element types: 16 bytes at any element boundary -----------------------
// Rows of an odd vocabulary start at any multiple of the element's size, so
// vectors are loaded and stored with that alignment (one unaligned 16-byte
// access each).
template <typename T> struct Elem;

template <> struct Elem<__hip_bfloat16> {
    static constexpr int N = 8;
    static DEV float get(u32 w, int half) {
        return __uint_as_float(half ? (w & 0xffff0000u) : (w << 16));
    }
    static DEV u32 put(float a, float b) {
        return (u32)f2bf(a) | ((u32)f2bf(b) << 16);
    }
};
template <> struct Elem<__half> {
    static constexpr int N = 8;
    static DEV float get(u32 w, int half) {
        return __half2float(__ushort_as_half((unsigned short)(half ? w >> 16 : w)));
    }
    static DEV u32 put(float a, float b) {
        return (u32)__half_as_ushort(__float2half(a)) |
               ((u32)__half_as_ushort(__float2half(b)) << 16);
    }
};
template <> struct Elem<float> {
    static constexpr int N = 4;
};

DEV float to_f(float v) { return v; }
DEV float to_f(__half v) { return __half2float(v); }
DEV float to_f(__hip_bfloat16 v) { return __bfloat162float(v); }
template <typename T> DEV T from_f(float v);
template <> DEV float from_f<float>(float v) { return v; }
template <> DEV __half from_f<__half>(float v) { return __float2half(v); }
template <> DEV __hip_bfloat16 from_f<__hip_bfloat16>(float v) {
    return __float2bfloat16(v);
}

template <typename T> struct Vec {
    static constexpr int N = Elem<T>::N;
    u32 w[4];
    DEV float get(int i) const {
        if constexpr (sizeof(T) == 4) return __uint_as_float(w[i]);
        else return Elem<T>::get(w[i >> 1], i & 1);
    }
    DEV void put(int i, float a, float b) {  // elements i and i + 1
        if constexpr (sizeof(T) == 4) {
            w[i] = __float_as_uint(a);
            w[i + 1] = __float_as_uint(b);
        } else {
            w[i >> 1] = Elem<T>::put(a, b);
        }
    }
};

// `at` counts elements from the row's start; lanes past its end see -inf
template <typename T>
DEV Vec<T> load_vec(const T *row, long at, long V) {
    constexpr int N = Vec<T>::N;
    Vec<T> v;
    if (at + N <= V) {
        __builtin_memcpy(v.w, row + at, 16);
    } else {
        float f[N];
#pragma unroll
        for (int i = 0; i < N; ++i)
            f[i] = at + i < V ? to_f(row[at + i]) : -INFINITY;
#pragma unroll
        for (int i = 0; i < N; i += 2) v.put(i, f[i], f[i + 1]);
    }
    return v;
}

template <typename T>
DEV void store_vec(T *row, long at, long V, const float *f) {
    constexpr int N = Vec<T>::N;
    if (at + N <= V) {
        Vec<T> v;
#pragma unroll
        for (int i = 0; i < N; i += 2) v.put(i, f[i], f[i + 1]);
        __builtin_memcpy(row + at, v.w, 16);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at + i < V) row[at + i] = from_f<T>(f[i]);
    }
}

template <typename T>
DEV const T *row_ptr(const VocabRows &g, int r) {
    const int o = r / g.inner, i = r - o * g.inner;
    return (const T *)g.base + (long)o * g.stride_o + (long)i * g.stride_i;
}

// orders a wave's LDS accesses; the hardware keeps a wave's own in order, so
// no instruction comes of it
DEV void wave_sync() {
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
}

DEV float exp2_hw(float v) { return __builtin_amdgcn_exp2f(v); }

// (x - m) in units of the exponent. The product form is exact against its
// own reference mc, which is off m*c by half a step; where that is no small
// part of the exponent (logits at a type's lowest or highest value) the
// difference is taken first.
DEV bool by_product(float mc) { return fabsf(mc) < 0x1p20f; }

// Not below -300: 2^-300 is 0 and (-inf) * 0 would be NaN.
DEV float diff2_safe(float x, float m, float mc, float c) {
    float d = by_product(mc) ? fmaf(x, c, -mc) : (x - m) * c;
    return d < -300.f ? -300.f : d;
}

DEV double block_sum_d(double v, double *lds) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) v += __shfl_xor(v, off, WAVE);
    __syncthreads();
    if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = v;
    __syncthreads();
    double r = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) r += lds[w];
    return r;
}

// ---- partials --------------------------------------------------------------
// One wave per stretch. Writes (m, s, t, s_in): s_in is the part of the sum
// that belongs to the teacher's entries (EXCL), and s then leaves it out:
// the rest of the mass is summed, not got as a difference, because a
// student that has learned leaves little of it.
template <typename T, bool ENT, bool EXCL>
__global__ __launch_bounds__(BLOCK) void vocab_partials(
    VocabRows g, const long *__restrict__ tokens, long ignore,
    const long *__restrict__ ids, int K, float c, float4 *__restrict__ part) {
    constexpr int N = Vec<T>::N;
    constexpr int SEG = WAVE * NVEC * N;
    __shared__ u32 bits[EXCL ? WAVES : 1][EXCL ? SEG / 32 : 1];
    const int lane = threadIdx.x % WAVE, wid = threadIdx.x / WAVE;
    const long total = (long)g.rows * g.nseg;
    for (long w = (long)blockIdx.x * WAVES + wid; w < total;
         w += (long)gridDim.x * WAVES) {
        const int r = (int)(w / g.nseg), seg = (int)(w - (long)r * g.nseg);
        if (tokens && tokens[r] == ignore) continue;
        const T *row = row_ptr<T>(g, r);
        const long lo = (long)seg * SEG;
        if (EXCL) {
            for (int i = lane; i < SEG / 32; i += WAVE) bits[wid][i] = 0;
            wave_sync();
            for (int k = lane; k < K; k += WAVE) {
                const long at = ids[(long)r * K + k] - lo;
                if (at >= 0 && at < SEG)
                    atomicOr(&bits[wid][at >> 5], 1u << (at & 31));
            }
            wave_sync();
        }
        Vec<T> v[NVEC];
#pragma unroll
        for (int j = 0; j < NVEC; ++j)
            v[j] = load_vec(row, lo + (long)(j * WAVE + lane) * N, g.V);
        float m = -INFINITY;
#pragma unroll
        for (int j = 0; j < NVEC; ++j)
#pragma unroll
            for (int i = 0; i < N; ++i) m = fmaxf(m, v[j].get(i));
        m = wave_max(m);
        const float mr = m == -INFINITY ? 0.f : m, mc = mr * c;
        float s = 0.f, t = 0.f, s_in = 0.f;
#pragma unroll
        for (int j = 0; j < NVEC; ++j) {
            u32 in = 0;
            if (EXCL) {
                const int at = (j * WAVE + lane) * N;
                in = (bits[wid][at >> 5] >> (at & 31)) & ((1u << N) - 1);
            }
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float d = diff2_safe(v[j].get(i), mr, mc, c);
                const float e = exp2_hw(d);
                if (EXCL && (in >> i & 1)) s_in += e;
                else s += e;
                if (ENT) t = fmaf(d, e, t);
            }
        }
        s = wave_sum(s);
        if (ENT) t = wave_sum(t);
        if (EXCL) s_in = wave_sum(s_in);
        if (lane == 0) part[w] = make_float4(m, s, t, s_in);
    }
}

// ---- join ------------------------------------------------------------------
struct RowStat {
    float m;           // largest logit, 0 where there is none
    double s, t, s_in; // against m*c itself
    double delta;      // m*c less its rounded value: 2^(x*c - mc) is
                       // 2^delta times too large
};

// every thread gets the row's statistics; sums in a fixed order, in 64 bits
DEV RowStat join_parts(const float4 *p, int nseg, float c, double *lds) {
    __shared__ float redm[WAVES];
    float m = -INFINITY;
    for (int i = threadIdx.x; i < nseg; i += BLOCK) m = fmaxf(m, p[i].x);
    m = block_max<BLOCK>(m, redm);
    RowStat st;
    st.m = m == -INFINITY ? 0.f : m;
    const float mc = st.m * c;
    const double exact = (double)st.m * c;
    st.delta = by_product(mc) ? exact - mc : 0.;
    double s = 0, t = 0, s_in = 0;
    for (int i = threadIdx.x; i < nseg; i += BLOCK) {
        const float4 q = p[i];
        const float qm = q.x == -INFINITY ? 0.f : q.x;
        // against each stretch's own rounded reference, where there is one
        const float qc = qm * c;
        double d = (by_product(qc) ? (double)qc : (double)qm * c) - exact;
        // adds nothing, but NaN stays NaN
        if (q.x == -INFINITY || d < -300) d = -300;
        const double f = exp2(d);
        s += q.y * f;
        s_in += q.w * f;
        t += (q.z + d * ((double)q.y + q.w)) * f;
    }
    st.s = block_sum_d(s, lds);
    st.s_in = block_sum_d(s_in, lds);
    st.t = block_sum_d(t, lds);
    return st;
}

// order of 32-bit floats as whole numbers; -0 counts as 0
DEV u32 order_of(float x) {
    const u32 b = __float_as_uint(x + 0.f);
    return b & 0x80000000u ? ~b : b | 0x80000000u;
}

DEV u64 block_max_u64(u64 v, u64 *lds) {
#pragma unroll
    for (int off = 32; off > 0; off >>= 1) {
        const u64 o = __shfl_xor(v, off, WAVE);
        v = o > v ? o : v;
    }
    __syncthreads();
    if (threadIdx.x % WAVE == 0) lds[threadIdx.x / WAVE] = v;
    __syncthreads();
    u64 r = lds[0];
#pragma unroll
    for (int w = 1; w < WAVES; ++w) r = lds[w] > r ? lds[w] : r;
    return r;
}

// stat[r] = (m, 1/s, H - ln s, 0) against the rounded m*c, what the gradient
// needs; 1/s is 0 where the row has no finite logit
template <typename T>
__global__ __launch_bounds__(BLOCK) void logprobs_join(
    VocabRows g, const float4 *__restrict__ part,
    const long *__restrict__ tokens, long ignore, int K, float c, double inv_t,
    float *__restrict__ logprobs, float *__restrict__ entropy,
    float *__restrict__ top_lp, long *__restrict__ top_ids,
    float4 *__restrict__ stat) {
    __shared__ double lds[WAVES];
    __shared__ u64 lds_k[WAVES];
    const float NEG = -INFINITY;
    for (int r = blockIdx.x; r < g.rows; r += gridDim.x) {
        const long tok = tokens ? tokens[r] : 0;
        if (tokens && tok == ignore) {
            if (threadIdx.x == 0) {
                logprobs[r] = 0.f;
                entropy[r] = 0.f;
                stat[r] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            for (int k = threadIdx.x; k < K; k += BLOCK) {
                top_lp[(long)r * K + k] = 0.f;
                top_ids[(long)r * K + k] = -1;
            }
            continue;
        }
        const T *row = row_ptr<T>(g, r);
        const RowStat st = join_parts(part + (long)r * g.nseg, g.nseg, c, lds);
        const bool none = st.s == 0, bad = !(st.s < INFINITY);
        const double ln_s = log(st.s);
        const float H = none ? 0.f
                        : bad ? NAN
                              : (float)(ln_s - 0.6931471805599453 * st.t / st.s);
        if (threadIdx.x == 0) {
            if (tokens) {
                float lp = NAN;
                if (tok >= 0 && tok < g.V && !bad)
                    lp = none ? NEG
                              : (float)(((double)to_f(row[tok]) - st.m) * inv_t -
                                        ln_s);
                logprobs[r] = lp;
            }
            entropy[r] = H;
            stat[r] = make_float4(
                st.m, none ? 0.f : (float)(exp2(-st.delta) / st.s),
                none ? 0.f
                     : (float)(-0.6931471805599453 *
                               (st.t / st.s + st.delta)),
                0.f);
        }
        u64 last = ~0ull;
        for (int k = 0; k < K; ++k) {
            u64 best = 0;
            for (long i = threadIdx.x; i < g.V; i += BLOCK) {
                const u64 key = (u64)order_of(to_f(row[i])) << 32 |
                                (0xffffffffu - (u32)i);
                if (key < last && key > best) best = key;
            }
            best = block_max_u64(best, lds_k);
            last = best;
            if (threadIdx.x == 0) {
                const u32 i = 0xffffffffu - (u32)best;
                const float x = to_f(row[i < g.V ? i : 0]);
                top_lp[(long)r * K + k] =
                    bad ? NAN
                        : none ? NEG
                               : (float)(((double)x - st.m) * inv_t - ln_s);
                top_ids[(long)r * K + k] = bad ? -1 : (long)i;
            }
        }
        __syncthreads();
    }
}

// stat[r] = (m, 1/s, a_in, a_out): the gradient of a student's logit is
// p_j a_in - sum of its q  inside the teacher's entries, p_j a_out outside.
// Both 0 mark a row without entries. q [rows, K] is kept for the gradient.
template <typename T>
__global__ __launch_bounds__(BLOCK) void distill_join(
    VocabRows g, const float4 *__restrict__ part,
    const float *__restrict__ tlp, const long *__restrict__ ids, int K,
    int bucket, float c, double inv_t, float *__restrict__ loss,
    float *__restrict__ q_out, float4 *__restrict__ stat) {
    __shared__ double lds[WAVES];
    for (int r = blockIdx.x; r < g.rows; r += gridDim.x) {
        const T *row = row_ptr<T>(g, r);
        // K <= BLOCK: one entry per thread
        const bool held = (int)threadIdx.x < K &&
                          ids[(long)r * K + threadIdx.x] >= 0;
        const long id = held ? ids[(long)r * K + threadIdx.x] : 0;
        const double l = held ? (double)tlp[(long)r * K + threadIdx.x] : 0.;
        double q = held ? exp(l) : 0.;
        const bool wrong = held && id >= g.V;
        const int any = __syncthreads_or(held ? 1 : 0);
        const int err = __syncthreads_or(wrong ? 1 : 0);
        double total = block_sum_d(q, lds);
        double q_rest = 0., log_norm = 0., mass;
        if (bucket) {
            q_rest = total < 1. ? 1. - total : 0.;
            mass = total + q_rest;
        } else {
            // not `total > 0`: NaN has to stay NaN
            log_norm = total == 0. ? 0. : log(total);
            q = total == 0. ? 0. : q / total;
            mass = total == 0. ? 0. : total / total;
        }
        if ((int)threadIdx.x < K) q_out[(long)r * K + threadIdx.x] = (float)q;
        if (!any || (!bucket && total == 0.)) {
            if (threadIdx.x == 0) {
                loss[r] = 0.f;
                stat[r] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            continue;
        }
        const RowStat st = join_parts(part + (long)r * g.nseg, g.nseg, c, lds);
        const double s = st.s + st.s_in;
        const bool none = s == 0, bad = !(s < INFINITY);
        const double ln_s = log(s);
        double term = 0.;
        if (held && !wrong && q != 0.) {
            const double x = (double)to_f(row[id]);
            const double lp = none || x == -INFINITY
                                  ? -INFINITY
                                  : (x - st.m) * inv_t - ln_s;
            term = q * ((l - log_norm) - lp);
        }
        double sum = block_sum_d(term, lds);
        double ratio = 0.;
        if (bucket && q_rest > 0.) {
            // entries that cover every token with mass leave no room for
            // the rest; what 32-bit log probabilities leave over by
            // rounding then counts as none
            const double p_rest = none ? 0. : st.s / s;
            if (p_rest > 0.) {
                sum += q_rest * (log(q_rest) - log(p_rest));
                ratio = q_rest / p_rest;
            } else if (q_rest > 0x1p-20) {
                sum = INFINITY;
            }
        }
        if (threadIdx.x == 0) {
            const bool nan = bad || err;
            loss[r] = nan ? NAN : (float)sum;
            stat[r] = make_float4(st.m,
                                  none ? 0.f : (float)(exp2(-st.delta) / s),
                                  nan ? NAN : (float)mass,
                                  nan ? NAN : (float)(mass - ratio));
        }
        __syncthreads();
    }
}

// ---- gradients -------------------------------------------------------------
// d x_j = p_j (a + b ln(p_j s)) + what is given for single tokens, one wave per
// stretch. Single tokens: a list of at most K entries of the row that fall
// into this stretch, compacted into LDS in the row's order, with one bit per
// element so that the rest of the stretch never looks at it. The same token
// given twice is added twice, in order.
template <typename T, bool DISTILL>
__global__ __launch_bounds__(BLOCK) void vocab_grad(
    VocabRows g, VocabGrad a, T *__restrict__ out) {
    constexpr int N = Vec<T>::N;
    constexpr int SEG = WAVE * NVEC * N;
    __shared__ u32 bits[WAVES][SEG / 32];
    __shared__ int list_at[WAVES][VOCAB_MAX_K + 1];
    __shared__ float list_val[WAVES][VOCAB_MAX_K + 1];
    const int lane = threadIdx.x % WAVE, wid = threadIdx.x / WAVE;
    const long total = (long)g.rows * g.nseg;
    for (long w = (long)blockIdx.x * WAVES + wid; w < total;
         w += (long)gridDim.x * WAVES) {
        const int r = (int)(w / g.nseg), seg = (int)(w - (long)r * g.nseg);
        const long lo = (long)seg * SEG;
        T *orow = out + (long)r * g.V;
        const float4 st = a.stat[r];
        bool skip = st.y == 0.f;
        if (DISTILL) skip = skip || (st.z == 0.f && st.w == 0.f);
        const long tok = !DISTILL && a.tokens ? a.tokens[r] : -1;
        if (!DISTILL && a.tokens && tok == a.ignore) skip = true;
        if (skip) {
            float zero[N] = {};
#pragma unroll
            for (int j = 0; j < NVEC; ++j) {
                const long at = lo + (long)(j * WAVE + lane) * N;
                store_vec(orow, at, g.V, zero);
            }
            continue;
        }
        for (int i = lane; i < SEG / 32; i += WAVE) bits[wid][i] = 0;
        wave_sync();
        // coefficients of p_j: a_in for listed tokens, a_out for the others
        float a_in, a_out, b = 0.f, scale = a.inv_t;
        int n = 0;
        if (DISTILL) {
            scale *= a.d_row[r];
            a_in = st.z;
            a_out = st.w;
        } else {
            float gs = 0.f;
            if (a.d_row && a.tokens) {
                const float gr = a.d_row[r];
                gs = tok >= 0 && tok < g.V ? gr : NAN;
                const long at = tok - lo;
                if (at >= 0 && at < SEG) {
                    if (lane == 0) {
                        bits[wid][at >> 5] |= 1u << (at & 31);
                        list_at[wid][0] = (int)at;
                        list_val[wid][0] = gr;
                    }
                    n = 1;
                }
            }
            float gk = 0.f;
            if (a.d_top)
                for (int k = lane; k < a.K; k += WAVE)
                    gk += a.d_top[(long)r * a.K + k];
            gs += wave_sum(gk);
            if (a.d_entropy) b = -a.d_entropy[r];
            a_in = a_out = b * st.z - gs;
        }
        wave_sync();
        const float *vals = DISTILL ? a.q : a.d_top;
        if (vals) {
            for (int k0 = 0; k0 < a.K; k0 += WAVE) {
                const int k = k0 + lane;
                const long at = k < a.K ? a.ids[(long)r * a.K + k] - lo : -1;
                const bool mine = at >= 0 && at < SEG && at + lo < g.V;
                const u64 who = __ballot(mine);
                if (mine) {
                    const int slot =
                        n + __popcll(who & ((1ull << lane) - 1));
                    const float val = vals[(long)r * a.K + k];
                    list_at[wid][slot] = (int)at;
                    list_val[wid][slot] = DISTILL ? -val : val;
                    atomicOr(&bits[wid][at >> 5], 1u << (at & 31));
                }
                n += __popcll(who);
            }
        }
        wave_sync();
        const T *row = row_ptr<T>(g, r);
        Vec<T> v[NVEC];
#pragma unroll
        for (int j = 0; j < NVEC; ++j)
            v[j] = load_vec(row, lo + (long)(j * WAVE + lane) * N, g.V);
        const float mc = st.x * a.c;
#pragma unroll
        for (int j = 0; j < NVEC; ++j) {
            const int at = (j * WAVE + lane) * N;
            const u32 in =
                (bits[wid][at >> 5] >> (at & 31)) & ((1u << N) - 1);
            float f[N];
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const float d = diff2_safe(v[j].get(i), st.x, mc, a.c);
                const float p = exp2_hw(d) * st.y;
                float k = a_out;
                if (!DISTILL) k = fmaf(b * 0.69314718f, d, k);
                else if (in >> i & 1) k = a_in;
                f[i] = p * k;
            }
            if (in) {
#pragma unroll
                for (int i = 0; i < N; ++i)
                    if (in >> i & 1)
                        for (int e = 0; e < n; ++e)
                            if (list_at[wid][e] == at + i)
                                f[i] += list_val[wid][e];
            }
#pragma unroll
            for (int i = 0; i < N; ++i) f[i] *= scale;
            store_vec(orow, lo + at, g.V, f);
        }
        wave_sync();
    }
}

// ---- launches --------------------------------------------------------------
// grids are capped so that threads stay far below 2^32; waves then stride
static int wave_grid(const VocabRows &g) {
    const long blocks = CDIV((long)g.rows * g.nseg, (long)WAVES);
    return (int)(blocks < (1l << 22) ? blocks : (1l << 22));
}
static int row_grid(const VocabRows &g) {
    return g.rows < (1 << 22) ? g.rows : (1 << 22);
}

template <typename T>
static void logprobs_fwd_t(const VocabRows &g, const VocabLogprobs &a,
                           hipStream_t stream) {
    const float c = (float)(1.4426950408889634 / a.temperature);
    hipLaunchKernelGGL((vocab_partials<T, true, false>), dim3(wave_grid(g)),
                       dim3(BLOCK), 0, stream, g, a.tokens, a.ignore, nullptr,
                       0, c, (float4 *)a.part);
    hipLaunchKernelGGL((logprobs_join<T>), dim3(row_grid(g)), dim3(BLOCK), 0,
                       stream, g, (const float4 *)a.part, a.tokens, a.ignore,
                       a.K, c, 1. / a.temperature, a.logprobs, a.entropy,
                       a.top_lp, a.top_ids, (float4 *)a.stat);
}

template <typename T>
static void distill_fwd_t(const VocabRows &g, const VocabDistill &a,
                          hipStream_t stream) {
    const float c = (float)(1.4426950408889634 / a.temperature);
    if (a.bucket)
        hipLaunchKernelGGL((vocab_partials<T, false, true>),
                           dim3(wave_grid(g)), dim3(BLOCK), 0, stream, g,
                           nullptr, 0, a.ids, a.K, c, (float4 *)a.part);
    else
        hipLaunchKernelGGL((vocab_partials<T, false, false>),
                           dim3(wave_grid(g)), dim3(BLOCK), 0, stream, g,
                           nullptr, 0, nullptr, 0, c, (float4 *)a.part);
    hipLaunchKernelGGL((distill_join<T>), dim3(row_grid(g)), dim3(BLOCK), 0,
                       stream, g, (const float4 *)a.part, a.teacher_lp, a.ids,
                       a.K, a.bucket, c, 1. / a.temperature, a.loss, a.q,
                       (float4 *)a.stat);
}

template <typename T>
static void grad_t(const VocabRows &g, const VocabGrad &a, int distill,
                   void *out, hipStream_t stream) {
    if (distill)
        hipLaunchKernelGGL((vocab_grad<T, true>), dim3(wave_grid(g)),
                           dim3(BLOCK), 0, stream, g, a, (T *)out);
    else
        hipLaunchKernelGGL((vocab_grad<T, false>), dim3(wave_grid(g)),
                           dim3(BLOCK), 0, stream, g, a, (T *)out);
}

extern "C" int vocab_segment(int dtype) {
    return WAVE * NVEC * (dtype == VOCAB_FP32 ? 4 : 8);
}

extern "C" void logprobs_fwd_launch(const VocabRows *g, const VocabLogprobs *a,
                                    int dtype, hipStream_t stream) {
    if (dtype == VOCAB_BF16) logprobs_fwd_t<__hip_bfloat16>(*g, *a, stream);
    else if (dtype == VOCAB_FP16) logprobs_fwd_t<__half>(*g, *a, stream);
    else logprobs_fwd_t<float>(*g, *a, stream);
}

extern "C" void distill_fwd_launch(const VocabRows *g, const VocabDistill *a,
                                   int dtype, hipStream_t stream) {
    if (dtype == VOCAB_BF16) distill_fwd_t<__hip_bfloat16>(*g, *a, stream);
    else if (dtype == VOCAB_FP16) distill_fwd_t<__half>(*g, *a, stream);
    else distill_fwd_t<float>(*g, *a, stream);
}

extern "C" void vocab_grad_launch(const VocabRows *g, const VocabGrad *a,
                                  int distill, void *out, int dtype,
                                  hipStream_t stream) {
    if (dtype == VOCAB_BF16) grad_t<__hip_bfloat16>(*g, *a, distill, out, stream);
    else if (dtype == VOCAB_FP16) grad_t<__half>(*g, *a, distill, out, stream);
    else grad_t<float>(*g, *a, distill, out, stream);
}
