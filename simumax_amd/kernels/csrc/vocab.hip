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
//   join:     one wave per row (one workgroup where top alternatives are
//             asked): statistics, loss;
//   grad:     one wave per stretch again: p from the statistics, plus what
//             the given tokens or the teacher's entries add.
// No floating-point atomics: the same input gives the same bits.
#include <hip/hip_fp16.h>

#include <type_traits>

#include "common.h"
#include "vocab.h"

#define BLOCK 256
#define WAVES (BLOCK / WAVE)
#define NVEC 8    // 16-byte vectors per lane and stretch
#define GROUP 64  // tokens per maximum kept for the top alternatives
#define CAP 512   // candidates for them that are ranked at once

typedef unsigned int u32;
typedef unsigned long long u64;

// ---- element types: 16 bytes at any element boundary -----------------------
// Rows of an odd vocabulary start at any multiple of the element's size, so
// vectors are loaded and stored with that alignment: one 16-byte access each,
// which the hardware takes at any address. Loads and stores of whole
// stretches are non-temporal: every byte is used once (read alone, 8192 rows
// of 128384 bf16: 6.9 TB/s, against 6.3 with ordinary loads; copied 5.5
// against 5.2).
typedef u32 u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_mem __attribute__((aligned(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Vec {
    static constexpr int N = 16 / sizeof(T);
    u32x4 w;

    DEV void load(const T *p) { w = *(const u32x4_mem *)p; }
    DEV void stream_in(const T *p) {
        w = __builtin_nontemporal_load((const u32x4_mem *)p);
    }
    DEV void stream_out(T *p) const {
        __builtin_nontemporal_store(w, (u32x4_mem *)p);
    }
    DEV float get(int i) const;
    DEV void put(int i, float a, float b);  // elements i and i + 1, i even
    // Largest and smallest bit pattern, as signed and unsigned numbers: of
    // floats of which one at least is not negative the first is the largest
    // float, of negative floats the second is. Packed, a half operation per
    // 16-bit element, and no unpacking.
    DEV void widen(s16x2 &hi, u16x2 &lo) const {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            const u32 x = w[k];  // a bit cast of w[k] itself reads w[0]
            hi = __builtin_elementwise_max(hi, __builtin_bit_cast(s16x2, x));
            lo = __builtin_elementwise_min(lo, __builtin_bit_cast(u16x2, x));
        }
    }
    DEV void widen(int &hi, u32 &lo) const {
#pragma unroll
        for (int k = 0; k < 4; ++k) {
            hi = max(hi, (int)w[k]);
            lo = min(lo, w[k]);
        }
    }
};

typedef __hip_bfloat16 bf16;

DEV float to_f(float v) { return v; }
DEV float to_f(__half v) { return __half2float(v); }
DEV float to_f(bf16 v) { return __bfloat162float(v); }
template <typename T> DEV T from_f(float v);
template <> DEV float from_f<float>(float v) { return v; }
template <> DEV __half from_f<__half>(float v) { return __float2half(v); }
template <> DEV bf16 from_f<bf16>(float v) { return __float2bfloat16(v); }

template <> DEV float Vec<float>::get(int i) const {
    return __uint_as_float(w[i]);
}
template <> DEV float Vec<bf16>::get(int i) const {
    return __uint_as_float(i & 1 ? w[i >> 1] & 0xffff0000u : w[i >> 1] << 16);
}
template <> DEV float Vec<__half>::get(int i) const {
    return __half2float(__ushort_as_half(
        (unsigned short)(i & 1 ? w[i >> 1] >> 16 : w[i >> 1])));
}
template <> DEV void Vec<float>::put(int i, float a, float b) {
    w[i] = __float_as_uint(a);
    w[i + 1] = __float_as_uint(b);
}
template <> DEV void Vec<bf16>::put(int i, float a, float b) {
    typedef __bf16 bf2 __attribute__((ext_vector_type(2)));
    const f32x2 f = {a, b};
    w[i >> 1] = __builtin_bit_cast(u32, __builtin_convertvector(f, bf2));
}
template <> DEV void Vec<__half>::put(int i, float a, float b) {
    typedef _Float16 h2 __attribute__((ext_vector_type(2)));
    const f32x2 f = {a, b};
    w[i >> 1] = __builtin_bit_cast(u32, __builtin_convertvector(f, h2));
}

// the two running patterns of Vec::widen, and what they say
template <typename T> struct Patterns {
    s16x2 hi = {-32768, -32768};
    u16x2 lo = {65535, 65535};
    DEV int top() const { return max((int)hi.x, (int)hi.y); }
    DEV u32 bottom() const { return min((u32)lo.x, (u32)lo.y); }
};
template <> struct Patterns<float> {
    int hi = -2147483647 - 1;
    u32 lo = 0xffffffffu;
    DEV int top() const { return hi; }
    DEV u32 bottom() const { return lo; }
};
template <typename T> DEV float from_pattern(u32 bits);
template <> DEV float from_pattern<float>(u32 b) { return __uint_as_float(b); }
template <> DEV float from_pattern<bf16>(u32 b) {
    return __uint_as_float(b << 16);
}
template <> DEV float from_pattern<__half>(u32 b) {
    return __half2float(__ushort_as_half((unsigned short)b));
}

template <typename T> DEV u32 pad_word() {  // -inf, once or twice
    return sizeof(T) == 4                       ? 0xff800000u
           : std::is_same<T, bf16>::value ? 0xff80ff80u : 0xfc00fc00u;
}

// A vector of which `past` elements lie behind the row's end, taken from the
// row's last 16 bytes: moved down, and -inf behind.
template <typename T> DEV void shift_in_pad(Vec<T> &v, int past) {
    const u32 pad = pad_word<T>();
    if constexpr (sizeof(T) == 2) {
        if (past & 1) {
#pragma unroll
            for (int k = 0; k < 4; ++k)
                v.w[k] = __builtin_amdgcn_alignbit(k < 3 ? v.w[k + 1] : pad,
                                                   v.w[k], 16);
        }
    }
    const int words = past * (int)sizeof(T) / 4;
    if (words & 1) v.w = (u32x4){v.w[1], v.w[2], v.w[3], pad};
    if (words & 2) v.w = (u32x4){v.w[2], v.w[3], pad, pad};
    if (words & 4) v.w = (u32x4){pad, pad, pad, pad};
}

// `at` counts elements from the row's start; elements past its end are -inf
template <typename T> DEV Vec<T> load_vec(const T *row, long at, long V) {
    constexpr int N = Vec<T>::N;
    Vec<T> v;
    if (V >= N) {
        v.load(row + min(at, V - N));
        shift_in_pad(v, (int)min(max(at + N - V, 0l), (long)N));
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

// a wave's stretch of a row; only a row's last one can be cut short
template <typename T>
DEV void load_stretch(const T *row, long lo, long V, int lane,
                      Vec<T> (&v)[NVEC]) {
    constexpr int N = Vec<T>::N;
    constexpr int SEG = WAVE * NVEC * N;
    if (lo + SEG <= V) {
        const T *p = row + lo + lane * N;
#pragma unroll
        for (int j = 0; j < NVEC; ++j) v[j].stream_in(p + j * WAVE * N);
    } else if (V >= N) {
        const int rest = (int)(V - lo);  // below SEG
#pragma unroll
        for (int j = 0; j < NVEC; ++j) {
            const int at = (j * WAVE + lane) * N;
            v[j].load(row + lo + min(at, rest - N));
        }
#pragma unroll
        for (int j = 0; j < NVEC; ++j) {
            const int at = (j * WAVE + lane) * N;
            shift_in_pad(v[j], min(max(at + N - rest, 0), N));
        }
    } else {
        v[0] = load_vec(row, (long)lane * N, V);
#pragma unroll
        for (int j = 1; j < NVEC; ++j) v[j].w = pad_word<T>();
    }
}

template <typename T>
DEV void store_vec(T *row, long at, long V, const float *f, bool whole) {
    constexpr int N = Vec<T>::N;
    Vec<T> v;
#pragma unroll
    for (int i = 0; i < N; i += 2) v.put(i, f[i], f[i + 1]);
    if (whole || at + N <= V) {  // whole: the same for all lanes
        v.stream_out(row + at);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at + i < V) {
                if constexpr (sizeof(T) == 4)
                    row[at + i] = __uint_as_float(v.w[i]);
                else
                    ((unsigned short *)row)[at + i] =
                        (unsigned short)(v.w[i >> 1] >> (i & 1) * 16);
            }
    }
}

template <typename T>
DEV const T *row_ptr(const VocabRows &g, int r) {
    const int o = r < g.inner ? 0 : r / g.inner, i = r - o * g.inner;
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

// sums and maxima over a wave, in every lane: within 16 lanes by data
// movement in the operand, then the four rows through scalar registers
template <int CTRL> DEV float dpp(float v) {
    return __int_as_float(__builtin_amdgcn_update_dpp(
        0, __float_as_int(v), CTRL, 0xf, 0xf, true));
}
#define DPP_XOR1 0xB1         // quad_perm [1, 0, 3, 2]
#define DPP_XOR2 0x4E         // quad_perm [2, 3, 0, 1]
#define DPP_HALF_MIRROR 0x141 // the other quad of 8
#define DPP_MIRROR 0x140      // the other 8 of 16
DEV float lane_f(float v, int lane) {
    return __int_as_float(
        __builtin_amdgcn_readlane(__float_as_int(v), lane));
}
DEV float sum_wave(float v) {
    v += dpp<DPP_XOR1>(v);
    v += dpp<DPP_XOR2>(v);
    v += dpp<DPP_HALF_MIRROR>(v);
    v += dpp<DPP_MIRROR>(v);
    return (lane_f(v, 0) + lane_f(v, 16)) + (lane_f(v, 32) + lane_f(v, 48));
}
template <int CTRL, typename I> DEV I dpp_i(I v) {
    return (I)__builtin_amdgcn_update_dpp(0, (int)v, CTRL, 0xf, 0xf, true);
}
// over aligned groups of LPG = 8 or 16 lanes
template <int LPG> DEV int group_max(int v) {
    v = max(v, dpp_i<DPP_XOR1>(v));
    v = max(v, dpp_i<DPP_XOR2>(v));
    v = max(v, dpp_i<DPP_HALF_MIRROR>(v));
    if (LPG == 16) v = max(v, dpp_i<DPP_MIRROR>(v));
    return v;
}
template <int LPG> DEV u32 group_min(u32 v) {
    v = min(v, dpp_i<DPP_XOR1>(v));
    v = min(v, dpp_i<DPP_XOR2>(v));
    v = min(v, dpp_i<DPP_HALF_MIRROR>(v));
    if (LPG == 16) v = min(v, dpp_i<DPP_MIRROR>(v));
    return v;
}
DEV int lane_i(int v, int lane) { return __builtin_amdgcn_readlane(v, lane); }
DEV int max_wave(int v) {
    v = group_max<16>(v);
    return max(max(lane_i(v, 0), lane_i(v, 16)),
               max(lane_i(v, 32), lane_i(v, 48)));
}
DEV u32 or_wave(u32 v) {
    v |= dpp_i<DPP_XOR1>(v);
    v |= dpp_i<DPP_XOR2>(v);
    v |= dpp_i<DPP_HALF_MIRROR>(v);
    v |= dpp_i<DPP_MIRROR>(v);
    return (u32)(lane_i(v, 0) | lane_i(v, 16) | lane_i(v, 32) | lane_i(v, 48));
}
DEV u32 min_wave(u32 v) {
    v = group_min<16>(v);
    return min(min((u32)lane_i(v, 0), (u32)lane_i(v, 16)),
               min((u32)lane_i(v, 32), (u32)lane_i(v, 48)));
}

DEV double lane_d(double v, int lane) {
    const u64 b = __builtin_bit_cast(u64, v);
    const u64 lo = (u32)lane_i((int)(u32)b, lane);
    const u64 hi = (u32)lane_i((int)(u32)(b >> 32), lane);
    return __builtin_bit_cast(double, hi << 32 | lo);
}
template <int CTRL> DEV double dpp_d(double v) {
    const u64 b = __builtin_bit_cast(u64, v);
    const u64 lo = dpp_i<CTRL>((u32)b), hi = dpp_i<CTRL>((u32)(b >> 32));
    return __builtin_bit_cast(double, hi << 32 | lo);
}
DEV double sum_wave_d(double v) {
    v += dpp_d<DPP_XOR1>(v);
    v += dpp_d<DPP_XOR2>(v);
    v += dpp_d<DPP_HALF_MIRROR>(v);
    v += dpp_d<DPP_MIRROR>(v);
    return (lane_d(v, 0) + lane_d(v, 16)) + (lane_d(v, 32) + lane_d(v, 48));
}
DEV float max_wave_f(float v) {
    v = fmaxf(v, dpp<DPP_XOR1>(v));
    v = fmaxf(v, dpp<DPP_XOR2>(v));
    v = fmaxf(v, dpp<DPP_HALF_MIRROR>(v));
    v = fmaxf(v, dpp<DPP_MIRROR>(v));
    return fmaxf(fmaxf(lane_f(v, 0), lane_f(v, 16)),
                 fmaxf(lane_f(v, 32), lane_f(v, 48)));
}

// Each lane's largest pattern of its vector j, over the LPG lanes of a group,
// to the group's lane j.
DEV int group_tops(const Vec<float> (&v)[NVEC], int lane) {
    int mine = 0;
#pragma unroll
    for (int j = 0; j < NVEC; ++j) {
        Patterns<float> p;
        v[j].widen(p.hi, p.lo);
        const int x = group_max<16>(p.top());
        if (lane % 16 == j) mine = x;
    }
    return mine;
}
// 16-bit types: two vectors to a register, and at every exchange a lane keeps
// the half that it is to end with: 15 operations for eight maxima over eight
// lanes, not 8 * 4.
template <typename T> DEV int group_tops(const Vec<T> (&v)[NVEC], int lane) {
    static_assert(NVEC == 8, "eight vectors, eight lanes");
    s16x2 two[4];
#pragma unroll
    for (int j = 0; j < 4; ++j) {
        Patterns<T> p, q;
        v[2 * j].widen(p.hi, p.lo);
        v[2 * j + 1].widen(q.hi, q.lo);
        const u32 a = __builtin_bit_cast(u32, p.hi);
        const u32 b = __builtin_bit_cast(u32, q.hi);
        // low halves of both, high halves of both
        const u32 lo = __builtin_amdgcn_perm(b, a, 0x05040100);
        const u32 hi = __builtin_amdgcn_perm(b, a, 0x07060302);
        two[j] = __builtin_elementwise_max(__builtin_bit_cast(s16x2, lo),
                                           __builtin_bit_cast(s16x2, hi));
    }
    const bool b0 = lane & 1, b1 = lane & 2, b2 = lane & 4;
    auto exchange = [](s16x2 keep, s16x2 give, auto ctrl) {
        const u32 o =
            dpp_i<decltype(ctrl)::value>(__builtin_bit_cast(u32, give));
        return __builtin_elementwise_max(keep, __builtin_bit_cast(s16x2, o));
    };
    // 7 - lane, then lane ^ 2, then lane ^ 1
    typedef std::integral_constant<int, DPP_HALF_MIRROR> Mirror;
    typedef std::integral_constant<int, DPP_XOR2> Xor2;
    typedef std::integral_constant<int, DPP_XOR1> Xor1;
    const s16x2 p0 = exchange(b2 ? two[2] : two[0], b2 ? two[0] : two[2],
                              Mirror());
    const s16x2 p1 = exchange(b2 ? two[3] : two[1], b2 ? two[1] : two[3],
                              Mirror());
    const s16x2 q = exchange(b1 ? p1 : p0, b1 ? p0 : p1, Xor2());
    const s16x2 x = exchange(q, q, Xor1());
    return b0 ? (int)x.y : (int)x.x;
}

// ---- partials --------------------------------------------------------------
// Workgroups go to the 8 XCDs in turn. Giving each XCD a run of consecutive
// stretches keeps neighbours, which share a cache line where rows are not
// aligned, behind one L2, and never gives an XCD the same columns of every
// row (8192 rows of 128257 bf16, read alone: 309 us, 394 us in plain order).
DEV u32 wave_index() {
    const u32 per = gridDim.x / 8;  // the grid is a multiple of 8
    const u32 b = (blockIdx.x % 8) * per + blockIdx.x / 8;
    return __builtin_amdgcn_readfirstlane(b * WAVES + threadIdx.x / WAVE);
}

// One wave per stretch. Writes (m, s, t, 0). With EXCL the sum leaves out the
// tokens that a teacher lists (m does not): the rest of the mass is summed,
// not got as a difference, because a student that has learned leaves little
// of it. Only vectors that hold such a token look at its bits. With GRP also the maximum of each GROUP
// consecutive tokens, for the search of the top alternatives.
//
// What bounds it: per element one unpacking, one product, one exponential,
// one or two sums and half an operation for the maximum, beside 2 or 4 bytes.
template <typename T, bool ENT, bool EXCL, bool GRP>
__global__ __launch_bounds__(BLOCK) void vocab_partials(
    VocabRows g, const long *__restrict__ tokens, long ignore,
    const long *__restrict__ ids, int K, float c, float4 *__restrict__ part,
    float *__restrict__ gmax) {
    constexpr int N = Vec<T>::N;
    constexpr int SEG = WAVE * NVEC * N;
    constexpr int LPG = GROUP / N;  // lanes per group: 8 or 16
    __shared__ u32 bits[EXCL ? WAVES : 1][EXCL ? SEG / 32 : 1];
    const int lane = threadIdx.x % WAVE;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const u32 total = (u32)g.rows * g.nseg;  // below 2^31, as is w's step
    for (u32 w = wave_index(); w < total; w += gridDim.x * WAVES) {
        const int r = w / (u32)g.nseg, seg = w - (u32)r * g.nseg;
        if (tokens && tokens[r] == ignore) continue;
        const T *row = row_ptr<T>(g, r);
        const long lo = (long)seg * SEG;
        // the ids before the stretch: loads arrive in order
        constexpr int EPL = EXCL ? VOCAB_MAX_K / WAVE : 1;
        long id[EPL];
        if (EXCL) {
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
                const int k = e * WAVE + lane;
                id[e] = k < K ? ids[(long)r * K + k] : -1;
            }
        }
        Vec<T> v[NVEC];
        load_stretch(row, lo, g.V, lane, v);
        // the tokens of this stretch that the teacher lists, one bit each
        u32 hit = 0;  // vectors of the stretch that hold one
        if (EXCL) {
            for (int i = lane; i < SEG / 32; i += WAVE) bits[wid][i] = 0;
            wave_sync();
#pragma unroll
            for (int e = 0; e < EPL; ++e) {
                const long at = id[e] - lo;
                if (at >= 0 && at < SEG) {
                    atomicOr(&bits[wid][at >> 5], 1u << (at & 31));
                    hit |= 1u << ((int)at / (WAVE * N));
                }
            }
            wave_sync();
            hit = or_wave(hit);
        }
        // the largest value, by bit patterns; a stretch (or a group) without
        // a value >= 0 is looked at a second time
        int top;
        u32 m_bits;
        if (GRP) {
            const int gm = group_tops(v, lane);
            u32 gbits = (u32)gm;
            const bool mine = lane % LPG < NVEC;
            if (__ballot(mine && gm < 0)) {
#pragma unroll
                for (int j = 0; j < NVEC; ++j) {
                    Patterns<T> p;
                    v[j].widen(p.hi, p.lo);
                    const u32 x = group_min<LPG>(p.bottom());
                    if (lane % LPG == j && gm < 0) gbits = x;
                }
            }
            if (mine) {
                // lane (group q of a vector, j) has group j * (64 / LPG) + q
                const int q = lane / LPG, j = lane % LPG;
                gmax[(long)w * (SEG / GROUP) + j * (WAVE / LPG) + q] =
                    from_pattern<T>(gbits);
            }
            top = max_wave(mine ? gm : -2147483647 - 1);
            m_bits = (u32)top;
            if (top < 0) m_bits = min_wave(mine ? gbits : 0xffffffffu);
        } else {
            Patterns<T> p;
#pragma unroll
            for (int j = 0; j < NVEC; ++j) v[j].widen(p.hi, p.lo);
            top = max_wave(p.top());
            m_bits = (u32)top;
            if (top < 0) {
                Patterns<T> n;
#pragma unroll
                for (int j = 0; j < NVEC; ++j) v[j].widen(n.hi, n.lo);
                m_bits = min_wave(n.bottom());
            }
        }
        const float m = from_pattern<T>(m_bits);
        const float mr = m == -INFINITY ? 0.f : m, mc = mr * c;
        float s = 0.f, t = 0.f;
        // one vector; the values stay packed until here
        auto sums = [&](const Vec<T> &x, int j, auto diff) {
            if (!EXCL || !(hit >> j & 1)) {
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const float d = diff(x.get(i)), e = exp2_hw(d);
                    s += e;
                    // 2^-300 is 0, and (-inf) * 0 would be NaN; NaN is in e
                    // already
                    if (ENT) t = fmaf(fmaxf(d, -300.f), e, t);
                }
            } else {
                const int at = (j * WAVE + lane) * N;
                const u32 in = bits[wid][at >> 5] >> (at & 31);
#pragma unroll
                for (int i = 0; i < N; ++i) {
                    const u32 e = __float_as_uint(exp2_hw(diff(x.get(i))));
                    // all ones where listed
                    const u32 mask = (u32)((int)(in << (31 - i)) >> 31);
                    s += __uint_as_float(e & ~mask);
                }
            }
        };
        if (by_product(mc)) {
#pragma unroll
            for (int j = 0; j < NVEC; ++j)
                sums(v[j], j, [&](float x) { return fmaf(x, c, -mc); });
        } else {
            // rare: read again, one vector at a time, rather than held twice
#pragma unroll 1
            for (int j = 0; j < NVEC; ++j)
                sums(load_vec(row, lo + (long)(j * WAVE + lane) * N, g.V), j,
                     [&](float x) { return (x - mr) * c; });
        }
        s = sum_wave(s);
        if (ENT) t = sum_wave(t);
        if (lane == 0) part[w] = make_float4(m, s, t, 0.f);
    }
}

// ---- join ------------------------------------------------------------------
struct RowStat {
    float m;           // largest logit, 0 where there is none
    double s, t;       // against m*c itself
    double delta;      // m*c less its rounded value: 2^(x*c - mc) is
                       // 2^delta times too large
};

// one wave joins a row's stretches, each lane's in order, in 64 bits
DEV RowStat join_parts(const float4 *p, int nseg, float c, int lane) {
    float m = -INFINITY;
    for (int i = lane; i < nseg; i += WAVE) m = fmaxf(m, p[i].x);
    m = max_wave_f(m);
    RowStat st;
    st.m = m == -INFINITY ? 0.f : m;
    const float mc = st.m * c;
    const double exact = (double)st.m * c;
    st.delta = by_product(mc) ? exact - mc : 0.;
    double s = 0, t = 0;
    for (int i = lane; i < nseg; i += WAVE) {
        const float4 q = p[i];
        const float qm = q.x == -INFINITY ? 0.f : q.x;
        // against each stretch's own rounded reference, where there is one
        const float qc = qm * c;
        double d = (by_product(qc) ? (double)qc : (double)qm * c) - exact;
        // adds nothing, but NaN stays NaN
        if (q.x == -INFINITY || d < -300) d = -300;
        const double f = exp2(d);
        s += q.y * f;
        t += (q.z + d * q.y) * f;
    }
    st.s = sum_wave_d(s);
    st.t = sum_wave_d(t);
    return st;
}

// ---- top alternatives ------------------------------------------------------
// Values as whole numbers of the same order (-0 counts as 0), without the low
// bits that the type never sets; 0 is below them all.
template <typename T> struct Order {
    static constexpr int LOW = sizeof(T) == 4                             ? 0
                               : std::is_same<T, __half>::value ? 13 : 16;
    static constexpr int BITS = 32 - LOW;
    static DEV u32 of(float x) {
        const u32 b = __float_as_uint(x + 0.f);
        return (b & 0x80000000u ? ~b : b | 0x80000000u) >> LOW;
    }
};

struct TopShared {
    u64 key[CAP];               // (order, ~index) of the candidates
    int group[VOCAB_MAX_K];     // groups that can hold alternatives
    int count[2][WAVES];        // of block_count, two turns
    int ties[32 * WAVES];
    int n_group, n_key;
};

// number of true predicates in the workgroup, given each wave's own. `turn`
// alternates between calls, so one barrier is enough.
DEV int block_count(int wave_count, TopShared &sh, int &turn) {
    if (threadIdx.x % WAVE == 0) sh.count[turn][threadIdx.x / WAVE] = wave_count;
    __syncthreads();
    int n = 0;
#pragma unroll
    for (int w = 0; w < WAVES; ++w) n += sh.count[turn][w];
    turn ^= 1;
    return n;
}

// calls f(order, index, valid) for every token of the chosen groups; all
// lanes take part in every call
template <typename T, typename F>
DEV void for_candidates(const T *row, long V, const TopShared &sh, int groups,
                        F f) {
    constexpr int N = Vec<T>::N, LPG = GROUP / N;
    for (int i = 0; i < groups * LPG; i += BLOCK) {
        const int slot = i + threadIdx.x;
        const bool on = slot < groups * LPG;
        const long at =
            on ? (long)sh.group[slot / LPG] * GROUP + slot % LPG * N : V;
        const Vec<T> v = load_vec(row, at, V);
#pragma unroll
        for (int k = 0; k < N; ++k)
            f(Order<T>::of(v.get(k)), (u32)(at + k), at + k < V);
    }
}

// The K largest of a row, (value down, index up), from its groups' maxima.
// The K groups of the largest (maximum, lowest index) hold them all: each of
// these has a token at least as good as any token of the others. The K-th
// maximum is found by bits; tokens of those groups that reach it are the
// candidates, hardly more than K in a row without structure; each one's rank
// is the number of better ones. Where more than CAP reach it (groups with
// many large tokens, or a vocabulary of few groups), a higher bound is
// searched among the tokens themselves, and, where one value alone has too
// many, a bound on the index. The whole takes NG maxima per thread.
template <typename T, int NG>
DEV void top_alternatives(const T *row, long V, const float *gmax, int K,
                          TopShared &sh, float *top_lp, long *top_ids,
                          double m, double inv_t, double ln_s, bool none) {
    const int tid = threadIdx.x, lane = tid % WAVE, wid = tid / WAVE;
    const int G = (int)((V + GROUP - 1) / GROUP);
    int turn = 0;
    if (tid == 0) sh.n_group = sh.n_key = 0;
    u32 key[NG];
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const int g = i * BLOCK + tid;
        key[i] = g < G ? Order<T>::of(gmax[g]) : 0;
    }
    u32 bound = 0;  // the K-th largest maximum, all bits below it 0
    int reach = G;  // how many reach it
    int KG = K;
    if (G <= K) {
        bound = 1;
        KG = G;
    } else {
        for (int bit = Order<T>::BITS - 1; bit >= 0; --bit) {
            const u32 b = bound | 1u << bit;
            int n = 0;
#pragma unroll
            for (int i = 0; i < NG; ++i) n += __popcll(__ballot(key[i] >= b));
            n = block_count(n, sh, turn);
            if (n >= K) {
                bound = b;
                reach = n;
                if (n == K) break;
            }
        }
    }
    // of the groups that equal the bound, those of lowest index
    int before[NG], quota = BLOCK * NG;
    if (reach > KG) {
        int above = 0;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            above += __popcll(__ballot(key[i] > bound));
            const int ties = __popcll(__ballot(key[i] == bound));
            if (lane == 0) sh.ties[i * WAVES + wid] = ties;
        }
        quota = KG - block_count(above, sh, turn);
        int run = 0;
#pragma unroll
        for (int i = 0; i < NG; ++i)
#pragma unroll
            for (int w = 0; w < WAVES; ++w) {
                if (w == wid) before[i] = run;
                run += sh.ties[i * WAVES + w];
            }
    } else {
        __syncthreads();  // n_group, n_key
#pragma unroll
        for (int i = 0; i < NG; ++i) before[i] = 0;
    }
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const u64 ties = __ballot(key[i] == bound);
        const int nth = before[i] + __popcll(ties & ((1ull << lane) - 1));
        if (key[i] > bound || (key[i] == bound && nth < quota) ||
            (reach <= KG && key[i] >= bound))
            sh.group[atomicAdd(&sh.n_group, 1)] = i * BLOCK + tid;
    }
    __syncthreads();
    u32 index_bound = 0xffffffffu;
    auto collect = [&](u32 order, u32 index, bool valid) {
        if (valid && (order > bound || (order == bound && index < index_bound))) {
            const int slot = atomicAdd(&sh.n_key, 1);
            if (slot < CAP) sh.key[slot] = (u64)order << 32 | ~index;
        }
    };
    for_candidates<T>(row, V, sh, KG, collect);
    __syncthreads();
    int n = sh.n_key;
    if (n > CAP) {
        bound = 0;
        for (int bit = Order<T>::BITS - 1; bit >= 0; --bit) {
            const u32 b = bound | 1u << bit;
            int c = 0;
            for_candidates<T>(row, V, sh, KG, [&](u32 order, u32, bool valid) {
                c += __popcll(__ballot(valid && order >= b));
            });
            c = block_count(c, sh, turn);
            if (c >= K) {
                bound = b;
                n = c;
                if (c <= CAP) break;
            }
        }
        if (n > CAP) {
            // more than CAP tokens share the K-th value: `need` of them, the
            // first ones
            int above = 0;
            for_candidates<T>(row, V, sh, KG, [&](u32 order, u32, bool valid) {
                above += __popcll(__ballot(valid && order > bound));
            });
            const int need = K - block_count(above, sh, turn);
            index_bound = 0;
            for (int bit = 30; bit >= 0; --bit) {
                const u32 b = index_bound | 1u << bit;
                int c = 0;
                for_candidates<T>(
                    row, V, sh, KG, [&](u32 order, u32 index, bool valid) {
                        c += __popcll(__ballot(valid && order == bound &&
                                               index < b));
                    });
                if (block_count(c, sh, turn) <= need) index_bound = b;
            }
        }
        if (tid == 0) sh.n_key = 0;
        __syncthreads();
        for_candidates<T>(row, V, sh, KG, collect);
        __syncthreads();
        n = sh.n_key;
    }
    for (int i = tid; i < n; i += BLOCK) {
        const u64 mine = sh.key[i];
        int rank = 0;
        for (int j = 0; j < n; ++j) rank += sh.key[j] > mine;
        if (rank < K) {
            const u32 index = ~(u32)mine;
            top_ids[rank] = (long)index;
            top_lp[rank] = none ? -INFINITY
                                : (float)(((double)to_f(row[index]) - m) *
                                              inv_t - ln_s);
        }
    }
    __syncthreads();
}

struct RowOut {
    double m, ln_s;
    bool none, bad;  // no finite logit; NaN or +inf among them
};

// One wave: a row's log probability, entropy and stat[r] =
// (m, 1/s, H - ln s, 0) against the rounded m*c, what the gradient needs;
// 1/s is 0 where the row has no finite logit.
template <typename T>
DEV RowOut logprobs_row(const VocabRows &g, const float4 *part, int r,
                        const long *tokens, float c, double inv_t,
                        float *logprobs, float *entropy, float4 *stat,
                        int lane, bool write) {
    const RowStat st = join_parts(part + (long)r * g.nseg, g.nseg, c, lane);
    RowOut o;
    o.m = st.m;
    o.none = st.s == 0;
    o.bad = !(st.s < INFINITY);
    o.ln_s = log(st.s);
    if (write && lane == 0) {
        if (tokens) {
            const long tok = tokens[r];
            float lp = NAN;
            if (tok >= 0 && tok < g.V && !o.bad)
                lp = o.none ? -INFINITY
                            : (float)(((double)to_f(row_ptr<T>(g, r)[tok]) -
                                       o.m) * inv_t - o.ln_s);
            logprobs[r] = lp;
        }
        const double ln2 = 0.6931471805599453, mean = st.t / st.s;
        entropy[r] = o.none ? 0.f
                     : o.bad ? NAN : (float)(o.ln_s - ln2 * mean);
        stat[r] = make_float4(
            st.m, o.none ? 0.f : (float)(exp2(-st.delta) / st.s),
            o.none ? 0.f : (float)(-ln2 * (mean + st.delta)), 0.f);
    }
    return o;
}

// without alternatives: one wave per row
template <typename T>
__global__ __launch_bounds__(BLOCK) void logprobs_join(
    VocabRows g, const float4 *__restrict__ part,
    const long *__restrict__ tokens, long ignore, float c, double inv_t,
    float *__restrict__ logprobs, float *__restrict__ entropy,
    float4 *__restrict__ stat) {
    const int lane = threadIdx.x % WAVE;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    for (u32 r = blockIdx.x * WAVES + wid; r < (u32)g.rows;
         r += gridDim.x * WAVES) {
        if (tokens && tokens[r] == ignore) {
            if (lane == 0) {
                logprobs[r] = 0.f;
                entropy[r] = 0.f;
                stat[r] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            continue;
        }
        logprobs_row<T>(g, part, (int)r, tokens, c, inv_t, logprobs, entropy,
                        stat, lane, true);
    }
}

// with alternatives: one workgroup per row
template <typename T, int NG>
__global__ __launch_bounds__(BLOCK) void logprobs_top_join(
    VocabRows g, const float4 *__restrict__ part,
    const float *__restrict__ gmax, const long *__restrict__ tokens,
    long ignore, int K, float c, double inv_t, float *__restrict__ logprobs,
    float *__restrict__ entropy, float *__restrict__ top_lp,
    long *__restrict__ top_ids, float4 *__restrict__ stat) {
    constexpr int GPS = WAVE * NVEC * Vec<T>::N / GROUP;  // per stretch
    __shared__ TopShared sh;
    const int lane = threadIdx.x % WAVE;
    for (int r = blockIdx.x; r < g.rows; r += gridDim.x) {
        float *lp_out = top_lp + (long)r * K;
        long *id_out = top_ids + (long)r * K;
        if (tokens && tokens[r] == ignore) {
            if (threadIdx.x == 0) {
                logprobs[r] = 0.f;
                entropy[r] = 0.f;
                stat[r] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            for (int k = threadIdx.x; k < K; k += BLOCK) {
                lp_out[k] = 0.f;
                id_out[k] = -1;
            }
            continue;
        }
        // every wave joins for itself
        const RowOut o = logprobs_row<T>(g, part, r, tokens, c, inv_t,
                                         logprobs, entropy, stat, lane,
                                         threadIdx.x < WAVE);
        if (o.bad) {
            for (int k = threadIdx.x; k < K; k += BLOCK) {
                lp_out[k] = NAN;
                id_out[k] = -1;
            }
        } else {
            top_alternatives<T, NG>(row_ptr<T>(g, r), g.V,
                                    gmax + (long)r * g.nseg * GPS, K, sh,
                                    lp_out, id_out, o.m, inv_t, o.ln_s,
                                    o.none);
        }
    }
}

// One wave per row, up to VOCAB_MAX_K / 64 entries per lane.
// stat[r] = (m, 1/s, a_in, a_out): the gradient of a student's logit is
// p_j a_in - sum of its q  inside the teacher's entries, p_j a_out outside.
// Both 0 mark a row without entries. q [rows, K] is kept for the gradient.
template <typename T>
__global__ __launch_bounds__(BLOCK) void distill_join(
    VocabRows g, const float4 *__restrict__ part,
    const float *__restrict__ tlp, const long *__restrict__ ids, int K,
    int bucket, float c, double inv_t, float *__restrict__ loss,
    float *__restrict__ q_out, float4 *__restrict__ stat) {
    constexpr int EPL = VOCAB_MAX_K / WAVE;
    constexpr int HASH = 2 * VOCAB_MAX_K;  // never more than half full
    __shared__ int seen[WAVES][HASH];
    const int lane = threadIdx.x % WAVE;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    for (u32 r = blockIdx.x * WAVES + wid; r < (u32)g.rows;
         r += gridDim.x * WAVES) {
        const T *row = row_ptr<T>(g, (int)r);
        long id[EPL];
        float l[EPL], x[EPL];
        double q[EPL], total = 0.;
        bool any = false, wrong = false;
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
            const int k = e * WAVE + lane;
            id[e] = -1;
            l[e] = x[e] = 0.f;
            if (k < K) {
                id[e] = ids[(long)r * K + k];
                l[e] = tlp[(long)r * K + k];
            }
        }
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
            const bool held = id[e] >= 0, in = id[e] < g.V;
            if (held && in) x[e] = to_f(row[id[e]]);
            any |= held;
            wrong |= held && !in;
            q[e] = 0.;
            if (__ballot(held)) q[e] = held ? exp((double)l[e]) : 0.;
            total += q[e];
        }
        any = __ballot(any) != 0;
        wrong = __ballot(wrong) != 0;
        total = sum_wave_d(total);
        double q_rest = 0., log_norm = 0., scale = 1., mass;
        if (bucket) {
            q_rest = total < 1. ? 1. - total : 0.;
            mass = total + q_rest;
        } else {
            // not `total > 0`: NaN has to stay NaN
            log_norm = total == 0. ? 0. : log(total);
            scale = total == 0. ? 0. : 1. / total;
            mass = total == 0. ? 0. : total / total;
        }
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
            q[e] *= scale;
            const int k = e * WAVE + lane;
            if (k < K) q_out[(long)r * K + k] = (float)q[e];
        }
        if (!any || (!bucket && total == 0.)) {
            if (lane == 0) {
                loss[r] = 0.f;
                stat[r] = make_float4(0.f, 0.f, 0.f, 0.f);
            }
            continue;
        }
        const RowStat st = join_parts(part + (long)r * g.nseg, g.nseg, c, lane);
        double s = st.s;
        if (bucket) {
            // the listed tokens' part, each token once
            for (int i = lane; i < HASH; i += WAVE) seen[wid][i] = -1;
            wave_sync();
            double s_in = 0.;
#pragma unroll
            for (int e = 0; e < EPL; ++e)
                if (id[e] >= 0 && id[e] < g.V) {
                    u32 at = ((u32)id[e] * 2654435761u) / (~0u / HASH + 1);
                    int old;
                    while ((old = atomicCAS(&seen[wid][at], -1, (int)id[e])) !=
                               -1 && old != (int)id[e])
                        at = (at + 1) % HASH;
                    if (old == -1) s_in += exp2(((double)x[e] - st.m) * c);
                }
            s += sum_wave_d(s_in);
        }
        const bool none = s == 0, bad = !(s < INFINITY);
        const double ln_s = log(s);
        double sum = 0.;
#pragma unroll
        for (int e = 0; e < EPL; ++e)
            if (id[e] >= 0 && id[e] < g.V && q[e] != 0.) {
                const double lp = none || x[e] == -INFINITY
                                      ? -INFINITY
                                      : ((double)x[e] - st.m) * inv_t - ln_s;
                sum += q[e] * (((double)l[e] - log_norm) - lp);
            }
        sum = sum_wave_d(sum);
        double ratio = 0.;
        if (bucket && q_rest > 0.) {
            // entries that cover every token with mass leave no room for
            // the rest; what 32-bit log probabilities leave over by
            // rounding then counts as none
            const double p_rest = none ? 0. : st.s / s;
            if (p_rest > 0.) {
                ratio = q_rest / p_rest;
                sum += q_rest * log(ratio);
            } else if (q_rest > 0x1p-20) {
                sum = INFINITY;
            }
        }
        if (lane == 0) {
            const bool nan = bad || wrong;
            loss[r] = nan ? NAN : (float)sum;
            stat[r] = make_float4(st.m,
                                  none ? 0.f : (float)(exp2(-st.delta) / s),
                                  nan ? NAN : (float)mass,
                                  nan ? NAN : (float)(mass - ratio));
        }
    }
}

// ---- gradients -------------------------------------------------------------
// d x_j = p_j (a + b ln(p_j s)) + what is given for single tokens, one wave per
// stretch, in one pass over packed registers: a product, an exponential and
// one or three more operations per element beside 4 or 8 bytes.
//
// Single tokens (the given one, alternatives with a gradient, a teacher's
// entries) are not looked for in the pass: the entries that fall into the
// stretch are gathered into LDS in the row's order, and after the stretch is
// written, and its stores have arrived, each one's lane computes its token
// anew and writes it once more. The same token given twice is added up by its
// first entry's lane, in order.
template <typename T, bool DISTILL>
__global__ __launch_bounds__(BLOCK) void vocab_grad(
    VocabRows g, VocabGrad a, T *__restrict__ out) {
    constexpr int N = Vec<T>::N;
    constexpr int SEG = WAVE * NVEC * N;
    __shared__ u32 bits_all[WAVES][SEG / 32];
    __shared__ int at_all[WAVES][VOCAB_MAX_K + 1];
    __shared__ float val_all[WAVES][VOCAB_MAX_K + 1];
    const int lane = threadIdx.x % WAVE;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    u32 *bits = bits_all[wid];
    int *list_at = at_all[wid];
    float *list_val = val_all[wid];
    const float *vals = DISTILL ? a.q : a.d_top;
    const u32 total = (u32)g.rows * g.nseg;  // below 2^31, as is w's step
    for (u32 w = wave_index(); w < total; w += gridDim.x * WAVES) {
        const int r = w / (u32)g.nseg, seg = w - (u32)r * g.nseg;
        const long lo = (long)seg * SEG;
        const bool whole = lo + SEG <= g.V;
        T *orow = out + (long)r * g.V;
        const float4 st = a.stat[r];
        bool skip = st.y == 0.f;
        if (DISTILL) skip = skip || (st.z == 0.f && st.w == 0.f);
        const long tok = !DISTILL && a.tokens ? a.tokens[r] : -1;
        if (!DISTILL && a.tokens && tok == a.ignore) skip = true;
        if (skip) {
            const float zero[N] = {};
#pragma unroll 1
            for (int j = 0; j < NVEC; ++j)
                store_vec(orow, lo + (long)(j * WAVE + lane) * N, g.V, zero,
                          whole);
            continue;
        }
        const T *row = row_ptr<T>(g, r);
        Vec<T> v[NVEC];
        load_stretch(row, lo, g.V, lane, v);
        // e = 2^((x - m) c) counts k_out (k_in where listed) + k_d * exponent
        int n = 0;
        float k_in, k_out, k_d = 0.f, scale = a.inv_t;
        if (DISTILL) {
            scale *= a.d_row[r];
            k_in = st.z;
            k_out = st.w;
        } else {
            float gs = 0.f;
            if (a.d_row && a.tokens) {
                const float gr = a.d_row[r];
                gs = tok >= 0 && tok < g.V ? gr : NAN;
                const long at = tok - lo;
                if (at >= 0 && at < SEG && tok < g.V) {
                    if (lane == 0) {
                        list_at[0] = (int)at;
                        list_val[0] = gr;
                    }
                    n = 1;
                }
            }
            if (a.d_top) {
                float gk = 0.f;
                for (int k = lane; k < a.K; k += WAVE)
                    gk += a.d_top[(long)r * a.K + k];
                gs += sum_wave(gk);
            }
            if (a.d_entropy) k_d = -a.d_entropy[r];
            k_in = k_out = k_d * st.z - gs;
            k_d *= 0.69314718f;
        }
        if (vals) {
            for (int k0 = 0; k0 < a.K; k0 += WAVE) {
                const int k = k0 + lane;
                const long at = k < a.K ? a.ids[(long)r * a.K + k] - lo : -1;
                const bool mine = at >= 0 && at < SEG && at + lo < g.V;
                const u64 who = __ballot(mine);
                if (mine) {
                    const int slot = n + __popcll(who & ((1ull << lane) - 1));
                    const float val = vals[(long)r * a.K + k];
                    list_at[slot] = (int)at;
                    list_val[slot] = DISTILL ? -val : val;
                }
                n += __popcll(who);
            }
        }
        wave_sync();
        const float mc = st.x * a.c, u = st.y * scale;
        const float u_out = k_out * u, u_d = k_d * u;
        const bool product = by_product(mc);
        auto grad = [&](float d, float uk) {
            // 2^-300 is 0, and (-inf) * 0 would be NaN
            if (!DISTILL) uk = fmaf(u_d, fmaxf(d, -300.f), uk);
            return exp2_hw(d) * uk;
        };
        if (product) {
#pragma unroll
            for (int j = 0; j < NVEC; ++j) {
                float f[N];
#pragma unroll
                for (int i = 0; i < N; ++i)
                    f[i] = grad(fmaf(v[j].get(i), a.c, -mc), u_out);
                store_vec(orow, lo + (long)(j * WAVE + lane) * N, g.V, f,
                          whole);
            }
        } else {
#pragma unroll 1
            for (int j = 0; j < NVEC; ++j) {
                const long at = lo + (long)(j * WAVE + lane) * N;
                const Vec<T> x = load_vec(row, at, g.V);
                float f[N];
#pragma unroll
                for (int i = 0; i < N; ++i)
                    f[i] = grad((x.get(i) - st.x) * a.c, u_out);
                store_vec(orow, at, g.V, f, whole);
            }
        }
        if (n > 0) {
            // is a token listed twice?
            u64 twice = 0;
            if (n > 1) {
                for (int i = lane; i < SEG / 32; i += WAVE) bits[i] = 0;
                wave_sync();
                for (int k0 = 0; k0 < n; k0 += WAVE) {
                    bool seen = false;
                    if (k0 + lane < n) {
                        const int at = list_at[k0 + lane];
                        const u32 bit = 1u << (at & 31);
                        seen = atomicOr(&bits[at >> 5], bit) & bit;
                    }
                    twice |= __ballot(seen);
                }
            }
            for (int k0 = 0; k0 < n; k0 += WAVE) {
                const int k = k0 + lane;
                const int at = k < n ? list_at[k] : -1;
                float val = k < n ? list_val[k] : 0.f;
                bool first = k < n;
                if (twice) {
                    val = 0.f;
                    for (int e = 0; e < n; ++e) {
                        const bool same = list_at[e] == at;
                        if (same) val += list_val[e];
                        if (same && e < k) first = false;
                    }
                }
                float f = 0.f;
                if (first) {
                    const float x = to_f(row[lo + at]);
                    f = fmaf(val, scale,
                             grad(product ? fmaf(x, a.c, -mc)
                                          : (x - st.x) * a.c,
                                  k_in * u));
                }
                // the stretch's own stores are to arrive first
                if (k0 == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                if (first) orow[lo + at] = from_f<T>(f);
            }
        }
        wave_sync();
    }
}

// ---- launches --------------------------------------------------------------
// grids are capped so that threads stay far below 2^32; waves then stride
static int wave_grid(const VocabRows &g) {
    const long blocks = CDIV((long)g.rows * g.nseg, (long)WAVES);
    return (int)(blocks < (1l << 22) ? CDIV(blocks, 8) * 8 : (1l << 22));
}
static int row_grid(long blocks) {
    return (int)(blocks < (1l << 22) ? blocks : (1l << 22));
}

template <typename T, int NG>
static void logprobs_top_join_t(const VocabRows &g, const VocabLogprobs &a,
                                float c, hipStream_t stream) {
    hipLaunchKernelGGL((logprobs_top_join<T, NG>), dim3(row_grid(g.rows)),
                       dim3(BLOCK), 0, stream, g, (const float4 *)a.part,
                       a.gmax, a.tokens, a.ignore, a.K, c, 1. / a.temperature,
                       a.logprobs, a.entropy, a.top_lp, a.top_ids,
                       (float4 *)a.stat);
}

template <typename T>
static void logprobs_fwd_t(const VocabRows &g, const VocabLogprobs &a,
                           hipStream_t stream) {
    const float c = (float)(1.4426950408889634 / a.temperature);
    if (a.K == 0) {
        hipLaunchKernelGGL((vocab_partials<T, true, false, false>),
                           dim3(wave_grid(g)), dim3(BLOCK), 0, stream, g,
                           a.tokens, a.ignore, nullptr, 0, c,
                           (float4 *)a.part, nullptr);
        hipLaunchKernelGGL((logprobs_join<T>),
                           dim3(row_grid(CDIV((long)g.rows, WAVES))),
                           dim3(BLOCK), 0, stream, g, (const float4 *)a.part,
                           a.tokens, a.ignore, c, 1. / a.temperature,
                           a.logprobs, a.entropy, (float4 *)a.stat);
        return;
    }
    hipLaunchKernelGGL((vocab_partials<T, true, false, true>),
                       dim3(wave_grid(g)), dim3(BLOCK), 0, stream, g,
                       a.tokens, a.ignore, nullptr, 0, c, (float4 *)a.part,
                       a.gmax);
    // maxima per thread; more than VOCAB_MAX_TOP_V tokens are refused before
    const long per = CDIV(CDIV(g.V, (long)GROUP), (long)BLOCK);
    if (per <= 4) logprobs_top_join_t<T, 4>(g, a, c, stream);
    else if (per <= 8) logprobs_top_join_t<T, 8>(g, a, c, stream);
    else if (per <= 16) logprobs_top_join_t<T, 16>(g, a, c, stream);
    else logprobs_top_join_t<T, 32>(g, a, c, stream);
}

template <typename T>
static void distill_fwd_t(const VocabRows &g, const VocabDistill &a,
                          hipStream_t stream) {
    const float c = (float)(1.4426950408889634 / a.temperature);
    if (a.bucket)
        hipLaunchKernelGGL((vocab_partials<T, false, true, false>),
                           dim3(wave_grid(g)), dim3(BLOCK), 0, stream, g,
                           nullptr, 0, a.ids, a.K, c, (float4 *)a.part,
                           nullptr);
    else
        hipLaunchKernelGGL((vocab_partials<T, false, false, false>),
                           dim3(wave_grid(g)), dim3(BLOCK), 0, stream, g,
                           nullptr, 0, nullptr, 0, c, (float4 *)a.part,
                           nullptr);
    hipLaunchKernelGGL((distill_join<T>),
                       dim3(row_grid(CDIV((long)g.rows, WAVES))), dim3(BLOCK),
                       0, stream, g, (const float4 *)a.part, a.teacher_lp, a.ids,
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
extern "C" int vocab_group(void) { return GROUP; }
static_assert(32 * BLOCK * GROUP == VOCAB_MAX_TOP_V, "limits agree");

extern "C" void logprobs_fwd_launch(const VocabRows *g, const VocabLogprobs *a,
                                    int dtype, hipStream_t stream) {
    if (dtype == VOCAB_BF16) logprobs_fwd_t<bf16>(*g, *a, stream);
    else if (dtype == VOCAB_FP16) logprobs_fwd_t<__half>(*g, *a, stream);
    else logprobs_fwd_t<float>(*g, *a, stream);
}

extern "C" void distill_fwd_launch(const VocabRows *g, const VocabDistill *a,
                                   int dtype, hipStream_t stream) {
    if (dtype == VOCAB_BF16) distill_fwd_t<bf16>(*g, *a, stream);
    else if (dtype == VOCAB_FP16) distill_fwd_t<__half>(*g, *a, stream);
    else distill_fwd_t<float>(*g, *a, stream);
}

extern "C" void vocab_grad_launch(const VocabRows *g, const VocabGrad *a,
                                  int distill, void *out, int dtype,
                                  hipStream_t stream) {
    if (dtype == VOCAB_BF16) grad_t<bf16>(*g, *a, distill, out, stream);
    else if (dtype == VOCAB_FP16) grad_t<__half>(*g, *a, distill, out, stream);
    else grad_t<float>(*g, *a, distill, out, stream);
}
