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
//   partials: one wave per stretch of 8 vectors of 16 bytes per lane, held in
//             registers: one read for the maximum and the sums;
//   join:     one wave per row (one workgroup where top alternatives are
//             asked): statistics, loss, the teacher's entries' gradients;
//   grad:     one wave per stretch of 4 vectors per lane: p from the
//             statistics, and what is given for single tokens.
// No floating-point atomics: the same input gives the same bits.
//
// A row is split over waves, not walked by one workgroup: 64 rows of 151936
// fill the card as 8192 do, and no wave waits for another. What is measured
// below are single launches back to back, of 8192 rows of 128257 bf16 where
// no size is given. On the same card reading alone reaches 7.0-7.4 TB/s, and
// copying 5.5-6.6 TB/s.
#include <hip/hip_fp16.h>

#include <type_traits>

#include "common.h"
#include "vocab.h"

#define BLOCK 256
#define WAVES (BLOCK / WAVE)
#define NVEC 8    // 16-byte vectors per lane and stretch
#define NGRAD 4   // the same in the gradient
#define GROUP 64  // tokens per maximum kept for the top alternatives
#define CAP 512   // candidates for them that are ranked at once

typedef unsigned int u32;
typedef unsigned long long u64;

// ---- element types: 16 bytes at any element boundary -----------------------
// Rows of an odd vocabulary start at any multiple of the element's size, so
// vectors are loaded and stored with that alignment: one 16-byte access each,
// which the hardware takes at any address.
typedef u32 u32x4 __attribute__((ext_vector_type(4)));
typedef u32x4 u32x4_mem __attribute__((aligned(2)));
typedef float f32x2 __attribute__((ext_vector_type(2)));
typedef short s16x2 __attribute__((ext_vector_type(2)));
typedef unsigned short u16x2 __attribute__((ext_vector_type(2)));

template <typename T> struct Vec {
    static constexpr int N = 16 / sizeof(T);
    u32x4 w;

    DEV void load(const T *p) { w = *(const u32x4_mem *)p; }
    DEV void store(T *p) const { *(u32x4_mem *)p = w; }
    DEV void stream_in(const T *p) {
        w = __builtin_nontemporal_load((const u32x4_mem *)p);
    }
    DEV void stream_out(T *p) const {
        __builtin_nontemporal_store(w, (u32x4_mem *)p);
    }
    DEV float get(int i) const;
    DEV void put(int i, float a, float b);  // elements i and i + 1, i even
    DEV float pick(int i) const {  // get, where i differs between lanes
        constexpr int PER = N / 4;
        const int k = i / PER;
        const u32 a = k & 1 ? w[1] : w[0], b = k & 1 ? w[3] : w[2];
        Vec<T> one;
        one.w[0] = k & 2 ? b : a;
        if constexpr (PER == 2) one.w[0] >>= (i & 1) * 16;
        return one.get(0);
    }
    DEV void drop(u32 in);  // -inf where `in` has the element's bit
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
template <typename T> struct Pattern { typedef unsigned short type; };
template <> struct Pattern<float> { typedef u32 type; };
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

template <typename T> DEV void Vec<T>::drop(u32 in) {
    constexpr int PER = N / 4;
#pragma unroll
    for (int k = 0; k < 4; ++k) {
        // all ones where dropped
        u32 mask = (u32)((int)(in << (31 - k * PER)) >> 31);
        if constexpr (PER == 2) {
            const u32 odd = (u32)((int)(in << (30 - k * PER)) >> 31);
            mask = (mask & 0xffffu) | odd << 16;
        }
        w[k] = (w[k] & ~mask) | (pad_word<T>() & mask);
    }
}

// A vector moved by `by` elements, down where positive, with -inf behind.
template <typename T> DEV void move_vec(Vec<T> &v, int by) {
    const u32 pad = pad_word<T>();
    if (by >= 0) {
        if constexpr (sizeof(T) == 2) {
            if (by & 1) {
#pragma unroll
                for (int k = 0; k < 4; ++k)
                    v.w[k] = __builtin_amdgcn_alignbit(
                        k < 3 ? v.w[k + 1] : pad, v.w[k], 16);
            }
        }
        const int words = by * (int)sizeof(T) / 4;
        if (words & 1) v.w = (u32x4){v.w[1], v.w[2], v.w[3], pad};
        if (words & 2) v.w = (u32x4){v.w[2], v.w[3], pad, pad};
        if (words & 4) v.w = (u32x4){pad, pad, pad, pad};
    } else {
        if constexpr (sizeof(T) == 2) {
            if (by & 1) {
#pragma unroll
                for (int k = 3; k >= 0; --k)
                    v.w[k] = __builtin_amdgcn_alignbit(
                        v.w[k], k > 0 ? v.w[k - 1] : pad, 16);
            }
        }
        const int words = -by * (int)sizeof(T) / 4;
        if (words & 1) v.w = (u32x4){pad, v.w[0], v.w[1], v.w[2]};
        if (words & 2) v.w = (u32x4){pad, pad, v.w[0], v.w[1]};
        if (words & 4) v.w = (u32x4){pad, pad, pad, pad};
    }
}

// `at` counts elements from the row's start, and may lie before it or behind
// its end: what is not in the row is -inf. A vector cut short is one load of
// the nearest whole one, moved.
template <typename T> DEV Vec<T> load_vec(const T *row, long at, long V) {
    constexpr int N = Vec<T>::N;
    const long near = min(max(at, 0l), max(V - N, 0l));
    Vec<T> v;
    if (V >= N) {
        v.load(row + near);
    } else {
        float f[N];
#pragma unroll
        for (int i = 0; i < N; ++i) f[i] = i < V ? to_f(row[i]) : -INFINITY;
#pragma unroll
        for (int i = 0; i < N; i += 2) v.put(i, f[i], f[i + 1]);
    }
    move_vec(v, (int)min(max(at - near, -(long)N), (long)N));
    return v;
}

// Stretches begin at a cache line (128 bytes) of the logits: a row's first one
// lies up to a line before the row. Whole lines are what the memory takes
// best: with stretches that began at the rows, the gradient of 8192 rows of
// 128257 bf16 took 830 us, and of 128384 tokens, whose rows all begin at a line,
// 698 us. Where the gradient's rows lie otherwise in their lines than the
// logits', it is the loads that gain by it: half of such rows 688 us, 738 with
// stretches at lines of the gradient.
DEV int before_row(const void *row, int size, u32 line) {
    return (int)((u32)(u64)row & line) / size;
}

// a wave's stretch of a row; only a row's first and last can be cut short
template <bool STREAM, typename T, int NV>
DEV void load_stretch(const T *row, long lo, long V, int lane,
                      Vec<T> (&v)[NV]) {
    constexpr int N = Vec<T>::N;
    constexpr int SEG = WAVE * NV * N;
    if (lo >= 0 && lo + SEG <= V) {
        const T *p = row + lo + lane * N;
#pragma unroll
        for (int j = 0; j < NV; ++j)
            if (STREAM) v[j].stream_in(p + j * WAVE * N);
            else v[j].load(p + j * WAVE * N);
    } else if (V >= N) {
        // as load_vec, in numbers relative to the stretch
        const int head = (int)max(-lo, 0l);
        const int last = (int)min(V - N - lo, (long)SEG);
        int by[NV];
#pragma unroll
        for (int j = 0; j < NV; ++j) {
            const int at = (j * WAVE + lane) * N;
            const int near = min(max(at, head), last);
            v[j].load(row + lo + near);
            by[j] = min(max(at - near, -N), N);
        }
#pragma unroll
        for (int j = 0; j < NV; ++j) move_vec(v[j], by[j]);
    } else {
        // the row is within the first vectors of its one stretch
#pragma unroll
        for (int j = 0; j < NV; ++j) v[j].w = pad_word<T>();
        v[0] = load_vec(row, lo + lane * N, V);
    }
}

template <bool STREAM, typename T>
DEV void store_vec(T *row, long at, long V, const float *f, bool whole) {
    constexpr int N = Vec<T>::N;
    Vec<T> v;
#pragma unroll
    for (int i = 0; i < N; i += 2) v.put(i, f[i], f[i + 1]);
    if (whole || (at >= 0 && at + N <= V)) {  // whole: the same for all lanes
        if (STREAM) v.stream_out(row + at);
        else v.store(row + at);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (at + i >= 0 && at + i < V) {
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

// One wave per stretch. Writes (m, s, t, 0). With EXCL as if the tokens that a
// teacher lists were not there: the rest of the mass is summed against its
// own maximum, not got as a difference, because a student that has learned
// leaves little of it. Only vectors that hold such a token look at its bits.
// With GRP also the maximum of each GROUP consecutive tokens, for the search
// of the top alternatives.
//
// What bounds it is the memory's read rate: 288-292 us (shortest and median
// launch; 7.2-7.3 TB/s), 294-309 with the entropy. Per element there are one
// unpacking, one product, one exponential, one or two sums and half an
// operation for the maximum, beside 2 or 4 bytes: the vector units issue in a
// fifth of the cycles. The group maxima's exchange and their stores take it
// from 147 us to 162-190 at 4096 rows (145-150 without the stores). 512 rows of
// 102400 fp32 with group maxima: 33-34 us (6.2-6.4 TB/s).
template <typename T, bool ENT, bool EXCL, bool GRP, bool STREAM>
__global__ __launch_bounds__(BLOCK) void vocab_partials(
    VocabRows g, u32 first, const long *__restrict__ tokens, long ignore,
    const long *__restrict__ ids, int K, float c, float4 *__restrict__ part,
    typename Pattern<T>::type *__restrict__ gmax) {
    constexpr int N = Vec<T>::N;
    constexpr int SEG = WAVE * NVEC * N;
    constexpr int LPG = GROUP / N;  // lanes per group: 8 or 16
    __shared__ u32 bits[EXCL ? WAVES : 1][EXCL ? SEG / 32 : 1];
    const int lane = threadIdx.x % WAVE;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const u32 w = first + wave_index();  // below 2^32
    if (w >= (u32)g.rows * g.nseg) return;
    const int r = w / (u32)g.nseg, seg = w - (u32)r * g.nseg;
    if (tokens && tokens[r] == ignore) return;
    const T *row = row_ptr<T>(g, r);
    const long lo = (long)seg * SEG - before_row(row, sizeof(T), g.line);
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
    load_stretch<STREAM>(row, lo, g.V, lane, v);
    // the tokens of this stretch that the teacher lists, one bit each
    u32 hit = 0;  // vectors of the stretch that hold one
    auto drop_listed = [&](Vec<T> &x, int j) {
        const int at = (j * WAVE + lane) * N;
        if (EXCL && hit >> j & 1) x.drop(bits[wid][at >> 5] >> (at & 31));
    };
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
#pragma unroll
        for (int j = 0; j < NVEC; ++j) drop_listed(v[j], j);
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
                (typename Pattern<T>::type)gbits;
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
    // one vector; the values stay packed until here. Summed by itself first:
    // beside a lane's token that has nearly all of a row, 7 terms each lose
    // what 32 bits lack, not 63
    auto sums = [&](const Vec<T> &x, auto diff) {
        float sv;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float d = diff(x.get(i)), e = exp2_hw(d);
            sv = i == 0 ? e : sv + e;
            // 2^-300 is 0, and (-inf) * 0 would be NaN; NaN is in e already
            if (ENT) t = fmaf(fmaxf(d, -300.f), e, t);
        }
        s += sv;
    };
    if (by_product(mc)) {
#pragma unroll
        for (int j = 0; j < NVEC; ++j)
            sums(v[j], [&](float x) { return fmaf(x, c, -mc); });
    } else {
        // rare: read again, one vector at a time, rather than held twice
#pragma unroll 1
        for (int j = 0; j < NVEC; ++j) {
            Vec<T> x = load_vec(row, lo + (long)(j * WAVE + lane) * N, g.V);
            drop_listed(x, j);
            sums(x, [&](float x) { return (x - mr) * c; });
        }
    }
    s = sum_wave(s);
    if (ENT) t = sum_wave(t);
    if (lane == 0) part[w] = make_float4(m, s, t, 0.f);
}

// ---- join ------------------------------------------------------------------
// 2^d and ln v in 64 bits, small: the library's take 60 registers more in
// kernels that live from their occupancy. 2^d by the power series of e^x for
// |x| <= ln 2 / 2, whose next term is below 2^-53; NaN stays NaN.
DEV double exp2_d(double d) {
    d = d < -2000. ? -2000. : d;
    const double i = rint(d), x = (d - i) * 0.6931471805599453;
    double p = 1. / 6227020800.;  // 1 / 13!
    p = fma(p, x, 1. / 479001600.);
    p = fma(p, x, 1. / 39916800.);
    p = fma(p, x, 1. / 3628800.);
    p = fma(p, x, 1. / 362880.);
    p = fma(p, x, 1. / 40320.);
    p = fma(p, x, 1. / 5040.);
    p = fma(p, x, 1. / 720.);
    p = fma(p, x, 1. / 120.);
    p = fma(p, x, 1. / 24.);
    p = fma(p, x, 1. / 6.);
    p = fma(p, x, 0.5);
    p = fma(p, x, 1.);
    p = fma(p, x, 1.);
    return __builtin_ldexp(p, (int)i);
}
// the 32-bit logarithm, and what it leaves over: for r = v / 2^y - 1, below
// 2^-18, ln v = y ln 2 + r - r^2 / 2 + r^3 / 3. For normal 32-bit v.
DEV double log_d(double v) {
    const double y = __builtin_amdgcn_logf((float)v);
    const double r = fma(v, exp2_d(-y), -1.);
    return fma(y, 0.6931471805599453, r - r * r * (0.5 - r * (1. / 3.)));
}

// sums of probabilities up to this one count as none
#define VOCAB_NO_MASS 1e-300

struct RowStat {
    float m;           // largest logit, 0 where there is none
    double s, t;       // against m*c itself
    double delta;      // m*c less its rounded value: 2^(x*c - mc) is
                       // 2^delta times too large
};

// one wave joins a row's stretches, each lane's in order, in 64 bits
DEV float4 first_part(const float4 *p, int nseg, int lane) {
    return lane < nseg ? p[lane] : make_float4(-INFINITY, 0.f, 0.f, 0.f);
}
DEV RowStat join_parts(float4 first, const float4 *p, int nseg, float c,
                       int lane) {
    float m = first.x;
    for (int i = lane + WAVE; i < nseg; i += WAVE) m = fmaxf(m, p[i].x);
    m = max_wave_f(m);
    RowStat st;
    st.m = m == -INFINITY ? 0.f : m;
    const float mc = st.m * c;
    const double exact = (double)st.m * c;
    st.delta = by_product(mc) ? exact - mc : 0.;
    double s = 0, t = 0;
    for (int i = lane; i < max(nseg, WAVE); i += WAVE) {
        const float4 q = i == lane ? first : i < nseg ? p[i] : first_part(p, 0, 0);
        const float qm = q.x == -INFINITY ? 0.f : q.x;
        // against each stretch's own rounded reference, where there is one
        const float qc = qm * c;
        double d = (by_product(qc) ? (double)qc : (double)qm * c) - exact;
        // adds nothing, but NaN stays NaN
        if (q.x == -INFINITY || d < -300) d = -300;
        const double f = exp2_d(d);
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
    static DEV float value(u32 order) {
        const u32 b = order << LOW;
        return __uint_as_float(b & 0x80000000u ? b ^ 0x80000000u
                                               : ~(b | ((1u << LOW) - 1)));
    }
};

#define GROUPS (VOCAB_MAX_K + VOCAB_MAX_K / 2)  // groups looked into at most

#define BINS (4 * BLOCK)

struct TopShared {
    u64 key[CAP];              // (order, ~index) of the candidates
    int group[GROUPS];         // groups that can hold alternatives
    u32 bin[BINS];             // counts of maxima
    int4 count[2][WAVES];      // of block_count, two turns
    int ties[32 * WAVES];
    u32 top[WAVES];
    int total[WAVES];
    u32 bound;
    int n_group, n_key, reach;
};

// sums over the workgroup of three numbers that each wave has. `turn`
// alternates between calls, so one barrier is enough.
DEV int3 block_count(int a, int b, int c, TopShared &sh, int &turn) {
    if (threadIdx.x % WAVE == 0)
        sh.count[turn][threadIdx.x / WAVE] = make_int4(a, b, c, 0);
    __syncthreads();
    int3 n = make_int3(0, 0, 0);
#pragma unroll
    for (int w = 0; w < WAVES; ++w) {
        const int4 o = sh.count[turn][w];
        n.x += o.x;
        n.y += o.y;
        n.z += o.z;
    }
    turn ^= 1;
    return n;
}

// The largest bound, by `bits` bits from the top, that at least `least` keys
// reach, two bits a turn; stops early where no more than `most` reach it.
// counter(a, b, c) gives a wave's numbers of keys >= a, >= b and >= c. `reach`
// starts with how many reach 0 and ends with how many reach the bound.
template <typename F>
DEV u32 search_bound(int bits, int least, int most, int &reach, TopShared &sh,
                     int &turn, F counter) {
    u32 bound = 0;
#pragma unroll 1
    for (int shift = (bits - 1) & ~1; shift >= 0; shift -= 2) {
        // of an odd number of bits the first turn has only one
        const bool two = shift + 1 < bits;
        int3 n = counter(bound + (1u << shift), bound + (2u << shift),
                         bound + (3u << shift));
        n = block_count(n.x, two ? n.y : 0, two ? n.z : 0, sh, turn);
        const int step = n.z >= least ? 3 : n.y >= least ? 2
                         : n.x >= least                  ? 1 : 0;
        bound += (u32)step << shift;
        reach = step == 3 ? n.z : step == 2 ? n.y : step == 1 ? n.x : reach;
        if (reach <= most) break;
    }
    return bound;
}

// inclusive sum over the lanes up to this one
DEV int scan_wave(int v) {
    v += __builtin_amdgcn_update_dpp(0, v, 0x111, 0xf, 0xf, true);  // row_shr:1
    v += __builtin_amdgcn_update_dpp(0, v, 0x112, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x114, 0xf, 0xf, true);
    v += __builtin_amdgcn_update_dpp(0, v, 0x118, 0xf, 0xf, true);
    // the last lane of each row of 16 to the next, of each half to the next
    v += __builtin_amdgcn_update_dpp(0, v, 0x142, 0xa, 0xf, false);
    v += __builtin_amdgcn_update_dpp(0, v, 0x143, 0xc, 0xf, false);
    return v;
}

// The same bound from one count of how far keys are below the largest, in
// steps of a bfloat16 (eight octaves: BINS = 1024): clear, add, find.
template <typename T, int NG>
DEV u32 bins_clear(const u32 (&key)[NG], TopShared &sh) {
    constexpr int FINE = 16 - Order<T>::LOW;
    const int tid = threadIdx.x;
    u32 top = 0;
#pragma unroll
    for (int i = 0; i < NG; ++i) top = max(top, key[i]);
    top >>= FINE;  // below 2^31 now: signed comparison serves
    top = (u32)max_wave((int)top);
    if (tid % WAVE == 0) sh.top[tid / WAVE] = top;
    *(int4 *)&sh.bin[tid * 4] = make_int4(0, 0, 0, 0);
    if (tid == 0) sh.reach = 0;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WAVES; ++w) top = max(top, sh.top[w]);
    return top;
}
template <typename T> DEV void bins_add(u32 key, u32 top, TopShared &sh) {
    const u32 below = top - (key >> (16 - Order<T>::LOW));
    if (key && below < BINS) atomicAdd(&sh.bin[below], 1u);
}
// False where fewer than K keys are that near, or where more than `most`
// reach the K-th's step and the type has finer ones.
template <typename T>
DEV bool bins_find(int K, int most, u32 top, u32 &bound, int &reach,
                   TopShared &sh) {
    constexpr int FINE = 16 - Order<T>::LOW;
    const int tid = threadIdx.x, lane = tid % WAVE, wid = tid / WAVE;
    __syncthreads();
    const int4 b = *(const int4 *)&sh.bin[tid * 4];
    const int own = b.x + b.y + b.z + b.w, upto = scan_wave(own);
    if (lane == WAVE - 1) sh.total[wid] = upto;
    __syncthreads();
    int before = upto - own;
#pragma unroll
    for (int w = 0; w < WAVES; ++w)
        if (w < wid) before += sh.total[w];
    if (before < K && before + own >= K) {
        // the K-th is one of this thread's four
        int n = before + b.x, at = 0;
        if (n < K) { n += b.y; at = 1; }
        if (n < K) { n += b.z; at = 2; }
        if (n < K) { n += b.w; at = 3; }
        sh.bound = (top - (tid * 4 + at)) << FINE;
        sh.reach = n;
    }
    __syncthreads();
    if (sh.reach == 0 || (FINE > 0 && sh.reach > most)) return false;
    bound = sh.bound;
    reach = sh.reach;
    return true;
}

// The K largest of a row, (value down, index up), from its groups' maxima.
// The K groups of the largest (maximum, lowest index) hold them all: each of
// these has a token at least as good as any token of the others. So a bound
// is searched that between K and 3/2 K (or 16 more) groups reach, or, where
// maxima are equal, exactly the K-th one, and then the first groups of those
// that equal it. Tokens of these groups that reach the bound are the
// candidates, hardly more than K in a row without structure; each one's rank
// is the number of better ones. Where more than CAP reach it (groups with
// many large tokens, or a vocabulary of few groups), a higher bound is
// searched among the tokens themselves, and, where one value alone has too
// many, a bound on the index. The whole takes NG maxima per thread.
//
// What bounds it is latency: barriers, and the groups' loads, of which
// AHEAD vectors per thread are under way together (waves wait in 61 % of their
// cycles). 4096 rows of 128257 with 64 alternatives 34-41 us (a search of the
// bound two bits at a time, without the bins, and loads one by one: 94), one
// row 6 us, 512 rows of 102400 fp32 with 128 alternatives 15-16 us.
template <typename T, int NG>
DEV void top_alternatives(const T *row, long g_V, int before, int G,
                          const u32 (&key)[NG], int K, TopShared &sh,
                          float *top_lp, long *top_ids) {
    constexpr int N = Vec<T>::N, LPG = GROUP / N;
    constexpr int AHEAD = 4;  // 8 and 16 were no faster
    const int tid = threadIdx.x, lane = tid % WAVE, wid = tid / WAVE;
    int turn = 0;
    if (tid == 0) sh.n_group = sh.n_key = 0;
    u32 bound = Order<T>::of(-INFINITY);  // 0 are keys of no group
    int reach = G;  // how many groups reach it
    const int most = min(K + max(K / 2, 16), GROUPS);
    const u32 top = bins_clear<T, NG>(key, sh);
    if (G > most) {
#pragma unroll
        for (int i = 0; i < NG; ++i) bins_add<T>(key[i], top, sh);
        if (!bins_find<T>(K, most, top, bound, reach, sh))
            bound = search_bound(Order<T>::BITS, K, most, reach, sh, turn,
                                 [&](u32 a, u32 b, u32 c) {
                                     int3 n = make_int3(0, 0, 0);
#pragma unroll
                                     for (int i = 0; i < NG; ++i) {
                                         n.x += __popcll(__ballot(key[i] >= a));
                                         n.y += __popcll(__ballot(key[i] >= b));
                                         n.z += __popcll(__ballot(key[i] >= c));
                                     }
                                     return n;
                                 });
    }
    if (reach > most) {
        // `bound` is the K-th maximum: of the groups that equal it, those of
        // lowest index
        int above = 0;
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            above += __popcll(__ballot(key[i] > bound));
            const int ties = __popcll(__ballot(key[i] == bound));
            if (lane == 0) sh.ties[i * WAVES + wid] = ties;
        }
        const int quota = K - block_count(above, 0, 0, sh, turn).x;
        // how many such groups come before each wave's i-th 64
        if (wid == 0) {
            int run = 0;
#pragma unroll
            for (int i = 0; i < NG * WAVES; i += WAVE) {
                const bool on = i + lane < NG * WAVES;
                const int own = on ? sh.ties[i + lane] : 0;
                const int upto = scan_wave(own);
                if (on) sh.ties[i + lane] = run + upto - own;
                run += lane_i(upto, WAVE - 1);
            }
        }
        __syncthreads();
#pragma unroll
        for (int i = 0; i < NG; ++i) {
            const u64 ties = __ballot(key[i] == bound);
            const int nth = sh.ties[i * WAVES + wid] +
                            __popcll(ties & ((1ull << lane) - 1));
            if (key[i] > bound || (key[i] == bound && nth < quota))
                sh.group[atomicAdd(&sh.n_group, 1)] = i * BLOCK + tid;
        }
        reach = K;
    } else {
        int own = 0;
#pragma unroll
        for (int i = 0; i < NG; ++i) own += key[i] >= bound;
        // one request for slots per wave
        const int upto = scan_wave(own);
        int slot = 0;
        if (lane == WAVE - 1) slot = atomicAdd(&sh.n_group, upto);
        slot = lane_i(slot, WAVE - 1) + upto - own;
#pragma unroll
        for (int i = 0; i < NG; ++i)
            if (key[i] >= bound) sh.group[slot++] = i * BLOCK + tid;
    }
    __syncthreads();
    // as many as were entered (of a row with NaN it can be fewer)
    reach = sh.n_group;
    const int slots = reach * LPG, V = (int)g_V;
    auto where = [&](int i) {
        const int slot = i + tid;
        return slot < slots
                   ? sh.group[slot / LPG] * GROUP + slot % LPG * N - before
                   : V;
    };
    // load_vec in two halves, so that loads can be under way together (of
    // at least one vector of tokens)
    auto nearest = [&](int at) {
        Vec<T> v;
        v.load(row + min(max(at, 0), V - N));
        return v;
    };
    auto moved = [&](Vec<T> v, int at) {
        const int by = min(max(at - min(max(at, 0), V - N), -N), N);
        if (__ballot(by != 0)) move_vec(v, by);
        return v;
    };
    auto vector = [&](int at) { return moved(nearest(at), at); };
    // candidates into LDS, one request for slots per vector that has any;
    // compared as floats, of which -0 equals 0
    u32 index_bound = 0xffffffffu;
    auto collect = [&](const Vec<T> &v, int at) {
        const float low = Order<T>::value(bound);
        u32 take = 0;
#pragma unroll
        for (int k = N - 1; k >= 0; --k)
            take = take << 1 | (v.get(k) >= low ? 1 : 0);
        take &= (1u << min(max(V - at, 0), N)) - 1;
        take &= ~0u << min(max(-at, 0), N);
        if (index_bound != 0xffffffffu) {
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (v.get(k) == low && (u32)at + k >= index_bound)
                    take &= ~(1u << k);
        }
        if (take) {
            int slot = atomicAdd(&sh.n_key, __popc(take));
            do {
                const int k = __ffs(take) - 1;
                take &= take - 1;
                if (slot < CAP)
                    sh.key[slot] = (u64)Order<T>::of(v.pick(k)) << 32 |
                                   ~((u32)at + k);
                ++slot;
            } while (take);
        }
    };
    auto collect_all = [&]() {
#pragma unroll 1
        for (int i0 = 0; i0 < slots; i0 += AHEAD * BLOCK) {
            Vec<T> v[AHEAD];
            int at[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) {
                at[i] = where(i0 + i * BLOCK);
                if (i0 + i * BLOCK < slots) v[i] = nearest(at[i]);
            }
#pragma unroll
            for (int i = 0; i < AHEAD; ++i)
                if (i0 + i * BLOCK < slots) collect(moved(v[i], at[i]), at[i]);
        }
    };
    if (V < N) {
        if (tid < V)
            sh.key[tid] = (u64)Order<T>::of(to_f(row[tid])) << 32 | ~(u32)tid;
        if (tid == 0) sh.n_key = V;
    } else if (G > most || V <= CAP) {
        collect_all();
    } else {
        // a vocabulary of few groups: their maxima have told nothing
        if (tid == 0) sh.n_key = CAP + 1;
    }
    __syncthreads();
    int n = sh.n_key;
    if (n > CAP) {
        // the wave's numbers of tokens of which the three predicates hold
        auto count = [&](auto a, auto b, auto c) {
            int3 n = make_int3(0, 0, 0);
#pragma unroll 1
            for (int i = 0; i < slots; i += BLOCK) {
                const int at = where(i);
                const Vec<T> x = vector(at);
#pragma unroll
                for (int k = 0; k < N; ++k) {
                    const bool in = at + k >= 0 && at + k < V;
                    const u32 order = Order<T>::of(x.get(k));
                    const u32 index = (u32)at + k;
                    n.x += __popcll(__ballot(in && a(order, index)));
                    n.y += __popcll(__ballot(in && b(order, index)));
                    n.z += __popcll(__ballot(in && c(order, index)));
                }
            }
            return n;
        };
        auto never = [](u32, u32) { return false; };
        auto count_above = [&]() {
            const int3 c = count(
                [&](u32 order, u32) { return order > bound; }, never, never);
            return block_count(c.x, 0, 0, sh, turn).x;
        };
        // a count of the tokens themselves, as of the maxima before
        bins_clear<T, NG>(key, sh);
#pragma unroll 1
        for (int i = 0; i < slots; i += BLOCK) {
            const int at = where(i);
            const Vec<T> x = vector(at);
#pragma unroll
            for (int k = 0; k < N; ++k)
                if (at + k >= 0 && at + k < V)
                    bins_add<T>(Order<T>::of(x.get(k)), top, sh);
        }
        int above = -1;
        if (!bins_find<T>(K, CAP, top, bound, n, sh)) {
            // fewer than K above the bound: it is the K-th value itself, as
            // where a mask leaves fewer than K tokens
            above = count_above();
            if (above < K)
                n = CAP + 1;
            else
                bound = search_bound(
                    Order<T>::BITS, K, CAP, n, sh, turn,
                    [&](u32 a, u32 b, u32 c) {
                        return count(
                            [&](u32 order, u32) { return order >= a; },
                            [&](u32 order, u32) { return order >= b; },
                            [&](u32 order, u32) { return order >= c; });
                    });
        }
        if (n > CAP && (above < 0 || above >= K)) above = count_above();
        if (n > CAP) {
            // more than CAP tokens with those that share the K-th value: of
            // these the first ones, `need` or as many more as are ranked too.
            // Two bits of the index a pass (3320 rows of 1570 fp32 of which
            // 5 % are not masked, 128 alternatives: 82 us, one bit a pass and
            // a search of the value before it 280)
            const int need = K - above;
            u32 from = 0;  // fewer than `need` come before it
#pragma unroll 1
            for (int shift = (31 - __clz(V)) & ~1; shift >= 0; shift -= 2) {
                const u32 step = 1u << shift;
                int3 c = count(
                    [&](u32 order, u32 index) {
                        return order == bound && index < from + step;
                    },
                    [&](u32 order, u32 index) {
                        return order == bound && index < from + 2 * step;
                    },
                    [&](u32 order, u32 index) {
                        return order == bound && index < from + 3 * step;
                    });
                c = block_count(c.x, c.y, c.z, sh, turn);
                const int m = c.x >= need ? c.x : c.y >= need ? c.y : c.z;
                const u32 steps = c.x >= need   ? 0
                                  : c.y >= need ? 1 : c.z >= need ? 2 : 3;
                from += steps * step;
                index_bound = from + step;  // enough come before it
                if (steps < 3 && above + m <= CAP) break;
            }
        }
        if (tid == 0) sh.n_key = 0;
        __syncthreads();
        collect_all();
        __syncthreads();
        n = sh.n_key;
    }
    // four lanes count the better ones of each candidate, a quarter each;
    // keys of 0 stand behind the candidates up to a multiple of 32
    if (tid < 32 && n + tid < CAP) sh.key[n + tid] = 0;
    __syncthreads();
    for (int i = tid / 4; i < (n + 3) / 4 * 4; i += BLOCK / 4) {
        const u64 mine = sh.key[min(i, CAP - 1)];
        int rank = 0;
        for (int j = tid % 4; j < n; j += 32)
#pragma unroll
            for (int k = 0; k < 8; ++k) rank += sh.key[j + 4 * k] > mine;
        rank += dpp_i<DPP_XOR1>(rank);
        rank += dpp_i<DPP_XOR2>(rank);
        if (i < n && rank < K && tid % 4 == 0) {
            top_ids[rank] = (long)(u32)~(u32)mine;
            top_lp[rank] = Order<T>::value((u32)(mine >> 32));
        }
    }
}

struct RowOut {
    double m, ln_s;
    bool none, bad;  // no finite logit; NaN or +inf among them
};

// a row's given token, its logit, and its first stretches: asked for early
template <typename T> struct RowIn {
    float4 first;
    float x;
    bool inside;  // the token is in the vocabulary
    DEV RowIn(const VocabRows &g, const float4 *part, int r,
              const long *tokens, int lane) {
        const long tok = tokens ? tokens[r] : -1;
        inside = tok >= 0 && tok < g.V;
        first = first_part(part + (long)r * g.nseg, g.nseg, lane);
        x = inside ? to_f(row_ptr<T>(g, r)[tok]) : 0.f;
    }
};

// One wave: a row's log probability, entropy and stat[r] =
// (m, 1/s, H - ln s, 0) against the rounded m*c, what the gradient needs;
// 1/s is 0 where the row has no finite logit.
template <typename T>
DEV RowOut logprobs_row(const RowIn<T> &in, const VocabRows &g,
                        const float4 *part, int r, float c, double inv_t,
                        float *logprobs, float *entropy, float4 *stat,
                        int lane) {
    const RowStat st =
        join_parts(in.first, part + (long)r * g.nseg, g.nseg, c, lane);
    RowOut o;
    o.m = st.m;
    o.none = st.s == 0;
    o.bad = !(st.s < INFINITY);
    o.ln_s = log_d(st.s);
    if (lane == 0) {
        if (logprobs) {
            float lp = NAN;
            if (in.inside && !o.bad)
                lp = o.none ? -INFINITY
                            : (float)(((double)in.x - o.m) * inv_t - o.ln_s);
            logprobs[r] = lp;
        }
        const double ln2 = 0.6931471805599453, mean = st.t / st.s;
        entropy[r] = o.none ? 0.f
                     : o.bad ? NAN : (float)(o.ln_s - ln2 * mean);
        stat[r] = make_float4(
            st.m, o.none ? 0.f : (float)(exp2_d(-st.delta) / st.s),
            o.none ? 0.f : (float)(-ln2 * (mean + st.delta)), 0.f);
    }
    return o;
}

// without alternatives: one wave per row, 7-8 us for 8192 rows; a workgroup
// per row, with its barriers, took 41
template <typename T>
__global__ __launch_bounds__(BLOCK) void logprobs_join(
    VocabRows g, u32 first, const float4 *__restrict__ part,
    const long *__restrict__ tokens, long ignore, float c, double inv_t,
    float *__restrict__ logprobs, float *__restrict__ entropy,
    float4 *__restrict__ stat) {
    const int lane = threadIdx.x % WAVE;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const u32 r = first + blockIdx.x * WAVES + wid;
    if (r >= (u32)g.rows) return;
    if (tokens && tokens[r] == ignore) {
        if (lane == 0) {
            logprobs[r] = 0.f;
            entropy[r] = 0.f;
            stat[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        return;
    }
    const RowIn<T> in(g, part, (int)r, tokens, lane);
    logprobs_row(in, g, part, (int)r, c, inv_t,
                 tokens ? logprobs : nullptr, entropy, stat, lane);
}

// with alternatives: one workgroup per row, NG group maxima per thread
template <typename T, int NG>
__global__ __launch_bounds__(BLOCK) void logprobs_top_join(
    VocabRows g, u32 first, const float4 *__restrict__ part,
    const typename Pattern<T>::type *__restrict__ gmax, const long *__restrict__ tokens,
    long ignore, int K, float c, double inv_t, float *__restrict__ logprobs,
    float *__restrict__ entropy, float *__restrict__ top_lp,
    long *__restrict__ top_ids, float4 *__restrict__ stat) {
    constexpr int GPS = WAVE * NVEC * Vec<T>::N / GROUP;  // per stretch
    __shared__ TopShared sh;
    __shared__ RowOut joined;
    __shared__ float lp[VOCAB_MAX_K];
    __shared__ long id[VOCAB_MAX_K];
    const int lane = threadIdx.x % WAVE;
    const int r = (int)(first + blockIdx.x);
    float *lp_out = top_lp + (long)r * K;
    long *id_out = top_ids + (long)r * K;
    // asked for before the token is known: a row left out has none, but
    // the space is there
    typename Pattern<T>::type gm[NG];
    const T *row = row_ptr<T>(g, r);
    const int before = before_row(row, sizeof(T), g.line);
    const int G = (int)((g.V + before + GROUP - 1) / GROUP);
#pragma unroll
    for (int i = 0; i < NG; ++i) {
        const int k = i * BLOCK + threadIdx.x;
        gm[i] = gmax[(long)r * g.nseg * GPS + min(k, G - 1)];
    }
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
        return;
    }
    u32 key[NG];
#pragma unroll
    for (int i = 0; i < NG; ++i)
        key[i] = i * BLOCK + (int)threadIdx.x < G ? Order<T>::of(from_pattern<T>(gm[i])) : 0;
    const RowIn<T> in(g, part, r, tokens, lane);
    top_alternatives<T, NG>(row, g.V, before, G, key, K, sh, lp, id);
    // the first wave joins, for all: here, where nothing else is held
    if (threadIdx.x < WAVE) {
        const RowOut own =
            logprobs_row(in, g, part, r, c, inv_t, tokens ? logprobs : nullptr,
                         entropy, stat, lane);
        if (lane == 0) joined = own;
    }
    __syncthreads();
    const RowOut o = joined;
    for (int k = threadIdx.x; k < K; k += BLOCK) {
        lp_out[k] = o.bad    ? NAN
                    : o.none ? -INFINITY
                             : (float)(((double)lp[k] - o.m) * inv_t - o.ln_s);
        id_out[k] = o.bad ? -1 : id[k];
    }
}

// One wave per row, up to VOCAB_MAX_K / 64 entries per lane. The gradient of a
// student's logit for a loss that counts 1 (and T = 1) is
//   p_j mass - q_j              of a token that the teacher lists,
//   p_j (mass - q_rest/p_rest)  of another, with q_rest = 0 without bucket.
// entry[r, k] = (id, the former), each token once: -1 where absent or not the
// token's first. stat[r] = (m, a, live, 0), where the latter is a 2^(x*c - mc)
// against the largest of the others: p_rest can be far below what 32 bits
// hold. live is 0 where the row has no gradient.
//
// What bounds it is the latency of the entries' logits, which lie anywhere
// (waves wait in 71 % of their cycles): 8192 rows with 128 entries 30-31 us, 4096
// with 64 entries 12 us.
template <typename T>
__global__ __launch_bounds__(BLOCK) void distill_join(
    VocabRows g, u32 first, const float4 *__restrict__ part,
    const float *__restrict__ tlp, const long *__restrict__ ids, int K,
    int bucket, float c, double inv_t, float *__restrict__ loss,
    int2 *__restrict__ entry, float4 *__restrict__ stat) {
    constexpr int EPL = VOCAB_MAX_K / WAVE;
    constexpr int HASH = 2 * VOCAB_MAX_K;  // never more than half full
    __shared__ int seen[WAVES][HASH];
    const int lane = threadIdx.x % WAVE;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    const u32 r = first + blockIdx.x * WAVES + wid;
    if (r >= (u32)g.rows) return;
    const T *row = row_ptr<T>(g, (int)r);
    const float4 *parts = part + (long)r * g.nseg;
    const float4 first_of = first_part(parts, g.nseg, lane);
    int id[EPL];  // -1 where absent or outside
    float l[EPL], x[EPL];
    double q[EPL], total = 0.;
    bool any = false, wrong = false;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
        const int k = e * WAVE + lane;
        const long i = k < K ? ids[(long)r * K + k] : -1;
        l[e] = k < K ? tlp[(long)r * K + k] : 0.f;
        any |= i >= 0;
        wrong |= i >= g.V;
        // (the low half of an id below -2^31 can be any number)
        id[e] = i >= 0 && i < g.V ? (int)i : -1;
        if (i < 0) l[e] = -INFINITY;
    }
#pragma unroll
    for (int e = 0; e < EPL; ++e) x[e] = id[e] >= 0 ? to_f(row[id[e]]) : 0.f;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
        q[e] = e * WAVE < K ? exp2_d(l[e] * 1.4426950408889634) : 0.;
        total += q[e];
    }
    any = __ballot(any) != 0;
    wrong = __ballot(wrong) != 0;
    total = sum_wave_d(total);
    double q_rest = 0., mass = total;
    if (bucket) {
        q_rest = total < 1. ? 1. - total : 0.;
        mass = total + q_rest;
    }
    if (!any || (!bucket && total <= VOCAB_NO_MASS)) {
#pragma unroll
        for (int e = 0; e < EPL; ++e)
            if (e * WAVE + lane < K)
                entry[(long)r * K + e * WAVE + lane] = make_int2(-1, 0);
        if (lane == 0) {
            loss[r] = 0.f;
            stat[r] = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        return;
    }

    // which entries are a token's first? By a table of the tokens seen.
    for (int i = lane; i < HASH; i += WAVE) seen[wid][i] = -1;
    wave_sync();
    bool own[EPL], twice = false;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
        own[e] = id[e] >= 0;
        if (own[e]) {
            u32 at = ((u32)id[e] * 2654435761u) / (~0u / HASH + 1);
            int old;
            while ((old = atomicCAS(&seen[wid][at], -1, id[e])) != -1 &&
                   old != id[e])
                at = (at + 1) % HASH;
            twice |= old != -1;
        }
    }
    if (!bucket) {
        mass = total / total;  // NaN stays NaN
        const double scale = 1. / total;
#pragma unroll
        for (int e = 0; e < EPL; ++e) q[e] *= scale;
    }
    double weight[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) weight[e] = q[e];
    if (__ballot(twice)) {
        // rare: the first in order has the sum of all, in order
#pragma unroll
        for (int e = 0; e < EPL; ++e) {
            double sum = 0.;
            bool before = false;
#pragma unroll
            for (int o = 0; o < EPL; ++o) {
#pragma unroll 1
                for (int i = 0; i < WAVE; ++i)
                    if (lane_i(id[o], i) == id[e]) {
                        sum += lane_d(q[o], i);
                        before |= o * WAVE + i < e * WAVE + lane;
                    }
            }
            weight[e] = sum;
            own[e] &= !before;
        }
    }
    // with bucket, of the tokens that are not listed
    const RowStat st = join_parts(first_of, parts, g.nseg, c, lane);
    double m = st.m, s = st.s, share = 1.;
    if (bucket) {
        // and the listed ones, each once, against the largest of all
        float high = -INFINITY;
#pragma unroll
        for (int e = 0; e < EPL; ++e)
            if (own[e]) high = fmaxf(high, x[e]);
        high = max_wave_f(high);
        if (st.s == 0) m = high == -INFINITY ? 0. : high;
        else m = fmax(m, (double)high);
        share = exp2_d((st.m - m) * c);
        double s_in = 0.;
#pragma unroll
        for (int e = 0; e < EPL; ++e)
            if (own[e]) s_in += exp2_d((x[e] - m) * c);
        s = sum_wave_d(s_in) + (st.s == 0 ? 0. : st.s * share);
    }
    const bool none = s == 0, bad = !(s < INFINITY), nan = bad || wrong;
    // entries that cover every token with mass leave no room for the rest;
    // what 32-bit log probabilities leave over by rounding then counts as
    // none
    const double p_rest = bucket && !none && st.s != 0 ? st.s * share / s : 0.;
    const bool open = q_rest > 0. && p_rest > VOCAB_NO_MASS;
    const double ratio = open ? q_rest / p_rest : 1.;
    const double ln_s = log_d(s), ln = log(bucket ? ratio : total);
    const double scale = none ? 0. : mass / s;
    double sum = 0.;
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
        if (e * WAVE >= K) break;
        const double lp = none || x[e] == -INFINITY
                              ? -INFINITY : (x[e] - m) * inv_t - ln_s;
        if (id[e] >= 0 && q[e] != 0.)
            sum += q[e] * ((l[e] - (bucket ? 0. : ln)) - lp);
        const double d = exp2_d((x[e] - m) * c) * scale;
        if (e * WAVE + lane < K)
            entry[(long)r * K + e * WAVE + lane] =
                make_int2(own[e] ? id[e] : -1,
                          __float_as_int(nan ? NAN : (float)(d - weight[e])));
    }
    sum = sum_wave_d(sum);
    if (open) sum += q_rest * ln;
    else if (bucket && q_rest > 0x1p-20) sum = INFINITY;
    if (lane == 0) {
        double a = mass * share / s;
        if (open) a -= q_rest / st.s;
        if (st.s == 0) a = 0.;
        loss[r] = nan ? NAN : (float)sum;
        stat[r] = make_float4(st.m, nan ? NAN : (float)(a * exp2_d(-st.delta)),
                              nan || !none ? 1.f : 0.f, 0.f);
    }
}

// ---- gradients -------------------------------------------------------------
// d x_j = p_j (a + b ln(p_j s)) + what is given for single tokens (in place of
// it for a teacher's entries), one wave per stretch, in one pass over packed
// registers: a product, an exponential and one or three more operations per
// element beside 4 or 8 bytes.
//
// Single tokens (the given one, alternatives with a gradient, a teacher's
// entries): those of the stretch are marked in LDS, a bit and a value each,
// while the stretch's loads are under way, and only vectors that hold one
// look there. Entries name a token once, the forward pass has seen to that.
//
// What bounds it is the memory, which takes reads and writes together best
// from few waves with little each: the values' place in LDS (33 KB) leaves
// four workgroups to a CU, and a stretch is half as long as in the forward
// pass. Copying alone took 765 us with 8 vectors per lane and eight
// workgroups, 703 us with 4 and four, 669 us with rows at cache lines. The
// gradient with a teacher's 128 entries takes 632-649 us (6.5-6.6 TB/s), of log
// probabilities of a batch cut to its first S positions, half of whose rows
// lie otherwise within their lines than the gradient's do, 689-695 us. Half the
// workgroups again (960 us) and half the vectors (1137 us) were slower.
template <typename T, bool DISTILL, bool STREAM_IN, bool STREAM_OUT>
__global__ __launch_bounds__(BLOCK) void vocab_grad(
    VocabRows g, u32 nseg, u32 first, float c, float inv_t,
    const float4 *__restrict__ stat, const float *__restrict__ d_row,
    const float *__restrict__ d_entropy, const long *__restrict__ tokens,
    long ignore, const int2 *__restrict__ entry, const float *__restrict__ d_top,
    const long *__restrict__ ids, int K, T *__restrict__ out) {
    constexpr int N = Vec<T>::N;
    constexpr int SEG = WAVE * NGRAD * N;
    constexpr int EPL = VOCAB_MAX_K / WAVE;
    __shared__ u32 bits_all[WAVES][SEG / 32];
    __shared__ __attribute__((aligned(16))) float value_all[WAVES][SEG];
    const int lane = threadIdx.x % WAVE;
    const int wid = __builtin_amdgcn_readfirstlane(threadIdx.x / WAVE);
    u32 *bits = bits_all[wid];
    float *value = value_all[wid];
    const u32 w = first + wave_index();  // below 2^32
    if (w >= (u32)g.rows * nseg) return;
    const int r = w / nseg, seg = w - r * nseg;
    T *orow = out + (long)r * g.V;
    const T *row = row_ptr<T>(g, r);
    const long lo = (long)seg * SEG - before_row(row, sizeof(T), 127);
    const bool whole = lo >= 0 && lo + SEG <= g.V;
    // the row's numbers come by scalar loads, which nothing queues behind
    const float4 st = stat[r];
    const long tok = !DISTILL && tokens ? tokens[r] : -1;
    const float g_row = d_row ? d_row[r] : 0.f;
    const float g_ent = !DISTILL && d_entropy ? d_entropy[r] : 0.f;
    bool skip = DISTILL ? st.z == 0.f : st.y == 0.f;
    if (!DISTILL && tokens && tok == ignore) skip = true;
    if (skip) {
        const float zero[N] = {};
#pragma unroll 1
        for (int j = 0; j < NGRAD; ++j)
            store_vec<STREAM_OUT>(orow, lo + (long)(j * WAVE + lane) * N, g.V,
                                  zero, whole);
        return;
    }
    for (int i = lane; i < SEG / 32; i += WAVE) bits[i] = 0;
    // entries before the stretch: loads arrive in order
    const bool entries = DISTILL || d_top;
    int2 pair[EPL];
    long id[EPL];
    float val[EPL];
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
        // nothing is done with them here: that would wait for each
        const long k = (long)r * K + min(e * WAVE + lane, K - 1);
        pair[e] = make_int2(-1, 0);
        id[e] = -1;
        val[e] = 0.f;
        if (entries && e * WAVE < K) {
            if (DISTILL) {
                pair[e] = entry[k];
            } else {
                id[e] = ids[k];
                val[e] = d_top[k];
            }
        }
    }
    Vec<T> v[NGRAD];
    load_stretch<STREAM_IN>(row, lo, g.V, lane, v);
    u32 at[EPL];  // of the stretch, SEG or more where not in it
#pragma unroll
    for (int e = 0; e < EPL; ++e) {
        const bool on = e * WAVE + lane < K;
        if (DISTILL) {
            id[e] = pair[e].x;
            val[e] = __int_as_float(pair[e].y);
        }
        const u64 off = id[e] - lo;
        at[e] = on && off < SEG && id[e] >= 0 ? (u32)off : SEG;
        if (!on) val[e] = 0.f;
    }

    // e = 2^((x - m) c) counts k_out + k_d * exponent
    float k_out = 1.f, k_d = 0.f, scale = inv_t;
    u32 tok_at = SEG;
    if (DISTILL) {
        scale *= g_row;
    } else {
        float gs = 0.f;
        if (d_row && tokens) {
            const bool inside = tok >= 0 && tok < g.V;
            gs = inside ? g_row : NAN;
            const u64 off = tok - lo;
            if (inside && off < SEG) tok_at = (u32)off;
        }
        if (d_top) {
            float gk = 0.f;
#pragma unroll
            for (int e = 0; e < EPL; ++e) gk += val[e];
            gs += sum_wave(gk);
        }
        k_d = -g_ent;
        k_out = k_d * st.z - gs;
        k_d *= 0.69314718f;
    }

    // mark the listed tokens, and note which vectors hold one
    u32 hit = 0;
    if (entries || tok_at < SEG) {
        wave_sync();  // the bits are clear
        bool found = false;  // the given token among the alternatives
        if (entries) {
#pragma unroll
            for (int e = 0; e < EPL; ++e)
                if (at[e] < SEG) {
                    if (!DISTILL && at[e] == tok_at) {
                        val[e] += g_row;
                        found = true;
                    }
                    atomicOr(&bits[at[e] >> 5], 1u << (at[e] & 31));
                    value[at[e]] = val[e] * scale;
                    hit |= 1u << (at[e] / (WAVE * N));
                }
        }
        if (!DISTILL && tok_at < SEG && __ballot(found) == 0 && lane == 0) {
            atomicOr(&bits[tok_at >> 5], 1u << (tok_at & 31));
            value[tok_at] = g_row * scale;
            hit |= 1u << (tok_at / (WAVE * N));
        }
        wave_sync();
        hit = or_wave(hit);
    }

    const float mc = st.x * c, u = st.y * scale;
    const float u_out = k_out * u, u_d = k_d * u;
    auto one = [&](const Vec<T> &x, int j, auto diff) {
        float f[N];
        const bool listed = hit >> j & 1;
        const int p = (j * WAVE + lane) * N;
        const u32 in = listed ? bits[p >> 5] >> (p & 31) : 0;
#pragma unroll
        for (int i = 0; i < N; ++i) {
            const float d = diff(x.get(i));
            // 2^-300 is 0, and (-inf) * 0 would be NaN
            const float k =
                DISTILL ? u_out : fmaf(u_d, fmaxf(d, -300.f), u_out);
            f[i] = exp2_hw(d) * k;
        }
        if (listed) {
#pragma unroll
            for (int i = 0; i < N; ++i)
                if (in >> i & 1)
                    f[i] = DISTILL ? value[p + i] : f[i] + value[p + i];
        }
        store_vec<STREAM_OUT>(orow, lo + p, g.V, f, whole);
    };
    if (by_product(mc)) {
#pragma unroll
        for (int j = 0; j < NGRAD; ++j)
            one(v[j], j, [&](float x) { return fmaf(x, c, -mc); });
    } else {
#pragma unroll 1
        for (int j = 0; j < NGRAD; ++j)
            one(load_vec(row, lo + (long)(j * WAVE + lane) * N, g.V), j,
                [&](float x) { return (x - st.x) * c; });
    }
}

// ---- launches --------------------------------------------------------------
// Whole stretches go past the caches (non-temporal) where they are too many
// for the 256 MB that stand before the memory, and through them where what
// ran before or comes after finds them there. Forward, backward and a sum of
// the gradient, on logits just written, bf16, with ordinary loads and stores
// / loads past the caches / both past them, in us:
//    64 MB   70 /  71 /  80      128 MB  108 / 114 / 131
//   192 MB  169 / 150 / 176      256 MB  225 / 210 / 221
//   512 MB  445 / 417 / 410     2048 MB 1598 / 1561 / 1539
#define STREAM_IN_ABOVE (144l << 20)
#define STREAM_OUT_ABOVE (384l << 20)

static long logits_bytes(const VocabRows &g, int size) {
    return (long)g.rows * g.V * size;
}

// More workgroups than MAX_GRID (threads stay far below 2^32) go in several
// launches: a loop in the kernels would keep constants and addresses in
// registers. Stretches' grids are a multiple of 8, see wave_index.
#define MAX_GRID (1l << 22)

template <typename F> static void launches(long blocks, int per, F f) {
    for (long b = 0; b < blocks; b += MAX_GRID)
        f((u32)(b * per), dim3((u32)(blocks - b < MAX_GRID ? blocks - b
                                                           : MAX_GRID)));
}
static long stretch_blocks(const VocabRows &g, u32 nseg) {
    return CDIV(CDIV((long)g.rows * nseg, (long)WAVES), 8) * 8;
}
static long row_blocks(const VocabRows &g) {
    return CDIV((long)g.rows, (long)WAVES);
}

// stretches (or groups) of a row; `shifted`: rows may begin within a line
static long vocab_stretches(long V, int size, int seg, bool shifted) {
    return CDIV(V + (shifted ? 127 / size : 0), (long)seg);
}

template <typename T, bool ENT, bool EXCL, bool GRP>
static void partials_t(const VocabRows &g, const long *tokens, long ignore,
                       const long *ids, int K, float c, float *part,
                       void *gmax, hipStream_t stream) {
    auto kernel = logits_bytes(g, sizeof(T)) > STREAM_IN_ABOVE
                      ? vocab_partials<T, ENT, EXCL, GRP, true>
                      : vocab_partials<T, ENT, EXCL, GRP, false>;
    launches(stretch_blocks(g, g.nseg), WAVES, [&](u32 first, dim3 grid) {
        hipLaunchKernelGGL(kernel, grid, dim3(BLOCK), 0, stream, g, first,
                           tokens, ignore, ids, K, c, (float4 *)part,
                           (typename Pattern<T>::type *)gmax);
    });
}

template <typename T, int NG>
static void logprobs_top_join_t(const VocabRows &g, const VocabLogprobs &a,
                                float c, hipStream_t stream) {
    launches(g.rows, 1, [&](u32 first, dim3 grid) {
        hipLaunchKernelGGL((logprobs_top_join<T, NG>), grid, dim3(BLOCK), 0,
                           stream, g, first, (const float4 *)a.part,
                           (const typename Pattern<T>::type *)a.gmax, a.tokens,
                           a.ignore, a.K, c, 1. / a.temperature, a.logprobs,
                           a.entropy, a.top_lp, a.top_ids, (float4 *)a.stat);
    });
}

template <typename T>
static void logprobs_fwd_t(const VocabRows &g, const VocabLogprobs &a,
                           hipStream_t stream) {
    const float c = (float)(1.4426950408889634 / a.temperature);
    if (a.K == 0) {
        partials_t<T, true, false, false>(g, a.tokens, a.ignore, nullptr, 0, c,
                                          a.part, nullptr, stream);
        launches(row_blocks(g), WAVES, [&](u32 first, dim3 grid) {
            hipLaunchKernelGGL((logprobs_join<T>), grid, dim3(BLOCK), 0,
                               stream, g, first, (const float4 *)a.part,
                               a.tokens, a.ignore, c, 1. / a.temperature,
                               a.logprobs, a.entropy, (float4 *)a.stat);
        });
        return;
    }
    partials_t<T, true, false, true>(g, a.tokens, a.ignore, nullptr, 0, c,
                                     a.part, a.gmax, stream);
    // maxima per thread, of a row that begins as late within a line as rows
    // can (the kernel counts groups from the line, as stretches are counted):
    // rows of 65535 bf16 have 1024 groups or 1025. More than VOCAB_MAX_TOP_V
    // are refused before
    const long groups =
        vocab_stretches(g.V, sizeof(T), GROUP, g.line != 0);
    const long per = CDIV(groups, (long)BLOCK);
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
        partials_t<T, false, true, false>(g, nullptr, 0, a.ids, a.K, c, a.part,
                                          nullptr, stream);
    else
        partials_t<T, false, false, false>(g, nullptr, 0, nullptr, 0, c,
                                           a.part, nullptr, stream);
    launches(row_blocks(g), WAVES, [&](u32 first, dim3 grid) {
        hipLaunchKernelGGL((distill_join<T>), grid, dim3(BLOCK), 0, stream, g,
                           first, (const float4 *)a.part, a.teacher_lp, a.ids,
                           a.K, a.bucket, c, 1. / a.temperature, a.loss,
                           (int2 *)a.entry,
                           (float4 *)a.stat);
    });
}

template <typename T>
static void grad_t(const VocabRows &g, const VocabGrad &a, int distill,
                   void *out, hipStream_t stream) {
    const long apart = g.stride_o | g.stride_i;  // its lowest bits are theirs
    const u32 nseg = (u32)vocab_stretches(
        g.V, sizeof(T), WAVE * NGRAD * Vec<T>::N,
        (long)(u64)g.base % 128 || apart * sizeof(T) % 128);
    const long bytes = logits_bytes(g, sizeof(T));
    auto kernel =
        bytes > STREAM_OUT_ABOVE ? (distill ? vocab_grad<T, true, true, true>
                                            : vocab_grad<T, false, true, true>)
        : bytes > STREAM_IN_ABOVE
            ? (distill ? vocab_grad<T, true, true, false>
                       : vocab_grad<T, false, true, false>)
            : (distill ? vocab_grad<T, true, false, false>
                       : vocab_grad<T, false, false, false>);
    launches(stretch_blocks(g, nseg), WAVES, [&](u32 first, dim3 grid) {
        hipLaunchKernelGGL(kernel, grid, dim3(BLOCK), 0, stream, g, nseg,
                           first, a.c, a.inv_t, (const float4 *)a.stat,
                           a.d_row, a.d_entropy, a.tokens, a.ignore,
                           (const int2 *)a.entry, a.d_top, a.ids, a.K,
                           (T *)out);
    });
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
