// k_append.cu -- packed token rows into the paged key-value cache, with the
// QK-RMSNorm and the rotation of query and key on the way.
//
// Per token row at position p, per query and key head x of 128 (the operation of
// src/cpu/qwen3_original.c:361-393, batched; without norm weights only the
// rotation):
//     y_i = w_i * (x_i / sqrtf(mean(x^2) + eps))
//     o_j      = y_j cos(a_j) - y_{j+64} sin(a_j)
//     o_{j+64} = y_j sin(a_j) + y_{j+64} cos(a_j),   a_j = p * theta^(-j/64), j < 64
// The key heads go to their page slots in the cache's type, the value heads are
// converted and stored beside them, the query heads go to q_out.
//
// Other rotations (TurnForm): the first `dim` elements of a head, as halves or as
// neighbouring pairs, cosine and sine times a gain, any frequencies.  A lane's four
// elements are chosen so that both elements of its two pairs are its own, and the
// rest of the head is dealt to the lanes beyond.
//
// A Q8_0 cache: s = max|o| / 127 over each 64 elements, codes o / s rounded half
// away from zero, with the operations of q3cu_quantize_q8 (the same codes and
// scales from the same f32 rows).  The maxima are taken over the warp by one
// instruction each; a lane stores two codes of each of its two element pairs.
//
// The angle is formed in binary64 as turns, p * (theta^(-j/64) / 2 pi) less its
// nearest whole number, so it is as exact at position 100,000 as at 0 (a
// binary32 product is off by up to 0.004 rad there); the remainder is carried
// as a pair of floats into sincospif and a first-order correction.  Sums are
// binary32; the one rounding to fewer bits is the store.
//
// Bound by memory: every element is read once and written once.  A warp takes
// one row, or with few rows a part of its heads, in batches of APPEND_HEADS
// heads of one kind: lane l holds elements 2l, 2l+1, 64+2l, 65+2l of each head,
// so both halves of a rotated pair are in one lane, a half row is one contiguous
// access, and the two angles of a lane, found once, serve all its heads.  The
// row is on its way to L2 while the warp finds its sequence, position and page.
// 4,096 rows (32/8 heads): f32 to bf16 28.2 us, 5.4 TB/s, bf16 to bf16 23.6 us, 4.3
// TB/s, f32 to f32 35.6 us, 5.7 TB/s, f32 to Q8_0 (bf16 queries) 29 us, 5.0 TB/s; one
// row: 3.0 us, into Q8_0 3.8 us.
#include "q3cu_paged.cuh"

#include <type_traits>

namespace q3 {

__device__ __forceinline__ void prefetch_l2(const void *p) { asm volatile("prefetch.global.L2 [%0];" :: "l"(p)); }

constexpr int APPEND_HEADS = 4, APPEND_WARPS = 8;
// Where part i of `parts` (at most 65,535) begins among `all` batches; a 64-bit division takes some hundred instructions.
__device__ __forceinline__ int part_of(int all, unsigned i, unsigned parts) {
    return all < 65536 ? int(unsigned(all) * i / parts) : int(uint64_t(all) * i / parts);
}

// Coherent loads: q_out may be q itself (a lane reads its elements before it stores them).
__device__ __forceinline__ float2 load_pair(const float *p) { return *reinterpret_cast<const float2 *>(p); }
__device__ __forceinline__ float2 load_pair(const uint16_t *p) {
    const uint32_t u = *reinterpret_cast<const uint32_t *>(p);
    return make_float2(bf16_to_f32(u & 0xffffu), bf16_to_f32(u >> 16));
}
// v as elements at, at + 1 of base.
enum AppendAs { AS_F32, AS_BF16, AS_Q8 };
template <AppendAs AS>
__device__ __forceinline__ void store_pair(void *base, int64_t at, float2 v) {
    if constexpr (AS == AS_BF16) *reinterpret_cast<uint32_t *>(static_cast<uint16_t *>(base) + at) = pack_bf16(v.x, v.y);
    else *reinterpret_cast<float2 *>(static_cast<float *>(base) + at) = v;
}

// Where a lane's elements lie in a head, two at lo and two at hi, and which of its two pairs are rotated: pair 0 is
// (lo, hi) and pair 1 (lo + 1, hi + 1), or with neighbouring pairs (lo, lo + 1) and (hi, hi + 1).
// WHOLE: the whole head by halves, so lo = 2 lane, hi = 64 + lo and all are rotated.
template <bool WHOLE> struct Place {
    __device__ __forceinline__ Place(int, int, bool) {}
    __device__ __forceinline__ int lo() const { return 2 * (threadIdx.x & 31); }
    __device__ __forceinline__ int hi() const { return 64 + lo(); }
    __device__ __forceinline__ int angle(int e) const { return lo() + e; }
    __device__ __forceinline__ bool turned(int) const { return true; }
    __device__ __forceinline__ bool paired() const { return false; }
};
template <> struct Place<false> {
    int lo_, hi_, half;
    bool pairs;
    __device__ __forceinline__ Place(int lane, int dim, bool p) : half(dim / 2), pairs(p) {
        const int beyond = lane - dim / 4;                   // lanes behind the rotated ones
        lo_ = pairs || beyond < 0 ? 2 * lane : dim + 2 * beyond;
        hi_ = pairs ? 64 + lo_ : beyond < 0 ? half + lo_ : dim + (HD - dim) / 2 + 2 * beyond;
    }
    __device__ __forceinline__ int lo() const { return lo_; }
    __device__ __forceinline__ int hi() const { return hi_; }
    __device__ __forceinline__ int angle(int e) const {      // which frequency, below 64
        return pairs ? (threadIdx.x & 31) + 32 * e : 2 * (threadIdx.x & 31) + e;
    }
    __device__ __forceinline__ bool turned(int e) const { return angle(e) < half; }
    __device__ __forceinline__ bool paired() const { return pairs; }
};
__device__ __forceinline__ void swap_inner(float2 &l, float2 &h) {
    const float x = l.y;
    l.y = h.x;
    h.x = x;
}

// A head's Q8_0 codes and scales from every lane's elements l (two at lo) and h (two at hi): elements `at` of base, scales
// at `scale`.
__device__ __forceinline__ void store_q8(void *base, int64_t at, float *scale, int lo, int hi, float2 l, float2 h) {
    const float a = amax_fold(amax_fold(0.0f, l.x), l.y), b = amax_fold(amax_fold(0.0f, h.x), h.y);
    const float low = fmaxf(lo < GS ? a : 0.0f, hi < GS ? b : 0.0f), high = fmaxf(lo < GS ? 0.0f : a, hi < GS ? 0.0f : b);
    // magnitudes compare as their bits do
    const Q8Scale g0 = q8_prepare(__uint_as_float(__reduce_max_sync(FULL, __float_as_uint(low))));
    const Q8Scale g1 = q8_prepare(__uint_as_float(__reduce_max_sync(FULL, __float_as_uint(high))));
    const Q8Scale gl = lo < GS ? g0 : g1, gh = hi < GS ? g0 : g1;
    // the fast codes of q8_encode_lane, a pair at a time; a lane near a tie, or of an exact group, does its four again
    uint32_t code[2];
    bool fix = gl.exact || gh.exact;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const float inv = i ? gh.inv : gl.inv;
        const f2 magic = pk2(12582912.0f, 12582912.0f), q = mul2(i ? pk2(h.x, h.y) : pk2(l.x, l.y), pk2(inv, inv));
        const f2 t = add2(q, magic), d = sub2(q, sub2(t, magic));
        float d0, d1, t0, t1;
        up2(d, d0, d1);
        up2(t, t0, t1);
        fix |= !(fabsf(d0) <= 0.49993896484375f) | !(fabsf(d1) <= 0.49993896484375f);
        code[i] = __byte_perm(__float_as_uint(t0), __float_as_uint(t1), 0x0040);
    }
    if (__builtin_expect(fix, 0)) {
        code[0] = q8_code_slow(l.x, gl.scale) | q8_code_slow(l.y, gl.scale) << 8;
        code[1] = q8_code_slow(h.x, gh.scale) | q8_code_slow(h.y, gh.scale) << 8;
    }
    uint8_t *p = static_cast<uint8_t *>(base) + at;
    *reinterpret_cast<uint16_t *>(p + lo) = uint16_t(code[0]);
    *reinterpret_cast<uint16_t *>(p + hi) = uint16_t(code[1]);
    if ((threadIdx.x & 31) == 0) *reinterpret_cast<float2 *>(scale) = make_float2(g0.scale, g1.scale);
}

// Up to APPEND_HEADS heads from x (the first head's first element), `step` elements apart where they go (`at`: the first
// one's first); turned by w if ROTATE, and normalised before if `norm` (the norm's weights are in w).
struct Turn { float2 c[2], s[2]; };                          // weight * cosine, weight * sine of both halves
template <typename E, AppendAs AS, bool ROTATE, bool WHOLE>
__device__ __forceinline__ void append_heads(const E *x, int n, bool norm, float eps, const Place<WHOLE> &place, const Turn &w,
                                             void *to, int64_t at, int64_t step, float *scale) {
    const int lo = place.lo(), hi = place.hi();
    float2 l[APPEND_HEADS], h[APPEND_HEADS];
#pragma unroll
    for (int i = 0; i < APPEND_HEADS; ++i) {
        l[i] = h[i] = make_float2(0.0f, 0.0f);
        if (i < n) {
            l[i] = load_pair(x + i * HD + lo);
            h[i] = load_pair(x + i * HD + hi);
        }
    }
    if constexpr (ROTATE) {
        float g[APPEND_HEADS] = {1.0f, 1.0f, 1.0f, 1.0f};
        if (norm) {
#pragma unroll
            for (int i = 0; i < APPEND_HEADS; ++i)
                g[i] = fmaf(l[i].x, l[i].x, fmaf(l[i].y, l[i].y, fmaf(h[i].x, h[i].x, h[i].y * h[i].y)));
#pragma unroll
            for (int o = 16; o > 0; o >>= 1)
#pragma unroll
                for (int i = 0; i < APPEND_HEADS; ++i) g[i] += __shfl_xor_sync(FULL, g[i], o);
#pragma unroll
            for (int i = 0; i < APPEND_HEADS; ++i) g[i] = rsqrtf(fmaf(g[i], 1.0f / HD, eps));
        }
#pragma unroll
        for (int i = 0; i < APPEND_HEADS; ++i) {
            if (place.paired()) swap_inner(l[i], h[i]);
            const float2 y = make_float2(g[i] * l[i].x, g[i] * l[i].y), z = make_float2(g[i] * h[i].x, g[i] * h[i].y);
            l[i] = make_float2(fmaf(y.x, w.c[0].x, -(z.x * w.s[1].x)), fmaf(y.y, w.c[0].y, -(z.y * w.s[1].y)));
            h[i] = make_float2(fmaf(y.x, w.s[0].x, z.x * w.c[1].x), fmaf(y.y, w.s[0].y, z.y * w.c[1].y));
            if constexpr (!WHOLE) {                          // the cosine is 1; a sine of 0 times infinity would be NaN
                if (!place.turned(0)) l[i].x = y.x * w.c[0].x, h[i].x = z.x * w.c[1].x;
                if (!place.turned(1)) l[i].y = y.y * w.c[0].y, h[i].y = z.y * w.c[1].y;
            }
            if (place.paired()) swap_inner(l[i], h[i]);
        }
    }
#pragma unroll
    for (int i = 0; i < APPEND_HEADS; ++i)
        if (i < n) {
            if constexpr (AS == AS_Q8) {
                store_q8(to, at + i * step, scale + i * (step / GS), lo, hi, l[i], h[i]);
            } else {
                store_pair<AS>(to, at + i * step + lo, l[i]);
                store_pair<AS>(to, at + i * step + hi, h[i]);
            }
        }
}

template <typename T, AppendAs QA, AppendAs CA, bool WHOLE>
__global__ void __launch_bounds__(APPEND_WARPS * 32, 4)
kv_append_kernel(const PagedKV c, const PagedSeqs b, int rows, const typename Elem<T>::type *q,
                 const typename Elem<T>::type *k, const typename Elem<T>::type *v, int64_t q_stride,
                 int64_t kv_stride, int n_heads, const float *__restrict__ q_norm, const float *__restrict__ k_norm,
                 const __grid_constant__ TurnFreq freq, const TurnForm form, float eps, void *q_out, uint32_t *status) {
    typedef typename Elem<T>::type E;
    __shared__ double turn[64];
    if (threadIdx.x < 64) turn[threadIdx.x] = freq.v[threadIdx.x];
    __syncthreads();
    griddep_wait();
    const int lane = threadIdx.x & 31, r = int(blockIdx.x) * APPEND_WARPS + int(threadIdx.x >> 5);
    if (r >= rows) return;
    // the row's batches: of query heads, of key heads, of value heads; this warp's are first .. last - 1
    const int qn = (n_heads + APPEND_HEADS - 1) / APPEND_HEADS, kn = (c.n_kv + APPEND_HEADS - 1) / APPEND_HEADS;
    // (into a Q8_0 cache the last ones, which take longest, begin first: 29 against 31 us for 4,096 rows; with a bf16 cache
    // that order is 1 to 2 us slower)
    const unsigned part = CA == AS_Q8 ? gridDim.y - 1 - blockIdx.y : blockIdx.y;
    const int first = part_of(qn + 2 * kn, part, gridDim.y), last = part_of(qn + 2 * kn, part + 1, gridDim.y);
    const E *qr = q + r * q_stride, *kr = k + r * kv_stride, *vr = v + r * kv_stride;
    constexpr int LINES = APPEND_HEADS * HD * int(sizeof(E)) / 128;        // 128-byte lines of a batch
    for (int i = lane + LINES * first; i < LINES * last; i += 32) {
        const int x = i / LINES, heads = x < qn ? n_heads : c.n_kv, at = x < qn ? x : x < qn + kn ? x - qn : x - qn - kn;
        const int e = at * APPEND_HEADS * HD + i % LINES * (128 / int(sizeof(E)));
        if (e < heads * HD) prefetch_l2((x < qn ? qr : x < qn + kn ? kr : vr) + e);
    }

    int pos;
    const int s = paged_row_of_warp(b, c, r, pos, status);
    if (s < 0) return;                                       // a row behind the last sequence
    if (pos < 0) return;                                     // padding, or beyond the table
    const int page = last > qn ? paged_page(b, c, s, pos, lane == 0 ? status : nullptr) : -1;
    const Place<WHOLE> place(lane, form.dim, form.pairs);
    float cs[2], sn[2];
#pragma unroll
    for (int e = 0; e < 2; ++e) {
        const double t = double(pos) * turn[place.angle(e)];
        const double half = 2.0 * (t - rint(t));             // half turns in [-1, 1]
        const float h = float(half), rest = 3.14159265f * float(half - double(h));
        float s0, c0;
        sincospif(h, &s0, &c0);
        sn[e] = fmaf(c0, rest, s0);
        cs[e] = fmaf(-s0, rest, c0);
        if constexpr (!WHOLE) {
            sn[e] = place.turned(e) ? sn[e] * form.gain : 0.0f;
            cs[e] = place.turned(e) ? cs[e] * form.gain : 1.0f;
        }
    }
    auto weighted = [&](const float *n) {
        Turn w;
        float2 f[2];
#pragma unroll
        for (int y = 0; y < 2; ++y)
            f[y] = n ? __ldg(reinterpret_cast<const float2 *>(n + (y ? place.hi() : place.lo()))) : make_float2(1.0f, 1.0f);
        if (place.paired()) swap_inner(f[0], f[1]);
#pragma unroll
        for (int y = 0; y < 2; ++y) {
            w.c[y] = make_float2(f[y].x * cs[0], f[y].y * cs[1]);
            w.s[y] = make_float2(f[y].x * sn[0], f[y].y * sn[1]);
        }
        return w;
    };
    Turn w = weighted(q_norm);
    for (int x = first; x < min(last, qn); ++x) {
        const int u = x * APPEND_HEADS;
        append_heads<E, QA, true, WHOLE>(qr + u * HD, n_heads - u, q_norm, eps, place, w, q_out,
                                         (int64_t(r) * n_heads + u) * HD, HD, nullptr);
    }
    if (page < 0) return;                                    // no keys or values here, or a bad page (flagged): none stored
    const int64_t at = paged_at(c, page, 0, pos), step = HD << c.page_shift;
    // the scales of head 0, those of head h h * (step / 64) further
    const int64_t sc = int64_t(page) * c.scale_stride + 2 * (pos & ((1 << c.page_shift) - 1));
    w = weighted(k_norm);
    for (int x = max(first, qn); x < min(last, qn + kn); ++x) {
        const int u = (x - qn) * APPEND_HEADS;
        append_heads<E, CA, true, WHOLE>(kr + u * HD, c.n_kv - u, k_norm, eps, place, w, c.k, at + u * step, step,
                                         c.k_scale + (sc + u * (step / GS)));
    }
    for (int x = max(first, qn + kn); x < last; ++x) {
        const int u = (x - qn - kn) * APPEND_HEADS;
        append_heads<E, CA, false, WHOLE>(vr + u * HD, c.n_kv - u, false, eps, place, w, c.v, at + u * step, step,
                                          c.v_scale + (sc + u * (step / GS)));
    }
}

cudaError_t launch_kv_append(const PagedKV &c, q3cu_dtype cache_dt, const PagedSeqs &b, int64_t rows, const void *q,
                             const void *k, const void *v, q3cu_dtype dt, int64_t q_stride, int64_t kv_stride,
                             int n_heads, const float *q_norm, const float *k_norm, const TurnFreq &freq,
                             const TurnForm &form, float eps, void *q_out, q3cu_dtype q_dt, uint32_t *status,
                             cudaStream_t stream, int sms) {
    // A row is split over warps while the rows alone are fewer than 32 warps per SM, and so that a warp has no more than 4
    // batches (6 of bf16 rows, whose batches are half the bytes): the warps that end last then have less to do by
    // themselves, for the angles found once more.  Whole rows a warp: 32,000 f32 rows (32/8 heads, Q8_0) 277 against 254
    // us, 9,000 88 against 84, 16,384 bf16 rows (bf16 cache) 82 against 72 (in threes 78); 16,384 bf16 rows (Q8_0) 109
    // against 111.
    const int64_t all = (n_heads + APPEND_HEADS - 1) / APPEND_HEADS + (c.n_kv + APPEND_HEADS - 1) / APPEND_HEADS * 2;
    const int64_t batches = all < 65535 ? all : 65535;       // a grid's height
    const int64_t most = dt == Q3CU_F32 ? 4 : 6, fill = (32 * int64_t(sms) + rows - 1) / rows, few = (batches + most - 1) / most;
    const int64_t parts = fill > few ? fill : few;
    const dim3 grid(unsigned((rows + APPEND_WARPS - 1) / APPEND_WARPS), unsigned(parts < batches ? parts : batches));
    const bool whole = form.dim == HD && !form.pairs && form.gain == 1.0f;
    auto go = [&](auto kernel, auto *typed) {
        typedef decltype(typed) P;
        return launch_dependent(kernel, grid, dim3(APPEND_WARPS * 32), 0, stream, c, b, int(rows), static_cast<P>(q),
                                static_cast<P>(k), static_cast<P>(v), q_stride, kv_stride, n_heads, q_norm, k_norm, freq,
                                form, eps, q_out, status);
    };
    auto cached = [&](auto type, auto qa, auto *typed) {     // by the cache's type and the rotation's form
        typedef decltype(type) T;
        constexpr AppendAs QA = decltype(qa)::value;
        if (cache_dt == Q3CU_Q8_0)
            return whole ? go(kv_append_kernel<T, QA, AS_Q8, true>, typed) : go(kv_append_kernel<T, QA, AS_Q8, false>, typed);
        if (cache_dt == Q3CU_BF16)
            return whole ? go(kv_append_kernel<T, QA, AS_BF16, true>, typed) : go(kv_append_kernel<T, QA, AS_BF16, false>, typed);
        return whole ? go(kv_append_kernel<T, QA, AS_F32, true>, typed) : go(kv_append_kernel<T, QA, AS_F32, false>, typed);
    };
    const std::integral_constant<AppendAs, AS_F32> f32;
    const std::integral_constant<AppendAs, AS_BF16> bf16;
    if (dt == Q3CU_F32) {
        const float *t = nullptr;
        return q_dt == Q3CU_F32 ? cached(float(), f32, t) : cached(float(), bf16, t);
    }
    const uint16_t *t = nullptr;
    return q_dt == Q3CU_F32 ? cached(bf16raw(), f32, t) : cached(bf16raw(), bf16, t);
}

// ---- reading rows back ------------------------------------------------------------------------
// The rows' keys and values as they are in the cache (Q8_0: code times scale), dense.  Bound by memory: a warp takes one
// row, or with few rows a part of its heads, READ_HEADS heads of k or of v at a time; a lane stores 16 bytes of a head, so
// that 32 lanes hold one head of an f32 result or two of a bf16 one.
// 8 sequences of up to 8,192 positions (8 kv heads), Q8_0 to bf16: 35.5 us, 4.6 TB/s (issue slots 68 % busy); a warp for k and one
// for v 37, four heads at a time the same; 300 positions to f32: 4 us.  From f32 and bf16 caches 5.4 to 5.7 and 4.7 to 4.9 TB/s.
constexpr int READ_HEADS = 8;
template <AppendAs CA, AppendAs AS>
__device__ __forceinline__ void read_heads(const void *pool, const float *scales, int64_t at, int64_t scale_at, int64_t step, int n,
                                           bool there, void *to) {
    constexpr int VEC = AS == AS_BF16 ? 8 : 4, SIDE = VEC / 4, LANES = HD / VEC;         // elements of a lane, heads at once
    typedef typename std::conditional<CA == AS_Q8, uint8_t, typename std::conditional<CA == AS_BF16, uint16_t, float>::type>::type E;
    const int lane = threadIdx.x & 31, mine = SIDE == 2 ? lane / LANES : 0, e = lane % LANES * VEC;
    const E *from = static_cast<const E *>(pool) + at + mine * step + e;
    const float *scale = scales + scale_at + mine * (step / GS) + e / GS;
    constexpr int N = READ_HEADS / SIDE;
    float4 x[N][SIDE];
    uint32_t code[N][SIDE];
    float s[N];
#pragma unroll
    for (int i = 0; i < N; ++i) {
#pragma unroll
        for (int y = 0; y < SIDE; ++y) x[i][y] = make_float4(0.0f, 0.0f, 0.0f, 0.0f), code[i][y] = 0x80808080u;
        s[i] = 0.0f;
        if (SIDE * i + mine >= n || !there) continue;
        const E *p = from + SIDE * i * step;
        if constexpr (CA == AS_Q8) {
            if constexpr (SIDE == 2) {
                const uint2 w = *reinterpret_cast<const uint2 *>(p);
                code[i][0] = w.x, code[i][1] = w.y;
            } else {
                code[i][0] = *reinterpret_cast<const uint32_t *>(p);
            }
            s[i] = scale[SIDE * i * (step / GS)];
        } else {
#pragma unroll
            for (int y = 0; y < SIDE; ++y) x[i][y] = load_quad(p + 4 * y);
        }
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
        if (SIDE * i + mine >= n) continue;
        if constexpr (CA == AS_Q8) {
            if (there)
#pragma unroll
                for (int y = 0; y < SIDE; ++y) {
                    const float4 f = q8_floats(code[i][y]);
                    x[i][y] = make_float4(s[i] * f.x, s[i] * f.y, s[i] * f.z, s[i] * f.w);
                }
        }
        if constexpr (SIDE == 2)
            *reinterpret_cast<uint4 *>(static_cast<uint16_t *>(to) + (SIDE * i + mine) * HD + e) =
                make_uint4(pack_bf16(x[i][0].x, x[i][0].y), pack_bf16(x[i][0].z, x[i][0].w), pack_bf16(x[i][1].x, x[i][1].y),
                           pack_bf16(x[i][1].z, x[i][1].w));
        else store_quad(static_cast<float *>(to) + i * HD + e, x[i][0]);
    }
}

template <AppendAs CA, AppendAs AS>
__global__ void __launch_bounds__(APPEND_WARPS * 32, 8)
kv_read_kernel(const PagedKV c, const PagedSeqs b, int rows, void *k, void *v, int64_t kv_stride, uint32_t *status) {
    griddep_wait();
    const int lane = threadIdx.x & 31, r = int(blockIdx.x) * APPEND_WARPS + int(threadIdx.x >> 5);
    if (r >= rows) return;
    int pos;
    const int s = paged_row_of_warp(b, c, r, pos, status);
    if (s < 0) return;                                       // a row behind the last sequence
    const int page = pos < 0 ? -1 : paged_page(b, c, s, pos, lane == 0 ? status : nullptr);
    const int64_t step = HD << c.page_shift, at = page < 0 ? 0 : paged_at(c, page, 0, pos);
    const int64_t sc = page < 0 || CA != AS_Q8 ? 0 : paged_scale_at(c, page, 0, pos);
    const int n = (c.n_kv + READ_HEADS - 1) / READ_HEADS;    // batches of k, and of v
    const int first = part_of(2 * n, blockIdx.y, gridDim.y), last = part_of(2 * n, blockIdx.y + 1, gridDim.y);
    constexpr int BYTES = AS == AS_BF16 ? 2 : 4;
    for (int x = first; x < last; ++x) {
        const bool side = x >= n;
        const int u = (side ? x - n : x) * READ_HEADS;
        read_heads<CA, AS>(side ? c.v : c.k, side ? c.v_scale : c.k_scale, at + u * step, sc + u * (step / GS), step,
                           c.n_kv - u, page >= 0, static_cast<uint8_t *>(side ? v : k) + (r * kv_stride + u * HD) * BYTES);
    }
}

cudaError_t launch_kv_read(const PagedKV &c, q3cu_dtype cache_dt, const PagedSeqs &b, int64_t rows, void *k, void *v,
                           q3cu_dtype dt, int64_t kv_stride, uint32_t *status, cudaStream_t stream, int sms) {
    // a row is split over warps while the rows alone are fewer than 32 warps per SM
    const int64_t all = 2 * ((int64_t(c.n_kv) + READ_HEADS - 1) / READ_HEADS), batches = all < 65535 ? all : 65535;
    const int64_t parts = rows >= 32 * sms ? 1 : (32 * int64_t(sms) + rows - 1) / rows;
    const dim3 grid(unsigned((rows + APPEND_WARPS - 1) / APPEND_WARPS), unsigned(parts < batches ? parts : batches));
    auto go = [&](auto kernel) {
        return launch_dependent(kernel, grid, dim3(APPEND_WARPS * 32), 0, stream, c, b, int(rows), k, v, kv_stride, status);
    };
    if (dt == Q3CU_F32)
        return cache_dt == Q3CU_Q8_0   ? go(kv_read_kernel<AS_Q8, AS_F32>)
               : cache_dt == Q3CU_BF16 ? go(kv_read_kernel<AS_BF16, AS_F32>)
                                       : go(kv_read_kernel<AS_F32, AS_F32>);
    return cache_dt == Q3CU_Q8_0   ? go(kv_read_kernel<AS_Q8, AS_BF16>)
           : cache_dt == Q3CU_BF16 ? go(kv_read_kernel<AS_BF16, AS_BF16>)
                                   : go(kv_read_kernel<AS_F32, AS_BF16>);
}

}  // namespace q3
