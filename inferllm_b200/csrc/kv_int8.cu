// Rows of keys and values in eight bits: rotated, rounded and written into the paged cache in one pass, and read back.
//
// A row is the d values of one position and kv head.  With a = max |x| over it, its scale is s = a / 127 and a value is kept as
// u = 128 + round(127 x / a) (ties to even), so that it stands for (u - 128) s: at most a / 254 from x, and the scale's rounding.  Pages: u
// [pages, kv heads, page_size, d] bytes, scales float32 [pages, kv heads, page_size] beside them.  The zero point of 128 keeps u
// unsigned: an attention kernel makes 1024 + u in half precision by putting the byte into the mantissa.
// One scale per row, not per page: rows come one at a time and are never rounded again.  A row whose largest value is below
// 2^-100 stands for zeros (s = 0; its quotients would leave float32), one with an infinity or a NaN reads back as NaN.
//
// The write does what rope_kv.cu does for a cache of wider rows (src/kern/naive/naive.cpp:389-414 for the rotation, src/core/op.cpp:414-416 for
// the rows' way into the cache; the reference keeps float32 rows only): pair (j, j + rot / 2) of every query and key head is turned by the position's angle,
// from a table; the arithmetic is float32, and keys and values are rounded once, to eight bits.  The queries leave in the
// activations' type, in a matrix of their own.
// Memory bounds it: a projection row is read once, 1 + 4 / d bytes per element are written.  A row belongs to the fewest lanes
// (8, 16 or 32) that hold it with eight channels each, so that the maximum is a few shuffles, and a thread keeps its channels'
// cos and sin for up to four heads of its token, whose loads are in flight together.
#include "common.cuh"

#define KQ_THREADS 256
#define KQ_TINY 7.888609e-31f       // 2^-100

// Four neighbouring channels, as they lie in memory and as numbers.
__device__ __forceinline__ void kq_numbers(uint2 u, float* f) {
    f[0] = __uint_as_float(u.x << 16);
    f[1] = __uint_as_float(u.x & 0xffff0000u);
    f[2] = __uint_as_float(u.y << 16);
    f[3] = __uint_as_float(u.y & 0xffff0000u);
}
__device__ __forceinline__ void kq_numbers(float4 u, float* f) { f[0] = u.x, f[1] = u.y, f[2] = u.z, f[3] = u.w; }
__device__ __forceinline__ void kq_store4(bf16* p, const float* f) {
    const __nv_bfloat162 a = __floats2bfloat162_rn(f[0], f[1]), b = __floats2bfloat162_rn(f[2], f[3]);
    *reinterpret_cast<uint2*>(p) = make_uint2(*reinterpret_cast<const unsigned*>(&a), *reinterpret_cast<const unsigned*>(&b));
}
__device__ __forceinline__ void kq_store4(float* p, const float* f) { *reinterpret_cast<float4*>(p) = make_float4(f[0], f[1], f[2], f[3]); }
template <typename TA, bool PARTIALS> struct KqFour { using Raw = float4; };
template <> struct KqFour<bf16, false> { using Raw = uint2; };

// of the projection at element `at`, or the sum of its K slices there
template <typename TA, bool PARTIALS>
__device__ __forceinline__ typename KqFour<TA, PARTIALS>::Raw kq_fetch4(const TA* __restrict__ x, const float* __restrict__ partials, int splits, long long stride, size_t at) {
    if constexpr (!PARTIALS) {
        return *reinterpret_cast<const typename KqFour<TA, PARTIALS>::Raw*>(x + at);
    } else {
        float4 f = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int z = 0; z < splits; z++) {
            const float4 p = *reinterpret_cast<const float4*>(partials + (size_t)z * stride + at);
            f.x += p.x, f.y += p.y, f.z += p.z, f.w += p.w;
        }
        return f;
    }
}
template <typename TA, bool PARTIALS>
__device__ __forceinline__ float kq_fetch1(const TA* __restrict__ x, const float* __restrict__ partials, int splits, long long stride, size_t at) {
    if (!PARTIALS) return to_f32(x[at]);
    float f = 0.f;
    for (int z = 0; z < splits; z++) f += partials[(size_t)z * stride + at];
    return f;
}

// LANES: lanes of a row, eight channels each.  WIDE (rot a multiple of 8): a lane of the rotated part has four channels and the four that they are turned with, so
// that it needs no other lane's and each of its cosines once (4,096 tokens of 32 + 16 heads of 128 take 22 us, floor 14, mostly instructions, 70 % of the issue slots; with eight
// neighbours a lane, and their partners fetched beside them, 3 us more).  Otherwise it has eight neighbours and fetches their partners one by one.  A block takes ROUNDS times
// KQ_THREADS / LANES heads of one token.
template <typename TA, bool PARTIALS, bool WIDE, int LANES, int ROUNDS>
__global__ void __launch_bounds__(KQ_THREADS, WIDE && !PARTIALS && sizeof(TA) == 2 ? 5 : 4)
kv_write_int8_kernel(const TA* __restrict__ qkv, const float* __restrict__ partials, int splits, long long split_stride, TA* __restrict__ q_out,
                     const float2* __restrict__ cs, const int* __restrict__ token_pos, const int* __restrict__ token_seq,
                     const int* __restrict__ block_table, int max_pages, int n_pages, unsigned char* __restrict__ kc, unsigned char* __restrict__ vc,
                     float* __restrict__ ksc, float* __restrict__ vsc, int nh, int nkv, int d, int rot, int page_size, int write_kv,
                     int table_positions, int* __restrict__ err) {
    pdl_grid_sync();
    constexpr int AT_ONCE = KQ_THREADS / LANES;
    const int t = blockIdx.x, c = threadIdx.x & (LANES - 1), half = rot >> 1, n_slots = nh + 2 * nkv;
    const bool active = c * 8 < d, turned = c * 8 < rot;
    const int ch0 = WIDE && turned ? c * 4 : c * 8, ch1 = WIDE && turned ? half + c * 4 : c * 8 + 4;
    // (the lanes of a row run together: its slot is the same for all of them, and shuffles stay within the row)
    const unsigned mask = LANES == 32 ? 0xffffffffu : ((1u << (LANES & 31)) - 1u) << ((threadIdx.x & 31) & ~(LANES - 1));
    const int s0 = blockIdx.y * (AT_ONCE * ROUNDS) + threadIdx.x / LANES, all = write_kv ? n_slots : nh;
    const size_t row0 = ((size_t)t * n_slots + s0) * d;
    // the rows first: where they go is looked up behind their loads
    typename KqFour<TA, PARTIALS>::Raw raw[ROUNDS][2];
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
        raw[i][0] = raw[i][1] = {};
        if (s0 + i * AT_ONCE >= all || !active) continue;
        raw[i][0] = kq_fetch4<TA, PARTIALS>(qkv, partials, splits, split_stride, row0 + i * (AT_ONCE * d) + ch0);
        raw[i][1] = kq_fetch4<TA, PARTIALS>(qkv, partials, splits, split_stride, row0 + i * (AT_ONCE * d) + ch1);
    }
    const int p = token_pos[t];
    if (p < 0 || (half > 0 && p >= table_positions)) {
        if (threadIdx.x == 0) atomicExch(err, 3);
        return;
    }
    int page = -1;
    const int logical = (int)((unsigned)p / (unsigned)page_size), offset = p - logical * page_size;
    if (write_kv) {
        if (logical < max_pages) page = block_table[(size_t)token_seq[t] * max_pages + logical];
        if (page < 0 || page >= n_pages) {
            if (threadIdx.x == 0) atomicExch(err, 2);
            page = -1;
        }
    }
    const int end = page < 0 ? nh : n_slots;         // queries come first
    float2 turn[4];
    if (WIDE && turned) {
        const float4 v0 = *reinterpret_cast<const float4*>(cs + (size_t)p * half + c * 4), v1 = *reinterpret_cast<const float4*>(cs + (size_t)p * half + c * 4 + 2);
        turn[0] = make_float2(v0.x, v0.y), turn[1] = make_float2(v0.z, v0.w), turn[2] = make_float2(v1.x, v1.y), turn[3] = make_float2(v1.z, v1.w);
    }
#pragma unroll
    for (int i = 0; i < ROUNDS; i++) {
        const int slot = s0 + i * AT_ONCE;
        if (slot >= end) break;
        const bool is_q = slot < nh, is_k = !is_q && slot < nh + nkv;
        float x[8];
        kq_numbers(raw[i][0], x);
        kq_numbers(raw[i][1], x + 4);
        if (turned && (is_q || is_k)) {
            if (WIDE) {
#pragma unroll
                for (int k = 0; k < 4; k++) {
                    const float a = x[k], b = x[k + 4];
                    x[k] = a * turn[k].x - b * turn[k].y;
                    x[k + 4] = a * turn[k].y + b * turn[k].x;
                }
            } else {
#pragma unroll
                for (int k = 0; k < 8; k++) {
                    const int ch = c * 8 + k, j = ch < half ? ch : ch - half;
                    if (ch >= rot) continue;
                    const float2 w = cs[(size_t)p * half + j];
                    const float y = kq_fetch1<TA, PARTIALS>(qkv, partials, splits, split_stride, row0 + i * (AT_ONCE * d) + (ch < half ? ch + half : j));
                    x[k] = ch < half ? x[k] * w.x - y * w.y : y * w.y + x[k] * w.x;
                }
            }
        }
        if (is_q) {
            TA* to = q_out + ((size_t)t * nh + slot) * d;
            if (active) {
                kq_store4(to + ch0, x);
                kq_store4(to + ch1, x + 4);
            }
            continue;
        }
        // the largest magnitude as bits: unsigned order is that of the values, with infinities and then NaNs above them
        unsigned top = 0;
#pragma unroll
        for (int k = 0; k < 8; k++) top = max(top, __float_as_uint(x[k]) & 0x7fffffffu);
#pragma unroll
        for (int o = LANES / 2; o > 0; o >>= 1) top = max(top, __shfl_xor_sync(mask, top, o));
        const float a = __uint_as_float(top);
        const bool finite = top < 0x7f800000u, tiny = finite && a < KQ_TINY;
        const float scale = !finite ? __uint_as_float(0x7fffffffu) : tiny ? 0.f : a / 127.f, inv = !finite || tiny ? 0.f : 1.f / a;
        const int hk = is_k ? slot - nh : slot - nh - nkv;
        const size_t row = ((size_t)page * nkv + hk) * page_size + offset;
        // u = 128 + round(127 x / a): (127 / 128) x / a, rounded once (the remainder of the first quotient corrects it: P. Markstein, 1990; with the reciprocal alone
        // exact halves, which rows of bfloat16 often hold, fell to either side: 0.13 % of their values), and 128 times that added to 1.5 x 2^23 + 128 in one rounding, whose sum's lowest byte it is
        unsigned u[8];
#pragma unroll
        for (int k = 0; k < 8; k++) {
            const float y = x[k] * 0.9921875f, q = y * inv;
            u[k] = __float_as_uint(fmaf(fmaf(fmaf(-q, a, y), inv, q), 128.f, 12583040.f));
        }
        unsigned lo = __byte_perm(__byte_perm(u[0], u[1], 0x0040), __byte_perm(u[2], u[3], 0x0040), 0x5410);
        unsigned hi = __byte_perm(__byte_perm(u[4], u[5], 0x0040), __byte_perm(u[6], u[7], 0x0040), 0x5410);
        if (!finite) lo = hi = 0x80808080u;
        if (active) {
            unsigned char* to = (is_k ? kc : vc) + row * d;
            *reinterpret_cast<unsigned*>(to + ch0) = lo;
            *reinterpret_cast<unsigned*>(to + ch1) = hi;
        }
        if (c == 0) (is_k ? ksc : vsc)[row] = scale;
    }
}

// rows of given positions, (u - 128) s in the activations' type: k, v [T, kv heads, d]; a position without a page reads back as NaN
template <typename TA>
__global__ void __launch_bounds__(KQ_THREADS)
kv_read_int8_kernel(const unsigned char* __restrict__ kc, const unsigned char* __restrict__ vc, const float* __restrict__ ksc, const float* __restrict__ vsc,
                    const int* __restrict__ token_pos, const int* __restrict__ token_seq, const int* __restrict__ block_table, int max_pages, int n_pages,
                    TA* __restrict__ k_out, TA* __restrict__ v_out, long long n, int nkv, int d, int page_size) {
    pdl_grid_sync();
    // a block takes pieces of eight channels of one position (blockIdx.x)
    const int pieces = d >> 3, i = blockIdx.y * KQ_THREADS + threadIdx.x;
    if (i >= nkv * pieces) return;
    const int hk = i / pieces, c = i - hk * pieces;
    const long long t = blockIdx.x;
    const int p = token_pos[t], logical = p < 0 ? max_pages : (int)((unsigned)p / (unsigned)page_size);
    const int page = logical < max_pages ? block_table[(size_t)token_seq[t] * max_pages + logical] : -1;
    const bool held = page >= 0 && page < n_pages;
    const size_t row = held ? ((size_t)page * nkv + hk) * page_size + (p - logical * page_size) : 0;
    const float nan = __uint_as_float(0x7fffffffu);
    auto one = [&](const unsigned char* cache, const float* scales, TA* out) {
        const uint2 v = *reinterpret_cast<const uint2*>(cache + row * d + c * 8);
        const float s = held ? scales[row] : nan;
        float f[8];
#pragma unroll
        for (int k = 0; k < 8; k++) f[k] = (float)((int)((k < 4 ? v.x : v.y) >> (8 * (k & 3)) & 255u) - 128) * s;
        store8(out + (t * nkv + hk) * d + c * 8, f);
    };
    one(kc, ksc, k_out);
    one(vc, vsc, v_out);
}

// qkv: the packed projection [T, (nh + 2 nkv) d] of dtype act_dtype, or (partials) its float32 K slices [splits][T][...], added in
// ascending order.  q_out [T, nh d].  kc, vc: one entry's pages; ksc, vsc their scales.  d a multiple of 8 up to 256; rot even, up to d;
// write_kv 0: the rotation alone.  err: 2 a position without a page, 3 one outside the table.
extern "C" int illm_kv_write_int8(const void* qkv, const float* partials, int splits, long long split_stride, void* q_out, const float* cos_sin,
                                  const int* token_pos, const int* token_seq, const int* block_table, int max_pages, long long n_pages, void* kc, void* vc,
                                  float* ksc, float* vsc, int act_dtype, int T, int nh, int nkv, int d, int rot, int page_size, int write_kv,
                                  int table_positions, int* err, void* stream) {
    if (T <= 0) return 0;
    if (nh <= 0 || nkv <= 0 || d <= 0 || d > 256 || (d & 7) || rot < 0 || rot > d || (rot & 1) || (rot > 0 && !cos_sin) || page_size <= 0 || max_pages <= 0 ||
        n_pages > 0x7fffffffLL || (act_dtype != ILLM_BF16 && act_dtype != ILLM_F32) || (partials ? splits < 1 : !qkv) || !q_out || !err)
        return ILLM_ERR_BAD_ARG;
    if (write_kv && (!kc || !vc || !ksc || !vsc || ((uintptr_t)kc & 7) || ((uintptr_t)vc & 7))) return ILLM_ERR_BAD_ARG;
    if (((uintptr_t)qkv & 15) || ((uintptr_t)partials & 15) || ((uintptr_t)q_out & 15) || ((uintptr_t)cos_sin & 15)) return ILLM_ERR_BAD_ARG;
    const int lanes = d <= 64 ? 8 : d <= 128 ? 16 : 32, at_once = KQ_THREADS / lanes;
    const int n_slots = nh + (write_kv ? 2 * nkv : 0), rounds_all = (n_slots + at_once - 1) / at_once;
    // several heads to a thread once that leaves eight blocks to every SM (4,096 tokens of 32 + 16 heads written and read back 29.2 us, one head to a thread 37.6; 8 tokens
    // of 32 + 64 heads 4.2 with one, 4.9 with four)
    const bool wide = (rot & 7) == 0;
    int rounds = 1;
    if (wide && !partials)
        while (rounds < 4 && rounds < rounds_all && (long long)T * ((rounds_all + rounds) / (rounds + 1)) >= 8LL * illm_sm_count()) rounds++;
    const dim3 grid((unsigned)T, (unsigned)((rounds_all + rounds - 1) / rounds));
    if (grid.y > 65535) return ILLM_ERR_BAD_ARG;
    cudaStream_t s = (cudaStream_t)stream;
#define KQ_RUN(TA, PART, W, L, N)                                                                                                               \
    illm_launch(kv_write_int8_kernel<TA, PART, W, L, N>, grid, dim3(KQ_THREADS), 0, s, (const TA*)qkv, partials, splits, split_stride, (TA*)q_out, \
                (const float2*)cos_sin, token_pos, token_seq, block_table, max_pages, (int)n_pages, (unsigned char*)kc, (unsigned char*)vc, ksc, vsc, nh, \
                nkv, d, rot, page_size, write_kv, table_positions, err)
#define KQ_LANES(TA, PART, W, N)                       \
    do {                                               \
        if (lanes == 8) KQ_RUN(TA, PART, W, 8, N);     \
        else if (lanes == 16) KQ_RUN(TA, PART, W, 16, N); \
        else KQ_RUN(TA, PART, W, 32, N);               \
    } while (0)
#define KQ_ROUNDS(TA)                                  \
    do {                                               \
        if (!wide) KQ_LANES(TA, false, false, 1);      \
        else if (rounds == 1) KQ_LANES(TA, false, true, 1); \
        else if (rounds == 2) KQ_LANES(TA, false, true, 2); \
        else if (rounds == 3) KQ_LANES(TA, false, true, 3); \
        else KQ_LANES(TA, false, true, 4);             \
    } while (0)
    if (partials) {
        if (act_dtype != ILLM_BF16) return ILLM_ERR_BAD_ARG;
        if (wide) KQ_LANES(bf16, true, true, 1);
        else KQ_LANES(bf16, true, false, 1);
    } else if (act_dtype == ILLM_BF16) {
        KQ_ROUNDS(bf16);
    } else {
        KQ_ROUNDS(float);
    }
#undef KQ_ROUNDS
#undef KQ_LANES
#undef KQ_RUN
    return illm_launch_status();
}

// k_out, v_out [n, nkv, d] of dtype `dtype`: the rows of n positions (token_pos, token_seq int32 [n]).
extern "C" int illm_kv_read_int8(const void* kc, const void* vc, const float* ksc, const float* vsc, const int* token_pos, const int* token_seq,
                                 const int* block_table, int max_pages, long long n_pages, void* k_out, void* v_out, int dtype, long long n, int nkv, int d,
                                 int page_size, void* stream) {
    if (n <= 0) return 0;
    if (nkv <= 0 || d <= 0 || d > 256 || (d & 7) || page_size <= 0 || max_pages <= 0 || n_pages <= 0 || n_pages > 0x7fffffffLL || !kc || !vc || !ksc || !vsc || ((uintptr_t)kc & 7) ||
        ((uintptr_t)vc & 7) || ((uintptr_t)k_out & 15) || ((uintptr_t)v_out & 15) || (dtype != ILLM_BF16 && dtype != ILLM_F32))
        return ILLM_ERR_BAD_ARG;
    const int items = nkv * (d / 8), threads = items >= KQ_THREADS ? KQ_THREADS : (items + 31) / 32 * 32;
    if (n > 0x7fffffffLL || items > 65535 * KQ_THREADS) return ILLM_ERR_BAD_ARG;
    const dim3 grid((unsigned)n, (unsigned)((items + KQ_THREADS - 1) / KQ_THREADS));
    cudaStream_t s = (cudaStream_t)stream;
    if (dtype == ILLM_BF16)
        illm_launch(kv_read_int8_kernel<bf16>, grid, dim3(threads), 0, s, (const unsigned char*)kc, (const unsigned char*)vc, ksc, vsc, token_pos,
                    token_seq, block_table, max_pages, (int)n_pages, (bf16*)k_out, (bf16*)v_out, n, nkv, d, page_size);
    else
        illm_launch(kv_read_int8_kernel<float>, grid, dim3(threads), 0, s, (const unsigned char*)kc, (const unsigned char*)vc, ksc, vsc, token_pos,
                    token_seq, block_table, max_pages, (int)n_pages, (float*)k_out, (float*)v_out, n, nkv, d, page_size);
    return illm_launch_status();
}
