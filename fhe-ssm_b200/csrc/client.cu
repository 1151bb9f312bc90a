// client.cu -- the client's token step on the GPU: the head product with a 4-bit table, the choice of
// the next token, and the look-up of the next embedding row in the same (tied) table.
//
// The server returns encrypted normed rows; the client decrypts them, applies the tied head in plaintext
// (the --dec-out side of gpu_real_model.cu:2444-2533), picks a token (spec_decode/decode_policy.py:37) and
// embeds it with a row of the same table (ml-eval/fhe_client.py:123-135).
//
// All three run on a stream of the caller's choice and read nothing of the context's chain or keys.  Only the
// product of several rows (k_q4_gemm) needs memory beside its operands; it takes it from the stream's pool.

#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <atomic>

namespace fhe {

// one value of a tensor whose type is known at run time (FHE_F32, FHE_F16, FHE_BF16)
__device__ __forceinline__ float ld_any(const void* p, int type, long long i) {
    if (type == FHE_F32) return static_cast<const float*>(p)[i];
    if (type == FHE_F16) return __half2float(static_cast<const __half*>(p)[i]);
    return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void st_any(void* p, int type, long long i, float v) {
    if (type == FHE_F32) static_cast<float*>(p)[i] = v;
    else if (type == FHE_F16) static_cast<__half*>(p)[i] = __float2half_rn(v);
    else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(v);
}

// Lets kernel K have all the shared memory a block can; asked of the driver once per GPU.
template <auto K>
static void client_smem(const Context& cx) {
    static std::atomic<uint64_t> done{0};
    const uint64_t bit = 1ull << cx.device;
    if (done.load(std::memory_order_relaxed) & bit) return;
    CUDA_CHECK(cudaFuncSetAttribute(K, cudaFuncAttributeMaxDynamicSharedMemorySize, 232448));
    done.fetch_or(bit, std::memory_order_relaxed);
}

// ---- products with a 4-bit table -----------------------------------------------------------
// W[i][c] = s[i][c / group] (q[i][c] - 8); out[r][i] = sum_c x[r][c] W[i][c].
//
// Within a group the sum is a product of whole numbers -8..7, which every 16-bit float holds exactly, with x; the
// scale is applied to the group's sum in float32.  x is cut into bf16 pieces that add up to it exactly (float32: 3 of 8
// bits, float16: 2, bf16: itself), each piece a column of the matrix product, so nothing is rounded before the
// float32 sums.  The group's sum is up to 2^10 times the largest value of x, which the scale would bring back into range but float32
// does not hold for values of 2^117 and more: a row that has one is cut 2^-16 times as large, and its output multiplied again.
//
// k_q4_mma: few columns (one row of x, or some).  What it must read is the table, so a warp streams 16 table rows through a
// shared-memory ring of its own (cp.async, no block barrier) and multiplies them on the tensor cores (m16n8k16: 16 table
// rows x 8 columns of pieces); with a CUDA-core product the unpacking and the float32 multiply-adds, 4 instructions
// a value, would cost more than the table's bytes.  Columns are permuted so that a 32-bit word of
// 8 values is a lane's share of two steps: the pairs (0,4), (1,5), (2,6), (3,7) come out of the word by one
// mask each.  Several warps share 16 rows where the table is short, each a part of the columns.
//
// One bfloat16 row on 50,304 x 1,024 at groups of 64 takes 11.6 us (27.5 MB: 2.4 TB/s, 37% of a copy's rate), on 16,384 x 4,096
// 16.2 us, on 4,096 x 1,024 4.1 us; 8 rows on 50,304 x 1,024 14.1 us.  About 3 us are the launch, x's pieces and the
// scales, a round trip each; then the loop, which waits for the table's bytes 3% of its time: instructions bound it,
// 54% of the issue slots and 51% of the integer pipe over the whole kernel (unpacking: 7 integer operations and 4 subtractions
// for 8 values), with the 24 warps an SM that the ring leaves room for.  More and smaller blocks cut x more often: 16,384 x
// 4,096 by 4 warps a tile takes 20.5 us.
constexpr int kQ4Warps = 8, kQ4Threads = 32 * kQ4Warps;
constexpr int kQ4Stage = 4;             // 32-column chunks of a stage
constexpr int kQ4Stages = 4;
constexpr int kQ4Pitch = kQ4Stage * 16 + 16;   // bytes of a row in a stage: 20 banks apart, 8 rows x 4 words meet all 32
constexpr int kQ4StageBytes = 16 * kQ4Pitch;
constexpr int kQ4RingBytes = 16 + kQ4Warps * kQ4Stages * kQ4StageBytes;   // before it a word: the rows that are large

struct Q4Args {
    fhe_q4 w;
    const void* x;
    int xt, terms, m;
    long long ldx;
    void* out;
    int ot;
    long long ldo;
    int ks_log2;     // 2^ks_log2 warps share a row tile's columns
    int kb_chunks;   // chunks of columns held at a time, in whole stages for each of these warps
    int units;       // scales that a warp holds for each row
    uint32_t group_magic;   // q4_group_magic
    int wide;        // rows of x start on 16-byte boundaries
    int scale_vec;   // a unit is a group, and rows of scales start on 16-byte boundaries
};

// The first bf16 piece of v (the high half of what is returned) and what is left of v: pieces are cut, not rounded, so none
// overflows; an infinity or NaN is all in the first.
__device__ __forceinline__ uint32_t q4_piece(float& v) {
    const uint32_t b = __float_as_uint(v);
    const bool finite = fabsf(v) < INFINITY;
    v = finite ? v - __uint_as_float(b & 0xffff0000u) : 0.f;
    return finite || !(b & 0x007fffffu) ? b : 0x7fff0000u;
}

template <class T>
__device__ __forceinline__ float q4_float(T v);
template <>
__device__ __forceinline__ float q4_float(float v) { return v; }
template <>
__device__ __forceinline__ float q4_float(__half v) { return __half2float(v); }
template <>
__device__ __forceinline__ float q4_float(__nv_bfloat16 v) { return __bfloat162float(v); }

constexpr float kQ4Big = 1.661534994731145e35f;   // 2^117
constexpr float kQ4Down = 1.f / 65536.f;

// Pieces of x's rows, chunks kb0..kb1 -> the product's operand [chunk][tile of 8 columns][lane], 16 bytes each:
// the lane's column (r TERMS + piece) and its 8 values, paired as q4_unpack pairs the table's.  DOWN: rows in the mask `down`
// are cut times kQ4Down.  True: the thread has met a value of kQ4Big or more, or one that is not finite.
template <class T, int TERMS, bool DOWN = false>
__device__ __forceinline__ bool q4_cut(const Q4Args& a, uint4* xs, int nt, int kb0, int kb1, uint32_t down = 0) {
    // a warp takes 8 chunks of a row at a time
    const int lane = threadIdx.x & 31, t = lane & 3;
    int r = threadIdx.x >> 5, ch = lane >> 2;
    bool large = false;
    for (;; r += kQ4Warps) {
        while (r >= a.m) r -= a.m, ch += 8;
        if (ch - (lane >> 2) >= kb1 - kb0) break;
        if (ch >= kb1 - kb0) continue;
        const int k = (kb0 + ch) * 32 + t * 8;
        const T* src = static_cast<const T*>(a.x) + r * a.ldx + k;
        if constexpr (TERMS == 1) {   // bfloat16 is its own piece
            const uint16_t* bits = reinterpret_cast<const uint16_t*>(src);
            uint4 u;
            if (a.wide && k + 8 <= a.w.cols) u = *reinterpret_cast<const uint4*>(bits);
            else {
                uint32_t p[8];
#pragma unroll
                for (int j = 0; j < 8; j++) p[j] = k + j < a.w.cols ? bits[j] : 0;
                u = make_uint4(p[0] | p[1] << 16, p[2] | p[3] << 16, p[4] | p[5] << 16, p[6] | p[7] << 16);
            }
            const auto larger = [](__nv_bfloat162 p, __nv_bfloat162 q) { return __hmax2(__habs2(p), __habs2(q)); };
            const auto two = [](const uint32_t& w) { return *reinterpret_cast<const __nv_bfloat162*>(&w); };
            const __nv_bfloat162 most = larger(larger(two(u.x), two(u.y)), larger(two(u.z), two(u.w)));
            // bit 15 of a half: 0x7a00, kQ4Big's bits, or more
            if (*reinterpret_cast<const uint32_t*>(&most) + 0x06000600u & 0x80008000u) large = true;
            if (DOWN && (down >> r & 1)) {
                const auto times = [](uint32_t w) {
                    return __byte_perm(__float_as_uint(__uint_as_float(w << 16) * kQ4Down),
                                       __float_as_uint(__uint_as_float(w & 0xffff0000u) * kQ4Down), 0x7632);
                };
                u = make_uint4(times(u.x), times(u.y), times(u.z), times(u.w));
            }
            xs[(ch * nt + (r >> 3)) * 32 + (r & 7) * 4 + t] =
                make_uint4(__byte_perm(u.x, u.z, 0x5410), __byte_perm(u.x, u.z, 0x7632), __byte_perm(u.y, u.w, 0x5410),
                           __byte_perm(u.y, u.w, 0x7632));
            continue;
        }
        float v[8];
        if (a.wide && k + 8 <= a.w.cols) {
            T u[8];
#pragma unroll
            for (int j = 0; j < (int)sizeof(T) * 8 / 16; j++)
                reinterpret_cast<uint4*>(u)[j] = reinterpret_cast<const uint4*>(src)[j];
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = q4_float(u[j]);
        } else {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] = k + j < a.w.cols ? q4_float(src[j]) : 0.f;
        }
        const auto cut = [&](auto piece) {
#pragma unroll
            for (int term = 0; term < TERMS; term++) {
                uint32_t p[8];
#pragma unroll
                for (int j = 0; j < 8; j++) p[j] = piece(v[j]);
                const int col = r * TERMS + term;
                xs[(ch * nt + (col >> 3)) * 32 + (col & 7) * 4 + t] =
                    make_uint4(__byte_perm(p[0], p[4], 0x7632), __byte_perm(p[1], p[5], 0x7632), __byte_perm(p[2], p[6], 0x7632),
                               __byte_perm(p[3], p[7], 0x7632));
            }
        };
        if (DOWN && (down >> r & 1)) {
#pragma unroll
            for (int j = 0; j < 8; j++) v[j] *= kQ4Down;
        }
        bool plain = true;
#pragma unroll
        for (int j = 0; j < 8; j++) plain = plain && fabsf(v[j]) < kQ4Big;
        if (plain) {   // 8 at a time: a test for each piece cost more than the cut
            cut([](float& f) {
                const uint32_t b = __float_as_uint(f);
                f -= __uint_as_float(b & 0xffff0000u);
                return b;
            });
        } else {
            large = true;
            cut(q4_piece);
        }
    }
    return large;
}

// The rows that have finite values of kQ4Big and more, in these chunks or before: into *big, and cut again times kQ4Down.  Returns
// those that are new.  By the whole block, and seldom: out of line, so that the way past it costs nothing.
template <class T, int TERMS>
__device__ __forceinline__ uint32_t q4_cut_large(const Q4Args& a, uint4* xs, int nt, int kb0, int kb1, uint32_t* big) {
    const uint32_t was = *big;
    __syncthreads();
    const int k0 = kb0 * 32, n = min(kb1 * 32, a.w.cols) - k0;
    for (int r = 0; r < a.m; r++) {
        bool found = false;
        for (int k = threadIdx.x; k < n; k += kQ4Threads) {
            const float v = fabsf(q4_float(static_cast<const T*>(a.x)[r * a.ldx + k0 + k]));
            found = found || (v >= kQ4Big && v < INFINITY);
        }
        if (found) atomicOr(big, 1u << r);
    }
    __syncthreads();
    const uint32_t now = *big;
    if (now) q4_cut<T, TERMS, true>(a, xs, nt, kb0, kb1, now);
    __syncthreads();
    return now ^ was;
}

// 8 values of 4 bits -> bf16 pairs (0,4), (1,5), (2,6), (3,7) of q - 8: 0x4300 is 128, its last bits count in ones
__device__ __forceinline__ void q4_unpack(uint32_t w, uint32_t* p) {
    const __nv_bfloat162 off = __floats2bfloat162_rn(136.f, 136.f);
#pragma unroll
    for (int i = 0; i < 4; i++) {
        const uint32_t v = (w >> (4 * i) & 0x000f000fu) | 0x43004300u;
        const __nv_bfloat162 d = __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), off);
        p[i] = *reinterpret_cast<const uint32_t*>(&d);
    }
}

__device__ __forceinline__ void q4_mma(float* d, const float* c, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                       uint32_t b0, uint32_t b1) {
    asm volatile(
        "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
        "{%10, %11, %12, %13};\n"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(c[0]), "f"(c[1]), "f"(c[2]), "f"(c[3]));
}

// Scales of 16 rows for `units` units of P chunks from chunk c0 -> sc[unit][row]; 0 past the last column.  src: the lane's row.
// Where a unit is a group and rows start on 16-byte boundaries, 16 bytes at a time: a load of single scales meets 16 rows'
// lines, and eight such loads a warp cost 128 of the L1's steps instead of 16.  `first`: the lane's first 16 bytes, asked for
// before x's pieces were cut, so that the two round trips are one.
template <class S, int P>
__device__ __forceinline__ void q4_scales(const Q4Args& a, const void* row, uint4 first, float* sc, int c0, int units, int chunks) {
    const int lane = threadIdx.x & 31, half = lane >> 4;
    const S* src = static_cast<const S*>(row);
    sc += lane & 15;
    if (a.scale_vec) {
        constexpr int V = 16 / sizeof(S);
        const int at = c0 / P, end = (chunks + P - 1) / P;
        uint4 q = first;
        const int e0 = (at & ~(V - 1)) + half * V;
        for (int e = e0; e < at + units; e += 2 * V) {
            S v[V];
            if (e + V <= end) {
                if (e != e0) q = *reinterpret_cast<const uint4*>(src + e);
                *reinterpret_cast<uint4*>(v) = q;
            } else {
#pragma unroll
                for (int j = 0; j < V; j++) v[j] = e + j < end ? src[e + j] : S(0.f);
            }
#pragma unroll
            for (int j = 0; j < V; j++)
                if (e + j >= at && e + j < at + units) sc[(e + j - at) * 16] = q4_float(v[j]);
        }
        return;
    }
#pragma unroll 4
    for (int u = half; u < units; u += 2) {
        const int ch = c0 + u * P;
        sc[u * 16] = ch < chunks ? q4_float(src[a.group_magic ? __umulhi(ch, a.group_magic) : ch]) : 0.f;
    }
}

// NT: tiles of 8 columns, which hold the pieces of all rows of x.  P: chunks after which the scale is applied, the largest of 1, 2, 4 that divides a group's.
template <int NT, int P>
__global__ void __launch_bounds__(kQ4Threads, 3) k_q4_mma(const __grid_constant__ Q4Args a) {
    extern __shared__ __align__(16) uint8_t qsm[];
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, g = lane >> 2, t = lane & 3;
    uint32_t* big = reinterpret_cast<uint32_t*>(qsm);
    uint8_t* ring = qsm + 16 + warp * (kQ4Stages * kQ4StageBytes);
    uint4* xs = reinterpret_cast<uint4*>(qsm + kQ4RingBytes);
    const int chunks = (a.w.cols + 31) / 32;
    const int ks = 1 << a.ks_log2, rows = 16 * kQ4Warps >> a.ks_log2;   // warps on a tile, table rows of a block
    const int row0 = blockIdx.x * rows + (warp >> a.ks_log2) * 16, kq = warp & (ks - 1);
    const int scale_bytes = a.w.scale_type == FHE_F32 ? 4 : 2;
    float* sc = reinterpret_cast<float*>(xs + a.kb_chunks * NT * 32) + warp * 16 * a.units;   // [unit][16 rows]
    if (tid == 0) *big = 0;
    float acc[NT][4];
#pragma unroll
    for (int n = 0; n < NT; n++)
#pragma unroll
        for (int j = 0; j < 4; j++) acc[n][j] = 0.f;
    // a lane copies 16 bytes of rows g and g + 8 a stage; rows past the end read the last one and are not stored
    const uint8_t* src0 = a.w.q + (long long)min(row0 + g, a.w.rows - 1) * a.w.ldq;
    const uint8_t* src1 = a.w.q + (long long)min(row0 + g + 8, a.w.rows - 1) * a.w.ldq;
    const uint32_t dst = (uint32_t)__cvta_generic_to_shared(ring) + g * kQ4Pitch + t * 16;
    const uint8_t* words = ring + g * kQ4Pitch + t * 4;

    for (int kb0 = 0; kb0 < chunks; kb0 += a.kb_chunks) {
        // the last block may pass the end: values and scales are 0 there
        const int kb1 = kb0 + a.kb_chunks, each = a.kb_chunks >> a.ks_log2, stages = each / kQ4Stage;
        const int c0 = kb0 + kq * each, c1 = c0 + each;
        auto fetch = [&](int s) {
            const int at = c0 + s * kQ4Stage + t;
            if (at < min(c1, chunks)) {
                const uint32_t d = dst + (s % kQ4Stages) * kQ4StageBytes;
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d), "l"(src0 + at * 16) : "memory");
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(d + 8 * kQ4Pitch), "l"(src1 + at * 16)
                             : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
        };
#pragma unroll
        for (int s = 0; s < kQ4Stages - 1; s++) fetch(s);
        const char* srow = static_cast<const char*>(a.w.scale) + min(row0 + (lane & 15), a.w.rows - 1) * a.w.lds * scale_bytes;
        uint4 first = make_uint4(0, 0, 0, 0);
        if (a.scale_vec) {
            const int v = 16 / scale_bytes, e = (c0 / P & ~(v - 1)) + (lane >> 4) * v;
            if (e + v <= (chunks + P - 1) / P) first = *reinterpret_cast<const uint4*>(srow + (size_t)e * scale_bytes);
        }
        __syncthreads();   // the previous block's pieces are read
        bool large = *big != 0;
        if (a.xt == FHE_F32) large |= q4_cut<float, 3>(a, xs, NT, kb0, kb1);
        else if (a.xt == FHE_F16) q4_cut<__half, 2>(a, xs, NT, kb0, kb1);
        else large |= q4_cut<__nv_bfloat16, 1>(a, xs, NT, kb0, kb1);
        if (a.w.scale_type == FHE_F16) q4_scales<__half, P>(a, srow, first, sc, c0, (c1 - c0) / P, chunks);
        else if (a.w.scale_type == FHE_BF16) q4_scales<__nv_bfloat16, P>(a, srow, first, sc, c0, (c1 - c0) / P, chunks);
        else q4_scales<float, P>(a, srow, first, sc, c0, (c1 - c0) / P, chunks);
        if (__syncthreads_or(large)) {
            const uint32_t more = a.xt == FHE_F32 ? q4_cut_large<float, 3>(a, xs, NT, kb0, kb1, big)
                                                  : q4_cut_large<__nv_bfloat16, 1>(a, xs, NT, kb0, kb1, big);
            // what was summed of the rows that are large from here on
#pragma unroll
            for (int n = 0; n < NT; n++)
#pragma unroll
                for (int j = 0; j < 4; j++)
                    if (more >> ((n * 8 + 2 * t + (j & 1)) / a.terms) & 1) acc[n][j] *= kQ4Down;
        }
        const uint4* xc = xs + (size_t)(c0 - kb0) * NT * 32 + lane;
        const float* su = sc + g;
#pragma unroll 4
        for (int s = 0; s < stages; s++) {
            fetch(s + kQ4Stages - 1);
            asm volatile("cp.async.wait_group %0;" ::"n"(kQ4Stages - 1) : "memory");
            __syncwarp();
            const uint8_t* st = words + (s % kQ4Stages) * kQ4StageBytes;
            constexpr float zero[4] = {0.f, 0.f, 0.f, 0.f};
            float c[NT][4];
#pragma unroll
            for (int ch = 0; ch < kQ4Stage; ch++) {
                uint32_t p[4], q[4];
                q4_unpack(*reinterpret_cast<const uint32_t*>(st + ch * 16), p);
                q4_unpack(*reinterpret_cast<const uint32_t*>(st + 8 * kQ4Pitch + ch * 16), q);
#pragma unroll
                for (int n = 0; n < NT; n++) {
                    const uint4 b = xc[(ch * NT + n) * 32];
                    q4_mma(c[n], ch % P == 0 ? zero : c[n], p[0], q[0], p[1], q[1], b.x, b.y);
                    q4_mma(c[n], c[n], p[2], q[2], p[3], q[3], b.z, b.w);
                }
                if (ch % P == P - 1) {
                    const float sg = su[ch / P * 16], sh = su[ch / P * 16 + 8];
#pragma unroll
                    for (int n = 0; n < NT; n++) {
                        acc[n][0] += sg * c[n][0];
                        acc[n][1] += sg * c[n][1];
                        acc[n][2] += sh * c[n][2];
                        acc[n][3] += sh * c[n][3];
                    }
                }
            }
            xc += kQ4Stage * NT * 32;
            su += kQ4Stage / P * 16;
            __syncwarp();
        }
        asm volatile("cp.async.wait_group 0;" ::: "memory");
    }
    // [warp][column][16 rows], then the pieces and the ks warps' parts are added up
    __syncthreads();
    float* so = reinterpret_cast<float*>(qsm + 16) + warp * (NT * 8 * 16);
#pragma unroll
    for (int n = 0; n < NT; n++) {
        so[(n * 8 + 2 * t) * 16 + g] = acc[n][0];
        so[(n * 8 + 2 * t + 1) * 16 + g] = acc[n][1];
        so[(n * 8 + 2 * t) * 16 + g + 8] = acc[n][2];
        so[(n * 8 + 2 * t + 1) * 16 + g + 8] = acc[n][3];
    }
    __syncthreads();
    const int rows_log2 = 7 - a.ks_log2;
    for (int i = tid; i < a.m << rows_log2; i += kQ4Threads) {
        const int r = i >> rows_log2, row = i & (rows - 1), at = blockIdx.x * rows + row;
        if (at >= a.w.rows) continue;
        const float* sp = reinterpret_cast<const float*>(qsm + 16) + ((row >> 4) << a.ks_log2) * (NT * 8 * 16) + (row & 15);
        float v = 0.f;
        for (int k = 0; k < ks; k++)
            for (int j = a.terms - 1; j >= 0; j--) v += sp[k * (NT * 8 * 16) + (r * a.terms + j) * 16];
        if (*big >> r & 1) v *= 1.f / kQ4Down;
        st_any(a.out, a.ot, (long long)r * a.ldo + at, v);
    }
}

// chunk / (chunks of a group) = chunk * magic >> 32 (both at most 2^15); 0: a group is a chunk
static uint32_t q4_group_magic(const fhe_q4& w) {
    const int gpc = std::min(w.group, FHE_Q4_MAX_COLS) / 32;
    return gpc == 1 ? 0u : (uint32_t)(((1ull << 32) + gpc - 1) / gpc);
}

template <int NT, int P>
static void q4_mma_launch(Context& cx, Q4Args a, cudaStream_t st) {
    const int tiles = (a.w.rows + 15) / 16, gpc = std::min(a.w.group, FHE_Q4_MAX_COLS) / 32;
    // warps enough to keep the loads in flight (8 an SM), but two stages of columns at least for each
    const int chunks = (a.w.cols + 31) / 32;
    a.ks_log2 = 0;
    while (a.ks_log2 < 3 && (tiles << a.ks_log2) < 148 * 8 && chunks >= (4 << a.ks_log2) * kQ4Stage) a.ks_log2++;
    // As many columns at a time as fit (512 bytes a chunk and tile of pieces, 512 a scale for 8 warps' rows), in equal blocks.  Two
    // blocks an SM where there are as many: one row on 16,384 x 4,096 took 18.1 us by 2,048 columns, 21.9 by all of them.
    const int each = kQ4Warps >> a.ks_log2, grid = (tiles + each - 1) / each;
    const int step = kQ4Stage << a.ks_log2, room = (grid > 148 ? 114704 : 213008) - kQ4RingBytes;
    const int fit = std::max(step, room / (512 * NT + 512 / P) / step * step), turns = (chunks + fit - 1) / fit;
    a.kb_chunks = ((chunks + turns - 1) / turns + step - 1) / step * step;
    a.units = (a.kb_chunks >> a.ks_log2) / P;
    a.scale_vec = gpc == P && (reinterpret_cast<uintptr_t>(a.w.scale) | (uintptr_t)a.w.lds * (a.w.scale_type == FHE_F32 ? 4 : 2)) % 16 == 0;
    a.group_magic = q4_group_magic(a.w);
    const size_t smem = kQ4RingBytes + (size_t)a.kb_chunks * NT * 512 + (size_t)a.units * kQ4Warps * 64;
    if (smem > 48 * 1024) client_smem<k_q4_mma<NT, P>>(cx);
    k_q4_mma<NT, P><<<grid, kQ4Threads, smem, st>>>(a);
    CUDA_CHECK(cudaGetLastError());
    cx.launches++;
}

template <int NT>
static void q4_mma_split(Context& cx, const Q4Args& a, cudaStream_t st) {
    const int gpc = a.w.group / 32;
    if (gpc % 2) q4_mma_launch<NT, 1>(cx, a, st);
    else if (gpc % 4) q4_mma_launch<NT, 2>(cx, a, st);
    else q4_mma_launch<NT, 4>(cx, a, st);
}

#include "q4_gemm.cuh"

template <int N, int KC, class XT>
static void q4_gemm_launch(Context& cx, QgArgs a, cudaStream_t st) {
    constexpr int kPieces = std::is_same<XT, float>::value ? 2 : 1, kSlot = N * 256 * kPieces;   // a job's 128 columns of x
    const int waves = (a.w.rows + 148 * kQgRowsMax - 1) / (148 * kQgRowsMax), xt = (a.m + N - 1) / N;
    a.block_rows = std::min(kQgRowsMax, ((a.w.rows + 148 * waves - 1) / (148 * waves) + 31) / 32 * 32);
    a.jobs = (a.w.cols + 127) / 128;
    a.part_jobs = a.jobs;
    // A short table of many columns: whole tiles, the columns in parts.  A job takes 0.5 us of a block, the sum of the parts a
    // launch: 64 float16 rows on 1,005 x 3,829 take 31.6 us in one part and 12.4 in 15.
    const int tiles = (a.w.rows + 127) / 128;
    if ((long long)tiles * xt * 2 <= 148 && a.jobs >= 12) {
        a.block_rows = 128;
        const int parts = std::min(148 / (tiles * xt), a.jobs / 2);
        a.part_jobs = (a.jobs + parts - 1) / parts;
    }
    const int parts = (a.jobs + a.part_jobs - 1) / a.part_jobs;
    a.slots = std::min({kQgSlotsMax, kQgXBytes / kSlot, a.part_jobs});
    // groups of a range, those past the last column's among them (zeros, but read)
    a.groups = (int)std::min(((long long)a.slots * 128 + a.w.group - 2) / a.w.group + 1,
                             ((long long)a.jobs * 128 + a.w.group - 1) / a.w.group);
    a.run = KC == 64 && a.w.group % 128 == 0 ? 2 : 1;
    const size_t smem = 2 * kQgStages * kQgStageBytes + (size_t)a.slots * kSlot + (size_t)a.groups * 1024 + N * sizeof(float) +
                        sizeof(QgBars);
    const size_t image = (size_t)xt * a.jobs * kSlot, powers = (size_t)xt * N * sizeof(float);
    const DevBuf work((image + powers + (parts > 1 ? (size_t)parts * a.m * a.w.rows * sizeof(float) : 0) + 7) / 8, st);
    a.image = reinterpret_cast<uint8_t*>(work.p);
    a.powers = reinterpret_cast<float*>(a.image + image);
    a.parts = parts > 1 ? reinterpret_cast<float*>(a.image + image + powers) : nullptr;
    client_smem<k_q4_gemm<N, KC, kPieces>>(cx);
    // by an ordinary launch: k_q4_gemm reads the table before it waits for this kernel, so it must not start before those ahead of it end
    k_q4_pack<N, KC, XT><<<xt * N, 128, 0, st>>>(a);
    CUDA_CHECK(cudaGetLastError());
    launch_pdl(cx, k_q4_gemm<N, KC, kPieces>, dim3((a.w.rows + a.block_rows - 1) / a.block_rows, xt, parts), dim3(kQgThreads),
               smem, st, a, cx.d_err);
    cx.launches += 2;
    if (parts > 1) {
        const dim3 grid((unsigned)std::min<long long>(592, ((long long)a.m * a.w.rows + 255) / 256));
        const auto sum = [&](auto* out) {
            using T = typename std::remove_pointer<decltype(out)>::type;
            launch_pdl(cx, k_q4_sum<T>, grid, dim3(256), 0, st, a.parts, parts, a.m, a.w.rows, out, a.ldo);
        };
        if (a.ot == FHE_F32) sum(static_cast<float*>(a.out));
        else if (a.ot == FHE_F16) sum(static_cast<__half*>(a.out));
        else sum(static_cast<__nv_bfloat16*>(a.out));
        cx.launches++;
    }
}
template <int N, class XT>
static void q4_gemm_group(Context& cx, const QgArgs& a, cudaStream_t st) {
    if (a.w.group % 64 == 0) q4_gemm_launch<N, 64, XT>(cx, a, st);
    else q4_gemm_launch<N, 32, XT>(cx, a, st);
}
template <class XT>
static void q4_gemm(Context& cx, const QgArgs& a, cudaStream_t st) {
    if (a.m <= 16) q4_gemm_group<16, XT>(cx, a, st);
    else if (a.m <= 32) q4_gemm_group<32, XT>(cx, a, st);
    else q4_gemm_group<64, XT>(cx, a, st);
}

static void q4_matvec(Context& cx, Q4Args a, cudaStream_t st) {
    const long long row = a.ldx * (a.xt == FHE_F32 ? 4 : 2);
    a.wide = (reinterpret_cast<uintptr_t>(a.x) | (uintptr_t)(a.m > 1 ? row : 0)) % 16 == 0;
    a.terms = a.xt == FHE_F32 ? 3 : a.xt == FHE_F16 ? 2 : 1;
    // By the columns of pieces, with which k_q4_mma grows (by tiles of 8 above all) and k_q4_gemm hardly does.  bfloat16 rows, us by
    // k_q4_mma and k_q4_gemm:
    //     50,304 x 1,024   8: 14.4, 17.8   9: 19.2, 18.1      16,384 x 4,096    8: 21.2, 22.0  10: 33.5, 21.9
    //     32,768 x 2,048   8: 18.5, 22.2  10: 21.6, 22.1       1,024 x 4,096    8:  9.2,  9.3  10: 13.3, 9.3
    // a small table, where k_q4_gemm's two launches weigh more, and groups of 32, where it adds up every 32 columns, on a long one:
    //      4,096 x 1,024  18:  8.2,  9.6      32,768 x 2,048, groups of 32  18: 31.8, 31.7  20: 32.2, 31.6
    const int pieces = a.m * a.terms;
    const int most = (a.w.rows < 16384 && a.w.cols < 1536) || (a.w.rows > 16384 && a.w.group % 64) ? 18 : 8;
    if (pieces > most) {
        const QgArgs q{a.w, a.x, a.m, a.ldx, a.out, a.ot, a.ldo, a.wide, 0, 0, 0, 0, 0, nullptr, 0, nullptr, nullptr,
                       cx.q4_waits < 0 ? kQgWaits : cx.q4_waits};
        if (a.xt == FHE_F32) q4_gemm<float>(cx, q, st);
        else if (a.xt == FHE_F16) q4_gemm<__half>(cx, q, st);
        else q4_gemm<__nv_bfloat16>(cx, q, st);
        return;
    }
    if (pieces <= 8) q4_mma_split<1>(cx, a, st);
    else if (pieces <= 16) q4_mma_split<2>(cx, a, st);
    else q4_mma_split<3>(cx, a, st);
}

// ---- rows of a 4-bit table by token id --------------------------------------------------------
// A thread takes 8 columns: one 32-bit load, one scale, 16 or 32 bytes out.  What it costs is one round trip for the token, one
// for its row and scale, and the output's bytes: 64 rows of 1,024 columns take 2.0 us, 2,048 rows 4.1 us (9.5 MB: 2.3 TB/s).
// A token outside the table gives zeros.
template <class T>
__global__ void __launch_bounds__(128) k_q4_rows(const fhe_q4 w, const int64_t* __restrict__ tokens, T* __restrict__ out,
                                                 long long ldo, uint32_t group_magic) {
    const int c = (blockIdx.y * 128 + threadIdx.x) * 8;
    if (c >= w.cols) return;
    const long long r = blockIdx.x;
    const int64_t t = tokens[r];
    float v[8];
    if (t >= 0 && t < w.rows) {
        const uint32_t q = *reinterpret_cast<const uint32_t*>(w.q + t * w.ldq + c / 2), ch = c / 32;
        const float s = ld_any(w.scale, w.scale_type, t * w.lds + (group_magic ? __umulhi(ch, group_magic) : ch));
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = (float)((int)(q >> (4 * j) & 15) - 8) * s;
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++) v[j] = 0.f;
    }
    T* o = out + r * ldo + c;
    __align__(16) T u[8];
#pragma unroll
    for (int j = 0; j < 8; j++) qg_store(&u[j], v[j]);
    if (c + 8 <= w.cols && reinterpret_cast<uintptr_t>(o) % 16 == 0) {
#pragma unroll
        for (int j = 0; j < (int)sizeof(T) / 2; j++) reinterpret_cast<uint4*>(o)[j] = reinterpret_cast<const uint4*>(u)[j];
    } else {
#pragma unroll
        for (int j = 0; j < 8; j++)
            if (c + j < w.cols) o[j] = u[j];
    }
}

template <class T>
static void q4_rows(Context& cx, const fhe_q4& w, const int64_t* tokens, int m, void* out, long long ldo, cudaStream_t st) {
    k_q4_rows<T><<<dim3(m, (w.cols + 1023) / 1024), 128, 0, st>>>(w, tokens, static_cast<T*>(out), ldo, q4_group_magic(w));
    CUDA_CHECK(cudaGetLastError());
    cx.launches++;
}

// ---- the choice of a token -----------------------------------------------------------------
// Per row of logits l (NaN counts as -inf), M = max l:
//   z = (l - M) / T (0 where l = M), e = exp(z), weight w = round(2^40 e), a whole number, so that sums of weights do
//   not depend on their order; tokens are ranked by l, equal ones by index;
//   kept: rank < top_k, sum of the weights ranked before < ceil(top_p * the top_k's sum), e >= min_p;
//   S = sum of the kept weights, the token is the first in index order whose running sum passes floor(u S).
//
// k_sample: a cluster of blocks per row, each with its part of the row in shared memory, so that the logits are read once.
// Nothing is sorted; some hundreds of tokens at most go to a list that one block selects from exactly.
//   top_k up to 1024: at least top_k tokens are no smaller than the top_k-th largest of the threads' own maxima, so the
//   list is what reaches that value, and everything else, exponentials included, is done on the list alone.
//   otherwise: e replaces the logits, and a histogram of it in 128 bins an octave (counts for top_k, 16 bits of
//   each e for top_p) tells the bins around the last kept token; their tokens are the list, the bins above are summed.
// 64 rows of 50,304 float32 logits at top_k 50 take 13.4 us (12.9 MB read: 1.0 TB/s), one such row at top_p 0.9 17.5; 64 bfloat16
// rows of 65,536 nearly equal ones at top_p 0.9, where every token has its exponential and its bin, 31 us, of which 14,000
// cycles are that pass (0.43 a token of the block's part) and the rest the cluster's syncs, the list's selection and the running sum.
// Parts of 32,768 logits and a cluster for the row, so that 64 rows of 50,304 are 128 blocks, one an SM.
// If the list overflows or the histogram's guess was off by more than a bin, one block selects on the row itself, by a radix search,
// while the cluster's others wait.  Equal logits overflow it, and flat rows without ties do where three bins, 1.2% to 2.3% of e at the
// cut, hold more than 2,560 tokens: 64 rows of 50,304 of standard deviation 0.3 at T 2 and top_p 0.5 take 192 us, one 175; one
// row of 262,144 of 0.6 at T 1.3 and top_p 0.6 1.17 ms (k_sample_long, whose blocks share the search, 0.20 for one token more).
constexpr int kSampleThreads = 1024, kSampleWarps = kSampleThreads / 32;
constexpr int kSampleRadix = 1024;              // bins of one step of the radix search
constexpr int kSamplePart = 32768;              // logits of a row that one block holds
constexpr int kSampleBins = 41 * 128 + 8;       // e from 1 down to 2^-41, below which a token has no weight
constexpr int kSampleList = 2560;
constexpr int kSampleClusterMax = 8;
constexpr float kSampleOne = 1099511627776.f;   // 2^40
// exp(-29) 2^40 = 0.28 rounds to no weight: what is further than 29 T below M is out
constexpr float kSampleReach = 29.f;

struct SampleArgs {
    const void* logits;
    long long ld;
    int type, rows, vocab;
    const float* u;
    const float *temperature, *top_p, *min_p;   // per row, or null: the one value
    const int32_t* top_k;
    float temperature1, top_p1, min_p1;
    int32_t top_k1;
    int64_t* token;
    float* logprob;
};

// larger for what is ranked first: the logit's bits in order, then the lower index
__device__ __forceinline__ uint64_t sample_rank_key(float x, uint32_t i) {
    const uint32_t b = __float_as_uint(x + 0.f);   // -0 and 0 are equal
    const uint32_t k = b & 0x80000000u ? ~b : b | 0x80000000u;
    return (uint64_t)k << 32 | (0xffffffffu - i);
}
__device__ __forceinline__ uint64_t sample_weight(float e) { return __float2ull_rn(e * kSampleOne); }
// bin 7: e = 1; bins 128 (i - 1) + 8 .. 128 i + 7: e from 2^(1 - i), not included, down to 2^-i
__device__ __forceinline__ int sample_bin(float e) { return (int)((0x3fffffffu - __float_as_uint(e)) >> 16) - 120; }
// e's bits are above this for the bins below b, and for no others
__device__ __forceinline__ uint32_t sample_bin_bits(int b) { return 0x3fffffffu - ((uint32_t)(b + 120) << 16); }
// a sum of the leading 16 bits of e, in bin b -> units of 2^-40
__device__ __forceinline__ uint64_t sample_bin_sum(uint64_t v, int b) {
    const int up = 40 - 15 - (b + 120) / 128;
    return up >= 0 ? v << up : v >> -up;
}

// sample_weight in two halves of 20 bits by float32 additions, for sums over many: the conversion to 64 bits is slow
__device__ __forceinline__ void sample_weight_add(float e, uint32_t& hi, uint32_t& lo) {
    const float b = e * 1048576.f, h = __fadd_rz(b, 8388608.f);           // its last bits: floor(b)
    const float l = __fmaf_rn(b - (h - 8388608.f), 1048576.f, 8388608.f);   // the rest, rounded to nearest even
    hi += __float_as_uint(h) - 0x4B000000u;
    lo += __float_as_uint(l) - 0x4B000000u;
}

struct SampleRow {
    const void* p;
    int type, v;
    float top, t, rt, reach;
    bool mul;   // t's reciprocal is far from the ends of float32, and M finite
    __device__ void set(const SampleArgs& a, int r) {
        p = static_cast<const uint8_t*>(a.logits) + (long long)r * a.ld * (a.type == FHE_F32 ? 4 : 2);
        type = a.type;
        v = a.vocab;
    }
    __device__ void scale(float top_, float t_) {
        top = top_;
        t = t_;
        rt = __frcp_rn(t_);
        reach = kSampleReach * t_;
        mul = t_ > 1e-30f && t_ < 1e30f && top_ < INFINITY;
    }
    __device__ float x(int i) const {
        const float a = ld_any(p, type, i);
        return a != a ? -INFINITY : a;
    }
    __device__ float z(float a) const { return a == top ? 0.f : __fdiv_rn(a - top, t); }
    __device__ bool counts(float a) const { return a == top || top - a <= reach; }
    // exp((a - M) / T), or 0 for a token without weight (below 2^-41; one half, which 2^-41 itself gives, rounds to the
    // even 0).  The quotient by the reciprocal and one correction of its exact remainder (Markstein 1990) is the rounded one; where
    // the difference is infinite it gives NaN, which has no weight either.
    __device__ __forceinline__ float e(float a) const {
        const float d = a - top;
        if (!mul) return a == top ? 1.f : e_cut(expf(__fdiv_rn(d, t)));
        const float q = d * rt;
        return e_cut(expf(__fmaf_rn(__fmaf_rn(-q, t, d), rt, q)));
    }
    __device__ __forceinline__ static float e_cut(float v) { return v >= 4.547473508864641e-13f ? v : 0.f; }
};

template <class T, class F>
__device__ T sample_reduce(T v, F f, T* sh) {
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    __syncthreads();
    if ((threadIdx.x & 31) == 0) sh[threadIdx.x >> 5] = v;
    __syncthreads();
    v = sh[threadIdx.x & 31];
    for (int o = 16; o; o >>= 1) v = f(v, __shfl_xor_sync(0xffffffffu, v, o));
    return v;
}
template <class T>
__device__ T sample_scan(T v) {   // inclusive, over a warp
    for (int o = 1; o < 32; o <<= 1) {
        const T n = __shfl_up_sync(0xffffffffu, v, o);
        if ((threadIdx.x & 31) >= o) v += n;
    }
    return v;
}
// inclusive over the block; sh: 32 values
template <class T>
__device__ T sample_block_scan(T v, T* sh) {
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    v = sample_scan(v);
    __syncthreads();
    if (lane == 31) sh[warp] = v;
    __syncthreads();
    const T w = sample_scan(sh[lane]);
    return v + (warp ? __shfl_sync(0xffffffffu, w, warp - 1) : T(0));
}

struct SampleRadix {
    uint64_t sum[kSampleRadix];
    uint32_t count[kSampleRadix];
    uint64_t key[32], wt[32];
    uint64_t red[32], red2[32];
    uint64_t got, before, before2;
    uint64_t mine;   // what a cluster's blocks show each other
    uint32_t n, at_count;
    int at;
};
struct SampleFound {
    uint64_t key, sum;   // the last kept token's rank key, and the sum of the weights down to it
};

// f over the values of the cluster's blocks, in their order; the same in every thread.  v is the same in a block.
template <class T, class F>
__device__ T sample_cluster(T v, F f, SampleRadix& sh) {
    static_assert(sizeof(T) <= sizeof(sh.mine), "");
    auto cluster = cooperative_groups::this_cluster();
    if (threadIdx.x == 0) *reinterpret_cast<T*>(&sh.mine) = v;
    cluster.sync();
    v = *reinterpret_cast<const T*>(&cluster.map_shared_rank(&sh, 0)->mine);
    for (unsigned b = 1; b < cluster.num_blocks(); b++) v = f(v, *reinterpret_cast<const T*>(&cluster.map_shared_rank(&sh, b)->mine));
    cluster.sync();
    return v;
}

// The token, in rank order, at which the running count (BY_COUNT) or sum of weights reaches `want` (>= 1); key 0 and the whole
// sum if none does.  each(f) calls f(rank key, weight()) for the calling thread's share of the tokens.  CLUSTER: the tokens are
// those of all the cluster's blocks, which call it together and all get the answer.
template <bool BY_COUNT, bool CLUSTER, class Each>
__device__ SampleFound sample_select(SampleRadix& sh, uint64_t want, Each each) {
    const int tid = threadIdx.x;
    const auto together = [] {
        if constexpr (CLUSTER) cooperative_groups::this_cluster().sync();
        else __syncthreads();
    };
    const auto smaller = [](uint64_t p, uint64_t q) { return min(p, q); };
    const auto larger = [](uint64_t p, uint64_t q) { return max(p, q); };
    uint64_t lo = ~0ull, hi = 0, before = 0;
    each([&](uint64_t k, auto) { lo = min(lo, k), hi = max(hi, k); });
    lo = sample_reduce(lo, smaller, sh.red);
    hi = sample_reduce(hi, larger, sh.red);
    if constexpr (CLUSTER) {
        lo = sample_cluster(lo, smaller, sh);
        hi = sample_cluster(hi, larger, sh);
    }
    if (hi == 0) return {0, 0};
    while (true) {
        // the tokens with keys in [lo, hi], in 1024 bins of equal width
        const int shift = max(0, 64 - __clzll((long long)(hi - lo)) - 10);
        sh.sum[tid] = 0;
        sh.count[tid] = 0;
        if (tid == 0) sh.at = -1, sh.n = 0;
        __syncthreads();
        each([&](uint64_t k, auto weight) {
            if (k < lo || k > hi) return;
            const int b = (int)((hi - k) >> shift);
            atomicAdd(&sh.count[b], 1u);
            atomicAdd((unsigned long long*)&sh.sum[b], (unsigned long long)weight());
        });
        together();
        uint64_t c = sh.count[tid], s = sh.sum[tid];
        if constexpr (CLUSTER) {
            auto cluster = cooperative_groups::this_cluster();
            for (unsigned b = 0; b < cluster.num_blocks(); b++) {
                if (b == cluster.block_rank()) continue;
                const SampleRadix* other = cluster.map_shared_rank(&sh, b);
                c += other->count[tid];
                s += other->sum[tid];
            }
            cluster.sync();   // the bins are read
        }
        const uint64_t sums = sample_block_scan(s, sh.red2);
        const uint64_t run = BY_COUNT ? sample_block_scan(c, sh.red) : sums, own = BY_COUNT ? c : s;
        if (run >= want && run - own < want) sh.at = tid, sh.at_count = c, sh.got = run - own, sh.before = before + sums - s;
        if (tid == kSampleRadix - 1) sh.before2 = before + sums;
        __syncthreads();
        const int at = sh.at;
        if (at < 0) return {0, sh.before2};
        want -= sh.got;
        before = sh.before;
        const uint32_t n = sh.at_count;
        // the bin's own range of keys
        const uint64_t top = hi - ((uint64_t)at << shift), bottom = top - ((1ull << shift) - 1);
        lo = bottom > top ? lo : max(lo, bottom);
        hi = top;
        if (n <= 32) {
            SampleRadix* list = &sh;   // the first block's
            if constexpr (CLUSTER) list = cooperative_groups::this_cluster().map_shared_rank(&sh, 0);
            each([&](uint64_t k, auto weight) {
                if (k < lo || k > hi) return;
                const uint32_t j = atomicAdd(&list->n, 1u);
                list->key[j] = k;
                list->wt[j] = weight();
            });
            together();
            if constexpr (CLUSTER) {
                if (list != &sh && tid < n) sh.key[tid] = list->key[tid], sh.wt[tid] = list->wt[tid];
                together();
            }
            if (tid < n) {
                uint64_t c = 0, s = 0;
                for (uint32_t l = 0; l < n; l++)
                    if (sh.key[l] > sh.key[tid]) c++, s += sh.wt[l];
                const uint64_t run = BY_COUNT ? c : s, own = BY_COUNT ? 1 : sh.wt[tid];
                if (run < want && run + own >= want) sh.got = sh.key[tid], sh.before2 = before + s + sh.wt[tid];
            }
            __syncthreads();
            const SampleFound f{sh.got, sh.before2};
            __syncthreads();
            return f;
        }
        __syncthreads();
    }
}

struct SampleSettings {
    float t, p, mp, u;
    int64_t k;
    __device__ SampleSettings(const SampleArgs& a, int r) {
        t = a.temperature ? a.temperature[r] : a.temperature1;
        p = a.top_p ? a.top_p[r] : a.top_p1;
        mp = a.min_p ? a.min_p[r] : a.min_p1;
        k = a.top_k ? a.top_k[r] : a.top_k1;
        u = fminf(fmaxf(a.u[r], 0.f), 1.f);     // a NaN: 0
        mp = mp > 0.f ? fminf(mp, 1.f) : 0.f;   // a NaN in the array: off
        if (!(t > 0.f)) t = 1.f, k = 1;
        t = fminf(t, 1e30f);
        if (k <= 0 || k >= a.vocab) k = 0;
    }
    // the running sum of weights that top_p asks for, of the top_k's sum s
    __device__ uint64_t limit(uint64_t s) const {
        const double w = ceil((double)p * (double)s);
        return w > 1.0 ? (uint64_t)w : 1;
    }
    __device__ uint64_t target(uint64_t s) const {
        const uint64_t v = (uint64_t)((double)u * (double)s);
        return v < s ? v : s - 1;
    }
};

// The first of a stretch [i0, i1) of tokens at which start + the running sum of kept(i) passes target, by one warp
template <class Kept>
__device__ int sample_walk(int i0, int i1, uint64_t start, uint64_t target, Kept kept) {
    const int lane = threadIdx.x & 31;
    for (int i = i0; i < i1; i += 32) {
        const uint64_t run = start + sample_scan(i + lane < i1 ? kept(i + lane) : 0ull);
        const uint32_t past = __ballot_sync(0xffffffffu, run > target);
        if (past) return i + __ffs(past) - 1;
        start = __shfl_sync(0xffffffffu, run, 31);
    }
    return -1;
}
__device__ __forceinline__ float sample_logprob(const SampleRow& row, int i, uint64_t total) {
    return row.z(row.x(i)) - (float)log((double)total / (double)kSampleOne);
}

// Rows longer than a cluster's shared memory: a cluster for each row, whose blocks read the logits again for every step.  A
// step is a few hundred instructions a token, so one block for a row of 300,000 took 1.9 ms; eight take 0.26.
__global__ void __launch_bounds__(kSampleThreads) k_sample_long(const SampleArgs a) {
    __shared__ SampleRadix sh;
    __shared__ float redf[32];
    auto cluster = cooperative_groups::this_cluster();
    const int nb = cluster.num_blocks(), rank = cluster.block_rank(), r = blockIdx.x / nb;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, first = rank * kSampleThreads + tid, step = nb * kSampleThreads;
    const SampleSettings set(a, r);
    SampleRow row;
    row.set(a, r);
    float top = -INFINITY;
    for (int i = first; i < row.v; i += step) top = fmaxf(top, row.x(i));
    const auto larger = [](float x, float y) { return fmaxf(x, y); };
    top = sample_cluster(sample_reduce(top, larger, redf), larger, sh);
    if (top == -INFINITY) {
        if (rank == 0 && tid == 0) a.token[r] = -1, a.logprob[r] = -INFINITY;
        return;
    }
    row.scale(top, set.t);
    auto each = [&](auto f) {
        for (int i = first; i < row.v; i += 4 * step) {   // four loads on their way
            float x[4];
#pragma unroll
            for (int j = 0; j < 4; j++) x[j] = i + j * step < row.v ? row.x(i + j * step) : -INFINITY;
#pragma unroll
            for (int j = 0; j < 4; j++)
                if (row.counts(x[j])) f(sample_rank_key(x[j], i + j * step), [&] { return sample_weight(row.e(x[j])); });
        }
    };
    uint64_t bound = 0;
    if (set.k) bound = sample_select<true, true>(sh, set.k, each).key;
    if (set.p < 1.f) {
        uint64_t s = 0;
        each([&](uint64_t k, auto weight) { s += k >= bound ? weight() : 0; });
        const auto plus = [](uint64_t x, uint64_t y) { return x + y; };
        s = sample_cluster(sample_reduce(s, plus, sh.red), plus, sh);
        bound = max(bound, sample_select<false, true>(sh, set.limit(s), each).key);
    }
    // a stretch of the row for each of the cluster's warps, in order
    const int warps = nb * kSampleWarps, per = (row.v + warps - 1) / warps;
    const int i0 = min(row.v, (rank * kSampleWarps + warp) * per), i1 = min(row.v, i0 + per);
    auto kept = [&](int i) -> uint64_t {
        const float x = row.x(i);
        if (!row.counts(x) || sample_rank_key(x, i) < bound) return 0;
        const float e = row.e(x);
        return e >= set.mp ? sample_weight(e) : 0;
    };
    uint64_t mine = 0;
    for (int i = i0 + lane; i < i1; i += 32) mine += kept(i);
    for (int o = 16; o; o >>= 1) mine += __shfl_xor_sync(0xffffffffu, mine, o);
    __syncthreads();
    if (lane == 0) sh.red[warp] = mine;
    __syncthreads();
    uint64_t own = 0, start = 0;
    for (int w = 0; w < kSampleWarps; w++) {
        if (w == warp) start = own;
        own += sh.red[w];
    }
    if (tid == 0) sh.mine = own;
    cluster.sync();
    uint64_t total = 0;
    for (int b = 0; b < nb; b++) {
        if (b == rank) start += total;
        total += cluster.map_shared_rank(&sh, b)->mine;
    }
    cluster.sync();   // a block leaves when the others have read it
    const uint64_t target = set.target(total);
    if (target < start || target >= start + mine) return;
    const int i = sample_walk(i0, i1, start, target, kept);
    if (lane == 0) a.token[r] = i, a.logprob[r] = sample_logprob(row, i, total);
}

// ---- selection from the list, by one block
constexpr int kSampleFew = 64, kSampleSmall = 256;
struct SampleList {
    // tokens: the logit, its index, e (-1: struck off)
    float x[kSampleList];
    uint32_t i[kSampleList];
    float e[kSampleList];
    uint32_t count[kSampleRadix], hi[kSampleRadix], lo[kSampleRadix];
    uint64_t few_key[kSampleFew], few_w[kSampleFew];
    uint64_t small_k[kSampleSmall], small_w[kSampleSmall];
    uint64_t red[32];
    uint64_t got, sum, before;
    uint32_t n, key_lo, key_hi;
    int at;
};
enum SamplePick { kByCount, kByWeight, kByIndex };

__device__ __forceinline__ uint32_t sample_order(float x) { return (uint32_t)(sample_rank_key(x, 0) >> 32); }

// Of the list's m tokens that are not struck off: the one, in rank order (kByIndex: in index order), at which the running count
// (kByCount) or sum of weights reaches want (>= 1).  Its rank key, or 0 if none does; *sum: the weights down to it (kByCount: all, if
// none does).
template <SamplePick BY>
__device__ uint64_t sample_pick(SampleList& l, uint32_t m, uint64_t want, uint64_t* sum) {
    const uint32_t tid = threadIdx.x, lane = tid & 31;
    bool by_order = BY != kByIndex;   // the search is on the logit's order first, then, among equal ones, on the index
    uint32_t equal = 0;
    uint64_t before = 0;
    const auto key = [&](uint32_t j) { return by_order ? sample_order(l.x[j]) : 0xffffffffu - l.i[j]; };
    const auto in = [&](uint32_t j) { return l.e[j] >= 0.f && (BY == kByIndex || by_order || sample_order(l.x[j]) == equal); };
    uint32_t lo = 0, hi = 0xffffffffu;
    if (m > kSampleFew) {
        while (true) {
            // the least and largest key from lo to hi
            if (tid == 0) l.key_lo = 0xffffffffu, l.key_hi = 0, l.at = -1;
            l.count[tid] = l.hi[tid] = l.lo[tid] = 0;
            __syncthreads();
            uint32_t a = 0xffffffffu, b = 0;
            for (uint32_t j = tid; j < m; j += kSampleThreads)
                if (in(j) && key(j) >= lo && key(j) <= hi) a = min(a, key(j)), b = max(b, key(j));
            a = __reduce_min_sync(0xffffffffu, a);
            b = __reduce_max_sync(0xffffffffu, b);
            if (lane == 0 && a <= b) atomicMin(&l.key_lo, a), atomicMax(&l.key_hi, b);
            __syncthreads();
            lo = l.key_lo;
            hi = l.key_hi;
            if (lo > hi) { *sum = before; return 0; }
            if (by_order && lo == hi) {   // many equal logits
                by_order = false;
                equal = hi;
                lo = 0, hi = 0xffffffffu;
                __syncthreads();
                continue;
            }
            // the tokens between them, in up to 1024 bins of equal width
            const int shift = max(0, 32 - __clz(hi - lo) - 10);
            for (uint32_t j = tid; j < m; j += kSampleThreads) {
                if (!in(j)) continue;
                const uint32_t k = key(j);
                if (k < lo || k > hi) continue;
                const uint32_t b = (hi - k) >> shift;
                const uint64_t w = sample_weight(l.e[j]);
                atomicAdd(&l.count[b], 1u);
                atomicAdd(&l.hi[b], (uint32_t)(w >> 20));        // the list's sums fit 32 bits in these halves
                atomicAdd(&l.lo[b], (uint32_t)w & 0xfffffu);
            }
            __syncthreads();
            const uint64_t w = ((uint64_t)l.hi[tid] << 20) + l.lo[tid], own = BY == kByCount ? l.count[tid] : w;
            const uint64_t run = sample_block_scan(own, l.red);
            if (run >= want && run - own < want) l.at = tid, l.got = run - own;
            if (tid == kSampleRadix - 1) l.sum = run;
            __syncthreads();
            const int at = l.at;
            if (at < 0) {
                if (BY == kByCount) {
                    uint64_t all = 0;
                    for (uint32_t j = tid; j < m; j += kSampleThreads) all += in(j) ? sample_weight(l.e[j]) : 0;
                    *sum = sample_reduce(all, [](uint64_t x, uint64_t y) { return x + y; }, l.red);
                } else {
                    *sum = before + l.sum;
                }
                __syncthreads();
                return 0;
            }
            want -= l.got;
            if (BY != kByCount) before += l.got;
            const uint32_t n = l.count[at], top = hi - ((uint32_t)at << shift), width = (1u << shift) - 1;
            lo = top - lo > width ? top - width : lo;
            hi = top;
            __syncthreads();
            if (n <= kSampleFew) break;
        }
    }
    // few: each against the others
    if (tid == 0) l.n = 0, l.got = 0, l.sum = before;
    __syncthreads();
    for (uint32_t j = tid; j < m; j += kSampleThreads) {
        if (!in(j) || key(j) < lo || key(j) > hi) continue;
        const uint32_t at = atomicAdd(&l.n, 1u);
        l.few_key[at] = BY == kByIndex ? 0xffffffffu - l.i[j] : sample_rank_key(l.x[j], l.i[j]);
        l.few_w[at] = sample_weight(l.e[j]);
    }
    __syncthreads();
    const uint32_t n = l.n;
    if (tid < n) {
        const uint64_t k = l.few_key[tid], w = l.few_w[tid];
        uint64_t c = 0, s = 0;
#pragma unroll 4
        for (uint32_t j = 0; j < n; j++)
            if (l.few_key[j] > k) c++, s += l.few_w[j];
        const uint64_t run = BY == kByCount ? c : s, own = BY == kByCount ? 1 : w;
        if (run < want && run + own >= want) l.got = k, l.sum = before + s + w;
    }
    __syncthreads();
    const uint64_t k = l.got;
    if (BY == kByCount) {
        // the weights down to it, whatever was left out of the few; all of them if no token is the one
        uint64_t all = 0;
        for (uint32_t j = tid; j < m; j += kSampleThreads)
            all += l.e[j] >= 0.f && sample_rank_key(l.x[j], l.i[j]) >= k ? sample_weight(l.e[j]) : 0;
        *sum = sample_reduce(all, [](uint64_t x, uint64_t y) { return x + y; }, l.red);
    } else {
        *sum = l.sum;
    }
    __syncthreads();
    return k;
}

constexpr int kSampleCoarse = kSampleBins / 8;   // the histogram in eighths, which blocks read of one another first
struct alignas(16) SampleShared {
    union {
        SampleList list;
        SampleRadix radix;   // where the list will not do
        uint32_t coarse_in[kSampleClusterMax][kSampleCoarse];   // before the list
    };
    uint64_t sum[kSampleClusterMax], above[kSampleClusterMax], part[kSampleClusterMax];   // each block writes its own to all
    float top[kSampleClusterMax], reach[kSampleClusterMax];
    uint32_t n[kSampleClusterMax];
    uint64_t bound, found;                  // block 0's answer
    int slow;
    uint64_t red[32];
    float redf[32];
    uint64_t want, guess, run_at;
    int at, lo;
    uint32_t listed, least;
    uint32_t warp_hi[kSampleWarps], warp_lo[kSampleWarps];
    alignas(16) uint32_t counts[kSampleBins], sums[kSampleBins];
    uint32_t coarse_counts[kSampleCoarse], coarse_sums[kSampleCoarse];
};
static_assert(sizeof(SampleShared) + (kSamplePart + 128) * sizeof(float) <= 232448, "a block's shared memory");

// n logits from row.p + first -> buf, as float32 without NaN; the calling thread's largest
template <class T>
__device__ __forceinline__ float sample_load(const SampleRow& row, int first, int n, float* buf) {
    const T* src = static_cast<const T*>(row.p) + first;
    constexpr int kVec = 16 / sizeof(T), kDeep = sizeof(T) == 4 ? 7 : 4;
    float top = -INFINITY;
    int done = 0;
    if (reinterpret_cast<uintptr_t>(src) % 16 == 0) {
        const int nv = n / kVec;
        for (int i = threadIdx.x; i < nv; i += kSampleThreads * kDeep) {
            uint4 v[kDeep];
#pragma unroll
            for (int d = 0; d < kDeep; d++)
                if (i + d * kSampleThreads < nv) v[d] = reinterpret_cast<const uint4*>(src)[i + d * kSampleThreads];
#pragma unroll
            for (int d = 0; d < kDeep; d++) {
                if (i + d * kSampleThreads >= nv) break;
                const T* u = reinterpret_cast<const T*>(&v[d]);
                float x[kVec];
#pragma unroll
                for (int j = 0; j < kVec; j++) {
                    x[j] = q4_float(u[j]);
                    if (x[j] != x[j]) x[j] = -INFINITY;
                    top = fmaxf(top, x[j]);
                }
#pragma unroll
                for (int j = 0; j < kVec; j += 4)
                    *reinterpret_cast<float4*>(buf + (size_t)(i + d * kSampleThreads) * kVec + j) =
                        make_float4(x[j], x[j + 1], x[j + 2], x[j + 3]);
            }
        }
        done = nv * kVec;
    }
    for (int i = done + threadIdx.x; i < n; i += kSampleThreads * 8) {
        T v[8];
#pragma unroll
        for (int d = 0; d < 8; d++)
            if (i + d * kSampleThreads < n) v[d] = src[i + d * kSampleThreads];
#pragma unroll
        for (int d = 0; d < 8; d++) {
            if (i + d * kSampleThreads >= n) break;
            float x = q4_float(v[d]);
            if (x != x) x = -INFINITY;
            top = fmaxf(top, x);
            buf[i + d * kSampleThreads] = x;
        }
    }
    return top;
}

// Value v of each block of the cluster, v at the same place of its SampleShared
template <class T>
__device__ __forceinline__ uint64_t sample_across(const cooperative_groups::cluster_group& cluster, T* v, int nb) {
    uint64_t sum = 0;
#pragma unroll
    for (int q = 0; q < kSampleClusterMax; q++)
        if (q < nb) sum += *cluster.map_shared_rank(v, q);
    return sum;
}

__global__ void __launch_bounds__(kSampleThreads) k_sample(const SampleArgs a) {
    namespace cg = cooperative_groups;
    extern __shared__ __align__(16) uint8_t ssm[];
    SampleShared& sh = *reinterpret_cast<SampleShared*>(ssm);
    SampleList& list = sh.list;
    float* buf = reinterpret_cast<float*>(ssm + sizeof(SampleShared));
    cg::cluster_group cluster = cg::this_cluster();
    const int nb = cluster.num_blocks(), rank = cluster.block_rank(), r = blockIdx.x / nb;
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    cluster.barrier_arrive();
    const SampleSettings set(a, r);
    const bool by_k = set.k != 0, by_p = set.p < 1.f;
    const auto larger = [](float x, float y) { return fmaxf(x, y); };
    const auto warp_sum = [&](uint64_t w) {
        for (int o = 16; o; o >>= 1) w += __shfl_xor_sync(0xffffffffu, w, o);
        return w;
    };
    const auto warps_sum = [&](uint64_t w) {   // of one value a warp, which stay in sh.red
        __syncthreads();
        if (lane == 0) sh.red[warp] = w;
        __syncthreads();
        return warp_sum(sh.red[lane]);
    };
    const auto block_sum = [&](uint64_t w) { return warps_sum(warp_sum(w)); };
    SampleRow row;
    row.set(a, r);
    const int part = ((row.v + nb - 1) / nb + 7) / 8 * 8, first = min(row.v, rank * part), n = min(row.v, first + part) - first;

    const float mine = a.type == FHE_F32   ? sample_load<float>(row, first, n, buf)
                       : a.type == FHE_F16 ? sample_load<__half>(row, first, n, buf)
                                           : sample_load<__nv_bfloat16>(row, first, n, buf);
    const int n4 = (n + 127) / 128 * 128;   // whole warps of four values a lane
    if (tid < n4 - n) buf[n + tid] = -INFINITY;
    float top = sample_reduce(mine, larger, sh.redf);
    // the least value that top_k threads' own maxima reach, to within a 1024th of their range
    bool few = by_k && set.k <= kSampleRadix;
    float reach = -INFINITY;
    if (few) {
        const float low = -sample_reduce(mine > -INFINITY ? -mine : -INFINITY, larger, sh.redf);
        list.count[tid] = 0;
        if (tid == 0) sh.at = -1, sh.least = 0xffffffffu;
        __syncthreads();
        const float width = top - low;
        int b = kSampleRadix;
        if (mine > -INFINITY) {
            b = mine == top ? 0 : (int)fminf((top - mine) / width * (kSampleRadix - 1), (float)(kSampleRadix - 1));
            atomicAdd(&list.count[b], 1u);
        }
        __syncthreads();
        const uint32_t own = list.count[tid], run = sample_block_scan(own, reinterpret_cast<uint32_t*>(sh.red));
        if (run >= set.k && run - own < set.k) sh.at = tid;
        __syncthreads();
        if (b <= sh.at) atomicMin(&sh.least, sample_order(mine));
        __syncthreads();
        if (sh.at >= 0) {
            const uint32_t o = sh.least;
            reach = __uint_as_float(o & 0x80000000u ? o ^ 0x80000000u : ~o);
        }
    }
    cluster.barrier_wait();   // every block runs
    if (tid < nb) {
        SampleShared* o = cluster.map_shared_rank(&sh, tid);
        o->top[rank] = top;
        o->reach[rank] = reach;
    }
    if (tid == 0) sh.listed = 0;
    cluster.sync();
    for (int b = 0; b < nb; b++) top = fmaxf(top, sh.top[b]), reach = fmaxf(reach, sh.reach[b]);
    if (top == -INFINITY) {   // in every block of the cluster
        if (rank == 0 && tid == 0) a.token[r] = -1, a.logprob[r] = -INFINITY;
        return;
    }
    row.scale(top, set.t);
    // each warp's stretch
    const int per = (n4 + 128 * kSampleWarps - 1) / (128 * kSampleWarps) * 128, i0 = min(n4, warp * per), i1 = min(n4, i0 + per);

    // token j of all blocks' lists, one after the other: the block's list and its place there
    const auto other = [&](uint32_t j, uint32_t& from) -> const SampleList* {
        int q = 0;
        while (j >= sh.n[q]) j -= sh.n[q++];
        from = j;
        return &cluster.map_shared_rank(&sh, q)->list;
    };
    if (few) {
        const auto take = [&](float x, int i) {
            if (x >= reach && x > -INFINITY) {
                const uint32_t j = atomicAdd(&sh.listed, 1u);
                if (j < kSampleList) list.x[j] = x, list.i[j] = first + i;
            }
        };
        for (int i = i0 + 4 * lane; i < i1; i += 128) {
            const float4 x = *reinterpret_cast<const float4*>(buf + i);
            if (fmaxf(fmaxf(x.x, x.y), fmaxf(x.z, x.w)) >= reach) take(x.x, i), take(x.y, i + 1), take(x.z, i + 2), take(x.w, i + 3);
        }
        __syncthreads();
        if (tid < nb) *cluster.map_shared_rank(&sh.n[rank], tid) = sh.listed;
        cluster.sync();
        uint32_t m = 0;
        for (int q = 0; q < nb; q++) m += sh.n[q];
        if (m <= kSampleList) {
            if (rank == 0) {
                for (uint32_t j = sh.n[0] + tid; j < m; j += kSampleThreads) {
                    uint32_t from;
                    const SampleList* o = other(j, from);
                    list.x[j] = o->x[from], list.i[j] = o->i[from];
                }
            }
            if (nb > 1) cluster.sync();
            if (rank) return;
            __syncthreads();
            uint64_t sum, total, pick;
            if (m <= kSampleSmall) {
                // Each token against the others, 4 to 32 threads a token: how many are ranked before it and their weights say
                // whether it is kept, the kept ones of lower index where its share of the sum begins.
                const int wide = m <= 32 ? 32 : m <= 64 ? 16 : m <= 128 ? 8 : 4;
                const uint32_t j = tid / wide, sub = tid & (wide - 1);
                if (tid < m) {
                    list.small_k[tid] = sample_rank_key(list.x[tid], list.i[tid]);
                    list.small_w[tid] = sample_weight(list.e[tid] = row.e(list.x[tid]));
                }
                __syncthreads();
                const uint64_t k = j < m ? list.small_k[j] : 0, w = j < m ? list.small_w[j] : 0;
                uint32_t c = 0;
                uint64_t s = 0;
                for (uint32_t l = sub; l < m; l += wide)
                    if (list.small_k[l] > k) c++, s += list.small_w[l];
                for (int o = wide / 2; o; o >>= 1) {
                    c += __shfl_xor_sync(0xffffffffu, c, o);
                    s += __shfl_xor_sync(0xffffffffu, s, o);
                }
                bool in = j < m && c < set.k;
                sum = block_sum(in && sub == 0 ? w : 0);
                in = in && (!by_p || s < set.limit(sum)) && list.e[j] >= set.mp;
                if (sub == 0 && j < m) list.small_w[j] = in ? w : 0;   // block_sum has waited for the readers
                total = block_sum(in && sub == 0 ? w : 0);
                const uint64_t target = set.target(total);
                s = 0;
                for (uint32_t l = sub; l < m; l += wide)
                    if ((uint32_t)list.small_k[l] > (uint32_t)k) s += list.small_w[l];
                for (int o = wide / 2; o; o >>= 1) s += __shfl_xor_sync(0xffffffffu, s, o);
                if (in && sub == 0 && s <= target && s + w > target) {
                    a.token[r] = list.i[j];
                    a.logprob[r] = sample_logprob(row, list.i[j], total);
                }
                return;
            }
            const auto strike = [&](uint64_t bound) {
                for (uint32_t j = tid; j < m; j += kSampleThreads)
                    if (sample_rank_key(list.x[j], list.i[j]) < bound) list.e[j] = -1.f;
                __syncthreads();
            };
            for (uint32_t j = tid; j < m; j += kSampleThreads) list.e[j] = row.e(list.x[j]);
            __syncthreads();
            uint64_t unused;
            strike(sample_pick<kByCount>(list, m, set.k, &sum));
            if (by_p) strike(sample_pick<kByWeight>(list, m, set.limit(sum), &sum));
            uint64_t w = 0;
            for (uint32_t j = tid; j < m; j += kSampleThreads) {
                if (list.e[j] < set.mp) list.e[j] = -1.f;
                if (list.e[j] > 0.f) w += sample_weight(list.e[j]);
            }
            total = block_sum(w);
            pick = sample_pick<kByIndex>(list, m, set.target(total) + 1, &unused);
            if (tid == 0) {
                const int i = (int)(0xffffffffu - (uint32_t)pick);
                a.token[r] = i;
                a.logprob[r] = sample_logprob(row, i, total);
            }
            return;
        }
    }

    // e in the logits' place; the histograms
    if (by_k || by_p)
        for (int b = tid; b < kSampleBins; b += kSampleThreads) sh.counts[b] = 0, sh.sums[b] = 0;
    if (tid < kSampleWarps) sh.warp_hi[tid] = sh.warp_lo[tid] = 0;
    __syncthreads();
    uint64_t all = 0;   // the whole sum
    uint32_t hi = 0, lo = 0;
    for (int i = i0 + 4 * lane; i < i1; i += 128) {
        const float4 x = *reinterpret_cast<const float4*>(buf + i);
        float e[4] = {row.e(x.x), row.e(x.y), row.e(x.z), row.e(x.w)};
        *reinterpret_cast<float4*>(buf + i) = make_float4(e[0], e[1], e[2], e[3]);
#pragma unroll
        for (int j = 0; j < 4; j++) {
            sample_weight_add(e[j] >= set.mp || by_p ? e[j] : 0.f, hi, lo);
            if (e[j] > 0.f) {
                if (by_k) atomicAdd(&sh.counts[sample_bin(e[j])], 1u);
                // 16 bits of e: a block's 2^15 tokens add up to less than 2^31
                if (by_p) atomicAdd(&sh.sums[sample_bin(e[j])], (__float_as_uint(e[j]) >> 8 & 0x7fffu) | 0x8000u);
            }
        }
    }
    // the weights of this warp's stretch: all of them if top_p needs their sum, else those that min_p keeps
    const auto stretch = [&](uint32_t hi, uint32_t lo) { return warp_sum(((uint64_t)hi << 20) + lo); };
    uint64_t warp_w = stretch(hi, lo);
    if (by_k || by_p) {
        const uint64_t s = warps_sum(warp_w);
        if (tid < kSampleCoarse) {
            const auto eight = [&](const uint32_t* h) {
                const uint4 u = reinterpret_cast<const uint4*>(h)[2 * tid], v = reinterpret_cast<const uint4*>(h)[2 * tid + 1];
                return u.x + u.y + u.z + u.w + v.x + v.y + v.z + v.w;
            };
            const uint32_t c = by_k ? eight(sh.counts) : 0, v = by_p ? eight(sh.sums) : 0;
            sh.coarse_counts[tid] = c;
            sh.coarse_sums[tid] = v;
            // what the first selection reads, to every block (loads across blocks take 500 cycles each way)
            for (int q = 0; q < nb; q++) cluster.map_shared_rank(&sh, q)->coarse_in[rank][tid] = by_k ? c : v;
        }
        if (tid < nb) *cluster.map_shared_rank(&sh.sum[rank], tid) = s;
        cluster.sync();
        for (int b = 0; b < nb; b++) all += sh.sum[b];
    }

    uint32_t cut = 0;   // kept are e with bits above this, and whatever the lists have not struck off
    bool summed = !by_k && (!by_p || set.mp == 0.f);   // warp_w follows what is kept as it is found
    // One selection.  The histogram tells a guess of the last kept token's bin; the tokens of that bin and its neighbours go to
    // the list, the weights above are summed, and block 0 selects.
    const auto locate = [&](bool by_count, uint64_t of) {
        const uint32_t* coarse = by_count ? sh.coarse_counts : sh.coarse_sums;
        const uint32_t* fine = by_count ? sh.counts : sh.sums;
        uint64_t own = 0;
        if (tid < kSampleCoarse) {
            if (by_count == by_k)
                for (int q = 0; q < nb; q++) own += sh.coarse_in[q][tid];
            else
                own = sample_across(cluster, &coarse[tid], nb);
            if (!by_count) own = sample_bin_sum(own, tid * 8);
        }
        const uint64_t run = sample_block_scan(own, sh.red);
        if (tid == 0) sh.at = -1, sh.listed = 0;
        if (tid == kSampleThreads - 1) {
            // what is asked for: top_k, or top_p's part of the sum; in the histogram's sums, which lack the bits below the leading
            // 16 of each all alike, a little less
            uint64_t want = set.k, guess = want;
            if (!by_count) {
                want = set.limit(of);
                const float lack = run < all ? (float)(all - run) / (float)all : 0.f;
                guess = want - (uint64_t)((float)want * lack);
                guess = guess < 1 ? 1 : guess > run ? run : guess;
            }
            sh.want = want;
            sh.guess = guess;
        }
        __syncthreads();
        const uint64_t want = sh.want, guess = sh.guess;
        if (run >= guess && run - own < guess) sh.at = tid, sh.run_at = run - own;
        __syncthreads();
        if (sh.at < 0) {   // no more than top_k have a weight: nothing is struck off
            __syncthreads();
            if (tid == 0) sh.found = all;
            __syncthreads();
            return;
        }
        if (warp == 0) {
            // the bin before the eighth's first (lane 0), its 8 bins (1 to 8)
            const int b = sh.at * 8 - 1 + lane;
            uint64_t v = lane < 9 && b >= 0 ? sample_across(cluster, &fine[b], nb) : 0;
            if (!by_count) v = sample_bin_sum(v, b);
            const uint64_t upto = sh.run_at - __shfl_sync(0xffffffffu, v, 0) + sample_scan(v);
            const uint32_t past = __ballot_sync(0xffffffffu, lane >= 1 && lane < 9 && upto >= guess);
            const int l = past ? __ffs(past) - 1 : 8;   // none: what single bins lose below 2^-40
            // one bin to either side: equal to the last place, exponentials need not be in their logits' order
            if (lane == l - 1) sh.lo = max(0, b), sh.run_at = upto - v;
        }
        __syncthreads();
        const int b0 = sh.lo, b1 = min(kSampleBins - 1, b0 + 2);
        const uint32_t above = sample_bin_bits(b0), in = max(cut, sample_bin_bits(b1 + 1));
        uint32_t hi = 0, lo = 0;
        for (int i = i0 + 4 * lane; i < i1; i += 128) {
            const float4 x = *reinterpret_cast<const float4*>(buf + i);
            const float e[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
            for (int j = 0; j < 4; j++) {
                const uint32_t bits = __float_as_uint(e[j]);
                sample_weight_add(bits > above ? e[j] : 0.f, hi, lo);
                if (bits > in && bits <= above) {
                    const uint32_t at = atomicAdd(&sh.listed, 1u);
                    if (at < kSampleList) list.i[at] = first + i + j, list.e[at] = e[j];
                }
            }
        }
        warp_w = stretch(hi, lo);
        const uint64_t s = warps_sum(warp_w);
        const uint32_t listed = min(sh.listed, (uint32_t)kSampleList);
        for (uint32_t j = tid; j < listed; j += kSampleThreads) list.x[j] = row.x(list.i[j]);
        if (tid < nb) {
            SampleShared* o = cluster.map_shared_rank(&sh, tid);
            o->above[rank] = s;
            o->n[rank] = sh.listed;
        }
        cluster.sync();
        if (rank == 0) {
            uint64_t over = 0, bound = 0, found = 0;
            uint32_t m = 0;
            for (int q = 0; q < nb; q++) over += sh.above[q], m += sh.n[q];
            bool slow = m > kSampleList || (!by_count && over >= want);
            if (!slow) {
                for (uint32_t j = sh.n[0] + tid; j < m; j += kSampleThreads) {
                    uint32_t from;
                    const SampleList* o = other(j, from);
                    list.x[j] = o->x[from], list.i[j] = o->i[from], list.e[j] = o->e[from];
                }
                __syncthreads();
                bound = by_count ? sample_pick<kByCount>(list, m, want - sh.run_at, &found)
                                 : sample_pick<kByWeight>(list, m, want - over, &found);
                found += over;
                slow = bound == 0;
            }
            if (slow) {
                const auto each = [&](auto f) {
                    for (int i = tid; i < row.v; i += kSampleThreads) {
                        const float x = row.x(i);
                        if (row.counts(x)) f(sample_rank_key(x, i), [&] { return sample_weight(row.e(x)); });
                    }
                };
                const SampleFound f = by_count ? sample_select<true, false>(sh.radix, want, each)
                                               : sample_select<false, false>(sh.radix, want, each);
                bound = f.key;
                found = f.sum;
            }
            if (tid < nb) {
                SampleShared* o = cluster.map_shared_rank(&sh, tid);
                o->bound = bound;
                o->found = found;
                o->slow = slow;
            }
        }
        cluster.sync();
        const uint64_t bound = sh.bound;
        if (sh.slow) {
            for (int i = i0 + lane; i < min(i1, n); i += 32)
                if (sample_rank_key(row.x(first + i), first + i) < bound) buf[i] = 0.f;
            summed = false;
        } else {
            for (uint32_t j = tid; j < listed; j += kSampleThreads) {
                const uint32_t i = list.i[j] - first;
                if (sample_rank_key(list.x[j], list.i[j]) < bound) {
                    buf[i] = 0.f;
                } else if (summed) {
                    const uint64_t w = sample_weight(list.e[j]);
                    atomicAdd(&sh.warp_hi[i / per], (uint32_t)(w >> 20));
                    atomicAdd(&sh.warp_lo[i / per], (uint32_t)w & 0xfffffu);
                }
            }
            cut = in;
        }
        __syncthreads();
    };
    if (by_k) locate(true, 0);
    if (by_p) locate(false, by_k ? sh.found : all);

    // the kept weights of each warp's stretch, block and cluster; the warp that the target falls to walks
    const auto kept = [&](float e) { return __float_as_uint(e) > cut && e >= set.mp ? e : 0.f; };
    if (summed) {
        warp_w += ((uint64_t)sh.warp_hi[warp] << 20) + sh.warp_lo[warp];
    } else {
        uint32_t hi = 0, lo = 0;
        for (int i = i0 + 4 * lane; i < i1; i += 128) {
            const float4 e = *reinterpret_cast<const float4*>(buf + i);
            sample_weight_add(kept(e.x), hi, lo);
            sample_weight_add(kept(e.y), hi, lo);
            sample_weight_add(kept(e.z), hi, lo);
            sample_weight_add(kept(e.w), hi, lo);
        }
        warp_w = stretch(hi, lo);
    }
    uint64_t total = warps_sum(warp_w);
    if (tid < nb) *cluster.map_shared_rank(&sh.part[rank], tid) = total;
    cluster.sync();
    total = 0;
    uint64_t start = 0;
    for (int b = 0; b < nb; b++) {
        if (b == rank) start = total;
        total += sh.part[b];
    }
    for (int w = 0; w < warp; w++) start += sh.red[w];   // warps_sum's
    const uint64_t target = set.target(total);
    if (target < start || target >= start + warp_w) return;
    for (int i = i0 + 4 * lane;; i += 128) {   // ends: the stretch's weights pass the target
        const float4 e = *reinterpret_cast<const float4*>(buf + i);
        const uint64_t w[4] = {sample_weight(kept(e.x)), sample_weight(kept(e.y)), sample_weight(kept(e.z)),
                               sample_weight(kept(e.w))};
        uint64_t run = start + sample_scan(w[0] + w[1] + w[2] + w[3]);
        const uint32_t past = __ballot_sync(0xffffffffu, run > target);
        if (past) {
            if (lane == __ffs(past) - 1) {
                int j = 3;
                while (run - w[j] > target) run -= w[j--];
                a.token[r] = first + i + j;
                a.logprob[r] = sample_logprob(row, first + i + j, total);
            }
            return;
        }
        start = __shfl_sync(0xffffffffu, run, 31);
    }
}

static void sample(Context& cx, const SampleArgs& a, cudaStream_t st) {
    // blocks for every SM, each with 1024 logits at least; a row has to fit its cluster
    int nb = 1;
    while (nb < kSampleClusterMax && (nb * kSamplePart < a.vocab || (a.rows * nb * 2 <= 148 && a.vocab >= 2048 * nb))) nb *= 2;
    const bool fits = a.vocab <= nb * kSamplePart;
    if (fits) client_smem<k_sample>(cx);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)a.rows * nb);
    cfg.blockDim = dim3(kSampleThreads);
    cfg.dynamicSmemBytes = fits ? sizeof(SampleShared) + (((size_t)a.vocab + nb - 1) / nb + 8 + 128) * sizeof(float) : 0;
    cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = nb;
    at[0].val.clusterDim.y = at[0].val.clusterDim.z = 1;
    cfg.attrs = at;
    cfg.numAttrs = 1;
    CUDA_CHECK(cudaLaunchKernelEx(&cfg, fits ? k_sample : k_sample_long, a));
    cx.launches++;
}

}  // namespace fhe

// ---- the C ABI --------------------------------------------------------------------------------
namespace {

int client_type_bytes(int type, const char* what) {
    if (type != FHE_F32 && type != FHE_F16 && type != FHE_BF16)
        throw fhe::Error(std::string(what) + ": unknown type", FHE_ERR_ARG);
    return type == FHE_F32 ? 4 : 2;
}

// device memory of the context's GPU, aligned to `align` bytes
void client_ptr(const fhe::Context& c, const void* p, size_t align, const char* what) {
    cudaPointerAttributes at{};
    if (!p) throw fhe::Error(std::string(what) + " is null", FHE_ERR_ARG);
    const cudaError_t e = cudaPointerGetAttributes(&at, p);
    if (e != cudaSuccess) {
        cudaGetLastError();
        throw fhe::Error(std::string("cannot query ") + what, FHE_ERR_ARG);
    }
    const bool dev = at.type == cudaMemoryTypeDevice || at.type == cudaMemoryTypeManaged;
    if (!dev || at.device != c.device)
        throw fhe::Error(std::string(what) + " is not device memory of the context's GPU", FHE_ERR_ARG);
    if (reinterpret_cast<uintptr_t>(p) % align)
        throw fhe::Error(std::string(what) + " is not " + std::to_string(align) + "-byte aligned", FHE_ERR_ARG);
}

void client_table(const fhe::Context& c, const fhe_q4* w) {
    REQUIRE(w, "null argument");
    // rows: the products count them, rounded up to their blocks' tiles, in 32 bits
    REQUIRE(w->rows >= 0 && w->rows <= FHE_Q4_MAX_ROWS && w->cols >= 1 && w->cols <= FHE_Q4_MAX_COLS,
            "q4 table: rows in 0..FHE_Q4_MAX_ROWS and cols in 1..FHE_Q4_MAX_COLS");
    REQUIRE(w->group >= 32 && w->group % 32 == 0, "q4 table: the group is a multiple of 32 columns");
    REQUIRE(w->ldq % 16 == 0 && w->ldq >= ((long long)w->cols + 31) / 32 * 16,
            "q4 table: rows are padded to a multiple of 16 bytes (32 columns)");
    REQUIRE(w->lds >= ((long long)w->cols + w->group - 1) / w->group, "q4 table: a scale for each group of a row");
    const int sb = client_type_bytes(w->scale_type, "q4 scales");
    if (!w->rows) return;
    client_ptr(c, w->q, 16, "q4 table");
    client_ptr(c, w->scale, sb, "q4 scales");
}

cudaStream_t client_stream(const fhe_ctx* cx, void* stream) {
    return stream ? static_cast<cudaStream_t>(stream) : cx->cx.stream;
}

// The context's GPU is the thread's current one for the length of a call, and the caller's again after it: these calls stand among
// torch's, which put theirs back.
struct ClientDevice {
    int was = -1;
    explicit ClientDevice(int device) {
        int now = -1;
        CUDA_CHECK(cudaGetDevice(&now));
        if (now == device) return;
        CUDA_CHECK(cudaSetDevice(device));
        was = now;
    }
    ~ClientDevice() {
        if (was >= 0) cudaSetDevice(was);
    }
    ClientDevice(const ClientDevice&) = delete;
};

}  // namespace

extern "C" int fhe_q4_matvec(fhe_ctx* cx, const fhe_q4* w, const void* x, int x_type, long long ldx, int m, void* out,
                             int out_type, long long ldo, void* stream) {
    return guard([&] {
        REQUIRE(cx, "null argument");
        client_table(cx->cx, w);
        const int xb = client_type_bytes(x_type, "x"), ob = client_type_bytes(out_type, "out");
        REQUIRE(m >= 0 && m <= FHE_Q4_MAX_M, "m in 0..FHE_Q4_MAX_M");
        REQUIRE(ldx >= w->cols || m <= 1, "x: rows are shorter than the table's columns");
        REQUIRE(ldo >= w->rows || m <= 1, "out: rows are shorter than the table's rows");
        if (m == 0 || w->rows == 0) return;
        client_ptr(cx->cx, x, xb, "x");
        client_ptr(cx->cx, out, ob, "out");
        const ClientDevice on(cx->cx.device);
        cudaStream_t st = client_stream(cx, stream);
        fhe::q4_matvec(cx->cx, fhe::Q4Args{*w, x, x_type, 0, m, ldx, out, out_type, ldo, 0, 0, 0, 0, 0, 0}, st);
    });
}

extern "C" int fhe_q4_rows(fhe_ctx* cx, const fhe_q4* w, const int64_t* tokens, int m, void* out, int out_type,
                           long long ldo, void* stream) {
    return guard([&] {
        REQUIRE(cx, "null argument");
        client_table(cx->cx, w);
        const int ob = client_type_bytes(out_type, "out");
        REQUIRE(m >= 0, "m is negative");
        REQUIRE(ldo >= w->cols || m <= 1, "out: rows are shorter than the table's columns");
        if (m == 0) return;
        client_ptr(cx->cx, tokens, 8, "tokens");
        client_ptr(cx->cx, out, ob, "out");
        const ClientDevice on(cx->cx.device);
        cudaStream_t st = client_stream(cx, stream);
        if (out_type == FHE_F32) fhe::q4_rows<float>(cx->cx, *w, tokens, m, out, ldo, st);
        else if (out_type == FHE_F16) fhe::q4_rows<__half>(cx->cx, *w, tokens, m, out, ldo, st);
        else fhe::q4_rows<__nv_bfloat16>(cx->cx, *w, tokens, m, out, ldo, st);
    });
}

extern "C" int fhe_sample(fhe_ctx* cx, const fhe_sample_cfg* cfg, const void* logits, int type, long long ld, int rows,
                          int vocab, const float* u, int64_t* token, float* logprob, void* stream) {
    return guard([&] {
        REQUIRE(cx && cfg, "null argument");
        const int b = client_type_bytes(type, "logits");
        REQUIRE(rows >= 0 && vocab >= 1, "sample: rows >= 0 and vocab >= 1");
        REQUIRE(vocab <= FHE_SAMPLE_MAX_VOCAB, "sample: the vocabulary is above FHE_SAMPLE_MAX_VOCAB");
        REQUIRE(ld >= vocab || rows <= 1, "logits: rows are shorter than the vocabulary");
        if (!cfg->temperature) REQUIRE(cfg->temperature_all >= 0.f && cfg->temperature_all <= 1e30f,
                                       "sample: temperature is a finite number >= 0");
        if (!cfg->top_k) REQUIRE(cfg->top_k_all >= 0, "sample: top_k >= 0 (0: off)");
        if (!cfg->top_p) REQUIRE(cfg->top_p_all > 0.f && cfg->top_p_all <= 1.f, "sample: top_p in (0, 1]");
        if (!cfg->min_p) REQUIRE(cfg->min_p_all >= 0.f && cfg->min_p_all <= 1.f, "sample: min_p in [0, 1]");
        if (rows == 0) return;
        client_ptr(cx->cx, logits, b, "logits");
        client_ptr(cx->cx, u, 4, "u");
        client_ptr(cx->cx, token, 8, "token");
        client_ptr(cx->cx, logprob, 4, "logprob");
        if (cfg->temperature) client_ptr(cx->cx, cfg->temperature, 4, "temperature");
        if (cfg->top_k) client_ptr(cx->cx, cfg->top_k, 4, "top_k");
        if (cfg->top_p) client_ptr(cx->cx, cfg->top_p, 4, "top_p");
        if (cfg->min_p) client_ptr(cx->cx, cfg->min_p, 4, "min_p");
        const ClientDevice on(cx->cx.device);
        cudaStream_t st = client_stream(cx, stream);
        fhe::SampleArgs a{logits, ld, type, rows, vocab, u, cfg->temperature, cfg->top_p, cfg->min_p, cfg->top_k,
                          cfg->temperature_all, cfg->top_p_all, cfg->min_p_all, cfg->top_k_all, token, logprob};
        fhe::sample(cx->cx, a, st);
    });
}
