// Orthogonalised updates: a list of float32 matrices U is replaced by an odd polynomial of each that moves its singular values towards
// one (Newton-Schulz iteration with the quintic the Muon optimiser uses), for the trained matrices of the segmentation networks.
//
//   X = U / (|U|_F + eps);   steps times:   A = X X^T,   X <- P X,   P = a I + b A + c A A           (X [m, n], m <= n: U or U^T)
//
// Flops per step: m^2 n + m^3 (two symmetric products, one triangle each) + 2 m^2 n.  The next step's A is P A P, symmetric as well, so several
// steps can stay on [m, m] matrices before their product is applied to X: done for wide matrices (or_group).
// The iteration magnifies small singular values by a per step, and with them whatever error the products leave (bfloat16 products: 1e-2 of
// the result after five steps, products of two bfloat16 halves 4e-5, float32 3e-6), so the products are float32-grade: every operand
// is kept as THREE bfloat16 planes, x = x0 + x1 + x2 (24 significant bits), and a product is the six plane products of weight 2^-16 or
// more, summed in float32 on the bfloat16 matrix cores -- six at 16 times the rate of the float32 matrix instructions.  The planes are
// written by the kernel that produces a matrix, once per element; the product kernels move bfloat16 only.
//
// All matrices of a group (or_group: two) go through each phase in ONE launch: a workgroup finds its matrix from the running tile counts of a table in the
// workspace.  The table travels in kernel arguments, one launch for 26 entries, so a captured graph keeps it.  Five steps of one matrix or of 26 of
// a group: 18 launches (near square), 20 (wide, 22 where long products are cut).
#include <algorithm>

#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 or_bf16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef short or_v4i16 __attribute__((ext_vector_type(4)));
typedef short or_v8i16 __attribute__((ext_vector_type(8)));
typedef uint32_t or_u32x4 __attribute__((ext_vector_type(4)));

constexpr int OR_NT = 512;                            // threads of a product workgroup
constexpr int OR_PAD = 64;                            // leading dimensions of the planes: multiples of it, zero-filled (the longest LDS stage)
constexpr int OR_SUM = 16384;                         // elements per workgroup of the norm
constexpr int OR_CHUNK = 26;                          // table entries per launch (kernel arguments: 4 KB)

enum { OR_P_SUM, OR_P_SPLIT, OR_P_GRAM, OR_P_SYM, OR_P_X, OR_PHASES };
enum { OR_B_X0, OR_B_X1, OR_B_A, OR_B_P0, OR_B_P1, OR_B_T, OR_B_Q, OR_BUFS };

struct OrMat {
    const float* src;
    float* dst;
    long long buf[OR_BUFS], sums, part;               // byte offsets of the planes, the norm's and the long products' partial sums in the workspace
    int rows, cols, m, n, ldx, lda;
    int splits, chunk;                                // pieces of the long axis in A = X X^T
    int first[OR_PHASES];                             // index of the matrix's first workgroup in each phase
    int pad;
};
struct OrChunk { OrMat mat[OR_CHUNK]; int base, count; };

__global__ void k_or_table(const OrChunk c, OrMat* __restrict__ table) {
    const int words = c.count * (int)(sizeof(OrMat) / 4);
    const int* s = reinterpret_cast<const int*>(c.mat);
    int* d = reinterpret_cast<int*>(table + c.base);
    for (int i = threadIdx.x; i < words; i += blockDim.x) d[i] = s[i];
}

// Workgroups are dealt to the eight dies in turn, each with an L2 of its own: die x takes every eighth group of OR_GROUP neighbouring tiles, so
// tiles that read the same rows mostly share an L2 (tile by tile over all dies the loads of a stage took longer than its products: 12 TB/s
// past the L2s); whole eighths of the list per die left the dies unequal work.
constexpr int OR_GROUP = 8;
__device__ __forceinline__ int or_tile() {
    const int w = blockIdx.x, whole = gridDim.x / (8 * OR_GROUP) * (8 * OR_GROUP);
    if (w >= whole) return w;
    const int i = w >> 3;
    return ((i / OR_GROUP) * 8 + (w & 7)) * OR_GROUP + i % OR_GROUP;
}

// the matrix workgroup `wg` of phase `ph` belongs to: the last one whose first workgroup is not behind it (one wave, 64 entries at a time)
__device__ __forceinline__ int or_find(const OrMat* __restrict__ table, int count, int ph, int wg) {
    int at = -1;
    for (int base = 0; base < count; base += 64) {
        const int i = base + (threadIdx.x & 63);
        const bool le = i < count && table[i].first[ph] <= wg;
        const unsigned long long mask = __ballot(le);
        at += __popcll(mask);
        if (mask != ~0ull) break;
    }
    return __builtin_amdgcn_readfirstlane(at);
}

// partial sums of squares in double (squares of small gradients leave float32's range), OR_SUM elements a workgroup
__global__ __launch_bounds__(256) void k_or_sum(const OrMat* __restrict__ table, int count, char* __restrict__ ws) {
    __shared__ double part[4];
    const OrMat& t = table[or_find(table, count, OR_P_SUM, blockIdx.x)];
    const int w = blockIdx.x - t.first[OR_P_SUM];
    const long long total = (long long)t.rows * t.cols, lo = (long long)w * OR_SUM, hi = min(total, lo + OR_SUM);
    double s = 0.0;
    const float* src = t.src;
#pragma unroll 8
    for (long long i = lo + threadIdx.x; i < hi; i += 256) {
        const double x = src[i];
        s = fma(x, x, s);
    }
    s = wave_sum(s);
    if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = s;
    __syncthreads();
    if (threadIdx.x == 0) reinterpret_cast<double*>(ws + t.sums)[w] = (part[0] + part[1]) + (part[2] + part[3]);
}

// LDS layouts.  K-contiguous operand: rows of BK values, the 16-byte chunks of a row permuted such that 8 rows of one chunk hit all banks.
template <int BK> __device__ __forceinline__ int or_row_at(int row, int chunk) { return row * BK + ((chunk ^ (BK == 32 ? (row >> 2) & 3 : (((row >> 1) & 1) << 2) | ((row >> 2) & 3))) << 3); }
// K-strided operand ([k][TB] as in memory): chunks permuted such that the 4 rows x 4 chunks of a transpose read hit all banks
template <int TB> __device__ __forceinline__ int or_col_at(int k, int chunk) {
    return k * TB + ((chunk ^ (TB == 128 ? ((k & 3) << 2) | ((k >> 2) & 3) : (((k >> 1) & 1) << 2) | ((k >> 2) & 3))) << 3);
}
template <int TB> __device__ __forceinline__ or_bf16x8 or_cols(const uint16_t* t, int k0, int c0, int lane) {
    const int i = lane & 15, k = k0 + 8 * (lane >> 5) + (i >> 2), c = c0 + (lane & 16) + 4 * (i & 3);
    typedef or_v4i16 __attribute__((address_space(3)))* lds_p;
    const or_v4i16 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(t + or_col_at<TB>(k, c >> 3) + (c & 7)));
    const or_v4i16 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(t + or_col_at<TB>(k + 4, c >> 3) + (c & 7)));
    const or_v8i16 v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
    return __builtin_bit_cast(or_bf16x8, v);
}

// 8 values -> one 16-byte store per plane
__device__ __forceinline__ void or_store8(uint16_t* p, long long plane, const float* v) {
    uint32_t w[3][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        float x = v[2 * i], y = v[2 * i + 1];
#pragma unroll
        for (int k = 0; k < 3; ++k) {
            w[k][i] = aadg_f2bf_pk(x, y);
            x -= __uint_as_float(w[k][i] << 16);
            y -= __uint_as_float(w[k][i] & 0xFFFF0000u);
        }
    }
#pragma unroll
    for (int k = 0; k < 3; ++k) *reinterpret_cast<uint4*>(p + k * plane) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
}
__device__ __forceinline__ void or_load8(const uint16_t* p, long long plane, float* v) {
    uint4 w[3];
#pragma unroll
    for (int k = 0; k < 3; ++k) w[k] = *reinterpret_cast<const uint4*>(p + k * plane);
    const uint32_t a[4] = {w[0].x, w[0].y, w[0].z, w[0].w}, b[4] = {w[1].x, w[1].y, w[1].z, w[1].w}, c[4] = {w[2].x, w[2].y, w[2].z, w[2].w};
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(a[i] << 16) + (__uint_as_float(b[i] << 16) + __uint_as_float(c[i] << 16));
        v[2 * i + 1] = __uint_as_float(a[i] & 0xFFFF0000u) + (__uint_as_float(b[i] & 0xFFFF0000u) + __uint_as_float(c[i] & 0xFFFF0000u));
    }
}

// X = U / (|U| + eps) as planes, 64 x 64 elements a workgroup, transposed through LDS where U is tall
__global__ __launch_bounds__(256) void k_or_planes(const OrMat* __restrict__ table, int count, char* __restrict__ ws, float eps) {
    __shared__ float tile[64][65];
    __shared__ float scale_s;
    const OrMat& t = table[or_find(table, count, OR_P_SPLIT, blockIdx.x)];
    const int m = t.m, n = t.n, ldx = t.ldx, cols = t.cols, tn = ldx / 64;
    const int w = blockIdx.x - t.first[OR_P_SPLIT], r0 = w / tn * 64, c0 = (w - w / tn * tn) * 64;
    const float* src = t.src;
    const bool tall = t.rows > t.cols;
    if (threadIdx.x < 64) {
        const int parts = (int)(((long long)t.rows * cols + OR_SUM - 1) / OR_SUM);
        const double* p = reinterpret_cast<const double*>(ws + t.sums);
        double s = 0.0;
        for (int i = threadIdx.x; i < parts; i += 64) s += p[i];
        s = wave_sum(s);
        if (threadIdx.x == 0) scale_s = (float)(1.0 / (sqrt(s) + (double)eps));
    }
    const int tx = threadIdx.x & 63, ty = threadIdx.x >> 6;
#pragma unroll
    for (int i = 0; i < 16; ++i) {
        const int y = ty + 4 * i;
        // X[r0 + y][c0 + tx]; tall: U[c0 + y][r0 + tx] = X[r0 + tx][c0 + y]
        if (!tall) tile[y][tx] = r0 + y < m && c0 + tx < n ? src[(long long)min(r0 + y, m - 1) * cols + min(c0 + tx, n - 1)] : 0.0f;
        else tile[tx][y] = c0 + y < n && r0 + tx < m ? src[(long long)min(c0 + y, n - 1) * cols + min(r0 + tx, m - 1)] : 0.0f;
    }
    __syncthreads();
    const float scale = scale_s;
    uint16_t* x = reinterpret_cast<uint16_t*>(ws + t.buf[OR_B_X0]);
    const long long plane = (long long)m * ldx;
#pragma unroll
    for (int i = 0; i < 2; ++i) {
        const int r = (threadIdx.x >> 3) + 32 * i, c = (threadIdx.x & 7) * 8;
        if (r0 + r >= m) continue;
        float v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) v[e] = tile[r][c + e] * scale;
        or_store8(x + (long long)(r0 + r) * ldx + c0 + c, plane, v);
    }
}

// what one product of a phase does: out = ca L R + cb E + cd I over the buffers of OrMat::buf (e < 0: no E).  Two of them: blockIdx.y.
struct OrOp { int l, r, o, e; float ca, cb, cd; };
struct OrOps { OrOp op[2]; };

// tile index -> (ti, tj), tj <= ti: w = ti (ti + 1) / 2 + tj
__device__ __forceinline__ void or_triangle(int w, int& ti, int& tj) {
    ti = (int)((sqrtf(8.0f * w + 1.0f) - 1.0f) * 0.5f);
    while (ti * (ti + 1) / 2 > w) --ti;
    while ((ti + 1) * (ti + 2) / 2 <= w) ++ti;
    tj = w - ti * (ti + 1) / 2;
}

// the finished tile, in LDS as float32 [TB][TB + 8], to the planes of a symmetric matrix: at (ti, tj), and mirrored at (tj, ti)
template <int TB>
__device__ __forceinline__ void or_store_symmetric(const OrMat& t, const float* tile, int ti, int tj, const OrOp& op, char* ws) {
    constexpr int TP = TB + 8, C8 = TB / 8;
    const int m = t.m, lda = t.lda;
    const long long plane = (long long)m * lda;
    uint16_t* out = reinterpret_cast<uint16_t*>(ws + t.buf[op.o]);
    const uint16_t* E = op.e < 0 ? nullptr : reinterpret_cast<const uint16_t*>(ws + t.buf[op.e]);
    const int i0 = ti * TB, j0 = tj * TB;
#pragma unroll 2
    for (int id = threadIdx.x; id < TB * C8; id += OR_NT) {
        const int r = id / C8, c = (id - r * C8) * 8, row = i0 + r, col = j0 + c;
        if (row >= m || col >= lda) continue;
        float v[8], e[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] = tile[r * TP + c + x] * op.ca;
        if (E != nullptr) {
            or_load8(E + (long long)row * lda + col, plane, e);
#pragma unroll
            for (int x = 0; x < 8; ++x) v[x] = fmaf(op.cb, e[x], v[x]);
        }
        if (op.cd != 0.0f) {
#pragma unroll
            for (int x = 0; x < 8; ++x) v[x] += row == col + x ? op.cd : 0.0f;
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] = col + x < m ? v[x] : 0.0f;
        or_store8(out + (long long)row * lda + col, plane, v);
    }
    if (ti == tj) return;
#pragma unroll 2
    for (int id = threadIdx.x; id < TB * C8; id += OR_NT) {                  // mirrored row = the tile's column: neighbouring lanes, neighbouring columns
        const int r8 = id / TB * 8, c = id - id / TB * TB, row = j0 + c, col = i0 + r8;
        if (row >= m || col >= lda) continue;
        float v[8], e[8];
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] = tile[(r8 + x) * TP + c] * op.ca;
        if (E != nullptr) {
            or_load8(E + (long long)row * lda + col, plane, e);
#pragma unroll
            for (int x = 0; x < 8; ++x) v[x] = fmaf(op.cb, e[x], v[x]);
        }
#pragma unroll
        for (int x = 0; x < 8; ++x) v[x] = col + x < m ? v[x] : 0.0f;
        or_store8(out + (long long)row * lda + col, plane, v);
    }
}

// One TB x TB tile of a product, 8 waves: 128: 64 x 32 each, stages of 32 values; 64: 32 x 32 each, two groups of four waves on the two
// halves of stages of 64 values (their sums meet in the tile).
//   PH = OR_GRAM: L = R = X (K = n, cut into t.splits pieces; more than one: the partial tile goes to the workspace for k_or_reduce), symmetric
//   PH = OR_SYM:  L, R symmetric matrices that commute, the product symmetric
//   PH = OR_X:    L symmetric, R = X, the K-strided operand (transpose reads); `last`: the result goes to the caller's matrix
// Of a symmetric product the tiles tj <= ti are computed and stored twice.  The lists are a few hundred tiles, a workgroup mostly has its CU for
// itself: two LDS buffers, one barrier a stage, the loads of the stage after the next in flight during the products.  Rows outside the
// matrix are read from its last row (their results are not stored); the contracted axis ends in zeros.
// The 53 matrices of the third and fourth stage of a SegFormer-B2 encoder: 1.43 ms for 149 Gflop, 0.63 PFLOP/s of bfloat16 products (0.10 of float32; a large
// float32 library product 0.15): a phase there is one to two rounds of tiles over the CUs, of which a product's last stores take a third (57 us for
// SYM: 18 stores, 32 the stages, 7 the rest).  Six large convolution matrices: 0.73 ms for 84 Gflop, 0.70 PFLOP/s.
enum { OR_GRAM, OR_SYM, OR_X };
template <int PH, int TB>
__global__ __launch_bounds__(OR_NT, 2) void k_or_mul(const OrMat* __restrict__ table, int count, char* __restrict__ ws, const OrOps ops, int last) {
    constexpr int BK = TB == 128 ? 32 : 64, CPR = BK / 8, WX = TB / 64, LR = 3 * TB * CPR / OR_NT;      // WX: 32-row blocks per wave; 16-byte chunks per thread and operand
    constexpr int TP = TB + 8, OPND = 3 * TB * BK, STAGE = 2 * OPND * 2, BYTES = 2 * STAGE > TB * TP * 4 ? 2 * STAGE : TB * TP * 4;
    __shared__ __attribute__((aligned(16))) char lds[BYTES];
    uint16_t* buf = reinterpret_cast<uint16_t*>(lds);                       // [2 stages][L, R][3 planes]
    constexpr int PHASE = PH == OR_GRAM ? OR_P_GRAM : PH == OR_SYM ? OR_P_SYM : OR_P_X;
    const int wg = or_tile();
    const OrMat& t = table[or_find(table, count, PHASE, wg)];
    const OrOp op = ops.op[blockIdx.y];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    int w = wg - t.first[PHASE], ti, tj, k_lo = 0, sp = 0;
    const uint16_t* L = reinterpret_cast<const uint16_t*>(ws + t.buf[op.l]);
    const uint16_t* R = reinterpret_cast<const uint16_t*>(ws + t.buf[op.r]);
    const int m = t.m, ldl = PH == OR_GRAM ? t.ldx : t.lda, ldr = PH == OR_SYM ? t.lda : t.ldx;
    int K = ldl;
    if (PH == OR_X) {
        const int tn = (t.ldx + TB - 1) / TB;
        ti = w / tn;
        tj = w - ti * tn;
    } else {
        if (PH == OR_GRAM) {
            sp = w % t.splits;
            w /= t.splits;
            k_lo = sp * t.chunk;
            K = min(K, k_lo + t.chunk);
        }
        or_triangle(w, ti, tj);
    }
    const long long pl_l = (long long)m * ldl, pl_r = (long long)m * ldr;
    const int i0 = ti * TB, j0 = tj * TB;
    const int wi = TB == 128 ? (wv >> 2) * 64 : (wv & 2) * 16, wj = TB == 128 ? (wv & 3) * 32 : (wv & 1) * 32, u0 = TB == 128 ? 0 : (wv >> 2) * 2;

    struct Regs { or_u32x4 l[LR], r[LR]; } ra, rb;                           // two stages under way
    auto fetch = [&](Regs& g, int k0) __attribute__((always_inline)) {
#pragma unroll
        for (int i = 0; i < LR; ++i) {
            const int id = tid + OR_NT * i;
            const int pl = id / (TB * CPR), q = id - pl * (TB * CPR), c = k0 + (q % CPR) * 8;
            g.l[i] = *reinterpret_cast<const or_u32x4*>(L + pl * pl_l + (long long)min(i0 + q / CPR, m - 1) * ldl + c);
            if (PH != OR_X) {
                g.r[i] = *reinterpret_cast<const or_u32x4*>(R + pl * pl_r + (long long)min(j0 + q / CPR, m - 1) * ldr + c);
            } else {
                const int pr = id / (BK * (TB / 8)), s = id - pr * (BK * (TB / 8));
                g.r[i] = *reinterpret_cast<const or_u32x4*>(R + pr * pl_r + (long long)min(k0 + s / (TB / 8), m - 1) * ldr + min(j0 + (s % (TB / 8)) * 8, ldr - 8));
            }
        }
    };
    auto stage = [&](const Regs& g, int b) __attribute__((always_inline)) {
        uint16_t *Ls = buf + b * 2 * OPND, *Rs = Ls + OPND;
#pragma unroll
        for (int i = 0; i < LR; ++i) {
            const int id = tid + OR_NT * i;
            const int pl = id / (TB * CPR), q = id - pl * (TB * CPR), at = pl * TB * BK + or_row_at<BK>(q / CPR, q % CPR);
            *reinterpret_cast<or_u32x4*>(&Ls[at]) = g.l[i];
            if (PH != OR_X) {
                *reinterpret_cast<or_u32x4*>(&Rs[at]) = g.r[i];
            } else {
                const int pr = id / (BK * (TB / 8)), s = id - pr * (BK * (TB / 8));
                *reinterpret_cast<or_u32x4*>(&Rs[pr * TB * BK + or_col_at<TB>(s / (TB / 8), s % (TB / 8))]) = g.r[i];
            }
        }
    };
    f32x16 acc[WX];
#pragma unroll
    for (int x = 0; x < WX; ++x)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[x][i] = 0.0f;
    auto multiply = [&](int b) __attribute__((always_inline)) {
        const uint16_t *Ls = buf + b * 2 * OPND, *Rs = Ls + OPND;
#pragma unroll
        for (int v = 0; v < 2; ++v) {
            const int u = u0 + v;
            or_bf16x8 l[3][WX], r[3];
#pragma unroll
            for (int p = 0; p < 3; ++p) {
#pragma unroll
                for (int x = 0; x < WX; ++x)
                    l[p][x] = __builtin_bit_cast(or_bf16x8, *reinterpret_cast<const or_u32x4*>(&Ls[p * TB * BK + or_row_at<BK>(wi + 32 * x + (lane & 31), 2 * u + h)]));
                if (PH != OR_X) r[p] = __builtin_bit_cast(or_bf16x8, *reinterpret_cast<const or_u32x4*>(&Rs[p * TB * BK + or_row_at<BK>(wj + (lane & 31), 2 * u + h)]));
                else r[p] = or_cols<TB>(&Rs[p * TB * BK], 16 * u, wj, lane);
            }
            // weights 2^-16, 2^-8, 1: the small ones first.  The six start from zero and their sum is added to the accumulator by the vector
            // unit: accumulating in the matrix instruction rounds 6 K / 16 times at the size of the whole sum and with a bias (3.7e-6
            // instead of 6e-7 of the result at K = 768)
            f32x16 d[WX] = {};
#pragma unroll
            for (int x = 0; x < WX; ++x) d[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(l[2][x], r[0], d[x], 0, 0, 0);
#pragma unroll
            for (int x = 0; x < WX; ++x) d[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(l[0][x], r[2], d[x], 0, 0, 0);
#pragma unroll
            for (int x = 0; x < WX; ++x) d[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(l[1][x], r[1], d[x], 0, 0, 0);
#pragma unroll
            for (int x = 0; x < WX; ++x) d[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(l[1][x], r[0], d[x], 0, 0, 0);
#pragma unroll
            for (int x = 0; x < WX; ++x) d[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(l[0][x], r[1], d[x], 0, 0, 0);
#pragma unroll
            for (int x = 0; x < WX; ++x) d[x] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(l[0][x], r[0], d[x], 0, 0, 0);
#pragma unroll
            for (int x = 0; x < WX; ++x)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[x][i] += d[x][i];
        }
    };
    // stage s is multiplied while s + 1 goes to the other buffer and s + 2, s + 3 are on their way (a trip past the L2, where the last phase's
    // workgroups of other dies left the data, takes longer than a stage's products); behind the end the last stage is read again, unused
    const int last_k = K - BK;
    fetch(ra, k_lo);
    fetch(rb, min(k_lo + BK, last_k));
    stage(ra, 0);
    __builtin_amdgcn_sched_barrier(0);                                        // (loads in the order in which the loop waits for them)
    fetch(ra, min(k_lo + 2 * BK, last_k));
    __syncthreads();
    int k0 = k_lo;
    for (; k0 + BK < K; k0 += 2 * BK) {
        stage(rb, 1);
        fetch(rb, min(k0 + 3 * BK, last_k));
        multiply(0);
        __syncthreads();
        stage(ra, 0);
        fetch(ra, min(k0 + 4 * BK, last_k));
        multiply(1);
        __syncthreads();
    }
    if (k0 < K) multiply(0);
    __syncthreads();
    // the tile goes through LDS (register i of half h = row 8 (i / 4) + 4 h + i % 4, lane & 31 = column: 2-byte stores of the planes straight from
    // the registers took longer than the product): pitch TB + 8 words, the two halves of a write 32 banks apart
    float* tile = reinterpret_cast<float*>(lds);
#pragma unroll
    for (int g = 0; g < (TB == 128 ? 1 : 2); ++g) {
        if (TB == 128 || (wv >> 2) == g) {
#pragma unroll
            for (int x = 0; x < WX; ++x)
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    float& at = tile[(wi + 32 * x + 8 * (i >> 2) + 4 * h + (i & 3)) * TP + wj + (lane & 31)];
                    at = g == 0 ? acc[x][i] : at + acc[x][i];
                }
        }
        __syncthreads();
    }
    if (PH == OR_GRAM && t.splits > 1) {
        float4* part = reinterpret_cast<float4*>(ws + t.part) + ((long long)w * t.splits + sp) * (TB * TB / 4);
        for (int id = tid; id < TB * TB / 4; id += OR_NT) {
            const int r = id / (TB / 4), c = (id - r * (TB / 4)) * 4;
            part[id] = *reinterpret_cast<const float4*>(&tile[r * TP + c]);
        }
        return;
    }
    if (PH != OR_X) {
        or_store_symmetric<TB>(t, tile, ti, tj, op, ws);
        return;
    }
    if (!last) {
        uint16_t* out = reinterpret_cast<uint16_t*>(ws + t.buf[op.o]);
        for (int id = tid; id < TB * (TB / 8); id += OR_NT) {
            const int r = id / (TB / 8), c = (id - r * (TB / 8)) * 8;
            if (i0 + r >= m || j0 + c >= t.ldx) continue;
            float v[8];
#pragma unroll
            for (int x = 0; x < 8; ++x) v[x] = tile[r * TP + c + x];
            or_store8(out + (long long)(i0 + r) * t.ldx + j0 + c, pl_r, v);
        }
        return;
    }
    const bool tall = t.rows > t.cols;
    for (int id = tid; id < TB * TB; id += OR_NT) {                             // lanes along the rows of the caller's matrix
        const int x = id / TB, y = id - x * TB, r = tall ? y : x, c = tall ? x : y;
        if (i0 + r < m && j0 + c < t.n) t.dst[tall ? (long long)(j0 + c) * t.cols + i0 + r : (long long)(i0 + r) * t.cols + j0 + c] = tile[r * TP + c];
    }
}

// joins the pieces of the long products A = X X^T in order
template <int TB>
__global__ __launch_bounds__(OR_NT) void k_or_reduce(const OrMat* __restrict__ table, int count, char* __restrict__ ws, const OrOps ops) {
    constexpr int TP = TB + 8;
    __shared__ __attribute__((aligned(16))) float tile[TB * TP];
    const int wg = or_tile();
    const OrMat& t = table[or_find(table, count, OR_P_SYM, wg)];
    if (t.splits == 1) return;                                                // (stored by the product itself)
    const int w = wg - t.first[OR_P_SYM];
    int ti, tj;
    or_triangle(w, ti, tj);
    const float4* part = reinterpret_cast<const float4*>(ws + t.part) + (long long)w * t.splits * (TB * TB / 4);
    for (int id = threadIdx.x; id < TB * TB / 4; id += OR_NT) {
        float4 s = part[id];
#pragma unroll 4
        for (int k = 1; k < t.splits; ++k) {
            const float4 x = part[(long long)k * (TB * TB / 4) + id];
            s.x += x.x; s.y += x.y; s.z += x.z; s.w += x.w;
        }
        const int r = id / (TB / 4), c = (id - r * (TB / 4)) * 4;
        *reinterpret_cast<float4*>(&tile[r * TP + c]) = s;
    }
    __syncthreads();
    or_store_symmetric<TB>(t, tile, ti, tj, ops.op[0], ws);
}

// ------------------------------------------------------------------------------------------------ host
constexpr int OR_MAX_SIDE = 1 << 16, OR_MAX_MATS = 4096;

struct OrLayout { size_t bytes; long long grid[OR_PHASES]; int n, tb_sym, tb_x; bool split; };

// Two groups, each with its own table and launches.
//   wide (n >= 2 m): the polynomial of two or three steps is taken on the Gram matrix, 13 m^3 + 6 m^2 n instead of 5 m^3 + 15 m^2 n flops
//   others: every step goes back to X.  On the Gram matrix small singular values carry the rounding of the large ones' squares, and a square
//   matrix has small ones: 3e-6 of the result instead of 5e-7 (64 x 64 noise; 1.1e-6 in plain float32), for no flops saved.
int or_group(const aadg_matrix& a) {
    const int64_t m = a.rows < a.cols ? a.rows : a.cols, n = (int64_t)a.rows + a.cols - m;
    return n >= 2 * m ? 1 : 0;
}

// The order of a group's table: most work first.  order: room for n entries; the number filled is returned
int64_t or_work(const aadg_matrix& a) {
    const int64_t m = a.rows < a.cols ? a.rows : a.cols;
    return m * ((int64_t)a.rows * a.cols + m * m);
}
int or_order(const aadg_matrix* mats, int n, int group, int* order) {
    int k = 0;
    for (int i = 0; i < n; ++i)
        if (or_group(mats[i]) == group) order[k++] = i;
    std::sort(order, order + k, [&](int x, int y) { return or_work(mats[x]) != or_work(mats[y]) ? or_work(mats[x]) > or_work(mats[y]) : x < y; });
    return k;
}

int or_check(const aadg_matrix* mats, int n) {
    if (mats == nullptr || n < 1 || n > OR_MAX_MATS) return AADG_E_BADARG;
    for (int i = 0; i < n; ++i) {
        if (mats[i].rows < 1 || mats[i].cols < 1) return AADG_E_BADARG;
        if (mats[i].rows > OR_MAX_SIDE || mats[i].cols > OR_MAX_SIDE || (long long)mats[i].rows * mats[i].cols > (1 << 28)) return AADG_E_UNSUPPORTED;
    }
    return 0;
}

// layout of a group behind byte `base` of the workspace: matrices order[0 .. k - 1]; fills the entries if `out` is given
int or_layout(const aadg_matrix* mats, const int* order, int k, size_t base, OrLayout& lay, OrMat* out) {
    // tiles of 128 (twice the products per LDS byte of 64) where a phase then still has a workgroup for every CU
    long long sym = 0, rect = 0;
    for (int i = 0; i < k; ++i) {
        const aadg_matrix& a = mats[order[i]];
        const long long m = a.rows < a.cols ? a.rows : a.cols, t = (m + 127) / 128;
        sym += t * (t + 1) / 2;
        rect += t * (((long long)a.rows + a.cols - m + 127) / 128);
    }
    lay.n = k;
    lay.tb_sym = sym >= 256 ? 128 : 64;
    lay.tb_x = rect >= 256 ? 128 : 64;
    sym = 0;
    for (int i = 0; i < k; ++i) {
        const aadg_matrix& a = mats[order[i]];
        const long long m = a.rows < a.cols ? a.rows : a.cols, t = (m + lay.tb_sym - 1) / lay.tb_sym;
        sym += t * (t + 1) / 2;
    }
    // pieces of the long axis: about two workgroups per CU, at least 512 values each (16 stages, as long as the join takes)
    const long long pieces = sym >= 512 ? 1 : sym > 0 ? (512 + sym - 1) / sym : 1;
    size_t at = base + aadg_align_up((size_t)k * sizeof(OrMat), 256);
    for (int p = 0; p < OR_PHASES; ++p) lay.grid[p] = 0;
    lay.split = false;
    for (int i = 0; i < k; ++i) {
        const aadg_matrix& a = mats[order[i]];
        OrMat t = {};
        t.src = a.src; t.dst = a.dst; t.rows = a.rows; t.cols = a.cols;
        t.m = t.rows < t.cols ? t.rows : t.cols;
        t.n = t.rows < t.cols ? t.cols : t.rows;
        t.ldx = (t.n + OR_PAD - 1) / OR_PAD * OR_PAD;
        t.lda = (t.m + OR_PAD - 1) / OR_PAD * OR_PAD;
        const long long parts = ((long long)t.rows * t.cols + OR_SUM - 1) / OR_SUM, tm = (t.m + lay.tb_sym - 1) / lay.tb_sym, ts = tm * (tm + 1) / 2;
        const long long xm = (t.m + lay.tb_x - 1) / lay.tb_x, xn = (t.ldx + lay.tb_x - 1) / lay.tb_x;
        long long sp = pieces < t.ldx / 512 ? pieces : t.ldx / 512;
        if (sp < 1) sp = 1;
        t.chunk = (int)aadg_align_up((size_t)((t.ldx + sp - 1) / sp), OR_PAD);
        t.splits = (t.ldx + t.chunk - 1) / t.chunk;
        lay.split = lay.split || t.splits > 1;
        const size_t px = aadg_align_up((size_t)3 * t.m * t.ldx * 2, 256), pa = aadg_align_up((size_t)3 * t.m * t.lda * 2, 256);
        for (int b = 0; b < OR_BUFS; ++b) { t.buf[b] = (long long)at; at += b == OR_B_X0 || b == OR_B_X1 ? px : pa; }
        t.sums = (long long)at; at += aadg_align_up((size_t)parts * 8, 256);
        t.part = (long long)at; at += t.splits > 1 ? (size_t)ts * t.splits * lay.tb_sym * lay.tb_sym * 4 : 0;
        const long long wgs[OR_PHASES] = {parts, (long long)((t.m + 63) / 64) * (t.ldx / 64), ts * t.splits, ts, xm * xn};
        for (int p = 0; p < OR_PHASES; ++p) {
            t.first[p] = (int)lay.grid[p];
            lay.grid[p] += wgs[p];
            if (lay.grid[p] > 0x7FFFFFFF) return AADG_E_UNSUPPORTED;
        }
        if (out != nullptr) out[i] = t;
    }
    lay.bytes = at - base;
    return 0;
}

struct OrRun {
    const OrLayout& lay;
    const OrMat* table;
    int n;
    char* ws;
    hipStream_t st;
    void gram(int x) const {
        const OrOps o = {{{x, x, OR_B_A, -1, 1.0f, 0.0f, 0.0f}}};
        const dim3 grid((unsigned)lay.grid[OR_P_GRAM]), join((unsigned)lay.grid[OR_P_SYM]);
        if (lay.tb_sym == 128) hipLaunchKernelGGL((k_or_mul<OR_GRAM, 128>), grid, dim3(OR_NT), 0, st, table, n, ws, o, 0);
        else hipLaunchKernelGGL((k_or_mul<OR_GRAM, 64>), grid, dim3(OR_NT), 0, st, table, n, ws, o, 0);
        if (!lay.split) return;
        if (lay.tb_sym == 128) hipLaunchKernelGGL((k_or_reduce<128>), join, dim3(OR_NT), 0, st, table, n, ws, o);
        else hipLaunchKernelGGL((k_or_reduce<64>), join, dim3(OR_NT), 0, st, table, n, ws, o);
    }
    void sym(const OrOps& o, int count) const {
        const dim3 grid((unsigned)lay.grid[OR_P_SYM], (unsigned)count);
        if (lay.tb_sym == 128) hipLaunchKernelGGL((k_or_mul<OR_SYM, 128>), grid, dim3(OR_NT), 0, st, table, n, ws, o, 0);
        else hipLaunchKernelGGL((k_or_mul<OR_SYM, 64>), grid, dim3(OR_NT), 0, st, table, n, ws, o, 0);
    }
    void sym(OrOp a) const { sym(OrOps{{a, a}}, 1); }
    void apply(int l, int x, int y, bool last) const {
        const OrOps o = {{{l, x, y, -1, 1.0f, 0.0f, 0.0f}}};
        const dim3 grid((unsigned)lay.grid[OR_P_X]);
        if (lay.tb_x == 128) hipLaunchKernelGGL((k_or_mul<OR_X, 128>), grid, dim3(OR_NT), 0, st, table, n, ws, o, last);
        else hipLaunchKernelGGL((k_or_mul<OR_X, 64>), grid, dim3(OR_NT), 0, st, table, n, ws, o, last);
    }
};

// group 1: blocks of two and three steps on the Gram matrix; group 0: blocks of one
int or_steps(const OrRun& run, int group, int steps, float a, float b, float c) {
    int x = OR_B_X0, y = OR_B_X1;
    for (int done = 0; done < steps;) {
        const int most = group == 0 ? 1 : done == 0 ? 2 : 3, block = steps - done < most ? steps - done : most;
        done += block;
        run.gram(x);
        int p = OR_B_P0, p2 = OR_B_P1, q = -1, free_q = OR_B_Q;                // q: the product of the block's P so far
        for (int k = 0; k < block; ++k) {
            run.sym({OR_B_A, OR_B_A, p, OR_B_A, c, b, a});                    // P = a I + b A + c A A
            const OrOp fold = {p, q, q < 0 ? -1 : (q == OR_B_Q ? OR_B_T : free_q), -1, 1.0f, 0.0f, 0.0f};        // Q <- P Q
            const OrOp half = {p, OR_B_A, OR_B_T, -1, 1.0f, 0.0f, 0.0f};       // T = P A
            const bool more = k + 1 < block;
            if (q < 0) {
                if (more) run.sym(half);
                q = p;
            } else if (more) {
                run.sym(OrOps{{half, fold}}, 2);
                q = fold.o;
            } else {
                run.sym(fold);
                q = fold.o;
            }
            if (more) run.sym({OR_B_T, p, OR_B_A, -1, 1.0f, 0.0f, 0.0f});      // A <- P A P
            const int s = p;
            p = p2;
            p2 = s;
        }
        run.apply(q, x, y, done == steps);
        const int s = x;
        x = y;
        y = s;
        AADG_LAUNCH_CHECK();
    }
    return 0;
}

}  // namespace

// the two groups' layouts, the second behind the first.  order: 2 n ints of scratch, the groups' matrices in table order
static int or_plan(const aadg_matrix* mats, int n, int* order, OrLayout* lay) {
    size_t base = 0;
    for (int g = 0; g < 2; ++g) {
        const int rc = or_layout(mats, order + g * n, or_order(mats, n, g, order + g * n), base, lay[g], nullptr);
        if (rc != 0) return rc;
        base += lay[g].bytes;
    }
    return 0;
}

extern "C" size_t aadg_orthogonalize_workspace_bytes(const aadg_matrix* mats_host, int n) {
    if (or_check(mats_host, n) != 0) return 0;
    int* order = (int*)malloc((size_t)n * 2 * sizeof(int));
    if (order == nullptr) return 0;
    OrLayout lay[2];
    const int rc = or_plan(mats_host, n, order, lay);
    free(order);
    return rc == 0 ? lay[0].bytes + lay[1].bytes : 0;
}

extern "C" int aadg_orthogonalize_f32(const aadg_matrix* mats_host, int n, int steps, float a, float b, float c, float eps, void* ws,
                                      size_t ws_bytes, void* stream) {
    int rc = or_check(mats_host, n);
    if (rc != 0) return rc;
    if (steps < 1 || steps > 64 || !(eps >= 0.0f)) return AADG_E_BADARG;
    for (int i = 0; i < n; ++i)
        if (mats_host[i].src == nullptr || mats_host[i].dst == nullptr || (uintptr_t)mats_host[i].src % 4 != 0 || (uintptr_t)mats_host[i].dst % 4 != 0)
            return AADG_E_BADARG;
    OrMat* entries = (OrMat*)malloc((size_t)n * (sizeof(OrMat) + 2 * sizeof(int)));
    if (entries == nullptr) return AADG_E_WORKSPACE;
    int* order = (int*)(entries + n);
    OrLayout lay[2];
    rc = or_plan(mats_host, n, order, lay);
    if (rc == 0 && (ws == nullptr || (uintptr_t)ws % 256 != 0 || ws_bytes < lay[0].bytes + lay[1].bytes)) rc = AADG_E_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    size_t base = 0;
    // every matrix is read (norms, planes) before any result is written: dst may be another group's src
    for (int pass = 0; pass < 2 && rc == 0; ++pass) {
        base = 0;
        for (int g = 0; g < 2 && rc == 0; ++g) {
            const int k = lay[g].n;
            OrMat* table = (OrMat*)((char*)ws + base);
            if (k > 0 && pass == 0) {
                or_layout(mats_host, order + g * n, k, base, lay[g], entries);
                for (int i = 0; i < k; i += OR_CHUNK) {
                    static_assert(sizeof(OrChunk) + sizeof(OrMat*) <= 4096, "kernel arguments");
                    OrChunk chunk = {};
                    chunk.base = i;
                    chunk.count = k - i < OR_CHUNK ? k - i : OR_CHUNK;
                    memcpy(chunk.mat, entries + i, (size_t)chunk.count * sizeof(OrMat));
                    hipLaunchKernelGGL(k_or_table, dim3(1), dim3(256), 0, st, chunk, table);
                }
                hipLaunchKernelGGL(k_or_sum, dim3((unsigned)lay[g].grid[OR_P_SUM]), dim3(256), 0, st, table, k, (char*)ws);
                hipLaunchKernelGGL(k_or_planes, dim3((unsigned)lay[g].grid[OR_P_SPLIT]), dim3(256), 0, st, table, k, (char*)ws, eps);
                const hipError_t e = hipGetLastError();
                if (e != hipSuccess) rc = (int)e;
            } else if (k > 0) {
                rc = or_steps(OrRun{lay[g], table, k, (char*)ws, st}, g, steps, a, b, c);
            }
            base += lay[g].bytes;
        }
    }
    free(entries);
    return rc;
}
