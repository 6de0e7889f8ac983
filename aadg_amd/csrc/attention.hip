// Softmax attention, forward and backward, for the transformer blocks of the SegFormer backbone (reference:
// models/mmseg/models/backbones/mix_transformer.py:86-100 `attn = (q @ k^T) * scale; softmax; attn @ v`).
//
//   s_ij = scale q_i . k_j            allowed(i, j): j < L_b  and  (not causal or j <= i + L_b - Nq)
//   lse_i = log sum_allowed exp s_ij  p_ij = exp(s_ij - lse_i)      o_i = sum_j p_ij v_j        (no allowed key: o_i = 0)
//   D_i = do_i . o_i                  ds_ij = p_ij (do_i . v_j - D_i)
//   dq_i = scale sum_j ds_ij k_j      dk_j = scale sum_i ds_ij q_i      dv_j = sum_i p_ij do_i
//
// The score matrix never reaches memory: the forward keeps a running maximum and sum per row (one pass over the keys) and leaves
// lse_i in base 2 (4 bytes a row), from which the backward recomputes p.
//
// Heads that share one key head (H = G r) are FOLDED into the rows: a workgroup of group g works on the R = r Nq rows
// (head g r + row / Nq, query row % Nq), so the keys are read once for all of them and the sums of dk / dv over the shared heads
// are part of the same accumulation.
//
// Matrix-core layout (one code for both types, template parameter T).  C of a 32 x 32 product: lane & 31 = column, register r of lane
// half h = row 8 (r / 4) + 4 h + r % 4.  The scores are taken TRANSPOSED where a lane must own a query (forward, dq: columns =
// queries, the row maximum and sum are in-register plus one exchange of the halves) and straight where a lane must own a key (dk,
// dv).  Either way the probabilities are the next product's B operand as they lie in the registers: the k slots of an MFMA are
// summed over, so any order of them is right as long as A uses the same one -- a B fragment made of C registers has slot (h, e) =
// row 4 h + e (and 8 + 4 h + e), and the A fragment is read from LDS for those rows.
//   bfloat16: v_mfma_f32_32x32x16_bf16, fragments of 8 values; the transposed A operand with ds_read_b64_tr_b16.
//   float32:  v_mfma_f32_32x32x2_f32, four per fragment of 4 values: exact float32 products (scores go through an exponential: a product
//             split in two bfloat16 halves, 2^-17 relative, would move p by |s| 2^-17).
// The probabilities and ds are rounded to bfloat16 for the second products of the bfloat16 kernels (half a step, 2^-8 relative, of
// factors whose partner is bfloat16 as well); maxima, sums, lse, D and every accumulator are float32.
#include "common.h"

namespace {

typedef __attribute__((ext_vector_type(8))) __bf16 at_bf16x8;
typedef __attribute__((ext_vector_type(16))) float f32x16;
typedef uint32_t at_u32x4 __attribute__((ext_vector_type(4)));
typedef short at_v4i16 __attribute__((ext_vector_type(4)));

__device__ __forceinline__ float at_exp2(float x) { return __builtin_amdgcn_exp2f(x); }     // v_exp_f32: 1 ulp, results below 2^-126 are 0

constexpr float AT_LAZY = 8.0f;                       // base-2 logarithm
constexpr float AT_LOG2E = 1.4426950408889634f;

struct AtStride { long long b, h, n; };               // elements: batch, head, row (the head dimension itself is contiguous)

struct AtArgs {
    const void *q, *k, *v, *o, *dout;
    void *out, *dq, *dk, *dv;                         // out: o (forward)
    const int* key_lengths;
    float* lse;                                       // [B, H, Nq] base-2 log-sum-exp; +inf for a row without keys
    float* delta;                                     // [B, H, Nq] D_i (backward)
    float *part, *ml;                                 // split partials: [splits][rows][d] and [splits][rows][2]
    AtStride sq, sk, sv, so, sdo, sdq, sdk, sdv;
    int B, H, G, Nq, Nk, d, causal, r, R;
    int tiles, splits, chunk;                         // row (or key) tiles per group, splits of the loop axis, its length per split
    float scale;
    unsigned mul;                                     // at_head
    int shift;
};

template <typename T> struct At;
template <> struct At<uint16_t> {
    static constexpr int KS = 16, CH = 8;             // values of the contracted axis per fragment; elements per 16 bytes
    typedef at_bf16x8 Frag;
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) { return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0); }
    static __device__ __forceinline__ Frag pack(const f32x16& c, int g) {
        const at_u32x4 p = {aadg_f2bf_pk(c[8 * g], c[8 * g + 1]), aadg_f2bf_pk(c[8 * g + 2], c[8 * g + 3]),
                            aadg_f2bf_pk(c[8 * g + 4], c[8 * g + 5]), aadg_f2bf_pk(c[8 * g + 6], c[8 * g + 7])};
        return __builtin_bit_cast(Frag, p);
    }
    // what pack() rounds off
    static __device__ __forceinline__ Frag rest(const f32x16& c, int g) {
        const at_u32x4 x = __builtin_bit_cast(at_u32x4, pack(c, g));
        at_u32x4 y;
#pragma unroll
        for (int i = 0; i < 4; ++i)
            y[i] = aadg_f2bf_pk(c[8 * g + 2 * i] - __uint_as_float(x[i] << 16), c[8 * g + 2 * i + 1] - __uint_as_float(x[i] & 0xFFFF0000u));
        return __builtin_bit_cast(Frag, y);
    }
    static __device__ __forceinline__ float dot(Frag a, Frag b, float s) {
        const at_u32x4 x = __builtin_bit_cast(at_u32x4, a), y = __builtin_bit_cast(at_u32x4, b);
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            s = fmaf(__uint_as_float(x[i] << 16), __uint_as_float(y[i] << 16), s);
            s = fmaf(__uint_as_float(x[i] & 0xFFFF0000u), __uint_as_float(y[i] & 0xFFFF0000u), s);
        }
        return s;
    }
    static __device__ __forceinline__ void store4(uint16_t* p, float a, float b, float c, float d) {
        *reinterpret_cast<uint2*>(p) = make_uint2(aadg_f2bf_pk(a, b), aadg_f2bf_pk(c, d));
    }
};
template <> struct At<float> {
    static constexpr int KS = 8, CH = 4;
    typedef aadg_f32x4 Frag;
    static __device__ __forceinline__ f32x16 mma(Frag a, Frag b, f32x16 c) {
#pragma unroll
        for (int e = 0; e < 4; ++e) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a[e], b[e], c, 0, 0, 0);
        return c;
    }
    static __device__ __forceinline__ Frag pack(const f32x16& c, int g) { return Frag{c[4 * g], c[4 * g + 1], c[4 * g + 2], c[4 * g + 3]}; }
    static __device__ __forceinline__ float dot(Frag a, Frag b, float s) {
#pragma unroll
        for (int i = 0; i < 4; ++i) s = fmaf(a[i], b[i], s);
        return s;
    }
    static __device__ __forceinline__ void store4(float* p, float a, float b, float c, float d) {
        *reinterpret_cast<float4*>(p) = make_float4(a, b, c, d);
    }
};

// A tile of rows x D in LDS, row-major.  bfloat16: rows 16 banks (mod 64) apart, the four 16-byte chunks of a group permuted by the number of the
// row's group of four: row reads (16 rows, one chunk) and transpose reads (4 rows, 4 neighbouring chunks) touch every bank once, and
// because the permutation stays within four chunks a fragment's address is one of two registers and an immediate (a permutation of
// whole rows took 40 address registers).
// float32: pitch D + 8 words (row reads of 16 bytes: 8 banks apart; column reads: the two halves, 4 rows apart, 32 banks apart).
template <typename T, int D> struct Tile;
template <int D> struct Tile<uint16_t, D> {
    static constexpr int PITCH = D == 32 ? 32 : D + 32;
    static __device__ __forceinline__ int at(int row, int chunk) { return row * PITCH + ((chunk ^ ((row >> 2) & 3)) << 3); }
    // rows row0 + (lane & 31), values KS u + 8 h .. + 7; row0 a multiple of 16
    static __device__ __forceinline__ at_bf16x8 rows(const uint16_t* t, int row0, int u, int lane) {
        const uint16_t* base = t + (lane & 31) * PITCH + (((2 * (u & 1) + (lane >> 5)) ^ ((lane >> 2) & 3)) << 3);
        return __builtin_bit_cast(at_bf16x8, *reinterpret_cast<const at_u32x4*>(base + row0 * PITCH + 32 * (u >> 1)));
    }
    // column c0 + (lane & 31), rows row0 + 4 h + {0..3} and row0 + 8 + 4 h + {0..3}, row0 a multiple of 16, c0 of 32: ds_read_b64_tr_b16 gives
    // lane i of 16 the 4 rows of column i; the lane passes the address of row i / 4, columns 4 (i % 4)
    static __device__ __forceinline__ at_bf16x8 cols(const uint16_t* t, int row0, int c0, int lane) {
        const int i = lane & 15, h = lane >> 5, ch = ((lane >> 3) & 2) + ((i >> 1) & 1);
        const uint16_t* p = t + (4 * h + (i >> 2)) * PITCH + 4 * (i & 1) + row0 * PITCH + c0;
        typedef at_v4i16 __attribute__((address_space(3)))* lds_p;
        const at_v4i16 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(p + ((ch ^ h) << 3)));
        const at_v4i16 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(p + ((ch ^ h ^ 2) << 3) + 8 * PITCH));
        typedef short v8i16 __attribute__((ext_vector_type(8)));
        const v8i16 v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
        return __builtin_bit_cast(at_bf16x8, v);
    }
};
template <int D> struct Tile<float, D> {
    static constexpr int PITCH = D + 8;
    static __device__ __forceinline__ int at(int row, int chunk) { return row * PITCH + (chunk << 2); }
    static __device__ __forceinline__ aadg_f32x4 rows(const float* t, int row0, int u, int lane) {
        return *reinterpret_cast<const aadg_f32x4*>(t + at(row0 + (lane & 31), 2 * u + (lane >> 5)));
    }
    static __device__ __forceinline__ aadg_f32x4 cols(const float* t, int row0, int c0, int lane) {
        const float* p = t + (row0 + 4 * (lane >> 5)) * PITCH + c0 + (lane & 31);
        return aadg_f32x4{p[0], p[PITCH], p[2 * PITCH], p[3 * PITCH]};
    }
};

// 16 bytes of row `row` (clamped into 0 .. n - 1), chunk c (clamped into the d values) of a strided matrix; at_keep zeroes what does not exist.  Two
// steps: the prefetched values are masked when they go to LDS, not where they are loaded (a select there waits for memory), and without a
// branch per load.
template <typename T> __device__ __forceinline__ at_u32x4 at_fetch(const T* base, long long stride, int row, int n, int c, int d) {
    return *reinterpret_cast<const at_u32x4*>(base + (long long)min(row, n - 1) * stride + min(c * At<T>::CH, d - At<T>::CH));
}
__device__ __forceinline__ at_u32x4 at_keep(at_u32x4 x, bool ok) {
    const uint32_t m = ok ? 0xFFFFFFFFu : 0u;
    return x & at_u32x4{m, m, m, m};
}
template <typename T> __device__ __forceinline__ at_u32x4 at_load(const T* base, long long stride, int row, int n, int c, int d) {
    return at_keep(at_fetch<T>(base, stride, row, n, c, d), row < n && c * At<T>::CH < d);
}

// head of a folded row within its group, row / Nq: the high half of row * mul, shifted (exact for row < 2^31: mul = ceil(2^(32 + shift) / Nq))
__device__ __forceinline__ int at_head(const AtArgs& a, int row) { return a.r == 1 ? 0 : a.Nq == 1 ? row : (int)(__umulhi((unsigned)row, a.mul) >> a.shift); }

// folded row -> element offset of a [B, H, Nq] strided matrix for group g
__device__ __forceinline__ long long at_row(const AtArgs& a, const AtStride& s, int b, int g, int row) {
    const int hr = at_head(a, row), i = row - hr * a.Nq;
    return b * s.b + (long long)(g * a.r + hr) * s.h + (long long)i * s.n;
}
__device__ __forceinline__ int at_query(const AtArgs& a, int row) { return row - at_head(a, row) * a.Nq; }

__device__ __forceinline__ int at_len(const AtArgs& a, int b) {
    return a.key_lengths == nullptr ? a.Nk : max(0, min(a.Nk, a.key_lengths[b]));
}

// keys a folded row sees: [0, at_limit)
__device__ __forceinline__ int at_limit(const AtArgs& a, int L, int row) {
    return a.causal ? max(0, min(L, at_query(a, row) + L - a.Nq + 1)) : L;
}

// the largest limit of rows [row0, row0 + n): the last one's, or L if the range holds the last query of a head
__device__ __forceinline__ int at_limit_max(const AtArgs& a, int L, int row0, int n) {
    const int last = min(row0 + n, a.R) - 1;
    if (!a.causal) return L;
    if (at_head(a, row0) != at_head(a, last)) return L;
    return at_limit(a, L, last);
}

// waves per SIMD the registers are budgeted for: two (256 registers), one for head widths over 64
template <typename T, int D> constexpr int at_min_waves() { return D == 128 ? 1 : 2; }

// keys per LDS tile: 64; 32 where the next tile's prefetch registers (2 BK D / threads values) would not fit beside the accumulators.  The one-wave float32
// backward (up to 32 rows or keys) is over its 256 registers all the same: k_attn_dkv<float, 64, 1> keeps 31 of them in memory, k_attn_dq<float, 64, 1>
// 16 ... 18, k_attn_dkv_pair<float, 128, 2> 6.
template <typename T, int D, int NW> constexpr int at_bk() { return NW == 1 || (sizeof(T) == 4 && D == 128) ? 32 : 64; }

// group and row tile of a workgroup.  Causal: by the length of the tiles' rows, all groups and heads side by side, the longest first, so that the
// launch does not end in long tiles; up to 512 workgroups, which all have a place at once where a CU takes two (number i and i + 256), the second half
// backwards, so that a CU has a long and a short one.  Two waves a SIMD is what bfloat16 width 128 and float32 width 64 run, the kernels that gain
// (two causal sequences of 4096, D = 128, forward and backward: 655 -> 600 us); bfloat16 widths of 64 and 32 have three and four (768 and 1024 places),
// float32 width 128 one, where the order is only another one.  (Tiles of a head: the r heads' in turn, exact where Nq is a multiple of the tile.)
__device__ __forceinline__ void at_row_tile(const AtArgs& a, int w, bool split, int& bg, int& tile) {
    if (!a.causal || split) {
        bg = w / a.tiles;
        tile = w - bg * a.tiles;
        return;
    }
    const int n = a.B * a.G, rank = w / n, half = (a.tiles + 1) / 2, per = a.tiles / a.r, rest = a.tiles - per * a.r;
    bg = w - rank * n;
    int i = gridDim.x > 512 || rank < half ? rank : a.tiles - 1 - (rank - half);
    tile = per * a.r + i;
    if (i < rest) return;
    i -= rest;
    const int q = i / a.r;
    tile = (i - q * a.r) * per + per - 1 - q;
}

// ------------------------------------------------------------------------------------------------ forward
// Workgroup: NW waves of 32 folded rows; keys in tiles of BK through LDS, the next tile's loads in registers during the products.
// Times in a loop of calls (single launches of the larger shapes take a tenth more under a profiler).  bfloat16, 48 x 16384 rows, 256 keys, D = 64: 98 us,
// 0.53 PFLOP/s: vector instructions issue in 0.66 of a CU's busy cycles (exponential, maximum, sum, packing: as many a score as D / 32 matrix
// instructions' share), the matrix units work in 0.26, waves wait 0.30 of their time -- no unit is at its limit.  Two causal sequences of 8192, 16 heads over
// 4, D = 128: 580 ... 607 us on two cards, 0.91 ... 0.95 PFLOP/s, vector 0.57, matrix 0.47 (800 us with each head's tiles in a row).  float32, 240 x 1024 rows, 256
// keys, D = 64: 155 us, 104 TFLOP/s of the 153 that a large float32 product reaches, matrix units 0.74.  A workgroup that holds all 256
// keys takes 88 us for the first case, but there is one to a CU and rows are cut into whole rounds of them (96 groups: 3/4 of the CUs), so this form
// serves every shape.  Two row blocks a wave take the same time.
template <typename T, int D, int NW, bool SPLIT>
__global__ __launch_bounds__(64 * NW, (at_min_waves<T, D>())) void k_attn_fwd(const AtArgs a) {
    typedef At<T> M;
    typedef Tile<T, D> L_;
    constexpr int BK = at_bk<T, D, NW>(), KS = M::KS, CH = M::CH, U = D / KS, CPR = D / CH, NT = 64 * NW, LD = BK * CPR / NT, DT = D / 32, PG = 16 / (KS / 2), KT = BK / 32;
    __shared__ __attribute__((aligned(16))) T Ks[BK * L_::PITCH];
    __shared__ __attribute__((aligned(16))) T Vs[BK * L_::PITCH];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int sp = SPLIT ? blockIdx.x % a.splits : 0;
    const int w = SPLIT ? blockIdx.x / a.splits : blockIdx.x;
    int bg, tile;
    at_row_tile(a, w, SPLIT, bg, tile);
    const int b = bg / a.G, g = bg - b * a.G;
    const int L = at_len(a, b);
    const int row0 = tile * 32 * NW + 32 * wv, row = row0 + (lane & 31);
    const bool live = row < a.R;
    const int k_lo = SPLIT ? sp * a.chunk : 0;
    const int wg_end = min(at_limit_max(a, L, tile * 32 * NW, 32 * NW), SPLIT ? k_lo + a.chunk : L);
    const int limit = live ? at_limit(a, L, row) : 0;
    const int wave_end = row0 < a.R ? at_limit_max(a, L, row0, 32) : 0;
    int wave_full = limit;                                                    // keys every row of the wave sees
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) wave_full = min(wave_full, __shfl_xor(wave_full, o, 64));
    wave_full = __builtin_amdgcn_readfirstlane(wave_full);

    const T* kb = (const T*)a.k + b * a.sk.b + (long long)g * a.sk.h;
    const T* vb = (const T*)a.v + b * a.sv.b + (long long)g * a.sv.h;
    typename M::Frag qf[U];
    {
        const T* qp = (const T*)a.q + at_row(a, a.sq, b, g, live ? row : 0);
#pragma unroll
        for (int u = 0; u < U; ++u) qf[u] = __builtin_bit_cast(typename M::Frag, at_load<T>(qp, 0, live ? 0 : 1, 1, 2 * u + h, a.d));
    }
    f32x16 acc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
    float m = -INFINITY, l = 0.0f;
    const float c = a.scale * AT_LOG2E;

    at_u32x4 rk[LD], rv[LD];
    auto fetch = [&](int k0) {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int id = tid + NT * i, rw = id / CPR, ch = id - rw * CPR;
            rk[i] = at_fetch<T>(kb, a.sk.n, k0 + rw, L, ch, a.d);
            rv[i] = at_fetch<T>(vb, a.sv.n, k0 + rw, L, ch, a.d);
        }
    };
    if (k_lo < wg_end) fetch(k_lo);
    for (int k0 = k_lo; k0 < wg_end; k0 += BK) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int id = tid + NT * i, rw = id / CPR, ch = id - rw * CPR;
            const bool ok = k0 + rw < L && ch * CH < a.d;
            *reinterpret_cast<at_u32x4*>(&Ks[L_::at(rw, ch)]) = at_keep(rk[i], ok);
            *reinterpret_cast<at_u32x4*>(&Vs[L_::at(rw, ch)]) = at_keep(rv[i], ok);
        }
        __syncthreads();
        if (k0 + BK < wg_end) fetch(k0 + BK);
        if (k0 >= wave_end) continue;                                         // (wave-uniform; the barriers above are reached by all)
        f32x16 s[KT];
#pragma unroll
        for (int t = 0; t < KT; ++t) {
#pragma unroll
            for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
#pragma unroll
            for (int u = 0; u < U; ++u) s[t] = M::mma(L_::rows(Ks, 32 * t, u, lane), qf[u], s[t]);
        }
        if (k0 + BK > wave_full) {
#pragma unroll
            for (int t = 0; t < KT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    s[t][i] = k0 + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3) < limit ? s[t][i] : -INFINITY;
        }
        // the reference value m of the exponentials follows the maximum only when that has grown by more than AT_LAZY: accumulator and sum
        // are rescaled in a few tiles instead of every one, p stays below 2^AT_LAZY
        float mx = s[0][0];
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) mx = fmaxf(mx, s[t][i]);
        mx = fmaxf(mx, __shfl_xor(mx, 32, 64)) * c;
        if (__any(mx > m + AT_LAZY)) {
            const float mn = fmaxf(m, mx), alpha = mn == -INFINITY ? 1.0f : at_exp2(m - mn);
            m = mn;
            l *= alpha;
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i) acc[t][i] *= alpha;
        }
        const float mc = m == -INFINITY ? 0.0f : m;
        float sum = 0.0f;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[t][i] = at_exp2(fmaf(s[t][i], c, -mc));
                sum += s[t][i];
            }
        l += sum;
#pragma unroll
        for (int t = 0; t < KT; ++t)
#pragma unroll
            for (int p = 0; p < PG; ++p) {
                const typename M::Frag pf = M::pack(s[t], p);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[dt] = M::mma(L_::cols(Vs, 32 * t + KS * p, 32 * dt, lane), pf, acc[dt]);
            }
    }
    l += __shfl_xor(l, 32, 64);
    if (!live) return;
    const long long flat = ((long long)b * a.G + g) * a.R + row;              // = (b H + head) Nq + query
    if (SPLIT) {
        const long long rows = (long long)a.B * a.G * a.R;
        if (h == 0) {
            a.ml[2 * (sp * rows + flat)] = m;
            a.ml[2 * (sp * rows + flat) + 1] = l;
        }
        float* op = a.part + (sp * rows + flat) * a.d;
#pragma unroll
        for (int t = 0; t < DT; ++t)
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int col = 32 * t + 8 * i + 4 * h;
                if (col < a.d) *reinterpret_cast<float4*>(op + col) = make_float4(acc[t][4 * i], acc[t][4 * i + 1], acc[t][4 * i + 2], acc[t][4 * i + 3]);
            }
        return;
    }
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);           // NaN stays
    T* op = (T*)a.out + at_row(a, a.so, b, g, row);
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = 32 * t + 8 * i + 4 * h;
            if (col < a.d) M::store4(op + col, acc[t][4 * i] * inv, acc[t][4 * i + 1] * inv, acc[t][4 * i + 2] * inv, acc[t][4 * i + 3] * inv);
        }
    if (h == 0 && a.lse != nullptr) a.lse[flat] = l == 0.0f ? INFINITY : m + log2f(l);
}

// joins the splits of the forward: one wave per row.  The lanes take the splits' (m, l) at once (at most 64 splits), then groups of d / 4 lanes
// take every 64 / (d / 4)-th split's partial row; a fixed order throughout.
template <typename T>
__global__ __launch_bounds__(256) void k_attn_join(const AtArgs a) {
    const long long rows = (long long)a.B * a.G * a.R, flat = (long long)blockIdx.x * 4 + (threadIdx.x >> 6);
    if (flat >= rows) return;
    const int lane = threadIdx.x & 63, per = a.d / 4, groups = 64 / per, grp = lane / per, col = (lane - grp * per) * 4;
    float ms = -INFINITY, ls = 0.0f;
    if (lane < a.splits) {
        const float2 x = *reinterpret_cast<const float2*>(a.ml + 2 * (lane * rows + flat));
        ls = x.y;
        if (ls != 0.0f) ms = x.x;                                             // l = 0: no key of this split, its partial row is not read
    }
    const float m = wave_max(ms);
    const float wgt = ls != 0.0f ? at_exp2(ms - m) : 0.0f;
    const float l = wave_sum(ls * wgt);
    float4 o = make_float4(0, 0, 0, 0);
    for (int s0 = 0; s0 < a.splits; s0 += groups) {
        const int s = s0 + grp;
        const float w = __shfl(wgt, s & 63, 64);
        if (grp < groups && s < a.splits && w != 0.0f) {
            const float4 x = *reinterpret_cast<const float4*>(a.part + (s * rows + flat) * a.d + col);
            o.x = fmaf(x.x, w, o.x); o.y = fmaf(x.y, w, o.y); o.z = fmaf(x.z, w, o.z); o.w = fmaf(x.w, w, o.w);
        }
    }
    float4 t = o;
    for (int k = 1; k < groups; ++k) {
        const int from = (lane + k * per) & 63;
        t.x += __shfl(o.x, from, 64); t.y += __shfl(o.y, from, 64); t.z += __shfl(o.z, from, 64); t.w += __shfl(o.w, from, 64);
    }
    if (grp != 0) return;
    const float inv = l > 0.0f ? 1.0f / l : (l == 0.0f ? 0.0f : l);           // NaN stays
    const long long bg = flat / a.R;
    const int b = (int)(bg / a.G), g = (int)(bg - (long long)b * a.G), row = (int)(flat - bg * a.R);
    At<T>::store4((T*)a.out + at_row(a, a.so, b, g, row) + col, t.x * inv, t.y * inv, t.z * inv, t.w * inv);
    if (lane == 0 && a.lse != nullptr) a.lse[flat] = l == 0.0f ? INFINITY : m + log2f(l);
}

// ------------------------------------------------------------------------------------------------ backward
// D_i = do_i . o_i, one 16-lane group per row, where dq, whose kernel leaves it, is not asked for and no row can need its correction
template <typename T>
__global__ __launch_bounds__(256) void k_attn_delta(const AtArgs a) {
    const long long rows = (long long)a.B * a.G * a.R, flat = (long long)blockIdx.x * 16 + (threadIdx.x >> 4);
    if (flat >= rows) return;
    const long long bg = flat / a.R;
    const int b = (int)(bg / a.G), g = (int)(bg - (long long)b * a.G), row = (int)(flat - bg * a.R);
    const T* op = (const T*)a.o + at_row(a, a.so, b, g, row);
    const T* gp = (const T*)a.dout + at_row(a, a.sdo, b, g, row);
    float s = 0.0f;
    typedef typename At<T>::Frag F;
    for (int c = threadIdx.x & 15; c * At<T>::CH < a.d; c += 16)
        s = At<T>::dot(*reinterpret_cast<const F*>(op + c * At<T>::CH), *reinterpret_cast<const F*>(gp + c * At<T>::CH), s);
#pragma unroll
    for (int o = 8; o > 0; o >>= 1) s += __shfl_xor(s, o, 64);
    if ((threadIdx.x & 15) == 0) a.delta[flat] = s;
}

// dq: the forward's walk over the keys with p recomputed; dq^T += K^T ds^T.  Leaves D_i for the dk / dv kernels.
// D_i = do_i . o_i carries o's rounding (half a bfloat16 step of |do||o|).  With few keys that is not small beside dp_j - D_i: for bfloat16 rows of
// up to 32 keys sum_j p_ij (dp_ij - D_i), zero but for that rounding, is added to D_i before the walk (two keys: gradients off by
// 0.0024 of their size, not 0.0045; ten: 0.0027, 0.0032).
// dS is rounded to the tensors' type for its products (at most 2^-8 of each term, which the sum over keys or rows averages: about the size of the
// result's own rounding).  Sequences of up to 32 keys, where few terms are averaged, and heads of up to 32 values, where D_i's rounding is largest beside dS,
// take what bfloat16 rounds off as a second product (every backward kernel: a sequence's gradients do not depend on its batch's padding).
// Three products a pair like the forward's two: two causal sequences of 4096, 8 heads over 2, D = 128: 160 us, 0.64 PFLOP/s.
template <typename T, int D, int NW, bool SPLIT>
__global__ __launch_bounds__(64 * NW, (at_min_waves<T, D>())) void k_attn_dq(const AtArgs a) {
    typedef At<T> M;
    typedef Tile<T, D> L_;
    constexpr int BK = at_bk<T, D, NW>(), KS = M::KS, CH = M::CH, U = D / KS, CPR = D / CH, NT = 64 * NW, LD = BK * CPR / NT, DT = D / 32, PG = 16 / (KS / 2), KT = BK / 32;
    __shared__ __attribute__((aligned(16))) T Ks[BK * L_::PITCH];
    __shared__ __attribute__((aligned(16))) T Vs[BK * L_::PITCH];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int sp = SPLIT ? blockIdx.x % a.splits : 0;
    const int w = SPLIT ? blockIdx.x / a.splits : blockIdx.x;
    int bg, tile;
    at_row_tile(a, w, SPLIT, bg, tile);
    const int b = bg / a.G, g = bg - b * a.G;
    const int L = at_len(a, b);
    const int row0 = tile * 32 * NW + 32 * wv, row = row0 + (lane & 31);
    const bool live = row < a.R;
    const int k_lo = SPLIT ? sp * a.chunk : 0;
    const int wg_end = min(at_limit_max(a, L, tile * 32 * NW, 32 * NW), SPLIT ? k_lo + a.chunk : a.dq == nullptr ? BK : L);      // (no dq: only D_i)
    const int limit = live ? at_limit(a, L, row) : 0;
    const int wave_end = row0 < a.R ? at_limit_max(a, L, row0, 32) : 0;
    int wave_full = limit;
#pragma unroll
    for (int o = 32; o > 0; o >>= 1) wave_full = min(wave_full, __shfl_xor(wave_full, o, 64));
    wave_full = __builtin_amdgcn_readfirstlane(wave_full);
    const T* kb = (const T*)a.k + b * a.sk.b + (long long)g * a.sk.h;
    const T* vb = (const T*)a.v + b * a.sv.b + (long long)g * a.sv.h;
    const long long flat = ((long long)b * a.G + g) * a.R + row;
    typename M::Frag qf[U], gf[U];
    {
        const T* qp = (const T*)a.q + at_row(a, a.sq, b, g, live ? row : 0);
        const T* gp = (const T*)a.dout + at_row(a, a.sdo, b, g, live ? row : 0);
#pragma unroll
        for (int u = 0; u < U; ++u) {
            qf[u] = __builtin_bit_cast(typename M::Frag, at_load<T>(qp, 0, live ? 0 : 1, 1, 2 * u + h, a.d));
            gf[u] = __builtin_bit_cast(typename M::Frag, at_load<T>(gp, 0, live ? 0 : 1, 1, 2 * u + h, a.d));
        }
    }
    const float lse = live ? a.lse[flat] : INFINITY;
    float dl = 0.0f;                                                          // D_i, left for the dk / dv kernel
    {
        const T* yp = (const T*)a.o + at_row(a, a.so, b, g, live ? row : 0);
#pragma unroll
        for (int u = 0; u < U; ++u)
            dl = M::dot(__builtin_bit_cast(typename M::Frag, at_load<T>(yp, 0, live ? 0 : 1, 1, 2 * u + h, a.d)), gf[u], dl);
        dl += __shfl_xor(dl, 32, 64);
    }
    const float c = a.scale * AT_LOG2E;
    f32x16 acc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
    at_u32x4 rk[LD], rv[LD];
    auto fetch = [&](int k0) {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int id = tid + NT * i, rw = id / CPR, ch = id - rw * CPR;
            rk[i] = at_fetch<T>(kb, a.sk.n, k0 + rw, L, ch, a.d);
            rv[i] = at_fetch<T>(vb, a.sv.n, k0 + rw, L, ch, a.d);
        }
    };
    if (k_lo < wg_end) fetch(k_lo);
    for (int k0 = k_lo; k0 < wg_end; k0 += BK) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int id = tid + NT * i, rw = id / CPR, ch = id - rw * CPR;
            const bool ok = k0 + rw < L && ch * CH < a.d;
            *reinterpret_cast<at_u32x4*>(&Ks[L_::at(rw, ch)]) = at_keep(rk[i], ok);
            *reinterpret_cast<at_u32x4*>(&Vs[L_::at(rw, ch)]) = at_keep(rv[i], ok);
        }
        __syncthreads();
        if (k0 + BK < wg_end) fetch(k0 + BK);
        if (k0 >= wave_end) continue;
        const bool edge = k0 + BK > wave_full;
        if (sizeof(T) == 2 && k0 == 0 && wave_full <= 32) {
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = 0.0f;
                dp[i] = -dl;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s = M::mma(L_::rows(Ks, 0, u, lane), qf[u], s);
                dp = M::mma(L_::rows(Vs, 0, u, lane), gf[u], dp);
            }
            float fix = 0.0f;
#pragma unroll
            for (int i = 0; i < 16; ++i) fix += 8 * (i >> 2) + 4 * h + (i & 3) < limit ? at_exp2(fmaf(s[i], c, -lse)) * dp[i] : 0.0f;
            fix += __shfl_xor(fix, 32, 64);
            dl += limit <= 32 ? fix : 0.0f;
        }
#pragma unroll
        for (int t = 0; t < KT; ++t) {
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                s[i] = 0.0f;
                dp[i] = -dl;
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s = M::mma(L_::rows(Ks, 32 * t, u, lane), qf[u], s);
                dp = M::mma(L_::rows(Vs, 32 * t, u, lane), gf[u], dp);
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) s[i] = at_exp2(fmaf(s[i], c, -lse)) * dp[i];
            if (edge) {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[i] = k0 + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3) < limit ? s[i] : 0.0f;
            }
#pragma unroll
            for (int p = 0; p < PG; ++p) {
                const typename M::Frag pf = M::pack(s, p);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[dt] = M::mma(L_::cols(Ks, 32 * t + KS * p, 32 * dt, lane), pf, acc[dt]);
                if constexpr (sizeof(T) == 2) {
                    if (D > 32 && L > 32) continue;
                    const typename M::Frag rf = M::rest(s, p);
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) acc[dt] = M::mma(L_::cols(Ks, 32 * t + KS * p, 32 * dt, lane), rf, acc[dt]);
                }
            }
        }
    }
    if (!live) return;
    if (h == 0 && sp == 0) a.delta[flat] = dl;
    if (a.dq == nullptr) return;
    const float sc = a.scale;
    T* op = (T*)a.dq + at_row(a, a.sdq, b, g, row);
    float* pp = SPLIT ? a.part + (sp * ((long long)a.B * a.G * a.R) + flat) * a.d : nullptr;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = 32 * t + 8 * i + 4 * h;
            if (col >= a.d) continue;
            const float x = acc[t][4 * i] * sc, y = acc[t][4 * i + 1] * sc, z = acc[t][4 * i + 2] * sc, q = acc[t][4 * i + 3] * sc;
            if (SPLIT) *reinterpret_cast<float4*>(pp + col) = make_float4(x, y, z, q);
            else M::store4(op + col, x, y, z, q);
        }
}

// order of the key tiles: the ones most rows see (causal: the first) first, and as in at_row_tile the second half backwards where every workgroup
// has a place at once
__device__ __forceinline__ int at_key_tile(const AtArgs& a, int rank) {
    const int half = (a.tiles + 1) / 2;
    return !a.causal || gridDim.x > 512 || rank < half ? rank : a.tiles - 1 - (rank - half);
}

// dk, dv: a wave owns 32 keys (its K and V fragments stay in registers) and walks the folded rows, BQ at a time through LDS;
// dv^T += dO^T P, dk^T += Q^T dS.  -D_i is the initial value of the dP accumulators.  (Head widths up to 64.)
// 48 x 16384 rows, 256 keys, D = 64, bfloat16: 172 us, 0.60 PFLOP/s (vector units; k_attn_dq 139 more: k_attn_bwd_short needs 206 for both).
template <typename T, int D, int NW, bool SPLIT>
__global__ __launch_bounds__(64 * NW, (at_min_waves<T, D>())) void k_attn_dkv(const AtArgs a) {
    typedef At<T> M;
    typedef Tile<T, D> L_;
    constexpr int BQ = NW == 1 || D == 128 || sizeof(T) == 4 ? 32 : 64, KS = M::KS, CH = M::CH, U = D / KS, CPR = D / CH, NT = 64 * NW;
    constexpr int LD = (BQ * CPR + NT - 1) / NT, DT = D / 32, PG = 16 / (KS / 2);
    __shared__ __attribute__((aligned(16))) T Qs[BQ * L_::PITCH];
    __shared__ __attribute__((aligned(16))) T Gs[BQ * L_::PITCH];
    __shared__ __attribute__((aligned(16))) float Ls[BQ], Ds[BQ];
    __shared__ __attribute__((aligned(16))) int Es[BQ];                       // key limit of each row
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int n = a.B * a.G * (SPLIT ? a.splits : 1), rank = blockIdx.x / n, w = blockIdx.x - rank * n;
    const int sp = SPLIT ? w % a.splits : 0, bg = SPLIT ? w / a.splits : w, tile = at_key_tile(a, rank), b = bg / a.G, g = bg - b * a.G;
    const int L = at_len(a, b);
    const int wg_key0 = tile * 32 * NW, key0 = wg_key0 + 32 * wv, key = key0 + (lane & 31);
    const T* kb = (const T*)a.k + b * a.sk.b + (long long)g * a.sk.h;
    const T* vb = (const T*)a.v + b * a.sv.b + (long long)g * a.sv.h;
    const float c = a.scale * AT_LOG2E;
    const int r_lo = SPLIT ? sp * a.chunk : 0, r_hi = wg_key0 < L ? (SPLIT ? min(a.R, r_lo + a.chunk) : a.R) : r_lo;      // (no key: nothing to walk)
    typename M::Frag kf[U], vf[U];
    if (wg_key0 < L) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            kf[u] = __builtin_bit_cast(typename M::Frag, at_load<T>(kb, a.sk.n, key, L, 2 * u + h, a.d));
            vf[u] = __builtin_bit_cast(typename M::Frag, at_load<T>(vb, a.sv.n, key, L, 2 * u + h, a.d));
        }
    }
    f32x16 ak[DT], av[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) ak[t][i] = av[t][i] = 0.0f;
    // first tile from q0 on with a row that sees a key of this workgroup
    // rows that see no key have zeros in LDS, whatever q, dO and D hold (0 x NaN in the products otherwise)
    const bool blind = a.causal && L < a.Nq;
    auto next = [&](int q0) {
        if (a.causal)
            while (q0 < r_hi && at_limit_max(a, L, q0, BQ) <= wg_key0) q0 += BQ;
        return q0;
    };
    at_u32x4 rq[LD], rg[LD];
    float r_lse = 0.0f, r_d = 0.0f;
    auto fetch = [&](int q0) {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int id = tid + NT * i, rw = id / CPR, ch = id - rw * CPR, rr = min(q0 + rw, r_hi - 1);
            rq[i] = at_fetch<T>((const T*)a.q + at_row(a, a.sq, b, g, rr), 0, 0, 1, ch, a.d);
            rg[i] = at_fetch<T>((const T*)a.dout + at_row(a, a.sdo, b, g, rr), 0, 0, 1, ch, a.d);
        }
        const long long f = ((long long)b * a.G + g) * a.R + min(q0 + (tid & (BQ - 1)), r_hi - 1);
        r_lse = a.lse[f];
        r_d = a.delta[f];
    };
    int q0 = next(r_lo);
    if (q0 < r_hi) fetch(q0);
    while (q0 < r_hi) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int id = tid + NT * i, rw = id / CPR, ch = id - rw * CPR;
            if (BQ * CPR % NT != 0 && id >= BQ * CPR) break;
            const bool ok = q0 + rw < r_hi && ch * CH < a.d && (!blind || at_limit(a, L, q0 + rw) > 0);
            *reinterpret_cast<at_u32x4*>(&Qs[L_::at(rw, ch)]) = at_keep(rq[i], ok);
            *reinterpret_cast<at_u32x4*>(&Gs[L_::at(rw, ch)]) = at_keep(rg[i], ok);
        }
        if (tid < BQ) {
            const bool ok = q0 + tid < r_hi;
            Ls[tid] = ok ? r_lse : INFINITY;
            const int e = ok ? at_limit(a, L, q0 + tid) : 0;
            Ds[tid] = e > 0 ? -r_d : 0.0f;
            Es[tid] = e;
        }
        __syncthreads();
        const int qn = next(q0 + BQ);
        if (qn < r_hi) fetch(qn);
        // a row that does not exist has lse = inf, i.e. p = 0: only the rows' limits can cut this wave's keys
        const bool edge = a.causal || key0 + 32 > L;
#pragma unroll
        for (int t = 0; t < BQ / 32; ++t) {
            f32x16 s, dp;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const aadg_f32x4 x = *reinterpret_cast<const aadg_f32x4*>(&Ds[32 * t + 8 * i + 4 * h]);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[4 * i + e] = 0.0f;
                    dp[4 * i + e] = x[e];
                }
            }
#pragma unroll
            for (int u = 0; u < U; ++u) {
                s = M::mma(L_::rows(Qs, 32 * t, u, lane), kf[u], s);
                dp = M::mma(L_::rows(Gs, 32 * t, u, lane), vf[u], dp);
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const aadg_f32x4 x = *reinterpret_cast<const aadg_f32x4*>(&Ls[32 * t + 8 * i + 4 * h]);
#pragma unroll
                for (int e = 0; e < 4; ++e) s[4 * i + e] = at_exp2(fmaf(s[4 * i + e], c, -x[e]));
            }
            if (edge) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int4 x = *reinterpret_cast<const int4*>(&Es[32 * t + 8 * i + 4 * h]);
                    const int lim[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        s[4 * i + e] = key < lim[e] ? s[4 * i + e] : 0.0f;
                        dp[4 * i + e] = key < lim[e] ? dp[4 * i + e] : 0.0f;
                    }
                }
            }
#pragma unroll
            for (int i = 0; i < 16; ++i) dp[i] *= s[i];
#pragma unroll
            for (int p = 0; p < PG; ++p) {
                const typename M::Frag pf = M::pack(s, p), df = M::pack(dp, p);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) {
                    av[dt] = M::mma(L_::cols(Gs, 32 * t + KS * p, 32 * dt, lane), pf, av[dt]);
                    ak[dt] = M::mma(L_::cols(Qs, 32 * t + KS * p, 32 * dt, lane), df, ak[dt]);
                }
                if constexpr (sizeof(T) == 2) {
                    if (D > 32 && L > 32) continue;
                    const typename M::Frag rf = M::rest(dp, p);
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) ak[dt] = M::mma(L_::cols(Qs, 32 * t + KS * p, 32 * dt, lane), rf, ak[dt]);
                }
            }
        }
        q0 = qn;
    }
    if (key >= a.Nk) return;
    const float sc = a.scale;
    const long long rows = (long long)a.B * a.G * a.Nk, flat = ((long long)b * a.G + g) * a.Nk + key;
    T* kp = (T*)a.dk + b * a.sdk.b + (long long)g * a.sdk.h + (long long)key * a.sdk.n;
    T* vp = (T*)a.dv + b * a.sdv.b + (long long)g * a.sdv.h + (long long)key * a.sdv.n;
    float* pk = SPLIT ? a.part + (2 * sp * rows + flat) * a.d : nullptr;
    float* pv = SPLIT ? pk + rows * a.d : nullptr;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = 32 * t + 8 * i + 4 * h;
            if (col >= a.d) continue;
            const float4 x = make_float4(ak[t][4 * i] * sc, ak[t][4 * i + 1] * sc, ak[t][4 * i + 2] * sc, ak[t][4 * i + 3] * sc);
            const float4 y = make_float4(av[t][4 * i], av[t][4 * i + 1], av[t][4 * i + 2], av[t][4 * i + 3]);
            if (SPLIT) {
                *reinterpret_cast<float4*>(pk + col) = x;
                *reinterpret_cast<float4*>(pv + col) = y;
            } else {
                M::store4(kp + col, x.x, x.y, x.z, x.w);
                M::store4(vp + col, y.x, y.y, y.z, y.w);
            }
        }
}

// dk, dv for head widths over 64: a PAIR of waves owns 32 keys and walks the folded rows, BQ at a time through LDS.  Wave 0 of a pair keeps the keys' K fragments, takes
// S = Q K^T, makes P and hands it over through LDS (lane to lane, float32), then accumulates dv^T += dO^T P; wave 1 keeps V, takes dP = dO V^T - D
// (-D_i is the initial value of its accumulators), makes dS = P dP and accumulates dk^T += Q^T dS.  Both halves are the same code on swapped
// operands and the same number of products; one wave doing both needs 2 D accumulator and D fragment registers and leaves a SIMD one
// wave (two causal sequences of 4096, 8 heads over 2, D = 128: 263 us, 0.52 PFLOP/s, vector 0.39, matrix 0.26 of the time; in pieces half as fine 365 us, 423 in
// one wave).
template <typename T, int D, int NW, bool SPLIT>
__global__ __launch_bounds__(64 * NW, 2) void k_attn_dkv_pair(const AtArgs a) {
    typedef At<T> M;
    typedef Tile<T, D> L_;
    constexpr int RT = sizeof(T) == 4 || NW == 2 ? 1 : 2, BQ = 32 * RT, NP = NW / 2, KS = M::KS, CH = M::CH, U = D / KS, CPR = D / CH, NT = 64 * NW;
    constexpr int LD = (BQ * CPR + NT - 1) / NT, DT = D / 32, PG = 16 / (KS / 2);
    __shared__ __attribute__((aligned(16))) T Xs[2 * BQ * L_::PITCH];         // Q, dO
    __shared__ __attribute__((aligned(16))) float Ps[RT * NP * 1024];
    __shared__ __attribute__((aligned(16))) float Ls[BQ], Ds[BQ];
    __shared__ __attribute__((aligned(16))) int Es[BQ];                       // key limit of each row
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5, pair = wv >> 1, role = wv & 1;
    const int n = a.B * a.G * (SPLIT ? a.splits : 1), rank = blockIdx.x / n, w = blockIdx.x - rank * n;
    const int sp = SPLIT ? w % a.splits : 0, bg = SPLIT ? w / a.splits : w, tile = at_key_tile(a, rank), b = bg / a.G, g = bg - b * a.G;
    const int L = at_len(a, b);
    const int wg_key0 = tile * 32 * NP, key0 = wg_key0 + 32 * pair, key = key0 + (lane & 31);
    const float c = a.scale * AT_LOG2E;
    const int r_lo = SPLIT ? sp * a.chunk : 0, r_hi = wg_key0 < L ? (SPLIT ? min(a.R, r_lo + a.chunk) : a.R) : r_lo;      // (no key: nothing to walk)
    typename M::Frag f[U];
    if (wg_key0 < L) {
        const T* base = role ? (const T*)a.v + b * a.sv.b + (long long)g * a.sv.h : (const T*)a.k + b * a.sk.b + (long long)g * a.sk.h;
        const long long step = role ? a.sv.n : a.sk.n;
#pragma unroll
        for (int u = 0; u < U; ++u) f[u] = __builtin_bit_cast(typename M::Frag, at_load<T>(base, step, key, L, 2 * u + h, a.d));
    }
    f32x16 acc[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) acc[t][i] = 0.0f;
    // first tile from q0 on with a row that sees a key of this workgroup
    // rows that see no key have zeros in LDS, whatever q, dO and D hold (0 x NaN in the products otherwise)
    const bool blind = a.causal && L < a.Nq;
    auto next = [&](int q0) {
        if (a.causal)
            while (q0 < r_hi && at_limit_max(a, L, q0, BQ) <= wg_key0) q0 += BQ;
        return q0;
    };
    at_u32x4 rq[LD], rg[LD];
    float r_lse = 0.0f, r_d = 0.0f;
    auto fetch = [&](int q0) {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int id = tid + NT * i, rw = id / CPR, ch = id - rw * CPR, rr = min(q0 + rw, r_hi - 1);
            rq[i] = at_fetch<T>((const T*)a.q + at_row(a, a.sq, b, g, rr), 0, 0, 1, ch, a.d);
            rg[i] = at_fetch<T>((const T*)a.dout + at_row(a, a.sdo, b, g, rr), 0, 0, 1, ch, a.d);
        }
        const long long e = ((long long)b * a.G + g) * a.R + min(q0 + (tid & (BQ - 1)), r_hi - 1);
        r_lse = a.lse[e];
        r_d = a.delta[e];
    };
    const T *X1 = Xs + role * BQ * L_::PITCH, *X2 = Xs + (1 - role) * BQ * L_::PITCH;
    aadg_f32x4* P = reinterpret_cast<aadg_f32x4*>(Ps) + pair * 256 + lane;
    // a row that does not exist has lse = inf, i.e. p = 0: only the rows' limits can cut this pair's keys
    const bool edge = a.causal || key0 + 32 > L;
    int q0 = next(r_lo);
    if (q0 < r_hi) fetch(q0);
    while (q0 < r_hi) {
        __syncthreads();
#pragma unroll
        for (int i = 0; i < LD; ++i) {
            const int id = tid + NT * i, rw = id / CPR, ch = id - rw * CPR;
            if (BQ * CPR % NT != 0 && id >= BQ * CPR) break;
            const bool ok = q0 + rw < r_hi && ch * CH < a.d && (!blind || at_limit(a, L, q0 + rw) > 0);
            *reinterpret_cast<at_u32x4*>(&Xs[L_::at(rw, ch)]) = at_keep(rq[i], ok);
            *reinterpret_cast<at_u32x4*>(&Xs[BQ * L_::PITCH + L_::at(rw, ch)]) = at_keep(rg[i], ok);
        }
        if (tid < BQ) {
            const bool ok = q0 + tid < r_hi;
            Ls[tid] = ok ? r_lse : INFINITY;
            const int e = ok ? at_limit(a, L, q0 + tid) : 0;
            Ds[tid] = e > 0 ? -r_d : 0.0f;
            Es[tid] = e;
        }
        __syncthreads();
        const int qn = next(q0 + BQ);
        if (qn < r_hi) fetch(qn);
        f32x16 s[RT];
#pragma unroll
        for (int t = 0; t < RT; ++t) {
            if (role) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const aadg_f32x4 x = *reinterpret_cast<const aadg_f32x4*>(&Ds[32 * t + 8 * i + 4 * h]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[t][4 * i + e] = x[e];
                }
            } else {
#pragma unroll
                for (int i = 0; i < 16; ++i) s[t][i] = 0.0f;
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int t = 0; t < RT; ++t) s[t] = M::mma(L_::rows(X1, 32 * t, u, lane), f[u], s[t]);
        if (!role) {
#pragma unroll
            for (int t = 0; t < RT; ++t) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const aadg_f32x4 x = *reinterpret_cast<const aadg_f32x4*>(&Ls[32 * t + 8 * i + 4 * h]);
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[t][4 * i + e] = at_exp2(fmaf(s[t][4 * i + e], c, -x[e]));
                }
                if (edge) {
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const int4 x = *reinterpret_cast<const int4*>(&Es[32 * t + 8 * i + 4 * h]);
                        const int lim[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                        for (int e = 0; e < 4; ++e) s[t][4 * i + e] = key < lim[e] ? s[t][4 * i + e] : 0.0f;
                    }
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) P[1024 / 4 * NP * t + 64 * i] = aadg_f32x4{s[t][4 * i], s[t][4 * i + 1], s[t][4 * i + 2], s[t][4 * i + 3]};
            }
        }
        __syncthreads();
        if (role) {
#pragma unroll
            for (int t = 0; t < RT; ++t)
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const aadg_f32x4 x = P[1024 / 4 * NP * t + 64 * i];
#pragma unroll
                    for (int e = 0; e < 4; ++e) s[t][4 * i + e] *= x[e];
                }
        }
#pragma unroll
        for (int t = 0; t < RT; ++t)
#pragma unroll
            for (int p = 0; p < PG; ++p) {
                const typename M::Frag pf = M::pack(s[t], p);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) acc[dt] = M::mma(L_::cols(X2, 32 * t + KS * p, 32 * dt, lane), pf, acc[dt]);
                if constexpr (sizeof(T) == 2) {
                    if (L > 32) continue;
                    const typename M::Frag rf = M::rest(s[t], p);
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) acc[dt] = M::mma(L_::cols(X2, 32 * t + KS * p, 32 * dt, lane), rf, acc[dt]);
                }
            }
        q0 = qn;
    }
    if (key >= a.Nk) return;
    const float sc = role ? a.scale : 1.0f;
    const long long rows = (long long)a.B * a.G * a.Nk, flat = ((long long)b * a.G + g) * a.Nk + key;
    T* out = role ? (T*)a.dk + b * a.sdk.b + (long long)g * a.sdk.h + (long long)key * a.sdk.n
                  : (T*)a.dv + b * a.sdv.b + (long long)g * a.sdv.h + (long long)key * a.sdv.n;
    float* part = SPLIT ? a.part + (2 * sp * rows + flat + (role ? 0 : rows)) * a.d : nullptr;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = 32 * t + 8 * i + 4 * h;
            if (col >= a.d) continue;
            const float4 x = make_float4(acc[t][4 * i] * sc, acc[t][4 * i + 1] * sc, acc[t][4 * i + 2] * sc, acc[t][4 * i + 3] * sc);
            if (SPLIT) *reinterpret_cast<float4*>(part + col) = x;
            else M::store4(out + col, x.x, x.y, x.z, x.w);
        }
}

// The whole backward in one walk over the rows, where a workgroup can hold every key (bfloat16, head widths 33 ... 64, at most 32 NW keys): five
// products instead of seven, and q, o, dO are read once.  Wave w owns keys 32 w ... + 31 as in k_attn_dkv; dS^T of all waves meets in LDS
// ([key][row], 72 bytes a key: 8-byte writes of neighbouring keys and the transpose reads spread over the banks), and dq^T = K^T dS^T is taken in
// 16 x 16 tiles (v_mfma_f32_16x16x32_bf16: every wave has its tiles over all keys, no sum across waves; its K^T fragments stay in registers).
// D_i comes from the rows on their way to LDS (eight neighbouring lanes hold a row).
// 48 x 16384 rows, 256 keys, D = 64: 207 us, 0.62 PFLOP/s (139 + 172 us in two walks); vector issue 0.41, LDS 0.38, matrix 0.32 of the time: two
// barriers a tile of 32 rows, which software pipelining over one barrier did not shorten.
template <int NW, bool SPLIT>
__global__ __launch_bounds__(64 * NW, 2) void k_attn_bwd_short(const AtArgs a) {
    typedef uint16_t T;
    typedef At<T> M;
    constexpr int D = 64, BQ = 32, KS = 16, U = D / KS, DT = D / 32, NS = NW, RH = NW == 8 ? 1 : 2, SP = 36;      // NS: 32-key steps; RH: row halves per wave; SP: dS^T pitch
    typedef Tile<T, D> L_;
    __shared__ __attribute__((aligned(16))) T Qs[BQ * L_::PITCH];
    __shared__ __attribute__((aligned(16))) T Gs[BQ * L_::PITCH];
    __shared__ __attribute__((aligned(16))) T Ss[32 * NW * SP];
    __shared__ __attribute__((aligned(16))) float Ls[BQ], Ds[BQ];
    __shared__ __attribute__((aligned(16))) int Es[BQ];
    const int tid = threadIdx.x, lane = tid & 63, wv = __builtin_amdgcn_readfirstlane(tid >> 6), h = lane >> 5;
    const int sp = SPLIT ? blockIdx.x % a.splits : 0, bg = SPLIT ? blockIdx.x / a.splits : blockIdx.x, b = bg / a.G, g = bg - b * a.G;
    const int L = at_len(a, b), Lc = max(L, 1);                               // (a sequence without keys reads key 0, masked)
    const int key0 = 32 * wv, key = key0 + (lane & 31);
    const T* kb = (const T*)a.k + b * a.sk.b + (long long)g * a.sk.h;
    const T* vb = (const T*)a.v + b * a.sv.b + (long long)g * a.sv.h;
    const float c = a.scale * AT_LOG2E;
    const int r_lo = SPLIT ? sp * a.chunk : 0, r_hi = SPLIT ? min(a.R, r_lo + a.chunk) : a.R;
    typename M::Frag kf[U], vf[U], kt[NS];
#pragma unroll
    for (int u = 0; u < U; ++u) {
        const bool ok = key < L && (2 * u + h) * 8 < a.d;
        kf[u] = __builtin_bit_cast(typename M::Frag, at_keep(at_fetch<T>(kb, a.sk.n, key, Lc, 2 * u + h, a.d), ok));
        vf[u] = __builtin_bit_cast(typename M::Frag, at_keep(at_fetch<T>(vb, a.sv.n, key, Lc, 2 * u + h, a.d), ok));
    }
    // K^T fragments of this wave's 16 columns: lane & 15 = column, eight keys per 16 lanes in the order the dS^T reads give: 8 (lane >> 4) + 0 ... 7
    const int dq0 = 16 * (wv & 3), rh0 = NW == 8 ? wv >> 2 : 0, kcol = dq0 + (lane & 15);
#pragma unroll
    for (int n = 0; n < NS; ++n) {
        uint32_t x[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const int kk = 32 * n + 8 * (lane >> 4) + e;
            const T val = kb[(long long)min(kk, Lc - 1) * a.sk.n + min(kcol, a.d - 1)];
            x[e] = kk < L && kcol < a.d ? val : 0;
        }
        const at_u32x4 y = {x[0] | x[1] << 16, x[2] | x[3] << 16, x[4] | x[5] << 16, x[6] | x[7] << 16};
        kt[n] = __builtin_bit_cast(typename M::Frag, y);
    }
    // up to 32 keys are all wave 0's: what bfloat16 rounds off dS takes the place of the empty keys 32 ... 63, beside the same K^T (wave 1 writes
    // its zeros over wave 2's)
    const bool few = L <= 32;
    const int skey = few && wv == 1 ? key + 32 : key;
    if (few) kt[1] = kt[0];
    f32x16 ak[DT], av[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 16; ++i) ak[t][i] = av[t][i] = 0.0f;
    // 256 chunks of each of q, dO, o per tile: eight waves split them (q | dO and o), four take all
    const bool has_q = NW == 4 || tid < 256, has_g = NW == 4 || tid >= 256;
    const int rw = (tid & 255) >> 3, ch = tid & 7;
    at_u32x4 rq = {}, rg = {}, ro = {};
    float r_lse = 0.0f;
    auto fetch = [&](int q0) {
        const int rr = min(q0 + rw, r_hi - 1);
        if (has_q) rq = at_fetch<T>((const T*)a.q + at_row(a, a.sq, b, g, rr), 0, 0, 1, ch, a.d);
        if (has_g) {
            rg = at_fetch<T>((const T*)a.dout + at_row(a, a.sdo, b, g, rr), 0, 0, 1, ch, a.d);
            ro = at_fetch<T>((const T*)a.o + at_row(a, a.so, b, g, rr), 0, 0, 1, ch, a.d);
        }
        r_lse = a.lse[((long long)b * a.G + g) * a.R + min(q0 + (tid & 31), r_hi - 1)];
    };
    const bool edge = a.causal || key0 + 32 > L;
    const bool blind = L == 0 || (a.causal && L < a.Nq);                      // rows that see no key: zeros in LDS as in k_attn_dkv
    fetch(r_lo);
    for (int q0 = r_lo; q0 < r_hi; q0 += BQ) {
        // (the last reads of Qs, Gs lie before the barrier in the middle of the last tile, those of Ss before the next barrier)
        const bool ok = q0 + rw < r_hi && ch * 8 < a.d && (!blind || at_limit(a, L, q0 + rw) > 0);
        if (has_q) *reinterpret_cast<at_u32x4*>(&Qs[L_::at(rw, ch)]) = at_keep(rq, ok);
        if (has_g) {
            const at_u32x4 x = at_keep(rg, ok);
            *reinterpret_cast<at_u32x4*>(&Gs[L_::at(rw, ch)]) = x;
            float dl = M::dot(__builtin_bit_cast(typename M::Frag, x), __builtin_bit_cast(typename M::Frag, at_keep(ro, ok)), 0.0f);
            dl += __shfl_xor(dl, 1, 64);
            dl += __shfl_xor(dl, 2, 64);
            dl += __shfl_xor(dl, 4, 64);
            if (ch == 0) Ds[rw] = -dl;
        }
        if (tid < BQ) {
            const bool live = q0 + tid < r_hi;
            Ls[tid] = live ? r_lse : INFINITY;
            Es[tid] = live ? at_limit(a, L, q0 + tid) : 0;
        }
        __syncthreads();
        if (q0 + BQ < r_hi) fetch(q0 + BQ);
        f32x16 s, dp;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const aadg_f32x4 x = *reinterpret_cast<const aadg_f32x4*>(&Ds[8 * i + 4 * h]);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                s[4 * i + e] = 0.0f;
                dp[4 * i + e] = x[e];
            }
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            s = M::mma(L_::rows(Qs, 0, u, lane), kf[u], s);
            dp = M::mma(L_::rows(Gs, 0, u, lane), vf[u], dp);
        }
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const aadg_f32x4 x = *reinterpret_cast<const aadg_f32x4*>(&Ls[8 * i + 4 * h]);
#pragma unroll
            for (int e = 0; e < 4; ++e) s[4 * i + e] = at_exp2(fmaf(s[4 * i + e], c, -x[e]));
        }
        if (edge) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const int4 x = *reinterpret_cast<const int4*>(&Es[8 * i + 4 * h]);
                const int lim[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    s[4 * i + e] = key < lim[e] ? s[4 * i + e] : 0.0f;
                    dp[4 * i + e] = key < lim[e] ? dp[4 * i + e] : 0.0f;
                }
            }
        }
#pragma unroll
        for (int i = 0; i < 16; ++i) dp[i] *= s[i];
        if (wv == 0 && __any(Es[lane & 31] <= 32)) {                          // rows whose keys are all this wave's: D_i corrected as in k_attn_dq
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                float fix = dp[i];
#pragma unroll
                for (int o = 16; o > 0; o >>= 1) fix += __shfl_xor(fix, o, 64);
                dp[i] -= Es[8 * (i >> 2) + 4 * h + (i & 3)] <= 32 ? s[i] * fix : 0.0f;
            }
        }
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const typename M::Frag pf = M::pack(s, p), df = M::pack(dp, p);
            const at_u32x4 dw = __builtin_bit_cast(at_u32x4, df);             // rows 16 p + 4 h + 0 ... 3 and + 8
            *reinterpret_cast<uint2*>(&Ss[skey * SP + 16 * p + 4 * h]) = make_uint2(dw[0], dw[1]);
            *reinterpret_cast<uint2*>(&Ss[skey * SP + 16 * p + 8 + 4 * h]) = make_uint2(dw[2], dw[3]);
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                av[dt] = M::mma(L_::cols(Gs, KS * p, 32 * dt, lane), pf, av[dt]);
                ak[dt] = M::mma(L_::cols(Qs, KS * p, 32 * dt, lane), df, ak[dt]);
            }
        }
        if (few && wv == 0) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const typename M::Frag rf = M::rest(dp, p);
                const at_u32x4 dw = __builtin_bit_cast(at_u32x4, rf);
                *reinterpret_cast<uint2*>(&Ss[(32 + key) * SP + 16 * p + 4 * h]) = make_uint2(dw[0], dw[1]);
                *reinterpret_cast<uint2*>(&Ss[(32 + key) * SP + 16 * p + 8 + 4 * h]) = make_uint2(dw[2], dw[3]);
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) ak[dt] = M::mma(L_::cols(Qs, KS * p, 32 * dt, lane), rf, ak[dt]);
            }
        }
        __syncthreads();
#pragma unroll
        for (int r = 0; r < RH; ++r) {
            const int rr0 = 16 * (rh0 + r);
            aadg_f32x4 y = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
            for (int n = 0; n < NS; ++n) {
                // B operand: lane & 15 = row, keys 32 n + 8 (lane >> 4) + 0 ... 7 (lane i of 16 passes key i / 4, rows 4 (i % 4), and gets 4 keys of row i)
                const T* q = &Ss[(32 * n + 8 * (lane >> 4) + ((lane & 15) >> 2)) * SP + rr0 + 4 * (lane & 3)];
                typedef at_v4i16 __attribute__((address_space(3)))* lds_p;
                const at_v4i16 v0 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(q)), v1 = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_p)(q + 4 * SP));
                typedef short v8i16 __attribute__((ext_vector_type(8)));
                const v8i16 v = {v0[0], v0[1], v0[2], v0[3], v1[0], v1[1], v1[2], v1[3]};
                y = __builtin_amdgcn_mfma_f32_16x16x32_bf16(kt[n], __builtin_bit_cast(at_bf16x8, v), y, 0, 0, 0);
            }
            const int row = q0 + rr0 + (lane & 15), col = dq0 + 4 * (lane >> 4);      // C: lane & 15 = row, register e = column 4 (lane >> 4) + e
            if (row < r_hi && col < a.d)
                M::store4((T*)a.dq + at_row(a, a.sdq, b, g, row) + col, y[0] * a.scale, y[1] * a.scale, y[2] * a.scale, y[3] * a.scale);
        }
    }
    if (key >= a.Nk) return;
    const float sc = a.scale;
    const long long rows = (long long)a.B * a.G * a.Nk, flat = ((long long)b * a.G + g) * a.Nk + key;
    T* kp = (T*)a.dk + b * a.sdk.b + (long long)g * a.sdk.h + (long long)key * a.sdk.n;
    T* vp = (T*)a.dv + b * a.sdv.b + (long long)g * a.sdv.h + (long long)key * a.sdv.n;
    float* pk = SPLIT ? a.part + (2 * sp * rows + flat) * a.d : nullptr;
    float* pv = SPLIT ? pk + rows * a.d : nullptr;
#pragma unroll
    for (int t = 0; t < DT; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int col = 32 * t + 8 * i + 4 * h;
            if (col >= a.d) continue;
            const float4 x = make_float4(ak[t][4 * i] * sc, ak[t][4 * i + 1] * sc, ak[t][4 * i + 2] * sc, ak[t][4 * i + 3] * sc);
            const float4 y = make_float4(av[t][4 * i], av[t][4 * i + 1], av[t][4 * i + 2], av[t][4 * i + 3]);
            if (SPLIT) {
                *reinterpret_cast<float4*>(pk + col) = x;
                *reinterpret_cast<float4*>(pv + col) = y;
            } else {
                M::store4(kp + col, x.x, x.y, x.z, x.w);
                M::store4(vp + col, y.x, y.y, y.z, y.w);
            }
        }
}

// sum of the splits' partials in split order, one lane per 4 values: out[b, head, n] = sum_s part[s * step + (b heads + head) n_rows + n];
// a second row of workgroups takes a second tensor, whose partials lie behind the first's
template <typename T>
__global__ __launch_bounds__(256) void k_attn_sum(const float* __restrict__ part, T* __restrict__ out0, AtStride s0, T* __restrict__ out1, AtStride s1, int B,
                                                  int heads, int n_rows, int d, int splits, long long step) {
    const int per = d / 4;
    const long long rows = (long long)B * heads * n_rows, id = (long long)blockIdx.x * 256 + threadIdx.x, flat = id / per;
    if (flat >= rows) return;
    const int col = (int)(id - flat * per) * 4;
    const float* p = part + (blockIdx.y ? rows * d : 0) + flat * d + col;
    float4 o = make_float4(0, 0, 0, 0);
#pragma unroll 4
    for (int i = 0; i < splits; ++i) {
        const float4 x = *reinterpret_cast<const float4*>(p + i * step);
        o.x += x.x; o.y += x.y; o.z += x.z; o.w += x.w;
    }
    const long long bh = flat / n_rows;
    const long long b = bh / heads, hh = bh - b * heads, n = flat - bh * n_rows;
    const AtStride s = blockIdx.y ? s1 : s0;
    At<T>::store4((blockIdx.y ? out1 : out0) + b * s.b + hh * s.h + n * s.n + col, o.x, o.y, o.z, o.w);
}

// ------------------------------------------------------------------------------------------------ host
constexpr int AT_TARGET_WAVES = 2048;

AtStride at_stride(const int64_t* s) { return AtStride{s[0], s[1], s[2]}; }

// 0, or the error of a descriptor the kernels do not take.  16-byte rows: every stride and pointer a multiple of 16 bytes.
int at_check(const aadg_attention_desc* s) {
    if (s == nullptr || s->dtype < 0 || s->dtype > 1 || s->B < 1 || s->H < 1 || s->G < 1 || s->Nq < 1 || s->Nk < 1 || s->d < 1) return AADG_E_BADARG;
    if (!(s->scale > 0.0f) || !(s->scale * AT_LOG2E < INFINITY)) return AADG_E_BADARG;
    if (s->H % s->G != 0) return AADG_E_BADARG;
    if (s->d % 8 != 0 || s->d > 128) return AADG_E_UNSUPPORTED;
    const int64_t r = s->H / s->G, R = r * s->Nq;
    if (R > (1 << 29) || s->Nk > (1 << 29) || (int64_t)s->B * s->H > (1 << 20)) return AADG_E_UNSUPPORTED;
    if ((int64_t)s->B * s->H * s->Nq / 4 >= 0x7FFFFFFF) return AADG_E_UNSUPPORTED;
    // grids: at most (rows or keys) / 32 tiles per group, 64 splits
    if ((int64_t)s->B * s->G * (((R > s->Nk ? R : s->Nk) + 31) / 32) * 64 > 0x7FFFFFFF) return AADG_E_UNSUPPORTED;
    if ((int64_t)s->B * s->H * s->Nq * (s->d / 4) / 256 >= 0x7FFFFFFF || (int64_t)s->B * s->G * s->Nk * (s->d / 4) / 256 >= 0x7FFFFFFF) return AADG_E_UNSUPPORTED;
    return 0;
}
bool at_aligned(const aadg_attention_desc* s, const void* p, const int64_t* st) {
    const int unit = s->dtype == 1 ? 8 : 4;
    return p != nullptr && (uintptr_t)p % 16 == 0 && st[0] % unit == 0 && st[1] % unit == 0 && st[2] % unit == 0;
}

struct AtPlan { int nw, tiles, splits, chunk; };

// Waves per workgroup by what there is to own (32 rows a wave).  Splits of the other axis, in units of `tile`.
// bfloat16: until the card has eight waves per CU.  The join is a launch of its own (4 us), so a split keeps what takes as long: 256 / D tiles (1 us a
// tile at D = 64); two where nearly nothing else runs (under a wave per four CUs) and a tile takes a trip to memory, not its
// products.  Causal key tiles differ in length: pieces of 2048 rows or more are cut twice as fine, so that a CU takes a new one
// when a short one ends (dk and dv of two sequences of 4096, 8 heads over 2, D = 128: 264 us instead of 373, the join 5 us more; with shorter
// pieces the join takes what that gains: 8 heads of 4096, D = 64: forward and backward 245 instead of 232).
// float32: one wave keeps a SIMD's matrix unit busy (a tile D / 20 us, a microsecond of latency), so the pieces run in rounds of one
// workgroup of four per CU, or four of one; a split costs the join and its partials (written and read at 4.7 TB/s).  The cheapest by that count.
AtPlan at_plan(const aadg_attention_desc* s, int own, int other, int tile, int small, bool keys) {
    AtPlan p;
    p.nw = own <= 32 * small ? small : 4;
    p.tiles = (own + 32 * p.nw - 1) / (32 * p.nw);
    const int64_t bg = (int64_t)s->B * s->G, waves = bg * p.tiles * p.nw;
    const int D = s->d <= 32 ? 32 : s->d <= 64 ? 64 : 128, n = (other + tile - 1) / tile;
    int64_t sp = 1;
    if (s->dtype == 1) {
        const int least = waves < 64 && D < 128 ? 2 : 256 / D;
        sp = std::min<int64_t>((AT_TARGET_WAVES + waves - 1) / waves, n / least);
        if (keys && s->causal && sp < (2 * AT_TARGET_WAVES + waves - 1) / waves && sp < n / 64)
            sp = std::min<int64_t>(n / 64, (2 * AT_TARGET_WAVES + waves - 1) / waves);
        sp = std::max<int64_t>(1, std::min<int64_t>(sp, 64));
    } else {
        const double part = (keys ? 16.0 : 8.0) * bg * (own / small) * s->d / 4.7e6;      // (own / small: the rows or keys that are written)
        double best = 0.0;
        for (int64_t x = 1; x <= 64 && x <= n; ++x) {
            const double cost = (double)((waves * x + 1023) / 1024 * ((n + x - 1) / x)) * (D / 20.0 + 1.0) + (x > 1 ? 4.0 + part * x : 0.0);
            if (x > 1 && cost >= best) continue;
            best = cost;
            sp = x;
        }
    }
    const int per = (int)((n + sp - 1) / sp);
    p.chunk = per * tile;
    p.splits = (n + per - 1) / per;
    return p;
}
AtPlan at_plan_rows(const aadg_attention_desc* s) { return at_plan(s, s->H / s->G * s->Nq, s->Nk, 64, 1, false); }
// (head widths over 64: a pair of waves has the 32 keys of a wave, so twice the keys are counted)
AtPlan at_plan_keys(const aadg_attention_desc* s) {
    const int f = s->d > 64 ? 2 : 1;
    return at_plan(s, f * s->Nk, s->H / s->G * s->Nq, 32, f, true);
}

// The one-walk backward: keys a workgroup can hold.  Splits of the rows by what they cost: a tile of 32 rows takes 2 us, the workgroups (one of eight
// waves or two of four to a CU) run in rounds, and every split writes and reads its dk and dv in float32 (4 us for the join, 4.7 TB/s).
bool at_is_short(const aadg_attention_desc* s) { return s->dtype == 1 && s->d > 32 && s->d <= 64 && s->Nk > 32 && s->Nk <= 256; }
AtPlan at_plan_short(const aadg_attention_desc* s) {
    AtPlan p;
    p.nw = s->Nk <= 128 ? 4 : 8;
    p.tiles = 1;
    const int64_t R = (int64_t)(s->H / s->G) * s->Nq, bg = (int64_t)s->B * s->G, n = (R + 31) / 32, slots = p.nw == 4 ? 512 : 256;
    const double join = 16.0 * bg * s->Nk * s->d / 4.7e6;
    double best = 0.0;
    for (int64_t sp = 1; sp <= 64 && sp <= n; ++sp) {
        const int64_t len = (n + sp - 1) / sp;
        const double cost = 2.0 * ((bg * sp + slots - 1) / slots) * len + (sp > 1 ? 4.0 + join * sp : 0.0);
        if (sp > 1 && cost >= best) continue;
        best = cost;
        p.chunk = (int)(len * 32);
        p.splits = (int)((n + len - 1) / len);
    }
    return p;
}

size_t at_fwd_bytes(const aadg_attention_desc* s) {
    const AtPlan p = at_plan_rows(s);
    return p.splits > 1 ? (size_t)p.splits * s->B * s->H * s->Nq * (s->d + 2) * 4 : 0;
}

void at_fill(AtArgs& a, const aadg_attention_desc* s, const int* key_lengths) {
    a.key_lengths = key_lengths;
    a.B = s->B; a.H = s->H; a.G = s->G; a.Nq = s->Nq; a.Nk = s->Nk; a.d = s->d; a.causal = s->causal != 0;
    a.r = s->H / s->G; a.R = a.r * s->Nq; a.scale = s->scale;
    // 2^shift < Nq <= 2^(shift + 1): mul < 2^32, and mul * Nq - 2^(32 + shift) < Nq <= 2^(shift + 1) keeps the quotient exact below 2^31
    a.shift = 0;
    while ((2ll << a.shift) < s->Nq) ++a.shift;
    a.mul = s->Nq == 1 ? 0 : (unsigned)(((1ull << (32 + a.shift)) + s->Nq - 1) / (unsigned)s->Nq);
    a.sq = at_stride(s->q_stride); a.sk = at_stride(s->k_stride); a.sv = at_stride(s->v_stride); a.so = at_stride(s->o_stride);
    a.sdo = at_stride(s->do_stride); a.sdq = at_stride(s->dq_stride); a.sdk = at_stride(s->dk_stride); a.sdv = at_stride(s->dv_stride);
}
void at_use(AtArgs& a, const AtPlan& p) { a.tiles = p.tiles; a.splits = p.splits; a.chunk = p.chunk; }

#define AT_LAUNCH(KERNEL, T, D, NW)                                                                                        \
    do {                                                                                                                   \
        const dim3 grid((unsigned)((long long)a.B * a.G * p.tiles * p.splits));                                            \
        if (p.splits > 1) hipLaunchKernelGGL((KERNEL<T, D, NW, true>), grid, dim3(64 * NW), 0, st, a);                     \
        else hipLaunchKernelGGL((KERNEL<T, D, NW, false>), grid, dim3(64 * NW), 0, st, a);                                 \
    } while (0)
#define AT_BY_NW(KERNEL, T, D, SMALL)                                                                                      \
    do {                                                                                                                   \
        if (p.nw == 4) AT_LAUNCH(KERNEL, T, D, 4);                                                                         \
        else AT_LAUNCH(KERNEL, T, D, SMALL);                                                                               \
    } while (0)
#define AT_BY_D(KERNEL, T, WIDE, SMALL)                                                                                    \
    do {                                                                                                                   \
        if (a.d <= 32) AT_BY_NW(KERNEL, T, 32, 1);                                                                         \
        else if (a.d <= 64) AT_BY_NW(KERNEL, T, 64, 1);                                                                    \
        else AT_BY_NW(WIDE, T, 128, SMALL);                                                                                \
    } while (0)

template <typename T> int at_forward(AtArgs& a, const AtPlan& p, hipStream_t st) {
    at_use(a, p);
    AT_BY_D(k_attn_fwd, T, k_attn_fwd, 1);
    AADG_LAUNCH_CHECK();
    if (p.splits > 1) {
        const long long n = (long long)a.B * a.H * a.Nq;
        hipLaunchKernelGGL(k_attn_join<T>, dim3((unsigned)((n + 3) / 4)), dim3(256), 0, st, a);
        AADG_LAUNCH_CHECK();
    }
    return 0;
}

template <typename T> int at_sum_kv(const AtArgs& a, int splits, hipStream_t st) {
    const long long nk = (long long)a.B * a.G * a.Nk, n = nk * (a.d / 4);
    hipLaunchKernelGGL(k_attn_sum<T>, dim3((unsigned)((n + 255) / 256), 2), dim3(256), 0, st, a.part, (T*)a.dk, a.sdk, (T*)a.dv, a.sdv, a.B, a.G, a.Nk,
                       a.d, splits, 2 * nk * a.d);
    AADG_LAUNCH_CHECK();
    return 0;
}

template <typename T> int at_backward(AtArgs& a, const aadg_attention_desc* s, hipStream_t st) {
    const long long rows = (long long)a.B * a.H * a.Nq;
    if (a.dq != nullptr && a.dk != nullptr && at_is_short(s)) {
        const AtPlan p = at_plan_short(s);
        at_use(a, p);
        const dim3 grid((unsigned)((long long)a.B * a.G * p.splits));
        if (p.nw == 8) {
            if (p.splits > 1) hipLaunchKernelGGL((k_attn_bwd_short<8, true>), grid, dim3(512), 0, st, a);
            else hipLaunchKernelGGL((k_attn_bwd_short<8, false>), grid, dim3(512), 0, st, a);
        } else {
            if (p.splits > 1) hipLaunchKernelGGL((k_attn_bwd_short<4, true>), grid, dim3(256), 0, st, a);
            else hipLaunchKernelGGL((k_attn_bwd_short<4, false>), grid, dim3(256), 0, st, a);
        }
        AADG_LAUNCH_CHECK();
        return p.splits > 1 ? at_sum_kv<T>(a, p.splits, st) : 0;
    }
    // (k_attn_delta has 16 threads a row and a launch less than 2^32 of them)
    if (a.dq != nullptr || rows >= 1ll << 28 || (sizeof(T) == 2 && (a.causal || a.key_lengths != nullptr || a.Nk <= 32))) {
        AtPlan p = at_plan_rows(s);
        if (a.dq == nullptr) p.splits = 1;                                    // only for D_i
        at_use(a, p);
        AT_BY_D(k_attn_dq, T, k_attn_dq, 1);
        AADG_LAUNCH_CHECK();
        if (p.splits > 1) {
            const long long n = rows * (a.d / 4);
            hipLaunchKernelGGL(k_attn_sum<T>, dim3((unsigned)((n + 255) / 256)), dim3(256), 0, st, a.part, (T*)a.dq, a.sdq, (T*)nullptr, a.sdq, a.B,
                               a.H, a.Nq, a.d, p.splits, rows * a.d);
            AADG_LAUNCH_CHECK();
        }
    } else {
        hipLaunchKernelGGL(k_attn_delta<T>, dim3((unsigned)((rows + 15) / 16)), dim3(256), 0, st, a);
        AADG_LAUNCH_CHECK();
    }
    if (a.dk != nullptr) {
        const AtPlan p = at_plan_keys(s);
        at_use(a, p);
        AT_BY_D(k_attn_dkv, T, k_attn_dkv_pair, 2);
        AADG_LAUNCH_CHECK();
        if (p.splits > 1) return at_sum_kv<T>(a, p.splits, st);
    }
    return 0;
}

size_t at_delta_bytes(const aadg_attention_desc* s) { return aadg_align_up((size_t)s->B * s->H * s->Nq * 4, 256); }

}  // namespace

extern "C" int aadg_attention_supported(const aadg_attention_desc* desc_host) { return at_check(desc_host) == 0 ? 1 : 0; }

extern "C" size_t aadg_attention_forward_workspace_bytes(const aadg_attention_desc* desc_host) {
    return at_check(desc_host) == 0 ? at_fwd_bytes(desc_host) : 0;
}

extern "C" size_t aadg_attention_backward_workspace_bytes(const aadg_attention_desc* desc_host) {
    if (at_check(desc_host) != 0) return 0;
    const AtPlan pk = at_plan_keys(desc_host), pq = at_plan_rows(desc_host), ps = at_plan_short(desc_host);
    const size_t row = (size_t)desc_host->d * 4;
    const int sk = at_is_short(desc_host) && ps.splits > pk.splits ? ps.splits : pk.splits;
    const size_t nk = sk > 1 ? (size_t)sk * 2 * desc_host->B * desc_host->G * desc_host->Nk * row : 0;
    const size_t nq = pq.splits > 1 ? (size_t)pq.splits * desc_host->B * desc_host->H * desc_host->Nq * row : 0;
    return at_delta_bytes(desc_host) + (nk > nq ? nk : nq);          // dq is joined before dk / dv reuse the partials
}

extern "C" int aadg_attention_forward(const aadg_attention_desc* desc_host, const void* q, const void* k, const void* v, const int* key_lengths,
                                      void* o, float* lse, void* ws, size_t ws_bytes, void* stream) {
    const int rc = at_check(desc_host);
    if (rc != 0) return rc;
    if (!at_aligned(desc_host, q, desc_host->q_stride) || !at_aligned(desc_host, k, desc_host->k_stride) ||
        !at_aligned(desc_host, v, desc_host->v_stride) || !at_aligned(desc_host, o, desc_host->o_stride)) return AADG_E_BADARG;
    const size_t need = at_fwd_bytes(desc_host);
    if (need > 0 && (ws == nullptr || (uintptr_t)ws % 16 != 0 || ws_bytes < need)) return AADG_E_WORKSPACE;
    AtArgs a = {};
    at_fill(a, desc_host, key_lengths);
    a.q = q; a.k = k; a.v = v; a.out = o; a.lse = lse;
    const AtPlan p = at_plan_rows(desc_host);
    a.part = (float*)ws;
    a.ml = a.part + (size_t)p.splits * a.B * a.H * a.Nq * a.d;
    return desc_host->dtype == 1 ? at_forward<uint16_t>(a, p, (hipStream_t)stream) : at_forward<float>(a, p, (hipStream_t)stream);
}

extern "C" int aadg_attention_backward(const aadg_attention_desc* desc_host, const void* q, const void* k, const void* v, const int* key_lengths,
                                       const void* o, const float* lse, const void* dout, void* dq, void* dk, void* dv, void* ws,
                                       size_t ws_bytes, void* stream) {
    const int rc = at_check(desc_host);
    if (rc != 0) return rc;
    if (!at_aligned(desc_host, q, desc_host->q_stride) || !at_aligned(desc_host, k, desc_host->k_stride) ||
        !at_aligned(desc_host, v, desc_host->v_stride) || !at_aligned(desc_host, o, desc_host->o_stride) ||
        !at_aligned(desc_host, dout, desc_host->do_stride) || lse == nullptr || (dk == nullptr) != (dv == nullptr)) return AADG_E_BADARG;
    if (dq != nullptr && !at_aligned(desc_host, dq, desc_host->dq_stride)) return AADG_E_BADARG;
    if (dk != nullptr && (!at_aligned(desc_host, dk, desc_host->dk_stride) || !at_aligned(desc_host, dv, desc_host->dv_stride))) return AADG_E_BADARG;
    if (dq == nullptr && dk == nullptr) return 0;
    if (ws == nullptr || (uintptr_t)ws % 16 != 0 || ws_bytes < aadg_attention_backward_workspace_bytes(desc_host)) return AADG_E_WORKSPACE;
    AtArgs a = {};
    at_fill(a, desc_host, key_lengths);
    a.q = q; a.k = k; a.v = v; a.o = o; a.lse = const_cast<float*>(lse); a.dout = dout; a.dq = dq; a.dk = dk; a.dv = dv;
    a.delta = (float*)ws;
    a.part = (float*)((char*)ws + at_delta_bytes(desc_host));
    return desc_host->dtype == 1 ? at_backward<uint16_t>(a, desc_host, (hipStream_t)stream) : at_backward<float>(a, desc_host, (hipStream_t)stream);
}
