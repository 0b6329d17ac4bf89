// The norms around a block in one pass: the norm after the block, its gate and
// the residual scale, and the norm before the next block.  Per row, in FP32,
//   y = block output, or sum_s w[t, s] * rows[inverse[t*k + s]]   (COMBINE)
//   z = post(y) * post_weight
//   s = residual_scale * r + block_scale * act(gate) * z          -> stream
//   n = pre(s) * pre_weight                                       -> normed
// with post, pre one of none, rms (v / sqrt(mean v^2 + eps)) and layer
// ((v - mean) / sqrt(var + eps), population variance).  s feeds the second
// norm unrounded; each output is rounded once.
// Bound by HBM (y or the k rows, r, s, n once each) or, for a few rows, by the
// chain load -> up to four block reductions -> store.  The row stays in
// registers between the reductions, so nothing is read twice.  12,450 rows of
// H = 2048 combined from k = 8, FP32 stream: 114 us (5.8 TB/s); of H = 4096 with a
// full sigmoid gate, layer and rms norm: 103 us (5.0 TB/s, issue slots); 64
// combined rows of 2048: 4.3 us; 3 rows of 5003: 5.0 us.  Many combined rows with an
// FP32 stream spill 48 bytes a thread, from L1, and other forms 8 or 16.
#include "pdx_common.cuh"

namespace pdx {

constexpr int kBnMaxH = 8192;      // eight values per thread, 1024 threads

struct BlockNormArgs {
    const uint16_t* y;            // [T, H], or the expert rows [y_rows, H] (COMBINE)
    const uint16_t* weights;      // [T, k] (COMBINE)
    const int32_t* inverse;       // [T, k] (COMBINE)
    int k, y_rows;
    const void* residual;         // [T, H] BF16 or FP32
    const uint16_t* post_weight;  // [H] or NULL
    const uint16_t* pre_weight;   // [H] or NULL
    const uint16_t* gate;         // NULL = 1
    int64_t gate_row, gate_col;   // element strides of the gate (0 = broadcast)
    int gate_sigmoid;
    int post, pre;
    float residual_scale, block_scale, eps;
    int H;
    void* stream;                 // residual's type, or NULL
    uint16_t* normed;             // or NULL
};

// Sum over the CTA in a fixed order.  Successive calls alternate between two
// halves of red[64], so one barrier a call is enough.
__device__ __forceinline__ float bn_block_sum(float v, float* red, int& turn) {
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    const int warps = static_cast<int>(blockDim.x >> 5);
    if (warps == 1) return v;
    float* r = red + 32 * turn;
    turn ^= 1;
    if (lane_id() == 0) r[threadIdx.x >> 5] = v;
    __syncthreads();
    v = static_cast<int>(lane_id()) < warps ? r[lane_id()] : 0.f;
#pragma unroll
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(0xffffffffu, v, off);
    return v;
}

// A thread's 8 CH values of a row of H: VEC, the aligned eight from 8 (tid + c
// blockDim) for every c < CH; else every blockDim-th value from tid (any H and
// alignment).  Values past H read as 0 and are not written.
template <bool VEC, int CH>
struct BnPlace {
    static constexpr int N = 8 * CH;
    int H;
    __device__ explicit BnPlace(int h) : H(h) {}
    __device__ __forceinline__ int col(int i) const {
        return VEC ? (static_cast<int>(threadIdx.x) + i / 8 * static_cast<int>(blockDim.x)) * 8 + i % 8
                   : static_cast<int>(threadIdx.x) + i * static_cast<int>(blockDim.x);
    }
    __device__ __forceinline__ bool in(int i) const { return col(VEC ? i & ~7 : i) < H; }
    __device__ __forceinline__ void clear(float (&v)[N]) const {   // values past H to 0
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (!in(i)) v[i] = 0.f;
    }
};

// Raw values, loaded early and converted where they are used.
template <bool VEC, int CH, typename T>
struct BnRaw {
    static constexpr int kVecs = static_cast<int>(sizeof(T)) / 2;   // 16-byte pieces of eight values
    uint4 q[VEC ? CH * kVecs : 1];
    T one[VEC ? 1 : 8 * CH];
    __device__ __forceinline__ void load(const BnPlace<VEC, CH>& at, const T* p) {
        if (VEC) {
#pragma unroll
            for (int c = 0; c < CH; ++c)
#pragma unroll
                for (int j = 0; j < kVecs; ++j)
                    q[c * kVecs + j] = at.in(8 * c) ? reinterpret_cast<const uint4*>(p + at.col(8 * c))[j]
                                                    : make_uint4(0, 0, 0, 0);
        } else {
#pragma unroll
            for (int i = 0; i < 8 * CH; ++i) one[i] = at.in(i) ? p[at.col(i)] : static_cast<T>(0);
        }
    }
    __device__ __forceinline__ float get(int i) const {
        if (!VEC) return sizeof(T) == 4 ? static_cast<float>(one[i]) : bits2f(static_cast<uint16_t>(one[i]));
        const int word = sizeof(T) == 4 ? i : i / 2;
        const uint4& v = q[word / 4];
        const uint32_t w = word % 4 == 0 ? v.x : (word % 4 == 1 ? v.y : (word % 4 == 2 ? v.z : v.w));
        if (sizeof(T) == 4) return __uint_as_float(w);
        return __uint_as_float(i & 1 ? w & 0xFFFF0000u : w << 16);
    }
};

template <bool VEC, int CH>
__device__ __forceinline__ void bn_store(const BnPlace<VEC, CH>& at, uint16_t* p, const float* v) {
    if (VEC) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (!at.in(8 * c)) continue;
            uint32_t w[4];
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const __nv_bfloat162 two = __floats2bfloat162_rn(v[8 * c + 2 * i], v[8 * c + 2 * i + 1]);
                w[i] = *reinterpret_cast<const uint32_t*>(&two);
            }
            *reinterpret_cast<uint4*>(p + at.col(8 * c)) = make_uint4(w[0], w[1], w[2], w[3]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8 * CH; ++i)
            if (at.in(i)) p[at.col(i)] = f2bits(v[i]);
    }
}
template <bool VEC, int CH>
__device__ __forceinline__ void bn_store(const BnPlace<VEC, CH>& at, float* p, const float* v) {
    if (VEC) {
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            if (!at.in(8 * c)) continue;
            float4* to = reinterpret_cast<float4*>(p + at.col(8 * c));
            to[0] = make_float4(v[8 * c], v[8 * c + 1], v[8 * c + 2], v[8 * c + 3]);
            to[1] = make_float4(v[8 * c + 4], v[8 * c + 5], v[8 * c + 6], v[8 * c + 7]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < 8 * CH; ++i)
            if (at.in(i)) p[at.col(i)] = v[i];
    }
}

// Normalise the row held in v (values past H are 0 and stay so).
template <bool VEC, int CH>
__device__ __forceinline__ void bn_norm(float (&v)[8 * CH], int how, bool weighted, const BnRaw<VEC, CH, uint16_t>& w,
                                        const BnPlace<VEC, CH>& at, float eps, float* red, int& turn) {
    constexpr int N = 8 * CH;
    if (how == PDX_NORM_NONE) return;
    const float inv_h = 1.0f / static_cast<float>(at.H);
    if (how == PDX_NORM_LAYER) {
        float s = 0.f;
#pragma unroll
        for (int i = 0; i < N; ++i) s += v[i];
        const float mean = bn_block_sum(s, red, turn) * inv_h;
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] -= mean;
        at.clear(v);
    }
    float q = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) q += v[i] * v[i];
    const float inv = rsqrtf(bn_block_sum(q, red, turn) * inv_h + eps);
    if (weighted) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= inv * w.get(i);
    } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= inv;
    }
}

// One CTA per row, 8 CH values a thread, at most MAXT threads.  EARLY (few rows,
// where the latency of a row counts): every load that does not depend on a
// reduction is issued before the first one, so a row costs one trip to memory
// and up to four block reductions.  Otherwise rows hide each other's latency and
// issue slots count (a reduction and the set-up cost a warp as much as the
// arithmetic of 8 values a lane, hence CH = 2), and how many rows fit an SM: the
// weights (and beside expert rows the gate) are loaded where they are used.
template <typename RES, bool COMBINE, bool VEC, int CH, int MAXT, bool EARLY>
__global__ void __launch_bounds__(MAXT, EARLY || MAXT == 1024 ? 1 : 1024 / MAXT) k_block_norm(BlockNormArgs a) {
    constexpr int N = 8 * CH;
    // expert rows loaded together; any-alignment rows take a register per value
    constexpr int kBatch = !VEC ? 2 : (EARLY && MAXT < 1024 ? 8 : 4);
    griddep_wait();
    griddep_launch();
    __shared__ float red[64];
    __shared__ int s_row[32];
    __shared__ float s_w[32];
    const int64_t t = blockIdx.x;
    const int H = a.H;
    const BnPlace<VEC, CH> at(H);
    int turn = 0;
    BnRaw<VEC, CH, RES> res;
    BnRaw<VEC, CH, uint16_t> yr, gate, post_w, pre_w;
    res.load(at, static_cast<const RES*>(a.residual) + t * H);
    if (!COMBINE && a.y) yr.load(at, a.y + t * H);
    const bool gate_rowwise = a.gate && a.gate_col == 1;
    if ((EARLY || !COMBINE) && gate_rowwise) gate.load(at, a.gate + t * a.gate_row);
    if (EARLY) {
        if (a.post_weight) post_w.load(at, a.post_weight);
        if (VEC && a.pre_weight) pre_w.load(at, a.pre_weight);
    }
    float v[N];
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = 0.f;
    if (COMBINE) {
        if (threadIdx.x < static_cast<unsigned>(a.k)) {
            int row = a.inverse[t * a.k + threadIdx.x];
            float w = bits2f(a.weights[t * a.k + threadIdx.x]);
            if (row < 0 || row >= a.y_rows) {
                raise_error(PDX_DEVERR_BAD_EXPERT);
                row = -1;
            }
            s_row[threadIdx.x] = row;
            s_w[threadIdx.x] = w;
        }
        __syncthreads();
        // FP32 sum in slot order
        for (int s0 = 0; s0 < a.k; s0 += kBatch) {
            BnRaw<VEC, CH, uint16_t> r[kBatch];
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (s0 + j < a.k && s_row[s0 + j] >= 0) r[j].load(at, a.y + static_cast<int64_t>(s_row[s0 + j]) * H);
#pragma unroll
            for (int j = 0; j < kBatch; ++j)
                if (s0 + j < a.k && s_row[s0 + j] >= 0) {
                    const float w = s_w[s0 + j];
#pragma unroll
                    for (int i = 0; i < N; ++i) v[i] += r[j].get(i) * w;
                }
        }
    } else if (a.y) {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = yr.get(i);
    }
    if (COMBINE || a.y) {
        if (!EARLY && a.post_weight) post_w.load(at, a.post_weight);
        bn_norm<VEC, CH>(v, a.post, a.post_weight != nullptr, post_w, at, a.eps, red, turn);
    }
    if (a.gate) {
        float g[N];
        if (gate_rowwise) {
            if (!EARLY && COMBINE) gate.load(at, a.gate + t * a.gate_row);
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = gate.get(i);
        } else {
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = at.in(i) ? bits2f(a.gate[t * a.gate_row + at.col(i) * a.gate_col]) : 0.f;
        }
        if (a.gate_sigmoid) {
#pragma unroll
            for (int i = 0; i < N; ++i) g[i] = __fdividef(1.0f, 1.0f + expf(-g[i]));   // 1 ulp reciprocal
        }
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] *= g[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) v[i] = a.residual_scale * res.get(i) + a.block_scale * v[i];
    at.clear(v);
    if (a.stream) bn_store(at, static_cast<RES*>(a.stream) + t * H, v);
    if (!a.normed) return;
    if (!(EARLY && VEC) && a.pre_weight) pre_w.load(at, a.pre_weight);
    bn_norm<VEC, CH>(v, a.pre, a.pre_weight != nullptr, pre_w, at, a.eps, red, turn);
    bn_store(at, a.normed + t * H, v);
}

}  // namespace pdx
