// The rotation of rows by their positions, as kernels take it.
#pragma once

#include "../../include/itak_hip_kv.h"
#include "internal.h"

#include <vector>

struct itak_rotation {
    itak_rotation_config cfg{};
    std::vector<double> frequencies;
    double amplitude = 1.0;
    double *turns_dev = nullptr;  // frequencies / (2 pi)
};

namespace itak {

// turns == null: no rotation.
struct RotationView {
    const double *turns;  // of a full circle, a position, per pair
    uint32_t half;        // pairs
    uint32_t interleaved;
    float amplitude;
};
inline RotationView rotation_view(const itak_rotation *r) {
    if (!r) return RotationView{nullptr, 0, 0, 1.0f};
    return RotationView{r->turns_dev, r->cfg.rotary_dim / 2, r->cfg.interleaved, float(r->amplitude)};
}
constexpr uint32_t kMostPairs = 128;

// (cos, sin) of pair i at a position, times the amplitude. The angle is taken in turns and loses its whole turns in 64 bits: an f32
// angle is off by 8e-3 rad at position 100,000. What is left is at most half a turn, and the f32 functions of it are within
// two units in the last place.
__device__ __forceinline__ float2 turn_of(const RotationView &r, double position, uint32_t i) {
    const double t = position * r.turns[i];
    const float part = float(t - rint(t));
    float s, c;
    sincospif(2.0f * part, &s, &c);
    return make_float2(c * r.amplitude, s * r.amplitude);
}

// One view of rows as kernels take it, strides in elements.
struct RowsView {
    void *data;
    uint64_t row_stride;
    uint64_t head_stride;
};

// An element type of tensors and pages: its ITAK_ELEM_* number, loads and stores of W elements as f32.
template <int ELEM>
struct Elem;
template <>
struct Elem<ITAK_ELEM_F32> {
    typedef float type;
    static __device__ __forceinline__ float to_f32(float x) { return x; }
    static __device__ __forceinline__ float from_f32(float x) { return x; }
};
template <>
struct Elem<ITAK_ELEM_F16> {
    typedef _Float16 type;
    static __device__ __forceinline__ float to_f32(_Float16 x) { return float(x); }
    static __device__ __forceinline__ _Float16 from_f32(float x) { return _Float16(x); }
};
template <>
struct Elem<ITAK_ELEM_BF16> {
    typedef __bf16 type;
    static __device__ __forceinline__ float to_f32(__bf16 x) { return float(x); }
    static __device__ __forceinline__ __bf16 from_f32(float x) { return __bf16(x); }
};

template <typename T, int W>
struct alignas(W * sizeof(T) < 16 ? W * sizeof(T) : 16) Piece {
    T v[W];
};

// The pieces of a head's channels that one thread takes each: W channels of the interleaved pairs or of the tail that is not
// turned, or W of a half and the W they turn with. W = 8 where types, strides and sizes let them be moved 16 bytes at a time,
// else 1 (2 for an interleaved pair).
struct HeadPieces {
    uint32_t turned;  // pieces of the turned part
    uint32_t all;
};
__host__ __device__ inline HeadPieces head_pieces(uint32_t head_dim, uint32_t half, uint32_t interleaved, uint32_t w) {
    const uint32_t per = interleaved && w > 1 ? w / 2 : w;  // pairs a piece
    const uint32_t turned = half / per;
    return HeadPieces{turned, turned + (head_dim - 2 * half) / w};
}
// Whether pieces of 8 fit a head.
inline bool pieces_of_8(uint32_t head_dim, uint32_t half, uint32_t interleaved) {
    return head_dim % 8 == 0 && (interleaved ? half % 4 == 0 : half % 8 == 0);
}

// Piece `piece` of a head: from src to dst, turned by cs[pair] (`sign` = -1: back). In place is fine: a piece is read whole
// before it is written, and no other piece shares its channels.
template <int FROM, int TO, int W>
__device__ __forceinline__ void move_piece(const typename Elem<FROM>::type *src, typename Elem<TO>::type *dst, uint32_t piece,
                                           const HeadPieces &pieces, uint32_t half, uint32_t interleaved, const float2 *cs,
                                           float sign) {
    typedef Elem<FROM> F;
    typedef Elem<TO> T;
    typedef Piece<typename F::type, W> In;
    typedef Piece<typename T::type, W> Out;
    if (piece >= pieces.turned) {  // the tail
        const uint32_t c = 2 * half + (piece - pieces.turned) * W;
        const In x = *reinterpret_cast<const In *>(src + c);
        Out y;
#pragma unroll
        for (int e = 0; e < W; ++e) {
            if constexpr (FROM == TO)
                y.v[e] = x.v[e];
            else
                y.v[e] = T::from_f32(F::to_f32(x.v[e]));
        }
        *reinterpret_cast<Out *>(dst + c) = y;
    } else if (interleaved && W > 1) {
        const uint32_t c = piece * W, pair = piece * (W / 2);
        const In x = *reinterpret_cast<const In *>(src + c);
        Out y;
#pragma unroll
        for (int e = 0; e < W; e += 2) {
            const float2 t = cs[pair + e / 2];
            const float a = F::to_f32(x.v[e]), b = F::to_f32(x.v[(e + 1) % W]), s = sign * t.y;
            y.v[e] = T::from_f32(a * t.x - b * s);
            y.v[(e + 1) % W] = T::from_f32(a * s + b * t.x);
        }
        *reinterpret_cast<Out *>(dst + c) = y;
    } else {
        const uint32_t c0 = interleaved ? 2 * piece : piece * W, c1 = interleaved ? c0 + 1 : c0 + half;
        const In x0 = *reinterpret_cast<const In *>(src + c0), x1 = *reinterpret_cast<const In *>(src + c1);
        Out y0, y1;
#pragma unroll
        for (int e = 0; e < W; ++e) {
            const float2 t = cs[piece * W + e];
            const float a = F::to_f32(x0.v[e]), b = F::to_f32(x1.v[e]), s = sign * t.y;
            y0.v[e] = T::from_f32(a * t.x - b * s);
            y1.v[e] = T::from_f32(a * s + b * t.x);
        }
        *reinterpret_cast<Out *>(dst + c0) = y0;
        *reinterpret_cast<Out *>(dst + c1) = y1;
    }
}

// The checks of a view (rotation.hip): null data, an unknown type, no heads, a first stride that lets rows run into one another.
struct ErrorState;
itak_status check_rows(ErrorState &e, const char *what, const itak_rows *v, uint64_t rows, uint64_t head_dim, bool written);
// With dense strides filled in.
RowsView rows_view(const itak_rows &v, uint64_t head_dim);
// Whether every run of 8 channels of a view starts on 16 bytes.
bool rows_on_16(const itak_rows &v, uint64_t head_dim);

// The device calls run on, for the length of a call.
class DeviceScope {
public:
    explicit DeviceScope(int device) {
        if (hipGetDevice(&before_) == hipSuccess && before_ != device) changed_ = (status_ = hipSetDevice(device)) == hipSuccess;
    }
    ~DeviceScope() {
        if (changed_) (void)hipSetDevice(before_);
    }
    DeviceScope(const DeviceScope &) = delete;
    hipError_t status() const { return status_; }

private:
    int before_ = 0;
    bool changed_ = false;
    hipError_t status_ = hipSuccess;
};

}  // namespace itak
