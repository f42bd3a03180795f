// The rotation of rows by their positions (rotary embedding), on its own: handles, checks and the kernel.
//
// y = a (x0 cos t - x1 sin t, x0 sin t + x1 cos t), t = position * f(pair): six operations for eight to sixteen bytes, so
// the kernel is bound by the bytes it moves, or by its launch where those are few. A workgroup serves one row (or a part of its heads):
// the row's up to 128 cosines and sines are worked out once, one a thread, and kept in LDS for all of its heads; the 64-bit
// reduction and the f32 sine and cosine, some sixty instructions, would cost more than the row's bytes if every head took them.
// 2,048 rows of 36 heads by 128 in f32, 75 MB: 13.5 us, 5.6 TB/s. One row: 2.0 us, of which 1.3 are a launch that does nothing.
#include "rotation.h"

#include "errors.h"
#include "rotation_table.h"

#include <new>

namespace itak {

namespace {

constexpr uint32_t kMostTensors = 4;
constexpr int kThreads = 256;
constexpr uint64_t kMostRows = (1u << 24) - 1;  // a workgroup a row: a launch's threads are counted in 32 bits

struct RotateArgs {
    RotationView r;
    const int64_t *positions;
    uint32_t head_dim;
    uint32_t pieces;      // of all the heads of a row
    uint32_t per_group;   // pieces one workgroup takes
    float sign;
    uint32_t tensors;
    uint32_t heads[kMostTensors];
    RowsView in[kMostTensors];
    RowsView out[kMostTensors];
};

template <int ELEM, int W>
__global__ __launch_bounds__(kThreads) void rotate_kernel(RotateArgs a) {
    typedef typename Elem<ELEM>::type T;
    __shared__ float2 cs[kMostPairs];
    const uint64_t row = blockIdx.x;
    const uint32_t tid = threadIdx.x;
    if (tid < a.r.half) cs[tid] = turn_of(a.r, double(a.positions[row]), tid);
    __syncthreads();
    const HeadPieces hp = head_pieces(a.head_dim, a.r.half, a.r.interleaved, W);
    const uint32_t first = blockIdx.y * a.per_group, end = min(first + a.per_group, a.pieces);
    for (uint32_t p = first + tid; p < end; p += kThreads) {
        uint32_t head = p / hp.all;
        const uint32_t piece = p - head * hp.all;
        uint32_t t = 0;
        while (t + 1 < a.tensors && head >= a.heads[t]) head -= a.heads[t++];
        const T *src = static_cast<const T *>(a.in[t].data) + row * a.in[t].row_stride + head * a.in[t].head_stride;
        T *dst = static_cast<T *>(a.out[t].data) + row * a.out[t].row_stride + head * a.out[t].head_stride;
        move_piece<ELEM, ELEM, W>(src, dst, piece, hp, a.r.half, a.r.interleaved, cs, a.sign);
    }
}

template <int W>
void launch_rotate(uint32_t elem, const RotateArgs &a, dim3 grid, hipStream_t stream) {
    if (elem == ITAK_ELEM_F32)
        launch_kernel(rotate_kernel<ITAK_ELEM_F32, W>, grid, kThreads, 0, stream, a);
    else if (elem == ITAK_ELEM_F16)
        launch_kernel(rotate_kernel<ITAK_ELEM_F16, W>, grid, kThreads, 0, stream, a);
    else
        launch_kernel(rotate_kernel<ITAK_ELEM_BF16, W>, grid, kThreads, 0, stream, a);
}

uint64_t elem_size(uint32_t elem) { return elem == ITAK_ELEM_F32 ? 4 : 2; }

}  // namespace

RowsView rows_view(const itak_rows &v, uint64_t head_dim) {
    if (v.row_stride == 0 && v.head_stride == 0) return RowsView{v.data, v.heads * head_dim, head_dim};
    return RowsView{v.data, v.row_stride, v.head_stride};
}

bool rows_on_16(const itak_rows &v, uint64_t head_dim) {
    const uint64_t mask = 16 / elem_size(v.elem) - 1;
    return head_dim % 8 == 0 && reinterpret_cast<uintptr_t>(v.data) % 16 == 0 && (v.row_stride & mask) == 0 &&
           (v.head_stride & mask) == 0;
}

itak_status check_rows(ErrorState &e, const char *what, const itak_rows *v, uint64_t rows, uint64_t head_dim, bool written) {
    if (!v) return set_error(e, ITAK_INVALID_ARGUMENT, what, 0, 0, 0, 0, "invalid argument: %s is null", what);
    if (v->elem > ITAK_ELEM_BF16)
        return set_error(e, ITAK_INVALID_ARGUMENT, what, v->elem, 0, 0, 0, "invalid argument: the type of %s is none of ITAK_ELEM_*", what);
    if (v->heads == 0) return set_error(e, ITAK_ZERO_DIMENSION, what, 0, 0, 0, 0, "heads of %s must be positive, got 0", what);
    if (rows && !v->data) return set_error(e, ITAK_INVALID_ARGUMENT, what, 0, 0, 0, 0, "invalid argument: %s has no data", what);
    if (reinterpret_cast<uintptr_t>(v->data) % elem_size(v->elem))
        return set_error(e, ITAK_INVALID_ARGUMENT, what, 0, 0, 0, 0, "invalid argument: %s does not start on one of its elements", what);
    const bool dense = v->row_stride == 0 && v->head_stride == 0;
    if (v->heads > (1u << 16) || v->row_stride > (1ull << 40) || v->head_stride > (1ull << 40))
        return size_overflow(e, what);
    // Two rows or heads of a view that is written may not meet: one of the two strides steps over a whole run of the other.
    if (written && !dense) {
        const uint64_t h = v->heads > 1 ? (v->heads - 1) * v->head_stride + head_dim : head_dim;
        const uint64_t r = rows > 1 ? (rows - 1) * v->row_stride + head_dim : head_dim;
        const bool heads_apart = v->heads == 1 || v->head_stride >= head_dim, rows_apart = rows <= 1 || v->row_stride >= head_dim;
        const bool nested = rows <= 1 || v->heads == 1 || v->row_stride >= h || v->head_stride >= r;
        if (!heads_apart || !rows_apart || !nested)
            return set_error(e, ITAK_INVALID_ARGUMENT, what, v->row_stride, v->head_stride, 0, 0,
                             "invalid argument: rows or heads of %s lie over one another", what);
    }
    return ITAK_OK;
}

}  // namespace itak

using namespace itak;

extern "C" {

itak_status itak_rotation_create(const itak_rotation_config *config, itak_rotation **out) {
    ErrorState &e = thread_error();
    if (!out) return invalid_argument(e, "out is null");
    *out = nullptr;
    if (!config) return invalid_argument(e, "config is null");
    if (const char *wrong = rotation_refusal(*config)) return invalid_argument(e, wrong);
    itak_rotation *r = nullptr;
    try {
        r = new itak_rotation;
        r->cfg = *config;
        r->frequencies = rotation_frequencies(*config);
        r->amplitude = rotation_amplitude(*config);
        std::vector<double> turns = r->frequencies;
        for (double &t : turns) t /= 2.0 * M_PI;
        const DeviceScope scope(config->device);
        hipError_t he = scope.status();
        const size_t bytes = turns.size() * sizeof(double);
        if (he == hipSuccess) he = hipMalloc(reinterpret_cast<void **>(&r->turns_dev), bytes);
        if (he == hipSuccess) he = hipMemcpy(r->turns_dev, turns.data(), bytes, hipMemcpyHostToDevice);
        if (he != hipSuccess) {
            (void)hipGetLastError();
            if (r->turns_dev) (void)hipFree(r->turns_dev);
            delete r;
            return hip_error(e, he, "place a rotation's frequencies");
        }
    } catch (const std::bad_alloc &) {
        delete r;
        return invalid_argument(e, "out of host memory");
    }
    *out = r;
    return ITAK_OK;
}

void itak_rotation_destroy(itak_rotation *rotation) {
    if (!rotation) return;
    const DeviceScope scope(rotation->cfg.device);
    (void)hipDeviceSynchronize();
    (void)hipFree(rotation->turns_dev);
    delete rotation;
}

itak_status itak_rotation_frequencies(const itak_rotation *rotation, double *frequencies_out, double *amplitude_out) {
    if (!rotation) return invalid_argument(thread_error(), "rotation is null");
    if (frequencies_out) std::copy(rotation->frequencies.begin(), rotation->frequencies.end(), frequencies_out);
    if (amplitude_out) *amplitude_out = rotation->amplitude;
    return ITAK_OK;
}

itak_status itak_rotate_device(const itak_rotation *rotation, void *hip_stream, uint64_t head_dim, uint64_t rows,
                               const int64_t *positions_dev, const itak_rows *inputs, const itak_rows *outputs,
                               uint32_t tensors, uint32_t inverse) {
    ErrorState &e = thread_error();
    if (!rotation) return invalid_argument(e, "rotation is null");
    if (tensors == 0 || tensors > kMostTensors) return invalid_argument(e, "tensors must be from 1 to 4");
    if (!inputs || !outputs) return invalid_argument(e, "inputs or outputs are null");
    if (inverse > 1) return invalid_argument(e, "inverse must be 0 or 1");
    const uint32_t rotary = rotation->cfg.rotary_dim;
    if (head_dim < rotary || head_dim > 1024)
        return set_error(e, ITAK_SHAPE_MISMATCH, "head_dim", rotary, head_dim, 0, 0,
                         "head_dim: got %llu, a rotation of %u channels needs that many and at most 1024", ULL(head_dim), rotary);
    if (rows > kMostRows) return size_overflow(e, "rows");
    if (rows && !positions_dev) return invalid_argument(e, "positions are null");
    bool by_8 = pieces_of_8(uint32_t(head_dim), rotary / 2, rotation->cfg.interleaved);
    RotateArgs a{};
    uint64_t heads = 0;
    for (uint32_t t = 0; t < tensors; ++t) {
        itak_status st = check_rows(e, "an input", inputs + t, rows, head_dim, false);
        if (st == ITAK_OK) st = check_rows(e, "an output", outputs + t, rows, head_dim, true);
        if (st != ITAK_OK) return st;
        if (inputs[t].elem != inputs[0].elem || outputs[t].elem != inputs[0].elem)
            return invalid_argument(e, "inputs and outputs are of several types");
        if (outputs[t].heads != inputs[t].heads) return shape_mismatch(e, "heads of an output", inputs[t].heads, outputs[t].heads);
        a.in[t] = rows_view(inputs[t], head_dim);
        a.out[t] = rows_view(outputs[t], head_dim);
        if (a.in[t].data == a.out[t].data && rows &&
            (a.in[t].row_stride != a.out[t].row_stride || a.in[t].head_stride != a.out[t].head_stride))
            return invalid_argument(e, "an output starts where its input does and is not the same view");
        by_8 = by_8 && rows_on_16(inputs[t], head_dim) && rows_on_16(outputs[t], head_dim);
        a.heads[t] = inputs[t].heads;
        heads += inputs[t].heads;
    }
    if (rows == 0) return ITAK_OK;
    a.r = rotation_view(rotation);
    a.positions = positions_dev;
    a.head_dim = uint32_t(head_dim);
    a.sign = inverse ? -1.0f : 1.0f;
    a.tensors = tensors;
    a.pieces = uint32_t(heads) * head_pieces(a.head_dim, a.r.half, a.r.interleaved, by_8 ? 8 : 1).all;
    // Few rows are cut into parts of their heads until the device has a workgroup a compute unit.
    const uint32_t whole = (a.pieces + kThreads - 1) / kThreads;
    const uint32_t parts = uint32_t(std::min<uint64_t>(whole, std::max<uint64_t>(1, 512 / rows)));
    a.per_group = (whole + parts - 1) / parts * kThreads;
    const dim3 grid(uint32_t(rows), (a.pieces + a.per_group - 1) / a.per_group);
    const DeviceScope scope(rotation->cfg.device);
    if (scope.status() != hipSuccess) return hip_error(e, scope.status(), "set the device");
    const hipStream_t stream = static_cast<hipStream_t>(hip_stream);
    if (by_8)
        launch_rotate<8>(inputs[0].elem, a, grid, stream);
    else
        launch_rotate<1>(inputs[0].elem, a, grid, stream);
    if (hipError_t he = hipGetLastError(); he != hipSuccess) return hip_error(e, he, "launch a rotation");
    return ITAK_OK;
}

}  // extern "C"
