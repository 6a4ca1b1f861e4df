// C++ host-side mirror of the ILGPU.Algorithms surface for radix sort, scan, reduce and
// histogram, bound to the C ABI of b200alg.h.  Header only; link with libb200alg and the CUDA
// runtime.
//
// The reference is C#; this mirror keeps its names, argument meaning, argument checks and
// exception kinds so that calling code reads like code written against ILGPU.Algorithms
// (paths inside the ILGPU source tree, Src/ILGPU.Algorithms):
//   delegates RadixSort / RadixSortPairs / Scan / Reduction / Histogram
//       RadixSortExtensions.cs:37-160, ScanExtensions.cs:52-76, ReductionExtensions.cs:30-35,
//       HistogramExtensions.cs:35-59
//   CreateRadixSort / CreateRadixSortPairs / CreateRadixSortProvider, temp-size helpers
//       RadixSortExtensions.cs:384-447, :1017-1437
//   CreateScan / CreateScanProvider / ComputeScanTempStorageSize, ScanKind
//       ScanExtensions.cs:27-38, :158-170, :930-991
//   CreateReduction / Reduce            ReductionExtensions.cs:135-309
//   Histogram / HistogramUnchecked      HistogramLaunchers.tt:52-101
//   operation structs                   ScanReduceOperations.tt, RadixSortOperations.tt
//   ArrayView / ArrayView1D / Stride1D  Src/ILGPU/ArrayView.cs, Runtime/ArrayViews.tt, Stride.cs
// The operators of a language model's training step (b200alg_embedding and what follows it) have no
// counterpart there and take the same form.
// There is no fallback path: every call ends in the CUDA library.
#pragma once

#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>

#include <cstdint>
#include <functional>
#include <limits>
#include <memory>
#include <stdexcept>
#include <string>
#include <type_traits>
#include <vector>

#include "b200alg.h"

namespace ILGPU {

// ---- exceptions (names of the .NET types the reference throws) ----------------------------
struct ArgumentNullException : std::invalid_argument { using std::invalid_argument::invalid_argument; };
struct ArgumentOutOfRangeException : std::out_of_range { using std::out_of_range::out_of_range; };
struct NotSupportedException : std::runtime_error { using std::runtime_error::runtime_error; };
struct InvalidOperationException : std::logic_error { using std::logic_error::logic_error; };

// Status of the native library -> exception (pattern: CuRandException.ThrowIfFailed,
// Runtime/Cuda/CuRandException.cs:98-103).
struct B200AlgException : std::runtime_error {
    int Status;
    explicit B200AlgException(int status)
        : std::runtime_error(std::string("b200alg: ") + b200alg_status_string(status) +
                             (status == B200ALG_CUDA_ERROR ? " [cudaError " + std::to_string(b200alg_last_cuda_error()) + "]" : "")),
          Status(status) {}
    static void ThrowIfFailed(int status) {
        switch (status) {
        case B200ALG_OK: return;
        case B200ALG_TOO_LARGE: throw NotSupportedException("NotSupportedArrayView64");
        case B200ALG_TEMP_TOO_SMALL: throw ArgumentOutOfRangeException("temp");
        case B200ALG_UNSUPPORTED: throw NotSupportedException(b200alg_status_string(status));
        default: throw B200AlgException(status);
        }
    }
};

// ---- element types ---------------------------------------------------------------------------
template <typename T> struct DTypeOf;
template <> struct DTypeOf<int8_t> { static constexpr int value = B200ALG_I8; };
template <> struct DTypeOf<uint8_t> { static constexpr int value = B200ALG_U8; };
template <> struct DTypeOf<int16_t> { static constexpr int value = B200ALG_I16; };
template <> struct DTypeOf<uint16_t> { static constexpr int value = B200ALG_U16; };
template <> struct DTypeOf<int32_t> { static constexpr int value = B200ALG_I32; };
template <> struct DTypeOf<uint32_t> { static constexpr int value = B200ALG_U32; };
template <> struct DTypeOf<int64_t> { static constexpr int value = B200ALG_I64; };
template <> struct DTypeOf<uint64_t> { static constexpr int value = B200ALG_U64; };
template <> struct DTypeOf<float> { static constexpr int value = B200ALG_F32; };
template <> struct DTypeOf<double> { static constexpr int value = B200ALG_F64; };

// ---- views -----------------------------------------------------------------------------------
namespace Stride1D {
struct Dense { static constexpr int64_t StrideExtent = 1; };
struct General { int64_t StrideExtent = 1; };
}  // namespace Stride1D

// ArrayView<T>: a dense span of device memory (Src/ILGPU/ArrayView.cs).
template <typename T> struct ArrayView {
    T *Pointer = nullptr;
    int64_t Length = 0;
    ArrayView() = default;
    ArrayView(T *pointer, int64_t length) : Pointer(pointer), Length(length) {}
    bool IsValid() const { return Pointer != nullptr; }
    int64_t LengthInBytes() const { return Length * (int64_t)sizeof(T); }
    ArrayView SubView(int64_t index, int64_t length) const {
        if (index < 0 || length < 0 || index + length > Length) throw ArgumentOutOfRangeException("index");
        return ArrayView(Pointer + index, length);
    }
    T *LoadEffectiveAddressAsPtr() const { return Pointer; }
};

// ArrayView1D<T, TStride>: `Length` elements, StrideExtent elements apart.
template <typename T, typename TStride = Stride1D::Dense> struct ArrayView1D {
    ArrayView<T> BaseView;
    TStride Stride;
    int64_t Length = 0;
    ArrayView1D() = default;
    ArrayView1D(ArrayView<T> base, int64_t length, TStride stride = TStride()) : BaseView(base), Stride(stride), Length(length) {}
    // dense views convert from ArrayView<T>
    template <typename S = TStride, typename = typename std::enable_if<std::is_same<S, Stride1D::Dense>::value>::type>
    ArrayView1D(ArrayView<T> base) : BaseView(base), Length(base.Length) {}
    bool IsValid() const { return BaseView.IsValid(); }
    int64_t StrideExtent() const { return Stride.StrideExtent; }
};

template <typename T> ArrayView1D<T, Stride1D::General> AsGeneral(ArrayView<T> base, int64_t stride) {
    const int64_t n = base.Length == 0 ? 0 : (base.Length - 1) / stride + 1;
    return ArrayView1D<T, Stride1D::General>(base, n, Stride1D::General{stride});
}

// ---- runtime plumbing: device, stream, buffers ---------------------------------------------------
class AcceleratorStream {
public:
    AcceleratorStream() : stream_(nullptr), owned_(false) {}  // default stream
    static AcceleratorStream Create() {
        AcceleratorStream s;
        if (cudaStreamCreateWithFlags(&s.stream_, cudaStreamNonBlocking) != cudaSuccess)
            throw InvalidOperationException("cudaStreamCreate failed");
        s.owned_ = true;
        return s;
    }
    AcceleratorStream(AcceleratorStream &&o) noexcept : stream_(o.stream_), owned_(o.owned_) { o.owned_ = false; }
    AcceleratorStream(const AcceleratorStream &) = delete;
    ~AcceleratorStream() { if (owned_) cudaStreamDestroy(stream_); }
    void *StreamPtr() const { return stream_; }  // CudaStream.StreamPtr
    void Synchronize() const { cudaStreamSynchronize(stream_); }
private:
    cudaStream_t stream_;
    bool owned_;
};

template <typename T> class MemoryBuffer1D {
public:
    explicit MemoryBuffer1D(int64_t length) : length_(length) {
        if (cudaMalloc(&ptr_, (size_t)(length < 1 ? 1 : length) * sizeof(T)) != cudaSuccess)
            throw InvalidOperationException("cudaMalloc failed");
    }
    MemoryBuffer1D(const MemoryBuffer1D &) = delete;
    ~MemoryBuffer1D() { cudaFree(ptr_); }
    ArrayView<T> View() const { return ArrayView<T>((T *)ptr_, length_); }
    int64_t Length() const { return length_; }
    void CopyFromCPU(const T *src) { cudaMemcpy(ptr_, src, (size_t)length_ * sizeof(T), cudaMemcpyHostToDevice); }
    void CopyToCPU(T *dst) const { cudaMemcpy(dst, ptr_, (size_t)length_ * sizeof(T), cudaMemcpyDeviceToHost); }
    void MemSetToZero() { cudaMemset(ptr_, 0, (size_t)length_ * sizeof(T)); }
private:
    void *ptr_ = nullptr;
    int64_t length_;
};

class Accelerator {
public:
    explicit Accelerator(int device = 0) : device_(device) {
        int count = 0;
        if (cudaGetDeviceCount(&count) != cudaSuccess || device >= count)
            throw InvalidOperationException("no such CUDA device: this path has no CPU fallback");
    }
    void Bind() const { cudaSetDevice(device_); }  // CudaAccelerator.cs:422-424
    void Synchronize() const { Bind(); cudaDeviceSynchronize(); }
    template <typename T> std::unique_ptr<MemoryBuffer1D<T>> Allocate1D(int64_t length) const {
        Bind();
        return std::unique_ptr<MemoryBuffer1D<T>>(new MemoryBuffer1D<T>(length));
    }
    int Device() const { return device_; }
private:
    int device_;
};

namespace Algorithms {

// ---- operations ------------------------------------------------------------------------------
enum class ScanKind { Inclusive, Exclusive };  // ScanExtensions.cs:27-38

namespace ScanReduceOperations {
template <typename TT, int OP> struct Operation {
    using T = TT;
    static constexpr int Op = OP;
    static T Identity() {
        return OP == B200ALG_ADD ? T(0) : (OP == B200ALG_MAX ? std::numeric_limits<T>::lowest() : std::numeric_limits<T>::max());
    }
};
#define B200ALG_DECLARE_SR_OPS(Name, Type)                      \
    using Add##Name = Operation<Type, B200ALG_ADD>;              \
    using Max##Name = Operation<Type, B200ALG_MAX>;              \
    using Min##Name = Operation<Type, B200ALG_MIN>;
B200ALG_DECLARE_SR_OPS(Int32, int32_t)
B200ALG_DECLARE_SR_OPS(Int64, int64_t)
B200ALG_DECLARE_SR_OPS(UInt32, uint32_t)
B200ALG_DECLARE_SR_OPS(UInt64, uint64_t)
B200ALG_DECLARE_SR_OPS(Float, float)
B200ALG_DECLARE_SR_OPS(Double, double)
#undef B200ALG_DECLARE_SR_OPS
}  // namespace ScanReduceOperations

namespace RadixSortOperations {
template <typename TT, bool DESCENDING> struct Operation {
    using T = TT;
    static constexpr int Order = DESCENDING ? B200ALG_SORT_DESCENDING : B200ALG_SORT_ASCENDING;
    static constexpr int NumBits = sizeof(TT) * 8;
};
#define B200ALG_DECLARE_SORT_OPS(Name, Type)            \
    using Ascending##Name = Operation<Type, false>;      \
    using Descending##Name = Operation<Type, true>;
B200ALG_DECLARE_SORT_OPS(Int8, int8_t)
B200ALG_DECLARE_SORT_OPS(UInt8, uint8_t)
B200ALG_DECLARE_SORT_OPS(Int16, int16_t)
B200ALG_DECLARE_SORT_OPS(UInt16, uint16_t)
B200ALG_DECLARE_SORT_OPS(Int32, int32_t)
B200ALG_DECLARE_SORT_OPS(UInt32, uint32_t)
B200ALG_DECLARE_SORT_OPS(Int64, int64_t)
B200ALG_DECLARE_SORT_OPS(UInt64, uint64_t)
B200ALG_DECLARE_SORT_OPS(Float, float)
B200ALG_DECLARE_SORT_OPS(Double, double)
#undef B200ALG_DECLARE_SORT_OPS
}  // namespace RadixSortOperations

// Named bin locators (the reference leaves the locator to user structs; see b200alg.h).
struct ModuloBinOperation {
    static constexpr int Locator = B200ALG_LOCATOR_MODULO;
    double Lo = 0.0, Hi = 1.0;
};
struct EqualWidthClampLocator {
    static constexpr int Locator = B200ALG_LOCATOR_EQUAL_WIDTH_CLAMP;
    double Lo, Hi;
    EqualWidthClampLocator(double lo, double hi) : Lo(lo), Hi(hi) {}
};

// ---- delegates -----------------------------------------------------------------------------------
template <typename T, typename TStride = Stride1D::Dense>
using RadixSort = std::function<void(const AcceleratorStream &, ArrayView1D<T, TStride>, ArrayView<int>)>;
template <typename TKey, typename TValue>
using RadixSortPairs = std::function<void(const AcceleratorStream &, ArrayView1D<TKey>, ArrayView1D<TValue>, ArrayView<int>)>;
template <typename T, typename TStrideIn = Stride1D::Dense, typename TStrideOut = Stride1D::Dense>
using Scan = std::function<void(const AcceleratorStream &, ArrayView1D<T, TStrideIn>, ArrayView1D<T, TStrideOut>, ArrayView<int>)>;
template <typename T, typename TStride = Stride1D::Dense>
using Reduction = std::function<void(const AcceleratorStream &, ArrayView1D<T, TStride>, ArrayView<T>)>;

namespace detail {
inline int64_t IntsFor(int64_t bytes) {
    const int64_t ints = (bytes + 3) / 4;
    if (ints > std::numeric_limits<int32_t>::max()) throw NotSupportedException("temporary storage exceeds the Index1D range");
    return ints;
}
inline void CheckTemp(const ArrayView<int> &temp, int64_t required_ints) {
    // TempViewManager (TempViewManager.cs:36-37, :84-112)
    if (!temp.IsValid()) throw ArgumentNullException("temp");
    if (temp.Length < required_ints) throw ArgumentOutOfRangeException("temp");
}
}  // namespace detail

// ---- temp sizing (in 32-bit ints, like the reference) --------------------------------------------
template <typename T, typename TRadixSortOperation>
inline int64_t ComputeRadixSortTempStorageSize(const Accelerator &, int64_t dataLength) {
    int64_t bytes = 0;
    B200AlgException::ThrowIfFailed(b200alg_radix_sort_temp_bytes(DTypeOf<T>::value, dataLength, 0, &bytes));
    return detail::IntsFor(bytes);
}
template <typename TKey, typename TValue, typename TRadixSortOperation>
inline int64_t ComputeRadixSortPairsTempStorageSize(const Accelerator &, int64_t dataLength) {
    int64_t bytes = 0;
    B200AlgException::ThrowIfFailed(b200alg_radix_sort_temp_bytes(DTypeOf<TKey>::value, dataLength, (int)sizeof(TValue), &bytes));
    return detail::IntsFor(bytes);
}
template <typename T> inline int64_t ComputeScanTempStorageSize(const Accelerator &, int64_t dataLength) {
    int64_t bytes = 0;
    B200AlgException::ThrowIfFailed(b200alg_scan_temp_bytes(DTypeOf<T>::value, dataLength, &bytes));
    return detail::IntsFor(bytes);
}

// ---- radix sort ------------------------------------------------------------------------------------
template <typename T, typename TStride, typename TRadixSortOperation>
inline RadixSort<T, TStride> CreateRadixSort(const Accelerator &accelerator) {
    static_assert(std::is_same<T, typename TRadixSortOperation::T>::value, "operation and element type differ");
    return [accelerator](const AcceleratorStream &stream, ArrayView1D<T, TStride> view, ArrayView<int> temp) {
        if (!view.IsValid()) throw ArgumentNullException("view");
        if (view.Length > std::numeric_limits<int32_t>::max()) throw NotSupportedException("NotSupportedArrayView64");
        detail::CheckTemp(temp, ComputeRadixSortTempStorageSize<T, TRadixSortOperation>(accelerator, view.Length));
        accelerator.Bind();
        B200AlgException::ThrowIfFailed(b200alg_radix_sort_keys(stream.StreamPtr(), view.BaseView.Pointer, view.Length,
                                                                view.StrideExtent(), DTypeOf<T>::value,
                                                                TRadixSortOperation::Order, temp.Pointer, temp.LengthInBytes()));
    };
}

template <typename TKey, typename TValue, typename TRadixSortOperation>
inline RadixSortPairs<TKey, TValue> CreateRadixSortPairs(const Accelerator &accelerator) {
    static_assert(std::is_same<TKey, typename TRadixSortOperation::T>::value, "operation and key type differ");
    return [accelerator](const AcceleratorStream &stream, ArrayView1D<TKey> keys, ArrayView1D<TValue> values, ArrayView<int> temp) {
        if (!keys.IsValid()) throw ArgumentNullException("keys");
        if (!values.IsValid()) throw ArgumentNullException("values");
        if (values.Length < keys.Length) throw ArgumentOutOfRangeException("values");
        if (keys.Length > std::numeric_limits<int32_t>::max()) throw NotSupportedException("NotSupportedArrayView64");
        detail::CheckTemp(temp, ComputeRadixSortPairsTempStorageSize<TKey, TValue, TRadixSortOperation>(accelerator, keys.Length));
        accelerator.Bind();
        B200AlgException::ThrowIfFailed(b200alg_radix_sort_pairs(stream.StreamPtr(), keys.BaseView.Pointer, values.BaseView.Pointer,
                                                                 keys.Length, DTypeOf<TKey>::value, (int)sizeof(TValue),
                                                                 TRadixSortOperation::Order, temp.Pointer, temp.LengthInBytes()));
    };
}

// Sequencers (Sequencer.cs:20-72, Sequencers.tt:26-38): element i is the index converted to T.
// Only these built-in, stateless ones cross the native boundary.
template <typename TValue> struct ISequencer { using T = TValue; };
struct IndexSequencer : ISequencer<int32_t> {};
struct Int8Sequencer : ISequencer<int8_t> {};
struct UInt8Sequencer : ISequencer<uint8_t> {};
struct Int16Sequencer : ISequencer<int16_t> {};
struct UInt16Sequencer : ISequencer<uint16_t> {};
struct Int32Sequencer : ISequencer<int32_t> {};
struct UInt32Sequencer : ISequencer<uint32_t> {};
struct Int64Sequencer : ISequencer<int64_t> {};
struct UInt64Sequencer : ISequencer<uint64_t> {};
struct FloatSequencer : ISequencer<float> {};
struct DoubleSequencer : ISequencer<double> {};

// The sequencer overload of CreateRadixSortPairs (RadixSortExtensions.cs:1017-1074): values
// entering the sort are sequencer.ComputeSequenceElement(i); `values` receives the result.
template <typename TKey, typename TValue, typename TSequencer>
using RadixSortPairsSequenced =
    std::function<void(const AcceleratorStream &, ArrayView1D<TKey>, ArrayView1D<TValue>, TSequencer, ArrayView<int>)>;
template <typename TKey, typename TValue, typename TSequencer, typename TRadixSortOperation>
inline RadixSortPairsSequenced<TKey, TValue, TSequencer> CreateRadixSortPairs(const Accelerator &accelerator) {
    static_assert(std::is_same<TKey, typename TRadixSortOperation::T>::value, "operation and key type differ");
    static_assert(std::is_same<TValue, typename TSequencer::T>::value, "sequencer and value type differ");
    return [accelerator](const AcceleratorStream &stream, ArrayView1D<TKey> keys, ArrayView1D<TValue> values, TSequencer,
                         ArrayView<int> temp) {
        if (!keys.IsValid()) throw ArgumentNullException("keys");
        if (!values.IsValid()) throw ArgumentNullException("values");
        if (keys.Length != values.Length) throw ArgumentOutOfRangeException("values");
        if (keys.Length > std::numeric_limits<int32_t>::max()) throw NotSupportedException("NotSupportedArrayView64");
        detail::CheckTemp(temp, ComputeRadixSortPairsTempStorageSize<TKey, TValue, TRadixSortOperation>(accelerator, keys.Length));
        accelerator.Bind();
        B200AlgException::ThrowIfFailed(b200alg_radix_sort_pairs_sequence(
            stream.StreamPtr(), keys.BaseView.Pointer, values.BaseView.Pointer, keys.Length, DTypeOf<TKey>::value,
            DTypeOf<TValue>::value, TRadixSortOperation::Order, temp.Pointer, temp.LengthInBytes()));
    };
}

// RadixSortProvider (RadixSortExtensions.cs:168-300): owns the temp buffer.
class RadixSortProvider {
public:
    RadixSortProvider(const Accelerator &accelerator, int64_t temp_ints)
        : accelerator_(accelerator), temp_(accelerator.Allocate1D<int>(temp_ints < 64 ? 64 : temp_ints)) {}
    template <typename T, typename TStride, typename TRadixSortOperation>
    std::function<void(const AcceleratorStream &, ArrayView1D<T, TStride>)> CreateRadixSort() {
        auto sort = Algorithms::CreateRadixSort<T, TStride, TRadixSortOperation>(accelerator_);
        ArrayView<int> temp = temp_->View();
        return [sort, temp](const AcceleratorStream &stream, ArrayView1D<T, TStride> view) { sort(stream, view, temp); };
    }
    template <typename TKey, typename TValue, typename TRadixSortOperation>
    std::function<void(const AcceleratorStream &, ArrayView1D<TKey>, ArrayView1D<TValue>)> CreateRadixSortPairs() {
        auto sort = Algorithms::CreateRadixSortPairs<TKey, TValue, TRadixSortOperation>(accelerator_);
        ArrayView<int> temp = temp_->View();
        return [sort, temp](const AcceleratorStream &stream, ArrayView1D<TKey> keys, ArrayView1D<TValue> values) {
            sort(stream, keys, values, temp);
        };
    }
private:
    Accelerator accelerator_;
    std::unique_ptr<MemoryBuffer1D<int>> temp_;
};
template <typename T, typename TRadixSortOperation>
inline RadixSortProvider CreateRadixSortProvider(const Accelerator &accelerator, int64_t dataLength) {
    return RadixSortProvider(accelerator, ComputeRadixSortTempStorageSize<T, TRadixSortOperation>(accelerator, dataLength));
}
template <typename TKey, typename TValue, typename TRadixSortOperation>
inline RadixSortProvider CreateRadixSortPairsProvider(const Accelerator &accelerator, int64_t dataLength) {
    return RadixSortProvider(accelerator, ComputeRadixSortPairsTempStorageSize<TKey, TValue, TRadixSortOperation>(accelerator, dataLength));
}

// ---- scan --------------------------------------------------------------------------------------------
template <typename T, typename TStrideIn, typename TStrideOut, typename TScanOperation>
inline Scan<T, TStrideIn, TStrideOut> CreateScan(const Accelerator &accelerator, ScanKind kind) {
    static_assert(std::is_same<T, typename TScanOperation::T>::value, "operation and element type differ");
    return [accelerator, kind](const AcceleratorStream &stream, ArrayView1D<T, TStrideIn> input,
                               ArrayView1D<T, TStrideOut> output, ArrayView<int> temp) {
        // order of the checks: ScanExtensions.cs:675-689
        if (!input.IsValid()) throw ArgumentNullException("input");
        if (!output.IsValid()) throw ArgumentNullException("output");
        if (output.Length < input.Length) throw ArgumentOutOfRangeException("output");
        if (input.Length > std::numeric_limits<int32_t>::max()) throw NotSupportedException("NotSupportedArrayView64");
        detail::CheckTemp(temp, ComputeScanTempStorageSize<T>(accelerator, input.Length));
        accelerator.Bind();
        B200AlgException::ThrowIfFailed(b200alg_scan(stream.StreamPtr(), input.BaseView.Pointer, input.StrideExtent(),
                                                     output.BaseView.Pointer, output.StrideExtent(), input.Length,
                                                     DTypeOf<T>::value, TScanOperation::Op, kind == ScanKind::Inclusive ? 1 : 0,
                                                     temp.Pointer, temp.LengthInBytes()));
    };
}

// ScanProvider (ScanExtensions.cs:84-142).
class ScanProvider {
public:
    ScanProvider(const Accelerator &accelerator, int64_t temp_ints)
        : accelerator_(accelerator), temp_(accelerator.Allocate1D<int>(temp_ints < 64 ? 64 : temp_ints)) {}
    template <typename T, typename TStrideIn, typename TStrideOut, typename TScanOperation>
    std::function<void(const AcceleratorStream &, ArrayView1D<T, TStrideIn>, ArrayView1D<T, TStrideOut>)> CreateScan(ScanKind kind) {
        auto scan = Algorithms::CreateScan<T, TStrideIn, TStrideOut, TScanOperation>(accelerator_, kind);
        ArrayView<int> temp = temp_->View();
        return [scan, temp](const AcceleratorStream &stream, ArrayView1D<T, TStrideIn> input, ArrayView1D<T, TStrideOut> output) {
            scan(stream, input, output, temp);
        };
    }
private:
    Accelerator accelerator_;
    std::unique_ptr<MemoryBuffer1D<int>> temp_;
};
template <typename T> inline ScanProvider CreateScanProvider(const Accelerator &accelerator, int64_t dataLength) {
    return ScanProvider(accelerator, ComputeScanTempStorageSize<T>(accelerator, dataLength));
}

// ---- reduce ------------------------------------------------------------------------------------------
template <typename T, typename TStride, typename TReduction>
inline Reduction<T, TStride> CreateReduction(const Accelerator &accelerator) {
    static_assert(std::is_same<T, typename TReduction::T>::value, "operation and element type differ");
    return [accelerator](const AcceleratorStream &stream, ArrayView1D<T, TStride> input, ArrayView<T> output) {
        // ReductionExtensions.cs:146-153
        if (!input.IsValid()) throw ArgumentNullException("input");
        if (input.Length < 1) throw ArgumentOutOfRangeException("input");
        if (!output.IsValid()) throw ArgumentNullException("output");
        if (output.Length < 1) throw ArgumentOutOfRangeException("output");
        accelerator.Bind();
        B200AlgException::ThrowIfFailed(b200alg_reduce(stream.StreamPtr(), input.BaseView.Pointer, input.StrideExtent(),
                                                       input.Length, DTypeOf<T>::value, TReduction::Op, output.Pointer));
    };
}

// Asynchronous overload with an output view (ReductionExtensions.cs:180-196).
template <typename T, typename TStride, typename TReduction>
inline void Reduce(const Accelerator &accelerator, const AcceleratorStream &stream, ArrayView1D<T, TStride> input, ArrayView<T> output) {
    CreateReduction<T, TStride, TReduction>(accelerator)(stream, input, output);
}
// Value-returning overload: allocates one element, reduces, copies back - which synchronises
// (ReductionExtensions.cs:198-216).
template <typename T, typename TStride, typename TReduction>
inline T Reduce(const Accelerator &accelerator, const AcceleratorStream &stream, ArrayView1D<T, TStride> input) {
    auto cell = accelerator.Allocate1D<T>(1);
    CreateReduction<T, TStride, TReduction>(accelerator)(stream, input, cell->View());
    T result;
    stream.Synchronize();
    cell->CopyToCPU(&result);
    return result;
}

// ---- histogram ---------------------------------------------------------------------------------------
template <typename T, typename TStride, typename TBinType, typename TLocator>
inline void Histogram(const Accelerator &accelerator, const AcceleratorStream &stream, ArrayView1D<T, TStride> view,
                      ArrayView<TBinType> histogram, ArrayView<int> histogramOverflow, const TLocator &locator) {
    // HistogramExtensions.cs:322-338
    if (!view.IsValid()) throw ArgumentNullException("view");
    if (!histogram.IsValid()) throw ArgumentNullException("histogram");
    if (!histogramOverflow.IsValid()) throw ArgumentNullException("histogramOverflow");
    if (view.Length > std::numeric_limits<int32_t>::max() || histogram.Length > std::numeric_limits<int32_t>::max())
        throw NotSupportedException("NotSupportedArrayView64");
    if (histogram.Length < 1) throw ArgumentOutOfRangeException("histogram");
    if (histogramOverflow.Length < 1) throw ArgumentOutOfRangeException("histogramOverflow");
    accelerator.Bind();
    B200AlgException::ThrowIfFailed(b200alg_histogram(stream.StreamPtr(), view.BaseView.Pointer, view.StrideExtent(), view.Length,
                                                      DTypeOf<T>::value, TLocator::Locator, locator.Lo, locator.Hi, histogram.Pointer,
                                                      histogram.Length, DTypeOf<TBinType>::value, histogramOverflow.Pointer));
}

template <typename T, typename TStride, typename TBinType, typename TLocator>
inline void HistogramUnchecked(const Accelerator &accelerator, const AcceleratorStream &stream, ArrayView1D<T, TStride> view,
                               ArrayView<TBinType> histogram, const TLocator &locator) {
    if (!view.IsValid()) throw ArgumentNullException("view");
    if (!histogram.IsValid()) throw ArgumentNullException("histogram");
    if (view.Length > std::numeric_limits<int32_t>::max() || histogram.Length > std::numeric_limits<int32_t>::max())
        throw NotSupportedException("NotSupportedArrayView64");
    if (histogram.Length < 1) throw ArgumentOutOfRangeException("histogram");
    accelerator.Bind();
    B200AlgException::ThrowIfFailed(b200alg_histogram(stream.StreamPtr(), view.BaseView.Pointer, view.StrideExtent(), view.Length,
                                                      DTypeOf<T>::value, TLocator::Locator, locator.Lo, locator.Hi, histogram.Pointer,
                                                      histogram.Length, DTypeOf<TBinType>::value, nullptr));
}

// ---- operators of a training step ------------------------------------------------------------------
// Element types float, __half and __nv_bfloat16; indices int32_t and int64_t.
template <typename T> struct ElementOf;
template <> struct ElementOf<float> { static constexpr int value = B200ALG_F32; };
template <> struct ElementOf<__half> { static constexpr int value = B200ALG_F16; };
template <> struct ElementOf<__nv_bfloat16> { static constexpr int value = B200ALG_BF16; };

// A matrix whose rows are dense and RowStride elements apart (ArrayView2D<T, Stride2D.DenseX>).
template <typename T> struct ArrayView2D {
    ArrayView<T> BaseView;
    int64_t Rows = 0, Width = 0, RowStride = 0;
    ArrayView2D() = default;
    ArrayView2D(ArrayView<T> base, int64_t rows, int64_t width, int64_t rowStride = -1)
        : BaseView(base), Rows(rows), Width(width), RowStride(rowStride < 0 ? width : rowStride) {
        if (rows < 0 || width < 0 || RowStride < width || (rows && base.Length < (rows - 1) * RowStride + width))
            throw ArgumentOutOfRangeException("extent");
    }
    bool IsValid() const { return BaseView.IsValid(); }
};

// One of a list of dense views of different element types.
struct ElementView {
    void *Pointer;
    int64_t Length;
    int DType;
    template <typename T> ElementView(ArrayView<T> view) : Pointer(view.Pointer), Length(view.Length), DType(ElementOf<T>::value) {}
};

template <typename TTable, typename TIndex, typename TOut>
using Embedding = std::function<void(const AcceleratorStream &, ArrayView2D<TTable>, ArrayView1D<TIndex>, ArrayView2D<TOut>, double)>;
template <typename TTable, typename TIndex, typename TOut>
inline Embedding<TTable, TIndex, TOut> CreateEmbedding(const Accelerator &accelerator) {
    return [accelerator](const AcceleratorStream &stream, ArrayView2D<TTable> table, ArrayView1D<TIndex> tokens, ArrayView2D<TOut> output,
                         double scale) {
        if (!table.IsValid()) throw ArgumentNullException("table");
        if (!tokens.IsValid()) throw ArgumentNullException("tokens");
        if (!output.IsValid()) throw ArgumentNullException("output");
        if (output.Width != table.Width || output.Rows < tokens.Length) throw ArgumentOutOfRangeException("output");
        accelerator.Bind();
        B200AlgException::ThrowIfFailed(b200alg_embedding(
            stream.StreamPtr(), table.BaseView.Pointer, table.Rows, table.Width, table.RowStride, ElementOf<TTable>::value, tokens.BaseView.Pointer,
            tokens.Length, tokens.StrideExtent(), DTypeOf<TIndex>::value, scale, output.BaseView.Pointer, output.RowStride, ElementOf<TOut>::value));
    };
}

inline int64_t ComputeEmbeddingGradientTempStorageSize(const Accelerator &, int64_t rows, int64_t width, int64_t dataLength) {
    int64_t bytes = 0;
    B200AlgException::ThrowIfFailed(b200alg_embedding_gradient_temp_bytes(rows, width, dataLength, &bytes));
    return detail::IntsFor(bytes);
}
template <typename TIndex, typename TUpstream, typename TTable>
using EmbeddingGradient =
    std::function<void(const AcceleratorStream &, ArrayView1D<TIndex>, ArrayView2D<TUpstream>, ArrayView2D<TTable>, ArrayView<int>, double)>;
template <typename TIndex, typename TUpstream, typename TTable>
inline EmbeddingGradient<TIndex, TUpstream, TTable> CreateEmbeddingGradient(const Accelerator &accelerator, bool accumulate = false) {
    return [accelerator, accumulate](const AcceleratorStream &stream, ArrayView1D<TIndex> tokens, ArrayView2D<TUpstream> outputGradient,
                                     ArrayView2D<TTable> tableGradient, ArrayView<int> temp, double scale) {
        if (!tokens.IsValid()) throw ArgumentNullException("tokens");
        if (!outputGradient.IsValid()) throw ArgumentNullException("outputGradient");
        if (!tableGradient.IsValid()) throw ArgumentNullException("tableGradient");
        if (outputGradient.Width != tableGradient.Width || outputGradient.Rows < tokens.Length) throw ArgumentOutOfRangeException("outputGradient");
        detail::CheckTemp(temp, ComputeEmbeddingGradientTempStorageSize(accelerator, tableGradient.Rows, tableGradient.Width, tokens.Length));
        accelerator.Bind();
        B200AlgException::ThrowIfFailed(b200alg_embedding_gradient(
            stream.StreamPtr(), tokens.BaseView.Pointer, tokens.Length, tokens.StrideExtent(), DTypeOf<TIndex>::value, outputGradient.BaseView.Pointer,
            outputGradient.RowStride, ElementOf<TUpstream>::value, scale, tableGradient.BaseView.Pointer, tableGradient.Rows, tableGradient.Width,
            tableGradient.RowStride, ElementOf<TTable>::value, accumulate ? 1 : 0, temp.Pointer, temp.LengthInBytes()));
    };
}

namespace detail {
struct ElementLists {
    std::vector<const void *> in;
    std::vector<void *> out;
    std::vector<int64_t> lengths;
    std::vector<int> types, out_types;
    ElementLists(const std::vector<ElementView> &views, const std::vector<ElementView> *outputs) {
        if (outputs && outputs->size() != views.size()) throw ArgumentOutOfRangeException("outputs");
        for (size_t i = 0; i < views.size(); ++i) {
            in.push_back(views[i].Pointer);
            lengths.push_back(views[i].Length);
            types.push_back(views[i].DType);
            if (!outputs) continue;
            if ((*outputs)[i].Length != views[i].Length) throw ArgumentOutOfRangeException("outputs");
            out.push_back((*outputs)[i].Pointer);
            out_types.push_back((*outputs)[i].DType);
        }
    }
};
}  // namespace detail

inline int64_t ComputeGradientNormTempStorageSize(const Accelerator &, int64_t numViews) {
    int64_t bytes = 0;
    B200AlgException::ThrowIfFailed(b200alg_gradient_norm_temp_bytes(numViews, &bytes));
    return detail::IntsFor(bytes);
}
inline void GradientNorm(const Accelerator &accelerator, const AcceleratorStream &stream, const std::vector<ElementView> &views, ArrayView<float> norm,
                         ArrayView<int> temp) {
    if (!norm.IsValid()) throw ArgumentNullException("norm");
    if (norm.Length < 1) throw ArgumentOutOfRangeException("norm");
    detail::CheckTemp(temp, ComputeGradientNormTempStorageSize(accelerator, (int64_t)views.size()));
    const detail::ElementLists l(views, nullptr);
    accelerator.Bind();
    B200AlgException::ThrowIfFailed(b200alg_gradient_norm(stream.StreamPtr(), l.in.data(), l.lengths.data(), l.types.data(), (int64_t)views.size(),
                                                          norm.Pointer, temp.Pointer, temp.LengthInBytes()));
}
// outputs == nullptr: in place.
inline void GradientClip(const Accelerator &accelerator, const AcceleratorStream &stream, const std::vector<ElementView> &views,
                         const std::vector<ElementView> *outputs, double maxNorm, ArrayView<float> norm, ArrayView<int> temp) {
    if (!norm.IsValid()) throw ArgumentNullException("norm");
    if (norm.Length < 1) throw ArgumentOutOfRangeException("norm");
    if (!(maxNorm >= 0.0)) throw ArgumentOutOfRangeException("maxNorm");
    detail::CheckTemp(temp, ComputeGradientNormTempStorageSize(accelerator, (int64_t)views.size()));
    const detail::ElementLists l(views, outputs);
    accelerator.Bind();
    B200AlgException::ThrowIfFailed(b200alg_gradient_clip(stream.StreamPtr(), l.in.data(), outputs ? l.out.data() : nullptr, l.lengths.data(),
                                                          l.types.data(), outputs ? l.out_types.data() : nullptr, (int64_t)views.size(), maxNorm,
                                                          norm.Pointer, temp.Pointer, temp.LengthInBytes()));
}
// By a norm that is in device memory already.
inline void GradientScale(const Accelerator &accelerator, const AcceleratorStream &stream, const std::vector<ElementView> &views,
                          const std::vector<ElementView> *outputs, double maxNorm, ArrayView<float> norm) {
    if (!norm.IsValid()) throw ArgumentNullException("norm");
    if (norm.Length < 1) throw ArgumentOutOfRangeException("norm");
    if (!(maxNorm >= 0.0)) throw ArgumentOutOfRangeException("maxNorm");
    const detail::ElementLists l(views, outputs);
    accelerator.Bind();
    B200AlgException::ThrowIfFailed(b200alg_gradient_scale(stream.StreamPtr(), l.in.data(), outputs ? l.out.data() : nullptr, l.lengths.data(),
                                                           l.types.data(), outputs ? l.out_types.data() : nullptr, (int64_t)views.size(),
                                                           norm.Pointer, maxNorm));
}

inline int64_t ComputeBalanceLossTempStorageSize(const Accelerator &, int64_t numExperts, int64_t dataLength) {
    int64_t bytes = 0;
    B200AlgException::ThrowIfFailed(b200alg_balance_loss_temp_bytes(numExperts, dataLength, &bytes));
    return detail::IntsFor(bytes);
}
namespace detail {
inline void CheckRouter(int64_t tokens, int64_t experts, const ArrayView<uint8_t> &mask, const ArrayView<int32_t> &counts) {
    if (mask.IsValid() && mask.Length < tokens) throw ArgumentOutOfRangeException("mask");
    if (!counts.IsValid()) throw ArgumentNullException("counts");
    if (counts.Length < experts + 1) throw ArgumentOutOfRangeException("counts");
}
}  // namespace detail
// mask: a byte per token, or an invalid view: all tokens count.
template <typename T, typename TIndex>
inline void BalanceLoss(const Accelerator &accelerator, const AcceleratorStream &stream, ArrayView2D<T> logits, ArrayView2D<TIndex> experts,
                        ArrayView<uint8_t> mask, double coefficient, ArrayView<float> loss, ArrayView<int32_t> counts, ArrayView<float> probabilities,
                        ArrayView<int> temp) {
    if (!logits.IsValid()) throw ArgumentNullException("logits");
    if (!experts.IsValid()) throw ArgumentNullException("experts");
    if (experts.Rows != logits.Rows) throw ArgumentOutOfRangeException("experts");
    detail::CheckRouter(logits.Rows, logits.Width, mask, counts);
    if (!loss.IsValid()) throw ArgumentNullException("loss");
    if (loss.Length < 1) throw ArgumentOutOfRangeException("loss");
    if (!probabilities.IsValid()) throw ArgumentNullException("probabilities");
    if (probabilities.Length < logits.Width) throw ArgumentOutOfRangeException("probabilities");
    detail::CheckTemp(temp, ComputeBalanceLossTempStorageSize(accelerator, logits.Width, logits.Rows));
    accelerator.Bind();
    B200AlgException::ThrowIfFailed(b200alg_balance_loss(
        stream.StreamPtr(), logits.BaseView.Pointer, logits.Rows, logits.Width, logits.RowStride, ElementOf<T>::value, experts.BaseView.Pointer,
        experts.Width, experts.RowStride, DTypeOf<TIndex>::value, mask.Pointer, coefficient, loss.Pointer, counts.Pointer, probabilities.Pointer,
        temp.Pointer, temp.LengthInBytes()));
}
template <typename T>
inline void BalanceLossGradient(const Accelerator &accelerator, const AcceleratorStream &stream, ArrayView2D<T> logits, ArrayView<uint8_t> mask,
                                ArrayView<int32_t> counts, int64_t choices, double coefficient, ArrayView<float> lossGradient,
                                ArrayView2D<T> logitsGradient, bool accumulate = false) {
    if (!logits.IsValid()) throw ArgumentNullException("logits");
    if (!logitsGradient.IsValid()) throw ArgumentNullException("logitsGradient");
    if (logitsGradient.Rows != logits.Rows || logitsGradient.Width != logits.Width) throw ArgumentOutOfRangeException("logitsGradient");
    detail::CheckRouter(logits.Rows, logits.Width, mask, counts);
    if (!lossGradient.IsValid()) throw ArgumentNullException("lossGradient");
    if (lossGradient.Length < 1) throw ArgumentOutOfRangeException("lossGradient");
    accelerator.Bind();
    B200AlgException::ThrowIfFailed(b200alg_balance_loss_gradient(
        stream.StreamPtr(), logits.BaseView.Pointer, logits.Rows, logits.Width, logits.RowStride, ElementOf<T>::value, mask.Pointer, counts.Pointer,
        choices, coefficient, lossGradient.Pointer, logitsGradient.BaseView.Pointer, logitsGradient.RowStride, accumulate ? 1 : 0));
}

}  // namespace Algorithms
}  // namespace ILGPU
