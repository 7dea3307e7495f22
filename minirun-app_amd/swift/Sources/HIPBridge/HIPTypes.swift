// Device buffers and errors of the bridge.  An HIPTensor stands where MLX
// passes an MLXArray: caller-owned device memory (or pinned host memory the
// device reads), a shape and element strides, no ownership.
import CMinirunHIP

public typealias HIPStream = UnsafeMutableRawPointer?  // hipStream_t; nil = the default stream

public struct HIPTensor {
    public var pointer: UnsafeMutableRawPointer
    public var shape: [Int]
    public var strides: [Int]  // elements
    public var dtype: mr_dtype

    public init(pointer: UnsafeMutableRawPointer, shape: [Int], strides: [Int]? = nil, dtype: mr_dtype) {
        self.pointer = pointer
        self.shape = shape
        self.dtype = dtype
        if let strides {
            self.strides = strides
        } else {  // row-major
            var s = [Int](repeating: 1, count: shape.count)
            var acc = 1
            for i in stride(from: shape.count - 1, through: 0, by: -1) {
                s[i] = acc
                acc *= shape[i]
            }
            self.strides = s
        }
    }

    public var raw: UnsafeRawPointer { UnsafeRawPointer(pointer) }
    public func bytes(_ n: Int) -> Int { n * (dtype == MR_U8 ? 1 : dtype == MR_F32 || dtype == MR_U32 || dtype == MR_I32 ? 4 : 2) }
}

/// What a C call cannot see of its pointers, checked before it.
extension HIPTensor {
    /// [rows, cols] (nil: any) with the values of a row next to each other.
    func needRows(_ name: String, _ rows: Int?, _ cols: Int?, dtype want: mr_dtype? = nil) throws {
        guard shape.count == 2, strides.count == 2, shape[0] == rows ?? shape[0], shape[1] == cols ?? shape[1] else {
            let size = { (n: Int?) in n.map { "\($0)" } ?? "any" }
            throw HIPError(status: MR_INVALID_SHAPE,
                           description: "\(name) must be [\(size(rows)), \(size(cols))], got \(shape)")
        }
        guard strides[1] == 1 || shape[1] == 1 else {
            throw HIPError(status: MR_INVALID_ARGUMENT, description: "\(name) must be contiguous in its last dimension")
        }
        try needType(name, want)
    }

    /// Of this shape (nil: any), without gaps.
    func needWhole(_ name: String, _ size: [Int]?, dtype want: mr_dtype? = nil) throws {
        guard shape == size ?? shape, strides.count == shape.count else {
            throw HIPError(status: MR_INVALID_SHAPE, description: "\(name) must be \(size ?? shape), got \(shape)")
        }
        var next = 1
        for axis in shape.indices.reversed() where !shape.contains(0) {
            guard strides[axis] == next || shape[axis] == 1 else {
                throw HIPError(status: MR_INVALID_ARGUMENT, description: "\(name) must be contiguous")
            }
            next *= shape[axis]
        }
        try needType(name, want)
    }

    private func needType(_ name: String, _ want: mr_dtype?) throws {
        guard dtype == want ?? dtype else {
            throw HIPError(status: MR_INVALID_DTYPE,
                           description: "\(name) has mr_dtype \(dtype.rawValue), not \(want?.rawValue ?? 0)")
        }
    }

    /// Row stride of a 2-D tensor; one row may have any.
    var rowStride: Int64 { Int64(shape[0] > 1 ? strides[0] : max(strides[0], shape[1])) }
}

/// A non-OK mr_status with the library's message for it (the reference's
/// wording where it has one: AffineBridgeError, DeepSeekV4Error).
public struct HIPError: Error, CustomStringConvertible {
    public let status: mr_status
    public let description: String

    static func check(_ st: mr_status) throws {
        guard st != MR_OK else { return }
        throw HIPError(status: st, description: String(cString: mr_get_last_error()))
    }
}

/// Library identity, e.g. "minirun-hip 0.1.0 gfx950".
public var hipBridgeVersion: String { String(cString: mr_version()) }
