// MXFP4 matrices on the device: the MXFP4Weights surface
// (Sources/MLXBridge/MXFP4Weights.swift:36-60) over mr_mxfp4_*.
import CMinirunHIP

/// MXFP4Weights.init(packed:scales:) (MLXBridge/MXFP4Weights.swift:36-60):
/// uint32 words of eight e2m1 numbers and one E8M0 byte per 32 inputs, checked
/// by mr_mxfp4_validate.
public struct HIPMXFP4Weights {
    public let desc: mr_mxfp4_matrix
    public let experts: Int?

    public init(packed: HIPTensor, scales: HIPTensor) throws {
        var ex: Int64 = 0, rows: Int64 = 0, cols: Int64 = 0
        let ps = packed.shape.map(Int64.init), ss = scales.shape.map(Int64.init)
        try HIPError.check(mr_mxfp4_validate(packed.dtype, Int32(ps.count), ps, scales.dtype, Int32(ss.count), ss,
                                             &ex, &rows, &cols))
        desc = mr_mxfp4_matrix(packed: packed.pointer.assumingMemoryBound(to: UInt32.self),
                               scales: scales.pointer.assumingMemoryBound(to: UInt8.self), rows: rows, cols: cols)
        experts = ex > 0 ? Int(ex) : nil
    }
}

/// Rows of bf16 or f32 to MXFP4, the storage of MLXBridge/MXFP4Weights.swift:36-60
/// (`packed` [rows, cols / 8] and `scales` [rows, cols / 32] are written).
public func hipMXFP4Quantize(_ x: HIPTensor, packed: HIPTensor, scales: HIPTensor, stream: HIPStream = nil) throws {
    try HIPError.check(mr_mxfp4_quantize(x.raw, x.dtype, Int64(x.shape[0]), Int64(x.shape[1]), Int64(x.strides[0]),
                                         packed.pointer.assumingMemoryBound(to: UInt32.self),
                                         scales.pointer.assumingMemoryBound(to: UInt8.self), stream))
}

/// The values of a matrix (MLXBridge/MXFP4Weights.swift:36-60) as f32 or bf16.
public func hipMXFP4Dequantize(_ w: HIPMXFP4Weights, into out: HIPTensor, stream: HIPStream = nil) throws {
    var d = w.desc
    d.rows *= Int64(w.experts ?? 1)
    try HIPError.check(mr_mxfp4_dequantize(&d, out.pointer, out.dtype, Int64(out.strides[out.strides.count - 2]), stream))
}

/// MXFP4 matmul (MLXBridge/MXFP4Weights.swift:36-60 holds the weight): y =
/// x . W^T for bf16 or f32 rows.
public func hipMXFP4MM(_ x: HIPTensor, _ w: HIPMXFP4Weights, into y: HIPTensor, stream: HIPStream = nil) throws {
    var d = w.desc
    try HIPError.check(mr_mxfp4_matmul(x.raw, x.dtype, Int32(x.shape[0]), Int64(x.strides[0]), &d, y.pointer, y.dtype,
                                       Int64(y.strides[0]), stream))
}

/// The same with x in MXFP4 (hipMXFP4Quantize's output) too.
public func hipMXFP4MM(quantized x: HIPMXFP4Weights, _ w: HIPMXFP4Weights, into y: HIPTensor,
                       stream: HIPStream = nil) throws {
    var dx = x.desc, dw = w.desc
    try HIPError.check(mr_mxfp4_matmul_quantized(&dx, &dw, y.pointer, y.dtype, Int64(y.strides[0]), stream))
}
