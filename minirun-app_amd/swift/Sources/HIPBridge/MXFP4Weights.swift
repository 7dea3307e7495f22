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
        try packed.needWhole("packed", nil)
        try scales.needWhole("scales", nil)
        desc = mr_mxfp4_matrix(packed: packed.pointer.assumingMemoryBound(to: UInt32.self),
                               scales: scales.pointer.assumingMemoryBound(to: UInt8.self), rows: rows, cols: cols)
        experts = ex > 0 ? Int(ex) : nil
    }

    /// One matrix, no stack, of `cols` columns.
    func needMatrix(_ name: String, cols: Int64? = nil) throws {
        guard experts == nil else {
            throw HIPError(status: MR_INVALID_SHAPE, description: "\(name) is a stack of experts, not one matrix")
        }
        guard desc.cols == cols ?? desc.cols else {
            throw HIPError(status: MR_INVALID_SHAPE,
                           description: "\(name) has \(desc.cols) columns, not \(cols ?? desc.cols)")
        }
    }
}

/// Rows of bf16 or f32 to MXFP4, the storage of MLXBridge/MXFP4Weights.swift:36-60
/// (`packed` [rows, cols / 8] and `scales` [rows, cols / 32] are written).
public func hipMXFP4Quantize(_ x: HIPTensor, packed: HIPTensor, scales: HIPTensor, stream: HIPStream = nil) throws {
    try x.needRows("x", nil, nil)
    try packed.needWhole("packed", [x.shape[0], x.shape[1] / 8], dtype: MR_U32)
    try scales.needWhole("scales", [x.shape[0], x.shape[1] / 32], dtype: MR_U8)
    try HIPError.check(mr_mxfp4_quantize(x.raw, x.dtype, Int64(x.shape[0]), Int64(x.shape[1]), x.rowStride,
                                         packed.pointer.assumingMemoryBound(to: UInt32.self),
                                         scales.pointer.assumingMemoryBound(to: UInt8.self), stream))
}

/// The values of a matrix (MLXBridge/MXFP4Weights.swift:36-60) as f32 or bf16, in
/// the weight's shape, or for a stack all rows in one; its matrices follow each
/// other at the row stride.
public func hipMXFP4Dequantize(_ w: HIPMXFP4Weights, into out: HIPTensor, stream: HIPStream = nil) throws {
    var d = w.desc
    d.rows *= Int64(w.experts ?? 1)
    let rows = Int(w.desc.rows), cols = Int(d.cols)
    var all = out  // the rows of all matrices
    if let experts = w.experts, out.shape.count != 2 {
        guard out.shape == [experts, rows, cols], out.strides.count == 3,
              experts == 1 || rows <= 1 || out.strides[0] == rows * out.strides[1] else {
            throw HIPError(status: MR_INVALID_SHAPE,
                           description: "out must be [\(experts), \(rows), \(cols)] with its rows at one stride, got \(out.shape)")
        }
        all = HIPTensor(pointer: out.pointer, shape: [experts * rows, cols], strides: [out.strides[1], out.strides[2]],
                        dtype: out.dtype)
        if rows == 1 { all.strides[0] = out.strides[0] }
    }
    try all.needRows("out", Int(d.rows), cols)
    try HIPError.check(mr_mxfp4_dequantize(&d, out.pointer, out.dtype, all.rowStride, stream))
}

/// MXFP4 matmul (MLXBridge/MXFP4Weights.swift:36-60 holds the weight): y =
/// x . W^T for bf16 or f32 rows.
public func hipMXFP4MM(_ x: HIPTensor, _ w: HIPMXFP4Weights, into y: HIPTensor, stream: HIPStream = nil) throws {
    var d = w.desc
    try w.needMatrix("w")
    try x.needRows("x", nil, Int(d.cols))
    try y.needRows("y", x.shape[0], Int(d.rows))
    try HIPError.check(mr_mxfp4_matmul(x.raw, x.dtype, Int32(clamping: x.shape[0]), x.rowStride, &d, y.pointer, y.dtype,
                                       y.rowStride, stream))
}

/// The same with x in MXFP4 (hipMXFP4Quantize's output) too.
public func hipMXFP4MM(quantized x: HIPMXFP4Weights, _ w: HIPMXFP4Weights, into y: HIPTensor,
                       stream: HIPStream = nil) throws {
    var dx = x.desc, dw = w.desc
    try w.needMatrix("w")
    try x.needMatrix("x", cols: dw.cols)
    try y.needRows("y", Int(dx.rows), Int(dw.rows))
    try HIPError.check(mr_mxfp4_matmul_quantized(&dx, &dw, y.pointer, y.dtype, y.rowStride, stream))
}
