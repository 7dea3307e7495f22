// Tokens in expert order and back, around products of all of an expert's rows
// at once; the reference runs its experts token by token
// (Sources/ModelAdapters/Loading/QwenExpertBackends.swift:77-260).
import CMinirunHIP

/// Pairs (token, slot) by expert: offsets [experts + 1], pairOfRow
/// [tokens * perToken], rowOfPair [tokens, perToken], all int32; -1 is none.
public struct HIPExpertOrder {
    public let offsets, pairOfRow, rowOfPair: HIPTensor
    public let experts: Int
    public var tokens: Int { rowOfPair.shape[0] }
    public var perToken: Int { rowOfPair.shape[1] }

    public init(offsets: HIPTensor, pairOfRow: HIPTensor, rowOfPair: HIPTensor, experts: Int) {
        self.offsets = offsets
        self.pairOfRow = pairOfRow
        self.rowOfPair = rowOfPair
        self.experts = experts
    }

    var pairs: Int { tokens * perToken }

    /// Whole int32 tensors of sizes that belong together.
    func needOrder() throws {
        guard rowOfPair.shape.count == 2, experts > 0 else {
            throw HIPError(status: MR_INVALID_SHAPE,
                           description: "rowOfPair must be [tokens, perToken] of one expert or more, got \(rowOfPair.shape) of \(experts)")
        }
        try rowOfPair.needWhole("rowOfPair", nil, dtype: MR_I32)
        try pairOfRow.needWhole("pairOfRow", [pairs], dtype: MR_I32)
        try offsets.needWhole("offsets", [experts + 1], dtype: MR_I32)
    }

    var rowMap: UnsafePointer<Int32> { UnsafePointer(rowOfPair.pointer.assumingMemoryBound(to: Int32.self)) }
}

/// Bytes of scratch hipExpertSort needs.
public func hipExpertSortWorkspaceSize(tokens: Int, perToken: Int, experts: Int) -> Int {
    mr_expert_sort_workspace_size(Int32(clamping: tokens), Int32(clamping: perToken), Int32(clamping: experts))
}

/// The stable order of the router's ids [tokens, perToken] by expert, into
/// `order` (QwenExpertBackends.swift:77-260 loops over them instead).
public func hipExpertSort(_ ids: HIPTensor, into order: HIPExpertOrder, workspace: UnsafeMutableRawPointer?,
                          workspaceBytes: Int, stream: HIPStream = nil) throws {
    try order.needOrder()
    try ids.needWhole("ids", [order.tokens, order.perToken], dtype: MR_I32)
    let int32 = { (t: HIPTensor) in t.pointer.assumingMemoryBound(to: Int32.self) }
    try HIPError.check(mr_expert_sort(UnsafePointer(int32(ids)), Int32(clamping: order.tokens),
                                      Int32(clamping: order.perToken), Int32(clamping: order.experts),
                                      int32(order.offsets), int32(order.pairOfRow), int32(order.rowOfPair), workspace,
                                      workspaceBytes, stream))
}

/// The tokens' rows in expert order.
public func hipExpertDispatch(_ x: HIPTensor, _ order: HIPExpertOrder, into rows: HIPTensor,
                              stream: HIPStream = nil) throws {
    try order.needOrder()
    try x.needRows("x", order.tokens, nil)
    try rows.needRows("rows", order.pairs, x.shape[1], dtype: x.dtype)
    try HIPError.check(mr_expert_dispatch(x.raw, x.dtype, Int32(clamping: order.tokens), Int64(x.shape[1]), x.rowStride,
                                          order.rowMap, Int32(clamping: order.perToken), rows.pointer, rows.rowStride,
                                          stream))
}

/// Each token's rows summed with the router's weights f32 [tokens, perToken]
/// (nil: ones, which is the gradient of hipExpertDispatch).
public func hipExpertCombine(_ rows: HIPTensor, _ order: HIPExpertOrder, weights: HIPTensor?, into out: HIPTensor,
                             stream: HIPStream = nil) throws {
    try order.needOrder()
    try rows.needRows("rows", order.pairs, nil)
    try out.needRows("out", order.tokens, rows.shape[1], dtype: rows.dtype)
    try weights?.needWhole("weights", [order.tokens, order.perToken], dtype: MR_F32)
    let w = weights.map { UnsafePointer($0.pointer.assumingMemoryBound(to: Float.self)) }
    try HIPError.check(mr_expert_combine(rows.raw, rows.dtype, rows.rowStride, Int64(rows.shape[1]), order.rowMap, w,
                                         Int32(clamping: order.tokens), Int32(clamping: order.perToken), out.pointer,
                                         out.rowStride, stream))
}

/// Gradients of hipExpertCombine: of the rows, and of the weights (nil: not
/// asked for).
public func hipExpertCombineBackward(_ dOut: HIPTensor, rows: HIPTensor, _ order: HIPExpertOrder, weights: HIPTensor?,
                                     dRows: HIPTensor?, dWeights: HIPTensor?, stream: HIPStream = nil) throws {
    try order.needOrder()
    try dOut.needRows("dOut", order.tokens, nil)
    try rows.needRows("rows", order.pairs, dOut.shape[1], dtype: dOut.dtype)
    try weights?.needWhole("weights", [order.tokens, order.perToken], dtype: MR_F32)
    try dRows?.needRows("dRows", order.pairs, dOut.shape[1], dtype: dOut.dtype)
    try dWeights?.needWhole("dWeights", [order.tokens, order.perToken], dtype: MR_F32)
    let w = weights.map { UnsafePointer($0.pointer.assumingMemoryBound(to: Float.self)) }
    let dw = dWeights.map { $0.pointer.assumingMemoryBound(to: Float.self) }
    try HIPError.check(mr_expert_combine_backward(dOut.raw, dOut.dtype, dOut.rowStride, Int64(dOut.shape[1]), rows.raw,
                                                  rows.rowStride, order.rowMap, w, Int32(clamping: order.tokens),
                                                  Int32(clamping: order.perToken), dRows?.pointer,
                                                  dRows?.rowStride ?? 0, dw, stream))
}

/// Each expert's rows times its own matrix of the stack `w`
/// (QwenExpertBackends.swift:143,244 multiply token by token): x is one bf16 or
/// f32 row per token, or per row of the order with `sortedRows`.
public func hipMXFP4ExpertMM(_ x: HIPTensor, _ w: HIPMXFP4Weights, _ order: HIPExpertOrder, sortedRows: Bool = false,
                             into y: HIPTensor, stream: HIPStream = nil) throws {
    try order.needOrder()
    try x.needRows("x", sortedRows ? order.pairs : order.tokens, Int(w.desc.cols))
    var a = mr_mxfp4_expert_args()
    a.x = x.raw
    a.x_dtype = x.dtype
    a.x_stride = x.rowStride
    a.x_rows = Int32(clamping: x.shape[0])
    try hipExpertMM(&a, w, order, sortedRows: sortedRows, into: y, stream: stream)
}

/// The same with x in MXFP4 (hipMXFP4Quantize's output).
public func hipMXFP4ExpertMM(quantized x: HIPMXFP4Weights, _ w: HIPMXFP4Weights, _ order: HIPExpertOrder,
                             sortedRows: Bool = false, into y: HIPTensor, stream: HIPStream = nil) throws {
    try order.needOrder()
    try x.needMatrix("x", cols: w.desc.cols)
    var a = mr_mxfp4_expert_args()
    a.x = UnsafeRawPointer(x.desc.packed)
    a.x_dtype = MR_U32
    a.x_scales = x.desc.scales
    a.x_rows = Int32(clamping: x.desc.rows)
    try hipExpertMM(&a, w, order, sortedRows: sortedRows, into: y, stream: stream)
}

private func hipExpertMM(_ a: inout mr_mxfp4_expert_args, _ w: HIPMXFP4Weights, _ order: HIPExpertOrder,
                         sortedRows: Bool, into y: HIPTensor, stream: HIPStream) throws {
    guard w.experts == order.experts else {
        throw HIPError(status: MR_INVALID_SHAPE,
                       description: "the weight has \(w.experts ?? 0) experts, the order \(order.experts)")
    }
    try y.needRows("y", order.pairs, Int(w.desc.rows))
    a.w = w.desc
    a.experts = Int32(clamping: order.experts)
    a.offsets = UnsafePointer(order.offsets.pointer.assumingMemoryBound(to: Int32.self))
    a.pair_of_row = sortedRows ? nil : UnsafePointer(order.pairOfRow.pointer.assumingMemoryBound(to: Int32.self))
    a.per_token = Int32(clamping: order.perToken)
    a.rows = Int32(clamping: order.pairs)
    a.y = y.pointer
    a.y_dtype = y.dtype
    a.y_stride = y.rowStride
    try HIPError.check(mr_mxfp4_expert_matmul(&a, stream))
}
