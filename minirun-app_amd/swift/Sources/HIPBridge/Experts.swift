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

    var rowMap: UnsafePointer<Int32> { UnsafePointer(rowOfPair.pointer.assumingMemoryBound(to: Int32.self)) }
}

/// Bytes of scratch hipExpertSort needs.
public func hipExpertSortWorkspaceSize(tokens: Int, perToken: Int, experts: Int) -> Int {
    mr_expert_sort_workspace_size(Int32(tokens), Int32(perToken), Int32(experts))
}

/// The stable order of the router's ids [tokens, perToken] by expert, into
/// `order` (QwenExpertBackends.swift:77-260 loops over them instead).
public func hipExpertSort(_ ids: HIPTensor, into order: HIPExpertOrder, workspace: UnsafeMutableRawPointer?,
                          workspaceBytes: Int, stream: HIPStream = nil) throws {
    let int32 = { (t: HIPTensor) in t.pointer.assumingMemoryBound(to: Int32.self) }
    try HIPError.check(mr_expert_sort(UnsafePointer(int32(ids)), Int32(order.tokens), Int32(order.perToken),
                                      Int32(order.experts), int32(order.offsets), int32(order.pairOfRow),
                                      int32(order.rowOfPair), workspace, workspaceBytes, stream))
}

/// The tokens' rows in expert order.
public func hipExpertDispatch(_ x: HIPTensor, _ order: HIPExpertOrder, into rows: HIPTensor,
                              stream: HIPStream = nil) throws {
    try HIPError.check(mr_expert_dispatch(x.raw, x.dtype, Int32(order.tokens), Int64(x.shape[1]), Int64(x.strides[0]),
                                          order.rowMap, Int32(order.perToken), rows.pointer, Int64(rows.strides[0]),
                                          stream))
}

/// Each token's rows summed with the router's weights f32 [tokens, perToken]
/// (nil: ones, which is the gradient of hipExpertDispatch).
public func hipExpertCombine(_ rows: HIPTensor, _ order: HIPExpertOrder, weights: HIPTensor?, into out: HIPTensor,
                             stream: HIPStream = nil) throws {
    let w = weights.map { UnsafePointer($0.pointer.assumingMemoryBound(to: Float.self)) }
    try HIPError.check(mr_expert_combine(rows.raw, rows.dtype, Int64(rows.strides[0]), Int64(rows.shape[1]),
                                         order.rowMap, w, Int32(order.tokens), Int32(order.perToken), out.pointer,
                                         Int64(out.strides[0]), stream))
}

/// Gradients of hipExpertCombine: of the rows, and of the weights (nil: not
/// asked for).
public func hipExpertCombineBackward(_ dOut: HIPTensor, rows: HIPTensor, _ order: HIPExpertOrder, weights: HIPTensor?,
                                     dRows: HIPTensor?, dWeights: HIPTensor?, stream: HIPStream = nil) throws {
    let w = weights.map { UnsafePointer($0.pointer.assumingMemoryBound(to: Float.self)) }
    let dw = dWeights.map { $0.pointer.assumingMemoryBound(to: Float.self) }
    try HIPError.check(mr_expert_combine_backward(dOut.raw, dOut.dtype, Int64(dOut.strides[0]), Int64(dOut.shape[1]),
                                                  rows.raw, Int64(rows.strides[0]), order.rowMap, w,
                                                  Int32(order.tokens), Int32(order.perToken), dRows?.pointer,
                                                  Int64(dRows?.strides[0] ?? 0), dw, stream))
}

/// Each expert's rows times its own matrix of the stack `w`
/// (QwenExpertBackends.swift:143,244 multiply token by token): x is one bf16 or
/// f32 row per token, or per row of the order with `sortedRows`.
public func hipMXFP4ExpertMM(_ x: HIPTensor, _ w: HIPMXFP4Weights, _ order: HIPExpertOrder, sortedRows: Bool = false,
                             into y: HIPTensor, stream: HIPStream = nil) throws {
    var a = mr_mxfp4_expert_args()
    a.x = x.raw
    a.x_dtype = x.dtype
    a.x_stride = Int64(x.strides[0])
    a.x_rows = Int32(x.shape[0])
    try hipExpertMM(&a, w, order, sortedRows: sortedRows, into: y, stream: stream)
}

/// The same with x in MXFP4 (hipMXFP4Quantize's output).
public func hipMXFP4ExpertMM(quantized x: HIPMXFP4Weights, _ w: HIPMXFP4Weights, _ order: HIPExpertOrder,
                             sortedRows: Bool = false, into y: HIPTensor, stream: HIPStream = nil) throws {
    var a = mr_mxfp4_expert_args()
    a.x = UnsafeRawPointer(x.desc.packed)
    a.x_dtype = MR_U32
    a.x_scales = x.desc.scales
    a.x_rows = Int32(x.desc.rows)
    try hipExpertMM(&a, w, order, sortedRows: sortedRows, into: y, stream: stream)
}

private func hipExpertMM(_ a: inout mr_mxfp4_expert_args, _ w: HIPMXFP4Weights, _ order: HIPExpertOrder,
                         sortedRows: Bool, into y: HIPTensor, stream: HIPStream) throws {
    guard w.experts == order.experts else {
        throw HIPError(status: MR_INVALID_SHAPE,
                       description: "the weight has \(w.experts ?? 0) experts, the order \(order.experts)")
    }
    a.w = w.desc
    a.experts = Int32(order.experts)
    a.offsets = UnsafePointer(order.offsets.pointer.assumingMemoryBound(to: Int32.self))
    a.pair_of_row = sortedRows ? nil : UnsafePointer(order.pairOfRow.pointer.assumingMemoryBound(to: Int32.self))
    a.per_token = Int32(order.perToken)
    a.rows = Int32(order.tokens * order.perToken)
    a.y = y.pointer
    a.y_dtype = y.dtype
    a.y_stride = Int64(y.strides[0])
    try HIPError.check(mr_mxfp4_expert_matmul(&a, stream))
}
