// Grouped-query attention between its projections: QwenAttention.forward
// (Sources/ModelAdapters/Model/QwenMoEModel.swift:193-264) for many sequences at
// once, keys and values in the pages of a cache.
import CMinirunHIP

/// The rotation of heads by their tokens' positions (DeepSeekV4Attention.swift:108-165
/// for adjacent pairs, QwenMoEModel.swift:223-228 for halves): device tables f32
/// [rows, pairs], positions int32 [tokens] (nil: token t by row t).
public struct HIPHeadRotation {
    public let cos, sin: HIPTensor
    public let positions: HIPTensor?
    public let firstColumn: Int
    public let halves: Bool

    public init(cos: HIPTensor, sin: HIPTensor, positions: HIPTensor? = nil, firstColumn: Int = 0, halves: Bool = false) {
        self.cos = cos
        self.sin = sin
        self.positions = positions
        self.firstColumn = firstColumn
        self.halves = halves
    }

    /// Whole tables of one shape, and a position for each token.
    func needRotation(_ tokens: Int) throws -> mr_rotary {
        guard cos.shape.count == 2 else {
            throw HIPError(status: MR_INVALID_SHAPE, description: "cos must be [rows, pairs], got \(cos.shape)")
        }
        try cos.needWhole("cos", nil, dtype: MR_F32)
        try sin.needWhole("sin", cos.shape, dtype: MR_F32)
        try positions?.needWhole("positions", [tokens], dtype: MR_I32)
        var r = mr_rotary()
        r.cos_t = UnsafePointer(cos.pointer.assumingMemoryBound(to: Float.self))
        r.sin_t = UnsafePointer(sin.pointer.assumingMemoryBound(to: Float.self))
        r.positions = positions.map { UnsafePointer($0.pointer.assumingMemoryBound(to: Int32.self)) }
        r.table_rows = Int64(cos.shape[0])
        r.dim = Int32(clamping: 2 * cos.shape[1])
        r.col0 = Int32(clamping: firstColumn)
        r.pairs = halves ? MR_ROPE_HALVES : MR_ROPE_ADJACENT
        return r
    }
}

/// Heads [tokens, heads, dim] of the queries or keys, with their norm's weight.
public struct HIPHeads {
    public let x: HIPTensor
    public let weight: HIPTensor?
    public let out: HIPTensor
    public let dOut: HIPTensor?
    public let dWeight: HIPTensor?

    /// `dOut` and `dWeight` belong to the gradients, whose `out` is that of `x`.
    public init(_ x: HIPTensor, weight: HIPTensor?, into out: HIPTensor, dOut: HIPTensor? = nil, dWeight: HIPTensor? = nil) {
        self.x = x
        self.weight = weight
        self.out = out
        self.dOut = dOut
        self.dWeight = dWeight
    }

    /// Checked against the call's sizes, as the C call takes them.
    func needRows(_ name: String, tokens: Int, dim: Int, x xType: mr_dtype, weight weightType: mr_dtype,
                  out outType: mr_dtype, backward: Bool) throws -> mr_head_rows {
        try x.needHeads(name, tokens, nil, dim, dtype: xType)
        try out.needHeads("out", tokens, x.shape[1], dim, dtype: outType)
        try weight?.needWhole("weight", [dim], dtype: weightType)
        var a = mr_head_rows()
        a.heads = Int32(clamping: x.shape[1])
        a.x = x.raw
        a.x_token_stride = Int64(x.strides[0])
        a.x_head_stride = Int64(x.strides[1])
        a.weight = weight?.raw
        a.out = out.pointer
        a.out_token_stride = Int64(out.strides[0])
        a.out_head_stride = Int64(out.strides[1])
        guard backward else { return a }
        guard let dOut else { throw HIPError(status: MR_INVALID_ARGUMENT, description: "\(name) has no dOut") }
        try dOut.needHeads("dOut", tokens, x.shape[1], dim, dtype: xType)
        try dWeight?.needWhole("dWeight", [dim], dtype: MR_F32)
        a.d_out = dOut.raw
        a.d_out_token_stride = Int64(dOut.strides[0])
        a.d_out_head_stride = Int64(dOut.strides[1])
        a.d_weight = dWeight?.pointer.assumingMemoryBound(to: Float.self)
        return a
    }
}

private func headNormArgs(_ q: HIPHeads, _ k: HIPHeads?, eps: Float, rotation: HIPHeadRotation?,
                          backward: Bool) throws -> mr_head_norm_args {
    try q.x.needHeads("q", nil, nil, nil)
    let tokens = q.x.shape[0], dim = q.x.shape[2]
    let weightType = (q.weight ?? k?.weight)?.dtype ?? MR_F32
    var a = mr_head_norm_args()
    a.tokens = Int32(clamping: tokens)
    a.dim = Int32(clamping: dim)
    a.x_dtype = q.x.dtype
    a.weight_dtype = weightType
    a.out_dtype = q.out.dtype
    a.eps = eps
    a.q = try q.needRows("q", tokens: tokens, dim: dim, x: q.x.dtype, weight: weightType, out: q.out.dtype, backward: backward)
    if let k {
        a.k = try k.needRows("k", tokens: tokens, dim: dim, x: q.x.dtype, weight: weightType, out: q.out.dtype,
                             backward: backward)
    }
    if let rotation { a.rope = try rotation.needRotation(tokens) }
    return a
}

/// RMSNorm of every head of q and k (Normalization.swift:15-19 per head) with the
/// rotation, in one pass (QwenMoEModel.swift:223-228).
public func hipHeadNormRope(_ q: HIPHeads, _ k: HIPHeads? = nil, eps: Float, rotation: HIPHeadRotation? = nil,
                            stream: HIPStream = nil) throws {
    var args = try headNormArgs(q, k, eps: eps, rotation: rotation, backward: false)
    try HIPError.check(mr_head_norm_rope(&args, stream))
}

/// Bytes of scratch hipHeadNormRopeBackward needs.
public func hipHeadNormRopeBackwardWorkspaceSize(_ q: HIPHeads, _ k: HIPHeads? = nil, eps: Float) throws -> Int {
    var args = try headNormArgs(q, k, eps: eps, rotation: nil, backward: true)
    return mr_head_norm_rope_backward_workspace_size(&args)
}

/// The gradients of hipHeadNormRope: `out` of the inputs, `dWeight` of the weights.
public func hipHeadNormRopeBackward(_ q: HIPHeads, _ k: HIPHeads? = nil, eps: Float, rotation: HIPHeadRotation? = nil,
                                    workspace: UnsafeMutableRawPointer?, workspaceBytes: Int,
                                    stream: HIPStream = nil) throws {
    var args = try headNormArgs(q, k, eps: eps, rotation: rotation, backward: true)
    args.workspace = workspace
    args.workspace_bytes = workspaceBytes
    try HIPError.check(mr_head_norm_rope_backward(&args, stream))
}

/// One layer's keys and values in pages [pages, kvHeads, pageSize, headDim]: bf16,
/// or MXFP4 words [.., headDim / 8] with scales [.., headDim / 32].
public struct HIPKVCache {
    public let keys, values: HIPTensor
    public let keyScales, valueScales: HIPTensor?
    public var pages: Int { keys.shape[0] }
    public var kvHeads: Int { keys.shape[1] }
    public var pageSize: Int { keys.shape[2] }
    public var headDim: Int { keys.shape[3] * (keyScales == nil ? 1 : 8) }
    let desc: mr_kv_cache

    public init(keys: HIPTensor, values: HIPTensor, keyScales: HIPTensor? = nil, valueScales: HIPTensor? = nil) throws {
        guard keys.shape.count == 4, (keyScales == nil) == (valueScales == nil) else {
            throw HIPError(status: MR_INVALID_SHAPE,
                           description: "a cache is keys and values [pages, kvHeads, pageSize, headDim], both with scales or neither")
        }
        let type = keyScales == nil ? MR_BF16 : MR_U32
        try keys.needPages("keys", keys.shape, dtype: type)
        try values.needPages("values", keys.shape, dtype: type)
        var d = mr_kv_cache()
        d.k = keys.pointer
        d.v = values.pointer
        d.pages = Int32(clamping: keys.shape[0])
        d.kv_heads = Int32(clamping: keys.shape[1])
        d.page_size = Int32(clamping: keys.shape[2])
        d.head_dim = Int32(clamping: keys.shape[3] * (keyScales == nil ? 1 : 8))
        d.page_stride = Int64(keys.strides[0])
        var same = keys.shape[0] < 2 || keys.strides[0] == values.strides[0]
        if let keyScales, let valueScales {
            let shape = Array(keys.shape[0..<3]) + [keys.shape[3] / 4]
            try keyScales.needPages("keyScales", shape, dtype: MR_U8)
            try valueScales.needPages("valueScales", shape, dtype: MR_U8)
            d.k_scales = keyScales.pointer.assumingMemoryBound(to: UInt8.self)
            d.v_scales = valueScales.pointer.assumingMemoryBound(to: UInt8.self)
            d.scale_page_stride = Int64(keyScales.strides[0])
            same = same && (keys.shape[0] < 2 || keyScales.strides[0] == valueScales.strides[0])
        }
        guard same else {
            throw HIPError(status: MR_INVALID_ARGUMENT, description: "keys and values must have one page stride")
        }
        self.keys = keys
        self.values = values
        self.keyScales = keyScales
        self.valueScales = valueScales
        desc = d
    }
}

/// New tokens' keys (normalised and rotated on the way) and values into the rows
/// `slots` int32 [tokens] of the cache (QwenMoEModel.swift:193-264 keeps them whole).
public func hipKVAppend(_ cache: HIPKVCache, keys: HIPTensor, values: HIPTensor, slots: HIPTensor, normalize: Bool = false,
                        normWeight: HIPTensor? = nil, eps: Float = 1e-6, rotation: HIPHeadRotation? = nil,
                        stream: HIPStream = nil) throws {
    try keys.needHeads("keys", nil, cache.kvHeads, cache.headDim)
    let tokens = keys.shape[0]
    try values.needHeads("values", tokens, cache.kvHeads, cache.headDim, dtype: keys.dtype)
    try slots.needWhole("slots", [tokens], dtype: MR_I32)
    try normWeight?.needWhole("normWeight", [cache.headDim])
    var a = mr_kv_append_args()
    a.cache = cache.desc
    a.tokens = Int32(clamping: tokens)
    a.k = keys.raw
    a.v = values.raw
    a.dtype = keys.dtype
    a.k_token_stride = Int64(keys.strides[0])
    a.k_head_stride = Int64(keys.strides[1])
    a.v_token_stride = Int64(values.strides[0])
    a.v_head_stride = Int64(values.strides[1])
    a.slots = UnsafePointer(slots.pointer.assumingMemoryBound(to: Int32.self))
    a.normalize = normalize ? 1 : 0
    a.norm_w = normWeight?.raw
    a.norm_w_dtype = normWeight?.dtype ?? MR_F32
    a.eps = eps
    if let rotation { a.rope = try rotation.needRotation(tokens) }
    try HIPError.check(mr_kv_append(&a, stream))
}

private func attentionArgs(_ q: HIPTensor, _ cache: HIPKVCache, pageTable: HIPTensor, lengths: HIPTensor, scale: Float,
                           queryOffsets: HIPTensor?, maxLength: Int, window: Int, sinks: HIPTensor?, into out: HIPTensor,
                           lse: HIPTensor?) throws -> mr_kv_attention_args {
    try q.needHeads("q", nil, nil, cache.headDim, dtype: MR_BF16)
    try pageTable.needRows("pageTable", nil, nil, dtype: MR_I32)
    let batch = pageTable.shape[0], tokens = q.shape[0], heads = q.shape[1]
    try lengths.needWhole("lengths", [batch], dtype: MR_I32)
    try queryOffsets?.needWhole("queryOffsets", [batch + 1], dtype: MR_I32)
    try sinks?.needWhole("sinks", [heads], dtype: MR_F32)
    try out.needHeads("out", tokens, heads, cache.headDim)
    try lse?.needWhole("lse", [tokens, heads], dtype: MR_F32)
    var a = mr_kv_attention_args()
    a.cache = cache.desc
    a.batch = Int32(clamping: batch)
    a.tokens = Int32(clamping: tokens)
    a.heads = Int32(clamping: heads)
    a.q = q.raw
    a.q_token_stride = Int64(q.strides[0])
    a.q_head_stride = Int64(q.strides[1])
    a.page_table = UnsafePointer(pageTable.pointer.assumingMemoryBound(to: Int32.self))
    a.page_table_stride = pageTable.rowStride
    a.max_pages = Int32(clamping: pageTable.shape[1])
    a.kv_lens = UnsafePointer(lengths.pointer.assumingMemoryBound(to: Int32.self))
    a.q_offsets = queryOffsets.map { UnsafePointer($0.pointer.assumingMemoryBound(to: Int32.self)) }
    a.max_kv_len = Int32(clamping: maxLength)
    a.window = Int32(clamping: window)
    a.scale = scale
    a.sinks = sinks.map { UnsafePointer($0.pointer.assumingMemoryBound(to: Float.self)) }
    a.out = out.pointer
    a.out_dtype = out.dtype
    a.out_token_stride = Int64(out.strides[0])
    a.out_head_stride = Int64(out.strides[1])
    a.lse = lse?.pointer.assumingMemoryBound(to: Float.self)
    return a
}

/// Bytes of scratch hipKVAttention needs for these arguments.
public func hipKVAttentionWorkspaceSize(_ q: HIPTensor, _ cache: HIPKVCache, pageTable: HIPTensor, lengths: HIPTensor,
                                        scale: Float, queryOffsets: HIPTensor? = nil, maxLength: Int = 0, window: Int = 0,
                                        sinks: HIPTensor? = nil, into out: HIPTensor, lse: HIPTensor? = nil) throws -> Int {
    var args = try attentionArgs(q, cache, pageTable: pageTable, lengths: lengths, scale: scale, queryOffsets: queryOffsets,
                                 maxLength: maxLength, window: window, sinks: sinks, into: out, lse: lse)
    return mr_kv_attention_workspace_size(&args)
}

/// Causal attention of q [tokens, heads, headDim] over the cached keys and values
/// (QwenMoEModel.swift:193-264): sequence b has `lengths[b]` keys in the pages
/// `pageTable[b]`, and the tokens queryOffsets[b] ..< queryOffsets[b + 1] (nil: token b).
public func hipKVAttention(_ q: HIPTensor, _ cache: HIPKVCache, pageTable: HIPTensor, lengths: HIPTensor, scale: Float,
                           queryOffsets: HIPTensor? = nil, maxLength: Int = 0, window: Int = 0, sinks: HIPTensor? = nil,
                           into out: HIPTensor, lse: HIPTensor? = nil, workspace: UnsafeMutableRawPointer?,
                           workspaceBytes: Int, stream: HIPStream = nil) throws {
    var args = try attentionArgs(q, cache, pageTable: pageTable, lengths: lengths, scale: scale, queryOffsets: queryOffsets,
                                 maxLength: maxLength, window: window, sinks: sinks, into: out, lse: lse)
    args.workspace = workspace
    args.workspace_bytes = workspaceBytes
    try HIPError.check(mr_kv_attention(&args, stream))
}
