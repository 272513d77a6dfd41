"use strict";
// RotaryEmbedding (ONNX opset 23): the heads of X [batch, heads, length, d] or [batch, length, heads * d] rotated by the angles of
// their tokens' positions, in one kernel.  The reference has no such operator; it would run the chain Split, Mul, Add, Concat
// (cpu split.ts:12-87, binary7.ts:24-75, concat.ts:21-84).
const { OperatorImpl } = require("../../../operatorImpl");
const { getAttrInt } = require("../../../operatorUtil");

class HipRotaryEmbedding extends OperatorImpl {
  constructor() {
    super("hip");
  }

  initialize(attribute) {
    super.initialize(attribute);
    this.interleaved = getAttrInt(attribute, "interleaved", 0);
    this.numHeads = getAttrInt(attribute, "num_heads", 0);
    this.rotary = getAttrInt(attribute, "rotary_embedding_dim", 0);
  }

  async run(context, inputs) {
    context.assertsHipTensorArray(inputs.filter((t) => t));
    const [x, cos, sin, positions] = inputs;
    for (const t of [x, cos, sin]) if (t.dataType !== "float32") throw new Error("RotaryEmbedding: only float32 is supported");
    if (positions && positions.dataType !== "int32") throw new Error("RotaryEmbedding: position_ids must be int32");
    if (x.ndim !== 3 && x.ndim !== 4) throw new Error("RotaryEmbedding: X must have 3 or 4 dimensions");
    const rows = x.ndim === 3, batch = x.dims[0], length = x.dims[rows ? 1 : 2], heads = rows ? this.numHeads : x.dims[1];
    if (rows && (heads <= 0 || x.dims[2] % heads !== 0)) throw new Error("RotaryEmbedding: num_heads must divide the last dimension of a 3-dimensional X");
    const d = rows ? x.dims[2] / heads : x.dims[3], rotary = this.rotary || d, half = rotary / 2;
    if (rotary % 2 !== 0 || rotary < 0 || rotary > d) throw new Error(`RotaryEmbedding: ${rotary} rotated elements of ${d}`);
    const table = positions ? [-1, half] : [batch, length, half];
    for (const t of [cos, sin])
      if (t.ndim !== table.length || t.dims.some((n, i) => (table[i] < 0 ? n !== cos.dims[i] : n !== table[i])))
        throw new Error(`RotaryEmbedding: cos_cache and sin_cache must be [${positions ? "positions" : `${batch}, ${length}`}, ${half}]`);
    if (positions && (positions.ndim !== 2 || positions.dims[0] !== batch || positions.dims[1] !== length))
      throw new Error(`RotaryEmbedding: position_ids must be [${batch}, ${length}]`);
    const output = context.emptyTensor(x.dims, "float32");
    if (x.length === 0) return [output];
    const rope = (offset, stride, head, c, s, p, tokens) =>
      context.native.rope(x.handle, offset, stride, head, output.handle, offset, stride, head, 0, 0, c.handle, s.handle, p ? p.handle : 0, tokens,
        heads, 0, d, rotary, half ? c.length / half : 0, this.interleaved ? 1 : 0, 0);
    if (rows) rope(0, heads * d, d, cos, sin, positions, batch * length);
    else if (batch === 1) rope(0, d, length * d, cos, sin, positions, length);
    else
      for (let b = 0; b < batch; b++) {
        // a batch's tokens are not at even distances from another's: it is a call of its own, with its own part of what is told for each token
        const part = (t, dataType, width) => {
          const own = context.emptyTensor([length * width], dataType);
          context.native.stridedCopy(t.handle, b * length * width, own.handle, 0, [length * width], [1], [1]);
          return own;
        };
        const own = positions ? [part(positions, "int32", 1)] : [part(cos, "float32", half), part(sin, "float32", half)];
        if (positions) rope(b * heads * length * d, d, length * d, cos, sin, own[0], length);
        else rope(b * heads * length * d, d, length * d, own[0], own[1], null, length);
        for (const t of own) t.dispose();
      }
    return [output];
  }
}

function getOpEntries() {
  return [{ opType: "RotaryEmbedding", backend: "hip", opsetMin: 23, factory: () => new HipRotaryEmbedding() }];
}
module.exports = { getOpEntries };
