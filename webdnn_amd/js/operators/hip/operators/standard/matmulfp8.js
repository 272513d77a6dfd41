"use strict";
// WebDNNHipMatMulFp8: a linear layer whose weights are held in 8 bits.  Inputs: X float32 [..., k]; W float8e4m3fn [n, k] (an
// initializer of ONNX type FLOAT8E4M3FN) with WScale float32 [ceil(n/128), ceil(k/128)], one scale for each 128 x 128 block;
// optionally a bias [n].  X is quantised in blocks of 1 x 128 on the way.  Attribute activation: "" or "Relu".
// The reference has no 8-bit operators; its MatMul is cpu matmul.ts:11-111.
const { OperatorImpl } = require("../../../operatorImpl");
const { getAttrString } = require("../../../operatorUtil");

const BLOCK = 128;
const blocks = (n) => Math.ceil(n / BLOCK);

class HipMatMulFp8 extends OperatorImpl {
  constructor() {
    super("hip");
  }

  initialize(attribute) {
    super.initialize(attribute);
    this.activation = getAttrString(attribute, "activation", "");
    if (this.activation !== "" && this.activation !== "Relu") throw new Error(`MatMulFp8: unknown activation ${this.activation}`);
  }

  async run(context, inputs) {
    context.assertsHipTensorArray(inputs);
    const [x, w, wScale, bias] = inputs;
    if (w.dataType !== "float8e4m3fn") throw new Error("MatMulFp8: the weights must be float8e4m3fn");
    for (const t of [x, wScale, bias]) if (t && t.dataType !== "float32") throw new Error("MatMulFp8: only float32 is supported");
    if (w.ndim !== 2 || x.ndim < 1 || x.dims[x.ndim - 1] !== w.dims[1]) throw new Error("MatMulFp8: inner dimensions differ");
    const [n, k] = w.dims, m = k ? x.length / k : x.dims.slice(0, -1).reduce((a, b) => a * b, 1);
    if (wScale.ndim !== 2 || wScale.dims[0] !== blocks(n) || wScale.dims[1] !== blocks(k)) throw new Error("MatMulFp8: one scale for each 128 x 128 block of the weights");
    if (bias && bias.length !== n) throw new Error("MatMulFp8: bias must have an element for each column");
    const q = context.emptyTensor([m, k], "float8e4m3fn"), scale = context.emptyTensor([m, blocks(k)], "float32");
    try {
      context.native.quantizeFp8(x.handle, q.handle, scale.handle, m, k, 1);
      const output = context.emptyTensor(x.dims.slice(0, -1).concat([n]), "float32");
      context.native.gemmFp8(q.handle, scale.handle, w.handle, wScale.handle, bias ? bias.handle : 0, output.handle, m, n, k,
        this.activation === "Relu" ? 1 : 0, 0);
      return [output];
    } finally {
      q.dispose();
      scale.dispose();
    }
  }
}

function getOpEntries() {
  return [{ opType: "WebDNNHipMatMulFp8", backend: "hip", opsetMin: 1, factory: () => new HipMatMulFp8() }];
}
module.exports = { getOpEntries };
