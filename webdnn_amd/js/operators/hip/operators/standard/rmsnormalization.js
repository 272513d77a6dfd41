"use strict";
// RMSNormalization (ONNX opset 23) over the last axis, alone or as what the hip fusion pass makes of Add -> RMSNormalization
// (the residual's addition of a decoder block).  The reference has no such operator; it would run the chain Mul, ReduceMean,
// Add, Sqrt, Div, Mul (cpu binary7.ts:24-75, reduce.ts:369-405, unary.ts:10-32).
const { OperatorImpl } = require("../../../operatorImpl");
const { getAttrFloat, getAttrInt, broadcastMulti } = require("../../../operatorUtil");

class HipRMSNormalization extends OperatorImpl {
  // withAdd: inputs (a, b, scale) -> (a + b, normalised sum)
  constructor(withAdd) {
    super("hip");
    this.withAdd = !!withAdd;
  }

  initialize(attribute) {
    super.initialize(attribute);
    this.axis = getAttrInt(attribute, "axis", -1);
    this.epsilon = getAttrFloat(attribute, "epsilon", 1e-5);
  }

  async run(context, inputs, nOutputs) {
    context.assertsHipTensorArray(inputs);
    for (const t of inputs) if (t.dataType !== "float32") throw new Error("RMSNormalization: only float32 is supported");
    if (nOutputs !== (this.withAdd ? 2 : 1)) throw new Error("RMSNormalization: unexpected number of outputs");
    if (!this.withAdd) return [this.normalise(context, inputs[0], inputs[1], null, null)];
    const [a, b, scale] = inputs;
    if (a.ndim === b.ndim && a.dims.every((d, i) => d === b.dims[i])) {
      const sum = context.emptyTensor(a.dims, "float32");
      return [sum, this.normalise(context, a, scale, b, sum)];
    }
    // a broadcasting addend: the Add kernel, as the separate node would
    const { dims, allStrides } = broadcastMulti([a.dims, b.dims]);
    const sum = context.emptyTensor(dims, "float32");
    context.native.binary(0, 0, a.handle, b.handle, sum.handle, dims, allStrides[0], allStrides[1]);
    return [sum, this.normalise(context, sum, scale, null, null)];
  }

  normalise(context, x, scale, skip, sum) {
    let axis = this.axis;
    if (axis < 0) axis += x.ndim;
    if (axis !== x.ndim - 1 || x.ndim < 1) throw new Error("RMSNormalization: only the last axis is supported");
    const len = x.dims[axis];
    if (scale.length !== len) throw new Error("RMSNormalization: scale must have the normalised length");
    const output = context.emptyTensor(x.dims, "float32");
    context.native.rmsnorm(x.handle, skip ? skip.handle : 0, scale.handle, sum ? sum.handle : 0, output.handle, 0, 0,
      len ? x.length / len : 0, len, this.epsilon);
    return output;
  }
}

function getOpEntries() {
  return [
    { opType: "RMSNormalization", backend: "hip", opsetMin: 23, factory: () => new HipRMSNormalization(false) },
    { opType: "WebDNNHipAddRMSNorm", backend: "hip", opsetMin: 1, factory: () => new HipRMSNormalization(true) },
  ];
}
module.exports = { getOpEntries };
