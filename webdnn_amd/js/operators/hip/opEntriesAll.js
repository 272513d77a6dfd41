"use strict";
// auto-generated by webdnn_amd/make_operator_entries.py

const { getOpEntries: getOpEntriesoperatorsstandardattention } = require("./operators/standard/attention");
const { getOpEntries: getOpEntriesoperatorsstandardbinary7 } = require("./operators/standard/binary7");
const { getOpEntries: getOpEntriesoperatorsstandardcast } = require("./operators/standard/cast");
const { getOpEntries: getOpEntriesoperatorsstandardconcat } = require("./operators/standard/concat");
const { getOpEntries: getOpEntriesoperatorsstandardconv } = require("./operators/standard/conv");
const { getOpEntries: getOpEntriesoperatorsstandardflatten } = require("./operators/standard/flatten");
const { getOpEntries: getOpEntriesoperatorsstandardgather } = require("./operators/standard/gather");
const { getOpEntries: getOpEntriesoperatorsstandardgemm } = require("./operators/standard/gemm");
const { getOpEntries: getOpEntriesoperatorsstandardglobalaveragepool } = require("./operators/standard/globalaveragepool");
const { getOpEntries: getOpEntriesoperatorsstandardlayernormalization } = require("./operators/standard/layernormalization");
const { getOpEntries: getOpEntriesoperatorsstandardmatmul } = require("./operators/standard/matmul");
const { getOpEntries: getOpEntriesoperatorsstandardmatmulfp8 } = require("./operators/standard/matmulfp8");
const { getOpEntries: getOpEntriesoperatorsstandardmaxpool } = require("./operators/standard/maxpool");
const { getOpEntries: getOpEntriesoperatorsstandardreducemean } = require("./operators/standard/reducemean");
const { getOpEntries: getOpEntriesoperatorsstandardreshape5 } = require("./operators/standard/reshape5");
const { getOpEntries: getOpEntriesoperatorsstandardrmsnormalization } = require("./operators/standard/rmsnormalization");
const { getOpEntries: getOpEntriesoperatorsstandardslice } = require("./operators/standard/slice");
const { getOpEntries: getOpEntriesoperatorsstandardsoftmax } = require("./operators/standard/softmax");
const { getOpEntries: getOpEntriesoperatorsstandardsplit } = require("./operators/standard/split");
const { getOpEntries: getOpEntriesoperatorsstandardsqueeze } = require("./operators/standard/squeeze");
const { getOpEntries: getOpEntriesoperatorsstandardtranspose } = require("./operators/standard/transpose");
const { getOpEntries: getOpEntriesoperatorsstandardunary } = require("./operators/standard/unary");
const { getOpEntries: getOpEntriesoperatorsstandardunsqueeze } = require("./operators/standard/unsqueeze");

function getOpEntries() {
  const entries = [];
  entries.push(...getOpEntriesoperatorsstandardattention());
  entries.push(...getOpEntriesoperatorsstandardbinary7());
  entries.push(...getOpEntriesoperatorsstandardcast());
  entries.push(...getOpEntriesoperatorsstandardconcat());
  entries.push(...getOpEntriesoperatorsstandardconv());
  entries.push(...getOpEntriesoperatorsstandardflatten());
  entries.push(...getOpEntriesoperatorsstandardgather());
  entries.push(...getOpEntriesoperatorsstandardgemm());
  entries.push(...getOpEntriesoperatorsstandardglobalaveragepool());
  entries.push(...getOpEntriesoperatorsstandardlayernormalization());
  entries.push(...getOpEntriesoperatorsstandardmatmul());
  entries.push(...getOpEntriesoperatorsstandardmatmulfp8());
  entries.push(...getOpEntriesoperatorsstandardmaxpool());
  entries.push(...getOpEntriesoperatorsstandardreducemean());
  entries.push(...getOpEntriesoperatorsstandardreshape5());
  entries.push(...getOpEntriesoperatorsstandardrmsnormalization());
  entries.push(...getOpEntriesoperatorsstandardslice());
  entries.push(...getOpEntriesoperatorsstandardsoftmax());
  entries.push(...getOpEntriesoperatorsstandardsplit());
  entries.push(...getOpEntriesoperatorsstandardsqueeze());
  entries.push(...getOpEntriesoperatorsstandardtranspose());
  entries.push(...getOpEntriesoperatorsstandardunary());
  entries.push(...getOpEntriesoperatorsstandardunsqueeze());
  return entries;
}

module.exports = { getOpEntries };
