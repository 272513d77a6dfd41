"use strict";
// Appends to a cache and attends over it through the N-API functions, as a JavaScript serving program would:
//   node cache_native.js case.json out.bin      (case.json: sizes and the operands' values; out.bin: the result, then the scales)
const fs = require("fs");
const path = require("path");
const native = require(path.join(__dirname, "..", "..", "webdnn_amd", "lib", "webdnn_hip.node"));

const c = JSON.parse(fs.readFileSync(process.argv[2], "utf-8"));
native.init(0);
const up = (data) => {
  const h = native.alloc(data.byteLength);
  native.write(h, 0, data);
  return h;
};
const cells = c.pages * c.kvHeads;
const kPages = up(new Uint8Array(cells * 64 * c.d).fill(0x7f)), vPages = up(new Uint8Array(cells * 64 * c.d).fill(0x7f));
const kScales = up(new Float32Array(cells).fill(1)), vScales = up(new Float32Array(cells).fill(1));
const table = up(Int32Array.from(c.table)), lens = up(Int32Array.from(c.lens)), starts = up(Int32Array.from(c.starts));
const q = up(Float32Array.from(c.q)), kv = up(Float32Array.from(c.kv));
const width = c.kvHeads * c.d, y = native.alloc(c.tokens * c.heads * c.d * 4);
native.cacheAppend(kv, 0, 2 * width, kv, width, 2 * width, kPages, kScales, vPages, vScales, table, lens, starts, c.seqs, c.tokens, c.kvHeads, c.d, c.pages, c.maxPages);
native.cacheAttention(q, 0, c.heads * c.d, kPages, kScales, vPages, vScales, table, lens, starts, y, c.seqs, c.tokens, c.heads, c.kvHeads, c.d, c.pages, c.maxPages, c.alpha);
const out = new Float32Array(c.tokens * c.heads * c.d), ks = new Float32Array(cells), vs = new Float32Array(cells);
native.read(y, 0, out);
native.read(kScales, 0, ks);
native.read(vScales, 0, vs);
fs.writeFileSync(process.argv[3], Buffer.concat([out, ks, vs].map((a) => Buffer.from(a.buffer))));
let refused = "";
try {
  native.cacheAttention(q, 0, c.heads * c.d, kPages, kScales, vPages, vScales, table, lens, starts, y, c.seqs, c.tokens, c.heads, c.kvHeads, 48, c.pages, c.maxPages, c.alpha);
} catch (error) {
  refused = error.message;
}
console.log(JSON.stringify({ refused }));
