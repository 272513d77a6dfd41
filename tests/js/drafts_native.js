"use strict";
// A step with drafted tokens through the N-API functions, as a JavaScript serving program would take it: queries and keys turned, appended, attended to as
// trees, verified, the accepted ones kept:
//   node drafts_native.js case.json out.bin   (out.bin: turned queries, attention's result, turned keys, the scales)
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
const ints = (a) => up(Int32Array.from(a)), floats = (a) => up(Float32Array.from(a));
const down = (h, n, Type) => {
  const a = new Type(n);
  native.read(h, 0, a);
  return a;
};
const cells = c.pages * c.kvHeads, d = c.d, width = (c.heads + 2 * c.kvHeads) * d, keys = c.kvHeads * d;
const kPages = up(new Uint8Array(cells * 64 * d).fill(0x7f)), vPages = up(new Uint8Array(cells * 64 * d).fill(0x7f));
const kScales = up(new Float32Array(cells).fill(1)), vScales = up(new Float32Array(cells).fill(1));
const table = ints(c.table), lens = ints(c.past), starts = ints(c.starts), positions = ints(c.positions), x = floats(c.x), cos = floats(c.cos), sin = floats(c.sin);
const cache = [kPages, kScales, vPages, vScales, table, lens];
const old = floats(c.old), oldTokens = c.oldStarts[c.seqs];
native.cacheAppend(old, 0, 2 * keys, old, keys, 2 * keys, ...cache, ints(c.oldStarts), c.seqs, oldTokens, c.kvHeads, d, c.pages, c.maxPages);
native.write(lens, 0, Int32Array.from(c.past.map((n, s) => n + c.starts[s + 1] - c.starts[s])));
const q = native.alloc(c.tokens * c.heads * d * 4), k = native.alloc(c.tokens * keys * 4), y = native.alloc(c.tokens * c.heads * d * 4);
native.rope(x, 0, width, d, q, 0, c.heads * d, d, 0, 0, cos, sin, positions, c.tokens, c.heads, 0, d, d, c.rows, 0, 0);
native.rope(x, c.heads * d, width, d, k, 0, keys, d, 0, 0, cos, sin, positions, c.tokens, c.kvHeads, 0, d, d, c.rows, 0, 0);
native.cacheAppendRope(x, c.heads * d, width, x, c.heads * d + keys, width, ...cache, starts, 0, cos, sin, positions, c.seqs, c.tokens, c.kvHeads, d, c.pages,
  c.maxPages, d, c.rows, 0, 0);
const mask = ints(c.mask);
const attend = (dim) => native.cacheAttentionTree(q, 0, c.heads * d, ...cache, starts, mask, y, c.seqs, c.tokens, c.heads, c.kvHeads, dim, c.pages, c.maxPages,
  c.words, c.alpha);
attend(d);
const next = native.alloc(c.seqs * 4), count = native.alloc(c.seqs * 4), taken = native.alloc(c.tokens * 4);
native.verifyDrafts(floats(c.p), 0, ints(c.drafted), ints(c.parents), floats(c.uniform), starts, next, count, taken, c.seqs, c.tokens, c.vocab);
native.cacheKeep(...cache, starts, taken, count, c.seqs, c.tokens, c.kvHeads, d, c.pages, c.maxPages);
const parts = [down(q, c.tokens * c.heads * d, Float32Array), down(y, c.tokens * c.heads * d, Float32Array), down(k, c.tokens * keys, Float32Array),
  down(kScales, cells, Float32Array), down(vScales, cells, Float32Array)];
fs.writeFileSync(process.argv[3], Buffer.concat(parts.map((a) => Buffer.from(a.buffer))));
let refused = "";
try {
  attend(48);
} catch (error) {
  refused = error.message;
}
const list = (h, n) => Array.from(down(h, n, Int32Array));
console.log(JSON.stringify({ refused, next: list(next, c.seqs), count: list(count, c.seqs), path: list(taken, c.tokens) }));
