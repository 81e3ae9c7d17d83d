'use strict';
// The operators of long caches through GPUOps: inputs and results as raw files of <dir>
// (tests/test_gpu_long_cache.py).
// Usage: node tests/js/long_cache.js <dir>
const fs = require('fs');
const path = require('path');
const rt = require('../../gemma4-js_amd/node/hip-runtime.js');

function main() {
  const dir = process.argv[2];
  const m = JSON.parse(fs.readFileSync(path.join(dir, 'meta.json'), 'utf8'));
  const device = rt.requestDevice(0);
  const load = (n) => rt.uploadBytes(device, new Uint8Array(fs.readFileSync(path.join(dir, `${n}.bin`))));
  const save = (n, buffer, bytes) => fs.writeFileSync(path.join(dir, `${n}.out`), Buffer.from(buffer.read(0, bytes)));
  const ops = new rt.GPUOps(device);
  const enc = device.createCommandEncoder();
  const k = load('k'), q = load('q');
  const cache = ops.kv4Cache(m.len, m.hd);
  ops.kv4Append(enc, cache, k, load('v'), m.len, 0);
  const weights = ops.emptyF32(m.len);
  save('y', ops.attentionKv4(enc, q, cache, m.rows, m.heads, m.len, m.len - m.rows, false, 0, weights), m.rows * m.heads * m.hd * 4);
  ops.attentionWeights(enc, q, k, m.rows, m.heads, m.hd, m.len, m.len - m.rows, false, 0, weights);
  save('weights', weights, m.len * 4);
  const rows = ops.cacheEvict(enc, weights, 1, m.len, m.keep, 2, 10);
  ops.cacheRows(enc, ops.kv4Planes(cache), rows, m.keep, 0, m.len);
  save('rows', rows, m.keep * 4);
  save('kept', weights, m.len * 4);
  const back = ops.kv4Read(enc, cache, 0, m.keep);
  save('kback', back.k, m.keep * m.hd * 4);
  save('vback', back.v, m.keep * m.hd * 4);
  let refused = '';
  try { ops.cacheEvict(enc, weights, 1, m.len, 5, 3, 3); } catch (e) { refused = e.message; }
  fs.writeFileSync(path.join(dir, 'out.json'), JSON.stringify({ refused }));
}

main();
