'use strict';
// The drafted-token operators through GPUOps: inputs and results as raw files of <dir>
// (tests/test_gpu_drafts.py).
// Usage: node tests/js/drafts.js <dir>
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
  const k = load('k'), v = load('v');
  const y = ops.attentionTree(enc, load('q'), k, v, m.nodes, m.heads, m.hd, m.prefix, load('parents'), true, m.window);
  save('y', y, m.nodes * m.heads * m.hd * 4);

  // the head in two chunks of the vocabulary; every fourth row is a node's state
  const n = m.nodes * m.heads, half = 1500;
  const E = new Uint8Array(fs.readFileSync(path.join(dir, 'E.bin')));
  const logits = ops.emptyF32(n * m.vocab);
  const x = load('x');
  for (const [at, rows] of [[0, half], [half, m.vocab - half]]) {
    const chunk = rt.uploadBytes(device, E.slice(at * m.hidden * 2, (at + rows) * m.hidden * 2));
    ops.headRows(enc, x, n, chunk, logits, at, m.vocab, rows, null, m.hidden);
  }
  const cuts = { temperature: 0.8, topK: 200, topP: 0.95 };
  const u = load('u'), states = ops.emptyF32(m.nodes * m.vocab);
  for (let j = 0; j < m.nodes; j++) {
    enc.copyBufferToBuffer(logits, j * m.heads * m.vocab * 4, states, j * m.vocab * 4, m.vocab * 4);
  }
  const { tokens, probs } = ops.sample(enc, states, m.nodes, m.vocab, u, cuts);
  save('tokens', tokens, m.nodes * 4);
  save('probs', probs, m.nodes * 4);

  ops.cacheRows(enc, [{ dst: k, src: k, width: m.hd }], load('rows'), 4, 10, m.cap);
  save('k', k, m.cap * m.hd * 4);
  let refused = '';
  try { ops.sample(enc, states, 1, m.vocab, u, { topP: 0 }); } catch (e) { refused = e.message; }
  fs.writeFileSync(path.join(dir, 'out.json'), JSON.stringify({ refused }));
}

main();
