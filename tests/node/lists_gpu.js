'use strict';
// GPU run of Sampler#sampleFiltered with allowedTokenIds, driven by
// tests/test_gpu_node_lists.py: reads a case directory, writes the results.
const assert = require('assert');
const fs = require('fs');
const path = require('path');
const sas = require(path.join(__dirname, '..', '..', 'shared_amd', 'js'));

const dir = process.argv[2];
function read(name, Type) {
  const b = fs.readFileSync(path.join(dir, name));
  const copy = new Uint8Array(b.byteLength);
  copy.set(b);
  return new Type(copy.buffer);
}
const m = JSON.parse(fs.readFileSync(path.join(dir, 'meta.json'), 'utf8'));
const s = new sas.Sampler(0);
try {
  const base = { logits: read('logits.f32', Float32Array), rows: m.rows, vocab: m.vocab, uniforms: read('u.f64', Float64Array), full: true };
  const listed = function (p, ids) { return Object.assign({}, p, { allowedTokenIds: ids }); };
  const lists = m.lists.map(function (l) { return new Uint32Array(l); });
  const run = function (name, params) {
    const out = s.sampleFiltered(Object.assign({}, base, { params: params }));
    fs.writeFileSync(path.join(dir, name + '_ids.u32'), Buffer.from(out.ids.buffer));
    fs.writeFileSync(path.join(dir, name + '_counts.i32'), Buffer.from(out.counts.buffer));
  };
  run('each', m.params.map(function (p, r) { return listed(p, lists[r]); }));
  run('shared', listed(m.params[1], lists[0]));
  run('same', m.params.map(function (p) { return listed(p, lists[0]); }));
  run('free', m.params);
  // as sampleRows: a list beside a mask, one longer than the vocabulary, one of another type
  const words = new Uint32Array(Math.ceil(m.vocab / 32)).fill(0xFFFFFFFF);
  const refused = function (opts, message) {
    assert.throws(function () { s.sampleFiltered(Object.assign({}, base, opts)); }, message);
  };
  refused({ params: listed(m.params[0], lists[0]), mask: words }, /allowedTokenIds and mask cannot both be given/);
  refused({ params: listed(m.params[0], new Uint32Array(m.vocab + 1)) }, /too many allowed token IDs/);
  refused({ params: m.params.map(function (p) { return listed(p, [1, 2]); }) }, /must be a Uint32Array/);
  console.log('[node] lists done');
} finally {
  s.close();
}
