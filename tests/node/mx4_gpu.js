'use strict';
// GPU run of the Node layer's MXFP4 calls, driven by tests/test_gpu_node_mx4.py:
// reads a case directory, writes the results.
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
function write(name, typed) {
  fs.writeFileSync(path.join(dir, name), Buffer.from(typed.buffer, typed.byteOffset, typed.byteLength));
}
const m = JSON.parse(fs.readFileSync(path.join(dir, 'meta.json'), 'utf8'));
const s = new sas.Sampler(0);
try {
  const up = function (name, Type) { const a = read(name, Type); return s.alloc(a.byteLength).upload(a); };
  const x = up('x.f32', Float32Array);
  const head = s.quantizeMx4({ x: up('w.u16', Uint16Array), xType: 'bf16', rows: m.vocab, dim: m.dim });
  const x4 = s.quantizeMx4({ x: x, rows: m.rows, dim: m.dim, out: s.allocMx4(m.rows, m.dim) });
  const logits = s.alloc(m.rows * m.vocab * 4);
  const out = function (name) { s.synchronize(); write(name, logits.download(new Float32Array(m.rows * m.vocab))); };
  s.projectMx4({ x: x, rows: m.rows, weight: head, out: logits, softcap: 30 });
  out('wide.f32');
  s.projectMx4({ x: x4, rows: m.rows, weight: head, out: logits });
  s.projectMx4({ x: x4, rows: m.rows, weight: head, out: logits, accumulate: true });
  out('twice.f32');
  const rows = s.alloc(m.ids * m.dim * 4);
  s.lookupMx4({ table: head, ids: up('ids.u32', Uint32Array), rows: m.ids, out: rows });
  s.synchronize();
  write('rows.f32', rows.download(new Float32Array(m.ids * m.dim)));
  const uniforms = read('u.f64', Float64Array);
  const r = s.lmHeadSample({ rows: m.rows, vocab: m.vocab, params: { temperature: 0.9, topK: 40, topP: 0.95 }, uniforms: uniforms,
    head: { hidden: x, weight: head, dim: m.dim, format: 'mx4' } });
  write('ids.out', r.ids);
  const steps = function (vocab) {
    return s.decodeStepsWithHead({ rows: m.rows, vocab: vocab, k: 2, params: { temperature: 0 }, hidden: function () { return x; },
      head: { weight: head, dim: m.dim, format: 'mx4' } });
  };
  write('greedy.out', Uint32Array.from(steps(m.vocab).map(function (row) { return row.ids[1]; })));
  let refused = 0;
  for (const f of [
    function () { s.quantizeMx4({ x: x, xType: 'f64', rows: 1, dim: 8 }); },
    function () { s.quantizeMx4({ x: x, rows: m.rows + 1, dim: m.dim }); },
    function () { s.quantizeMx4({ x: x, rows: m.rows, dim: m.dim, out: s.allocMx4(1, m.dim) }); },
    function () { s.lookupMx4({ table: head, rows: m.vocab + 1, out: s.alloc((m.vocab + 1) * m.dim * 4) }); },
    function () { s.lookupMx4({ table: head, rows: 2, out: s.alloc(4) }); },
    function () { s.projectMx4({ x: x, xType: 'f16', rows: 1, weight: head, out: logits }); },
    function () { s.projectMx4({ x: x, rows: 1, weight: logits, out: logits }); },
    function () { s.projectMx4({ x: s.allocMx4(1, 32), rows: 1, weight: head, out: logits }); },
    function () { s.projectMx4({ x: x, rows: m.rows, weight: head, out: s.alloc(16) }); },
    function () { s.lmHeadSample({ rows: 1, vocab: m.vocab, params: {}, head: { hidden: x, weight: logits, dim: m.dim, format: 'mx4' } }); },
    function () { s.lmHeadSample({ rows: 1, vocab: m.vocab + 1, params: {}, head: { hidden: x, weight: head, dim: m.dim, format: 'mx4' } }); },
    function () { steps(m.vocab + 1); },
  ]) {
    try { f(); } catch (e) { refused++; }
  }
  if (refused !== 12) throw new Error('refusals: ' + refused);
  console.log('[node] mx4 done');
} finally {
  s.close();
}
