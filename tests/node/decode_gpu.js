'use strict';
// GPU run of Sampler#project and #sampleFiltered, driven by
// tests/test_gpu_node_decode.py: reads a case directory, writes the results.
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
  const logits = s.alloc(m.rows * m.vocab * 4);
  s.project({ x: up('x.f32', Float32Array), rows: m.rows, dim: m.dim, weight: up('w.u16', Uint16Array), outDim: m.vocab, out: logits,
    adapters: { a: up('a.u16', Uint16Array), b: up('b.u16', Uint16Array), count: m.adapters, rank: m.rank },
    rowAdapter: up('which.i32', Int32Array), softcap: 30 });
  s.synchronize();
  write('logits.f32', logits.download(new Float32Array(m.rows * m.vocab)));
  const uniforms = read('u.f64', Float64Array);
  const one = s.sampleFiltered({ logits: logits, rows: m.rows, vocab: m.vocab, params: m.params[0], uniforms: uniforms, full: true });
  write('one_ids.u32', one.ids);
  write('one_probs.f64', one.probs);
  const each = s.sampleFiltered({ logits: logits, rows: m.rows, vocab: m.vocab, params: m.params, uniforms: uniforms,
    mask: read('mask.u32', Uint32Array), full: true });
  write('each_ids.u32', each.ids);
  write('each_counts.i32', each.counts);
  let refused = 0;
  for (const bad of [{ logitsType: 'f64' }, { uniforms: undefined }, { params: [{}, {}] }, { rows: m.rows + 1, uniforms: new Float64Array(m.rows + 1) },
    { mask: new Uint32Array(5) }]) {
    try { s.sampleFiltered(Object.assign({ logits: logits, rows: m.rows, vocab: m.vocab, params: {}, uniforms: uniforms }, bad)); } catch (e) { refused++; }
  }
  try { s.project({ x: logits, rows: 1, dim: 12, outDim: 4, out: logits }); } catch (e) { refused++; }
  for (const out of [s.alloc(4), undefined]) {
    try { s.project({ x: logits, rows: 2, dim: 64, weight: logits, outDim: 64, out: out }); } catch (e) { refused++; }
  }
  if (refused !== 8) throw new Error('refusals: ' + refused);
  console.log('[node] decode done');
} finally {
  s.close();
}
