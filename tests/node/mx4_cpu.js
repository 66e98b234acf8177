'use strict';
// CPU checks of the Node layer's MXFP4 calls (no GPU): a call that fails leaves no
// memory behind, and freed buffers are refused.
const assert = require('assert');
const path = require('path');
const sas = require(process.env.SAS_JS_DIR || path.join(__dirname, '..', '..', 'shared_amd', 'js'));

function buffer(bytes, freed) {
  const b = Object.create(sas.DeviceBuffer.prototype);
  b.bytes = bytes;
  b.ptr = freed ? null : 4096n;
  b.free = function () { this.ptr = null; };
  return b;
}

// A sampler without a device: `room` allocations succeed, the next one throws;
// calls into the library throw (there is no handle).
function fake(room) {
  const s = Object.create(sas.Sampler.prototype);
  s.made = [];
  s._idle = function () { return null; };
  s._handle = function () { return null; };
  s.alloc = function (bytes) {
    if (s.made.length === room) throw new Error('out of device memory');
    s.made.push(buffer(bytes));
    return s.made[s.made.length - 1];
  };
  return s;
}
const left = function (s) { return s.made.filter(function (b) { return b.ptr !== null; }).length; };

{
  const s = fake(1);
  assert.throws(function () { s.allocMx4(4, 64); }, /out of device memory/);
  assert.strictEqual(left(s), 0);
  console.log('ok a table whose scales find no room frees its codes');
}
{
  const s = fake(10);
  assert.throws(function () { s.quantizeMx4({ x: buffer(1024), rows: 4, dim: 64 }); });
  assert.strictEqual(s.made.length, 2);
  assert.strictEqual(left(s), 0);
  const out = s.allocMx4(4, 64);
  assert.throws(function () { s.quantizeMx4({ x: buffer(1024), rows: 4, dim: 64, out: out }); });
  assert.strictEqual(left(s), 2);
  console.log('ok a quantisation that fails frees the table it made, and no other');
}
{
  const s = fake(10), table = s.allocMx4(8, 64);
  const freed = /freed/;
  assert.throws(function () { s.lookupMx4({ table: table, ids: buffer(16, true), rows: 4, out: buffer(1024) }); }, freed);
  assert.throws(function () { s.lookupMx4({ table: table, rows: 4, out: buffer(1024, true) }); }, freed);
  assert.throws(function () { s.quantizeMx4({ x: buffer(1024, true), rows: 4, dim: 64 }); }, freed);
  assert.throws(function () { s.projectMx4({ x: buffer(1024, true), rows: 4, weight: table, out: buffer(128) }); }, freed);
  table.free();
  assert.throws(function () { s.lookupMx4({ table: table, ids: buffer(16), rows: 4, out: buffer(1024) }); }, freed);
  assert.throws(function () { s.projectMx4({ x: buffer(1024), rows: 4, weight: table, out: buffer(128) }); }, freed);
  assert.throws(function () { s.projectMx4({ x: table, rows: 4, weight: s.allocMx4(8, 64), out: buffer(128) }); }, freed);
  const head = { hidden: buffer(1024), weight: table, dim: 64, format: 'mx4' };
  assert.throws(function () { s._describeHead({ rows: 1, vocab: 8, head: head }); }, freed);
  console.log('ok freed buffers and tables are refused');
}
