'use strict';
// CPU checks of the Node layer's MXFP4 calls (no GPU): a call that fails leaves no
// memory behind.
const assert = require('assert');
const path = require('path');
const sas = require(process.env.SAS_JS_DIR || path.join(__dirname, '..', '..', 'shared_amd', 'js'));

function buffer(bytes) {
  const b = Object.create(sas.DeviceBuffer.prototype);
  b.bytes = bytes;
  b.ptr = 4096n;
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
