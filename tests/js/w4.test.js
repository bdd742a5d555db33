'use strict';
// The Node classes of a forward with 8-bit activations, on the CPU: names, extents against device buffers, weights'
// images.  Runs over a stand-in for the HIP runtime (tests/fake_hip.cc, preloaded), whose launches do nothing.
const assert = require('assert');
const path = require('path');
const pkg = require(path.join(__dirname, '..', '..', 'qwen3-embedding-webgpu-prepacked_amd', 'js'));
const { DeviceContext, EightBitRows, FourBitMatmul, prepacked } = pkg;

const cases = [];
function test(name, fn) { cases.push({ name, fn }); }
const TOO_FAR = { name: 'RangeError', message: /exceed the device buffer/ };

let ctx;

test('rows into 8 bits: every tensor is held to its buffer', () => {
  ctx = new DeviceContext(0);
  const x = ctx.alloc(5 * 64 * 2), r = ctx.alloc(5 * 64 * 2), sum = ctx.alloc(5 * 64 * 2), weight = ctx.alloc(64 * 4);
  const rows = new EightBitRows(ctx, 5, 64);
  rows.quantize(x, 5);
  rows.quantize(x, 0);
  rows.quantize(x, 2, { xStride: 128, xOffset: 256, dtype: 'bf16' });
  rows.rmsnorm(x, weight, 5);
  rows.rmsnorm(x, weight, 5, { residual: r, sum, eps: 1e-5 });
  rows.rmsnorm(x, weight, 5, { residual: r, sum: x });
  rows.rmsnorm(x, weight, 2, { residual: r, residualStride: 128, sum: r });
  assert.throws(() => rows.quantize(x, 6), TOO_FAR);
  assert.throws(() => rows.quantize(x, 5, { xStride: 72 }), TOO_FAR);
  assert.throws(() => rows.quantize(x, 5, { xOffset: 16 }), TOO_FAR);
  assert.throws(() => rows.quantize(x, 5, { codesStride: 72 }), TOO_FAR);
  assert.throws(() => rows.quantize(x, 5, { dtype: 'f32' }), /unknown dtype f32/);
  assert.throws(() => rows.quantize(x, -1), /qattn error -1.*rows/);
  assert.throws(() => rows.quantize(x, 2, { xStride: 68 }), /qattn error -1.*stride/);
  assert.throws(() => rows.rmsnorm(x, ctx.alloc(63 * 4), 5), TOO_FAR);
  assert.throws(() => rows.rmsnorm(x, weight, 5, { residual: r, sum, sumStride: 72 }), TOO_FAR);
  assert.throws(() => rows.rmsnorm(x, weight, 5, { residual: r, residualOffset: 2, sum }), TOO_FAR);
  assert.throws(() => rows.rmsnorm(x, weight, 5, { residual: r }), /qattn error -1.*residual and sum/);
  assert.throws(() => rows.rmsnorm(x, weight, 5, { eps: 'small' }), { name: 'TypeError' });
  assert.throws(() => new EightBitRows(ctx, 5, 60).quantize(x, 5), /qattn error -1.*width/);
  x.destroy();
  assert.throws(() => rows.quantize({ handle: x.handle }, 5), { name: 'TypeError' });
  rows.destroy();
});

test('4-bit weights are laid out on the host', () => {
  const image = (kind, ...args) => ctx.addon.w4Image(kind, ...args);
  const k = 64, n = 3;
  const codes = new Uint8Array(n * k / 2).map((_, i) => (i * 37) & 255), groups = new Uint8Array(n * k / 32).fill(11 | (8 << 4));
  const scales = Float32Array.from([1, 2, -0.5]);
  const packed = image('pack', k, n, codes, groups, scales);
  assert.strictEqual(packed.length, 1024 + 64 + 64);  // one tile of 16 rows, one block of 128 columns
  // record (group g, row r): columns j and j + 16 of the group in byte j
  const code = (row, col) => (codes[row * k / 2 + (col >> 1)] >> (col & 1 ? 4 : 0)) & 15;
  for (let row = 0; row < n; row += 1)
    for (let g = 0; g < 2; g += 1)
      for (let j = 0; j < 16; j += 1)
        assert.strictEqual(packed[256 * g + 16 * row + j], code(row, 32 * g + j) | (code(row, 32 * g + j + 16) << 4));
  assert.strictEqual(packed[1024 + 4 * 2 + 1], 11 | (8 << 4));
  assert.strictEqual(new Float32Array(packed.buffer, 1024 + 64, 3)[2], -0.5);
  assert.strictEqual(image('quantize', 32, 2, new Float32Array(64).fill(1)).length, 1024 + 64 + 64);
  assert.throws(() => image('pack', 48, n, codes, groups, scales), { name: 'RangeError', message: /no 4-bit weight/ });
  assert.throws(() => image('pack', k, n, codes.subarray(1), groups, scales), { name: 'RangeError', message: /other sizes/ });
  assert.throws(() => image('pack', k, n, codes, groups), { name: 'TypeError' });
  assert.throws(() => image('pack', k, n, codes, groups.map(() => 15 | (15 << 4)), scales), /qattn error -1/);
  assert.throws(() => image('quantize', 32, 2, new Float32Array(63)), { name: 'RangeError', message: /another size/ });
  assert.throws(() => image('quantize', 32, 2, new Float32Array(64).fill(NaN)), /qattn error -1/);
  assert.throws(() => image('q4', 32, 32, new Uint8Array(639)), { name: 'RangeError', message: /fewer weights/ });
  assert.throws(() => image('q5', 32, 32, new Uint8Array(640)), { name: 'TypeError' });
  assert.throws(() => image('q4', 32, -1, new Uint8Array(640)), { name: 'TypeError' });
});

test('products: rows, weights and results are held to their buffers', () => {
  const matmul = new FourBitMatmul(ctx);
  const weight = matmul.quantize(new Float32Array(64 * 96).fill(0.5), 64, 96);
  assert.deepStrictEqual([weight.k, weight.n, weight.buffer.bytes], [64, 96, 6 * 1152]);
  const rows = new EightBitRows(ctx, 5, 64), y = ctx.alloc(5 * 96 * 2);
  matmul.run(rows, 5, weight, y);
  matmul.run(rows, 0, weight, y);
  matmul.run(rows, 4, weight, y, { yStride: 104, yOffset: 16, dtype: 'bf16' });
  assert.throws(() => matmul.run(rows, 6, weight, y), TOO_FAR);
  assert.throws(() => matmul.run(rows, 5, weight, y, { yOffset: 16 }), TOO_FAR);
  assert.throws(() => matmul.run(rows, 5, weight, y, { wBytes: 6 * 1152 + 1 }), TOO_FAR);
  assert.throws(() => matmul.run(rows, 5, weight, y, { wBytes: 6 * 1152 - 1 }), /qattn error -1.*w_bytes/);
  assert.throws(() => matmul.run(rows, 4, weight, y, { yStride: 100 }), /qattn error -1.*ldy/);
  assert.throws(() => matmul.run(new EightBitRows(ctx, 5, 32), 5, weight, y), /rows of 32 codes meet weights of 64/);
  assert.throws(() => matmul.runSwiglu(rows, 5, weight, y), /no \[gate \| up\]/);
  const both = matmul.quantize(new Float32Array(64 * 128).fill(0.5), 64, 128);
  matmul.runSwiglu(rows, 5, both, y);
  assert.throws(() => matmul.runSwiglu(rows, 5, both, y, { yStride: 56 }), /qattn error -1/);
  const foreign = new DeviceContext(0);
  assert.throws(() => new FourBitMatmul(foreign).run(rows, 5, weight, y), /another context/);
  foreign.destroy();
  // a tensor of a model file
  const q4 = new Uint8Array(2 * 32 * 18).fill(0x88);
  const part = prepacked.packQ40Tile32('t', [{ name: 't', k: 64, n: 32, bytes: q4 }]);
  const file = prepacked.buildPrepackedFile('0'.repeat(64), 1, {}, [part]);
  const model = prepacked.parsePrepackedModel(file.buffer.slice(file.byteOffset, file.byteOffset + file.byteLength));
  const t = matmul.upload(model, 't');
  assert.deepStrictEqual([t.k, t.n], [64, 32]);
  assert.throws(() => matmul.upload(model, 'u'), /no tensor u/);
  ctx.destroy();
});

(async () => {
  let failed = 0;
  for (const c of cases) {
    try {
      await c.fn();
      console.log(`ok - ${c.name}`);
    } catch (error) {
      failed += 1;
      console.log(`not ok - ${c.name}\n  ${error && error.stack}`);
    }
  }
  console.log(`${cases.length - failed}/${cases.length} passed`);
  process.exit(failed ? 1 : 0);
})();
