'use strict';
// The Node classes of the operators behind one shared prefix, on the CPU: names, extents against device
// buffers, lifetimes.  Runs over a stand-in for the HIP runtime (tests/fake_hip.cc, preloaded), whose
// launches do nothing.
const assert = require('assert');
const path = require('path');
const pkg = require(path.join(__dirname, '..', '..', 'qwen3-embedding-webgpu-prepacked_amd', 'js'));
const { DeviceContext, RotaryPositions, PagedKvCache, SharedPrefixAttention } = pkg;

const cases = [];
function test(name, fn) { cases.push({ name, fn }); }
const TOO_FAR = { name: 'RangeError', message: /exceed the device buffer/ };

let ctx;

test('rotary positions: every tensor is held to its buffer', () => {
  ctx = new DeviceContext(0);
  const rope = new RotaryPositions(ctx);
  const q = ctx.alloc(5 * 512 * 2), k = ctx.alloc(5 * 256 * 2), out = ctx.alloc(5 * 512 * 2), at = ctx.alloc(5 * 4);
  const go = (change = {}, block = {}) => rope.run(Object.assign(
    { q: Object.assign({ x: q, heads: 4 }, block), k: { x: k, heads: 2 }, positions: at, tokens: 5 }, change));
  go();
  go({}, { out });
  go({ tokens: 0 });
  go({ tokens: 3 }, { xOffset: 2 * 1024 });
  go({ layout: 'interleaved', scaling: 'yarn', factor: 4, dtype: 'bf16', rotaryDim: 64, inverse: true });
  assert.throws(() => go({ tokens: 6 }), TOO_FAR);
  assert.throws(() => go({}, { xStride: 513 }), TOO_FAR);
  assert.throws(() => go({}, { out, outStride: 513 }), TOO_FAR);
  assert.throws(() => go({}, { xOffset: 2 }), TOO_FAR);
  assert.throws(() => go({}, { heads: 5 }), TOO_FAR);
  assert.throws(() => go({ k: { x: k, heads: 3 } }), TOO_FAR);
  assert.throws(() => go({ positionsOffset: 4 }), TOO_FAR);
  assert.throws(() => go({}, { xOffset: -2 }), { name: 'RangeError' });
  assert.throws(() => go({ layout: 'both' }), /unknown layout both/);
  assert.throws(() => go({ scaling: 'ntk' }), /unknown scaling ntk/);
  assert.throws(() => go({ dtype: 'f32' }), /unknown dtype f32/);
  assert.throws(() => go({ rotaryDim: 3 }), /qattn error -1.*rotary_dim/);
  assert.throws(() => go({ theta: 'big' }), { name: 'TypeError' });
  assert.throws(() => go({ positions: undefined }), /missing positions/);
  const handle = q.handle;
  for (const b of [q, k, out, at]) b.destroy();
  assert.throws(() => ctx.addon.rope(ctx.handle, { q: { x: handle, heads: 4 }, positions: handle, tokens: 5 }), /freed/);
});

test('the paged cache: rows and slots are held to their buffers', () => {
  for (const format of ['16bit', 'e4m3', 'int8']) {
    const cache = new PagedKvCache(ctx, { pages: 4, pageSize: 16, kvHeads: 2, headDim: 64, format });
    const k = ctx.alloc(7 * 128 * 2), v = ctx.alloc(7 * 128 * 2), slots = ctx.alloc(7 * 8);
    cache.write(k, v, slots, 7);
    cache.read(slots, 7, k, v);
    cache.write(k, v, slots, 3, { kStride: 256, kOffset: 32 });
    assert.throws(() => cache.write(k, v, slots, 8), TOO_FAR);
    assert.throws(() => cache.write(k, v, slots, 4, { vStride: 384 }), TOO_FAR);
    assert.throws(() => cache.read(slots, 7, k, v, { kOffset: 16 }), TOO_FAR);
    assert.throws(() => cache.read(slots, 7, k, v, { slotsOffset: 8 }), TOO_FAR);
    assert.throws(() => cache.read(slots, 4, k, v, { vStride: 132 }), /qattn error -1.*stride/);
    cache.desc.pages = 5;
    assert.throws(() => cache.write(k, v, slots, 7), TOO_FAR);
    cache.desc.pages = 4;
    cache.destroy();
    assert.throws(() => cache.write(k, v, slots, 7), /freed/);
    for (const b of [k, v, slots]) b.destroy();
  }
  assert.throws(() => new PagedKvCache(ctx, { pages: 1, pageSize: 16, format: 'int4' }), /unknown cache format/);
});

test('shared attention: batches and tensors are held to the buffers', () => {
  const cache = new PagedKvCache(ctx, { pages: 8, pageSize: 16, kvHeads: 2, headDim: 64, format: 'int8' });
  const q = ctx.alloc(10 * 256 * 2), o = ctx.alloc(10 * 256 * 2), rows = ctx.alloc(20 * 128 * 2);
  const attention = new SharedPrefixAttention(ctx);
  const batch = { cuSeqlens: [0, 4, 10], ownLengths: [4, 16], prefixPages: [0, 3], prefixLength: 20 };
  const options = { qHeads: 4, k: rows, v: rows };
  const make = (b = {}, change = {}) => attention.createRun(q, o, cache, Object.assign({}, batch, b), Object.assign({}, options, change));
  const run = make();
  assert.strictEqual(run.info.tokens, 10);
  assert.strictEqual(run.info.keys, 40);
  attention.encode(run);
  attention.updateRun(run, Object.assign({}, batch, { cuSeqlens: [0, 1, 2] }));
  assert.strictEqual(run.info.tokens, 2);
  const paged = make({ cuSeqlens: [0, 1], ownLengths: [33], ownPages: [1, 7, 2] });
  attention.updateRun(paged, { cuSeqlens: [0, 2], ownLengths: [40], ownPages: [1, 7, 2] });
  assert.throws(() => attention.updateRun(run, Object.assign({}, batch, { cuSeqlens: [0, 4, 11] })), TOO_FAR);
  assert.throws(() => attention.updateRun(run, Object.assign({}, batch, { ownLengths: [5, 16] })), TOO_FAR);
  assert.throws(() => attention.updateRun(run, Object.assign({}, batch, { prefixLength: 33 })), /fewer pages/);
  assert.throws(() => attention.updateRun(paged, { cuSeqlens: [0, 1], ownLengths: [33], ownPages: [1, 7] }), /fewer pages/);
  assert.throws(() => attention.updateRun(paged, { cuSeqlens: [0, 1], ownLengths: [33], ownPages: [1, 7, 8] }), /qattn error -1.*own_pages/);
  assert.throws(() => attention.updateRun(run, { cuSeqlens: [0, 1], ownLengths: [3, 4] }), { name: 'TypeError' });
  assert.throws(() => attention.updateRun(run, { cuSeqlens: [0, 1], ownLengths: [3], ownPages: [1] }), /qattn error -1.*own_pages/);
  assert.strictEqual(paged.info.keys, 40);  // the plan of before the refusals
  attention.destroyRun(paged);
  assert.throws(() => make({ cuSeqlens: [0, 5, 11] }), TOO_FAR);
  assert.throws(() => make({}, { qStride: 264 }), TOO_FAR);
  assert.throws(() => make({}, { oOffset: 16 }), TOO_FAR);
  assert.throws(() => make({}, { kStride: 136 }), TOO_FAR);
  assert.throws(() => make({}, { k: undefined, v: undefined }), /own keys need/);
  assert.throws(() => make({}, { mask: 'full' }), /unknown mask/);
  assert.throws(() => make({}, { qHeads: 3 }), /qattn error -1.*q_heads/);
  // rebinding: another cache of the geometry; a smaller buffer is refused
  const other = new PagedKvCache(ctx, { pages: 8, pageSize: 16, kvHeads: 2, headDim: 64, format: 'int8' });
  const wider = new PagedKvCache(ctx, { pages: 8, pageSize: 32, kvHeads: 2, headDim: 64, format: 'int8' });
  const small = ctx.alloc(256);
  attention.updateRun(run, batch);
  attention.rebindRun(run, q, o, other, { k: rows, v: rows });
  attention.encode(run);
  assert.throws(() => attention.rebindRun(run, small, o, other, { k: rows, v: rows }), TOO_FAR);
  // the run remembers its batch, whatever becomes of the arrays
  const cu = Int32Array.from(batch.cuSeqlens);
  attention.updateRun(run, Object.assign({}, batch, { cuSeqlens: cu }));
  cu.fill(0);
  assert.throws(() => attention.rebindRun(run, small, o, other, { k: rows, v: rows }), TOO_FAR);
  assert.throws(() => attention.rebindRun(run, q, o, other, { k: small, v: rows }), TOO_FAR);
  assert.throws(() => attention.rebindRun(run, q, o, wider, { k: rows, v: rows }), /qattn error -1/);
  // the cache of before the rebinding may go, the bound one may not
  cache.destroy();
  attention.encode(run);
  other.destroy();
  assert.throws(() => attention.encode(run), /freed/);
  attention.destroyRun(run);
  assert.throws(() => ctx.addon.encodeSharedRun(run.handle), { name: 'TypeError' });
  for (const b of [q, o, rows, small]) b.destroy();
  wider.destroy();
});

test('runs end with their context', () => {
  const cache = new PagedKvCache(ctx, { pages: 2, pageSize: 16 });
  const q = ctx.alloc(4096), o = ctx.alloc(4096);
  const attention = new SharedPrefixAttention(ctx);
  const run = attention.createRun(q, o, cache, { cuSeqlens: [0, 1], ownLengths: [1], ownPages: [1], prefixPages: [0], prefixLength: 16 });
  const foreign = new DeviceContext(0);
  assert.throws(() => new RotaryPositions(foreign).run({ q: { x: q, heads: 16 }, positions: o, tokens: 1 }), /another context/);
  foreign.destroy();
  ctx.destroy();
  assert.throws(() => attention.encode(run), /destroyed/);
  attention.destroyRun(run);
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
