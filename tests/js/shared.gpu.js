'use strict';
// A prefix kept once and a batch behind it, through the Node classes: its keys into a paged cache, the
// batch's q and k rotated, attention over both.  Usage: node shared.gpu.js <workdir> (tests/test_gpu_shared_js.py
// wrote the inputs and checks the outputs).
const fs = require('fs');
const path = require('path');
const pkg = require(path.join(__dirname, '..', '..', 'qwen3-embedding-webgpu-prepacked_amd', 'js'));
const { DeviceContext, RotaryPositions, PagedKvCache, SharedPrefixAttention } = pkg;

const work = process.argv[2];
const { prefix, lengths, pageSize, pages, format } = JSON.parse(fs.readFileSync(path.join(work, 'case.json')));
const bytes = (name) => new Uint8Array(fs.readFileSync(path.join(work, `${name}.bin`)));
const save = (name, buffer) => fs.writeFileSync(path.join(work, `${name}.bin`), Buffer.from(buffer.read(new Uint8Array(buffer.bytes))));

const ctx = new DeviceContext(0);
const upload = (data) => { const b = ctx.alloc(data.byteLength); b.write(data); return b; };
const tokens = lengths.reduce((a, b) => a + b, 0);
const cu = [0];
for (const n of lengths) cu.push(cu[cu.length - 1] + n);

const kept = [upload(bytes('prefix_k')), upload(bytes('prefix_v'))];
const qkv = upload(bytes('qkv'));  // [tokens, 2048 + 1024 + 1024]
const prefixPages = pages.slice(0, Math.ceil(prefix / pageSize));
const slots = new BigInt64Array(prefix);
for (let i = 0; i < prefix; i += 1) slots[i] = BigInt(prefixPages[Math.floor(i / pageSize)] * pageSize + (i % pageSize));
const positions = new Int32Array(tokens);
lengths.forEach((n, s) => { for (let i = 0; i < n; i += 1) positions[cu[s] + i] = prefix + i; });

const cache = new PagedKvCache(ctx, { pages: pages.length, pageSize, format });
const dSlots = upload(slots), dPositions = upload(positions);
cache.write(kept[0], kept[1], dSlots, prefix);
const q = ctx.alloc(tokens * 4096), k = ctx.alloc(tokens * 2048), o = ctx.alloc(tokens * 4096);
new RotaryPositions(ctx).run({
  q: { x: qkv, out: q, heads: 16, xStride: 4096 }, k: { x: qkv, out: k, heads: 8, xStride: 4096, xOffset: 4096 },
  positions: dPositions, tokens,
});
const attention = new SharedPrefixAttention(ctx);
const run = attention.createRun(q, o, cache, { cuSeqlens: Int32Array.from(cu), ownLengths: Int32Array.from(lengths), prefixPages, prefixLength: prefix },
  { k, v: qkv, vOffset: 2 * (2048 + 1024), vStride: 4096 });
attention.encode(run);
const backK = ctx.alloc(prefix * 2048), backV = ctx.alloc(prefix * 2048);
cache.read(dSlots, prefix, backK, backV);
ctx.synchronize();
save('q', q);
save('k', k);
save('o', o);
save('back_k', backK);
save('back_v', backV);
console.log(JSON.stringify(run.info));
attention.destroyRun(run);
cache.destroy();
ctx.destroy();
