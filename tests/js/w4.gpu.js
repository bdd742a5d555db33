'use strict';
// Norm, product, gate/up product and the way back into 8 bits through the Node classes.
// Usage: node w4.gpu.js <workdir> (tests/test_gpu_w4_js.py wrote the inputs and checks the outputs).
const fs = require('fs');
const path = require('path');
const pkg = require(path.join(__dirname, '..', '..', 'qwen3-embedding-webgpu-prepacked_amd', 'js'));
const { DeviceContext, EightBitRows, FourBitMatmul } = pkg;

const work = process.argv[2];
const { tokens, width, features, n, dtype } = JSON.parse(fs.readFileSync(path.join(work, 'case.json')));
const bytes = (name) => new Uint8Array(fs.readFileSync(path.join(work, `${name}.bin`)));
const floats = (name) => new Float32Array(bytes(name).slice().buffer);
const save = (name, buffer) => fs.writeFileSync(path.join(work, `${name}.bin`), Buffer.from(buffer.read(new Uint8Array(buffer.bytes))));

const ctx = new DeviceContext(0);
const upload = (data) => { const b = ctx.alloc(data.byteLength); b.write(data); return b; };
const x = upload(bytes('x')), r = upload(bytes('r')), gains = upload(bytes('gains'));
const matmul = new FourBitMatmul(ctx);
const gateUp = matmul.quantize(floats('gate_up'), width, 2 * features);
const down = matmul.quantize(floats('down'), features, n);

const rows = new EightBitRows(ctx, tokens, width), inner = new EightBitRows(ctx, tokens, features);
const ffn = ctx.alloc(tokens * features * 2), yStride = Math.ceil(n / 8) * 8, y = ctx.alloc(tokens * yStride * 2);
y.write(new Uint8Array(y.bytes));
rows.rmsnorm(x, gains, tokens, { residual: r, sum: r, dtype });
matmul.runSwiglu(rows, tokens, gateUp, ffn, { dtype });
inner.quantize(ffn, tokens, { dtype });
matmul.run(inner, tokens, down, y, { yStride, dtype });
ctx.synchronize();
save('sum', r);
save('codes', rows.codes);
save('scales', rows.scales);
save('ffn', ffn);
save('inner_codes', inner.codes);
save('inner_scales', inner.scales);
save('y', y);
rows.destroy();
inner.destroy();
ctx.destroy();
