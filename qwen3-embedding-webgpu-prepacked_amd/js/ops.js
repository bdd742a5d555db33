'use strict';
// Attention operator over libqattn.so, mirroring the reference's CausalAttentionKernel
// (src/webgpu/ops.ts:318-345):
//   createRun(q, k, v, output, batch, sequence, qHeads = 16, kvHeads = 8, valueStride = 1024,
//             valueOffset = 0) -> AttentionRun      (padded [batch, sequence] layout, ops.ts:327)
//   encode(run)                                     (ops.ts:344; the stream is the context's)
//   destroyRun(run)                                 (the run's owned buffers, model.ts:108-111)
// plus createVarlenRun(q, k, v, output, cuSeqlens, options) for packed sequences and
// updateRun(run, cuSeqlens) to re-plan a run for the next batch of the same tensors.
// Buffers are device buffers from DeviceContext.alloc().  The mask is the reference's
// always-on 176-token prefix + 432-token local window (ops.ts:206) unless options say otherwise.

const { loadAddon } = require('./addon');

const MASK = { causal: 0, 'prefix-local': 1 };

function maskCode(name) {
  if (!(name in MASK)) throw new Error(`unknown mask ${name}; expected 'causal' or 'prefix-local'`);
  return MASK[name];
}

class DeviceBuffer {
  constructor(context, bytes) {
    this.context = context;
    this.bytes = bytes;
    this.handle = context.addon.alloc(context.handle, bytes);
  }
  write(typedArray, byteOffset = 0) { this.context.addon.write(this.handle, typedArray, byteOffset); }
  read(typedArray, byteOffset = 0) { this.context.addon.read(this.handle, typedArray, byteOffset); return typedArray; }
  destroy() {
    if (this.handle) this.context.addon.free(this.handle);
    this.handle = null;
  }
}

// One device (reference: requestWebGPUDevice, src/webgpu/device.ts:6-24).
class DeviceContext {
  constructor(device = 0) {
    this.addon = loadAddon();
    this.handle = this.addon.createContext(device);
  }
  info() { return this.addon.deviceName(this.handle); }
  alloc(bytes) { return new DeviceBuffer(this, bytes); }
  synchronize() { this.addon.synchronize(this.handle); }
  synchronizeAsync() { return this.addon.synchronizeAsync(this.handle); }
  destroy() {
    if (this.handle) this.addon.destroyContext(this.handle);
    this.handle = null;
  }
}

class CausalAttentionKernel {
  constructor(context) {
    this.context = context;
  }

  // Padded layout exactly as the reference plans it: batch sequences of `sequence` rows each.
  createRun(q, k, v, output, batch, sequence, qHeads = 16, kvHeads = 8, valueStride = 1024, valueOffset = 0, options = {}) {
    if (qHeads !== 16 || kvHeads !== 8) throw new Error('only 16 query heads over 8 KV heads (Qwen3-Embedding-0.6B) are supported');
    const cuSeqlens = new Int32Array(batch + 1);
    for (let b = 0; b < batch; b += 1) cuSeqlens[b + 1] = cuSeqlens[b] + sequence;
    return this.createVarlenRun(q, k, v, output, cuSeqlens, Object.assign({ valueStride, valueOffset }, options));
  }

  // Packed varlen layout: sequence i is rows cuSeqlens[i]..cuSeqlens[i+1]-1.
  createVarlenRun(q, k, v, output, cuSeqlens, options = {}) {
    const desc = {
      q: q.handle, k: k.handle, v: v.handle, o: output.handle,
      qRowStride: options.queryStride || 2048,
      kRowStride: options.keyStride || 1024,
      vRowStride: options.valueStride || 1024,
      oRowStride: options.outputStride || 2048,
      vOffset: options.valueOffset || 0,
      cuSeqlens: Int32Array.from(cuSeqlens),
      mask: maskCode(options.mask || 'prefix-local'),
      prefix: options.prefix === undefined ? 176 : options.prefix,
      window: options.window === undefined ? 432 : options.window,
      flags: options.batchInvariant ? 1 : 0,
    };
    if (options.lastRows) desc.oLast = options.lastRows.handle;
    const addon = this.context.addon;
    const handle = addon.createRun(this.context.handle, desc);
    return { handle, info: addon.runInfo(handle), cuSeqlens: desc.cuSeqlens };
  }

  // A new batch for a run's tensors: re-plans the work list in place (qattn_run_update), so one
  // run created at a plan's capacity serves every batch of that plan.
  updateRun(run, cuSeqlens) {
    const cu = Int32Array.from(cuSeqlens);
    this.context.addon.updateRun(run.handle, cu);
    run.cuSeqlens = cu;
    run.info = this.context.addon.runInfo(run.handle);
  }

  encode(run) { this.context.addon.encode(run.handle); }

  destroyRun(run) {
    if (run.handle) this.context.addon.destroyRun(run.handle);
    run.handle = null;
  }
}

// The projection over a `.wgpack` Q4_0 tensor (the reference's compact batch matmul,
// src/webgpu/quant-matmul.ts:267-307, and its `matmul(input, name, rows, output)` helper):
// upload(model, name) places a parsed file's q4_0-tile32-compact tensor [K, N] on the device as
// it is stored; run(x, rows, y) computes y = x W^T for fp16 rows x [rows, K] into y [rows, N].
class CompactQ4Matmul {
  constructor(context) {
    this.context = context;
  }

  upload(model, name) {
    const t = model.tensors.get(name);
    if (!t) throw new Error(`prepacked model has no tensor ${name}`);
    if (t.storage !== 'q4_0-tile32-compact') throw new Error(`${name} is not a compact Q4_0 tensor`);
    const [k, n] = t.dimensions;
    const buffer = this.context.alloc(t.byteLength);
    buffer.write(new Uint8Array(model.buffer, t.byteOffset, t.byteLength));
    return { name, k, n, buffer };
  }

  run(x, rows, weight, y, options = {}) {
    const ldx = options.inputStride === undefined ? weight.k : options.inputStride;
    const ldy = options.outputStride === undefined ? weight.n : options.outputStride;
    this.context.addon.q4Matmul(this.context.handle, x.handle, ldx, rows, weight.k, weight.buffer.handle,
      weight.buffer.bytes, weight.n, y.handle, ldy);
  }
}

// ---- requests behind one shared prefix (no counterpart in the reference, which recomputes an
// instruction's tokens with every request): a prefix's keys and values are kept in a PagedKvCache, a batch
// is rotated to the positions that follow them, and attends to both.

const DTYPE = { f16: 0, bf16: 1 };
const KV_FORMAT = { '16bit': 0, e4m3: 1, int8: 2 };
const ROPE_LAYOUT = { half: 0, interleaved: 1 };
const ROPE_SCALING = { plain: 0, linear: 1, yarn: 2 };

function codeOf(table, name, what) {
  if (!Object.prototype.hasOwnProperty.call(table, name)) {
    throw new Error(`unknown ${what} ${name}; expected ${Object.keys(table).map((k) => `'${k}'`).join(', ')}`);
  }
  return table[name];
}
const handleOf = (buffer) => (buffer ? buffer.handle : undefined);

// Rotary positions: run({ q, k, positions, tokens, ... }) turns the head vectors of q and k
// ({ x, heads, out, xStride, outStride, xOffset, outOffset }; without `out` in place) by their token's
// position (Int32 on the device).
class RotaryPositions {
  constructor(context) {
    this.context = context;
  }

  run(options) {
    const block = (b) => b && Object.assign({}, b, { x: handleOf(b.x), out: handleOf(b.out) });
    this.context.addon.rope(this.context.handle, Object.assign({}, options, {
      q: block(options.q), k: block(options.k), positions: handleOf(options.positions),
      dtype: codeOf(DTYPE, options.dtype || 'f16', 'dtype'),
      layout: codeOf(ROPE_LAYOUT, options.layout || 'half', 'layout'),
      scaling: codeOf(ROPE_SCALING, options.scaling || 'plain', 'scaling'),
      inverse: options.inverse ? 1 : 0,
    }));
  }
}

// A paged cache of K and V and its device memory: slot s is row s % pageSize of page
// floor(s / pageSize).
class PagedKvCache {
  constructor(context, { pages, pageSize, kvHeads = 8, headDim = 128, dtype = 'f16', format = '16bit' }) {
    this.context = context;
    Object.assign(this, { pages, pageSize, kvHeads, headDim, dtype, format });
    const codes = codeOf(KV_FORMAT, format, 'cache format');
    const vectors = pages * pageSize * kvHeads;
    this.buffers = {
      k: context.alloc(vectors * headDim * (codes ? 1 : 2)),
      v: context.alloc(vectors * headDim * (codes ? 1 : 2)),
      kScale: codes ? context.alloc(vectors * 4) : null,
      vScale: codes ? context.alloc(vectors * 4) : null,
    };
    this.desc = {
      pages, pageSize, kvHeads, headDim, dtype: codeOf(DTYPE, dtype, 'dtype'), format: codes,
      k: this.buffers.k.handle, v: this.buffers.v.handle,
      kScale: handleOf(this.buffers.kScale), vScale: handleOf(this.buffers.vScale),
    };
  }

  // Rows of K and V ({ kStride, vStride, kOffset, vOffset }) into the slots of a device array of BigInt64;
  // a slot outside the cache writes nothing.
  write(k, v, slots, tokens, options = {}) {
    this.context.addon.kvWrite(this.context.handle, this.desc,
      Object.assign({}, options, { k: k.handle, v: v.handle, slots: slots.handle, tokens }));
  }

  // Slots back into rows; a slot outside the cache gives zeros.
  read(slots, tokens, k, v, options = {}) {
    this.context.addon.kvRead(this.context.handle, this.desc,
      Object.assign({}, options, { k: k.handle, v: v.handle, slots: slots.handle, tokens }));
  }

  destroy() {
    for (const b of Object.values(this.buffers)) if (b) b.destroy();
  }
}

// Attention of a batch of sequences behind one shared prefix.
//   batch: { cuSeqlens, ownLengths, prefixPages, prefixLength, ownPages }; without ownPages the own keys
//   are the rows of options.k and options.v
class SharedPrefixAttention {
  constructor(context) {
    this.context = context;
  }

  createRun(q, output, cache, batch, options = {}) {
    const desc = Object.assign({}, options, batch, {
      q: q.handle, o: output.handle, cache: cache.desc, k: handleOf(options.k), v: handleOf(options.v),
      mask: maskCode(options.mask || 'causal'),
    });
    const addon = this.context.addon;
    const handle = addon.createSharedRun(this.context.handle, desc);
    return { handle, info: addon.sharedRunInfo(handle) };
  }

  // The next batch (a step later): new lengths and pages for the same tensors.
  updateRun(run, batch) {
    this.context.addon.updateSharedRun(run.handle, batch);
    run.info = this.context.addon.sharedRunInfo(run.handle);
  }

  // Other tensors of the same strides and another cache of the same geometry (the next layer's).
  rebindRun(run, q, output, cache, options = {}) {
    this.context.addon.rebindSharedRun(run.handle, Object.assign({}, options, {
      q: q.handle, o: output.handle, cache: cache.desc, k: handleOf(options.k), v: handleOf(options.v),
    }));
  }

  encode(run) { this.context.addon.encodeSharedRun(run.handle); }

  destroyRun(run) {
    if (run.handle) this.context.addon.destroySharedRun(run.handle);
    run.handle = null;
  }
}

module.exports = {
  DeviceContext, DeviceBuffer, CausalAttentionKernel, CompactQ4Matmul, RotaryPositions, PagedKvCache,
  SharedPrefixAttention, MASK,
};
