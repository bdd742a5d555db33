// Type declarations of the Node attention-path package (js/index.js).  The engine and plugin
// interfaces match src/webgpu/embedding-engine.ts:1-13 of the reference.

export interface TokenizerResult {
  input_ids: { tolist(): number[][] };
}
export type TokenizerLike = (text: string) => TokenizerResult;

export interface EmbeddingPlan {
  run(ids: Uint32Array, lengths: Uint32Array): Promise<Float32Array[]>;
  /** Optional split of run(): a plan that has both gets up to two batches in flight from the
   *  engine (the next is packed and enqueued while one runs); results still resolve in order. */
  enqueue?(ids: Uint32Array, lengths: Uint32Array): unknown;
  complete?(ticket: unknown): Promise<Float32Array[]>;
}
export interface EmbeddingRuntime {
  /** 'varlen': the engine packs requests back to back (ids.length === sum(lengths)). */
  packing?: 'padded' | 'varlen';
  createPlan(batch: number, sequence: number): EmbeddingPlan;
}

export class Qwen3EmbeddingEngine {
  constructor(runtime: EmbeddingRuntime, tokenizer: TokenizerLike, maxBatchSize?: number,
              batchWindowMs?: number, eosToken?: number);
  readonly maxBatchSize: number;
  readonly batchWindowMs: number;
  readonly eosToken: number;
  embed(text: string): Promise<Float32Array>;
}

export function packPadded(tokenLists: number[][], eosToken: number): { ids: Uint32Array; lengths: Uint32Array; sequence: number };
export function packVarlen(tokenLists: number[][]): { ids: Uint32Array; lengths: Uint32Array; sequence: number };
export function cuSeqlensOf(lengths: ArrayLike<number>): Int32Array;

export type MaskName = 'causal' | 'prefix-local';

export class DeviceBuffer {
  readonly bytes: number;
  write(data: ArrayBufferView, byteOffset?: number): void;
  read<T extends ArrayBufferView>(data: T, byteOffset?: number): T;
  destroy(): void;
}

export class DeviceContext {
  constructor(device?: number);
  info(): { name: string; computeUnits: number };
  alloc(bytes: number): DeviceBuffer;
  synchronize(): void;
  synchronizeAsync(): Promise<void>;
  destroy(): void;
}

export interface RunInfo {
  tokens: number; pairs: number; flops: number; bytes: number;
  workItems: number; blockQueries: number; tilePairs: number; slots: number; splitItems: number;
}
export interface AttentionRun { handle: unknown; info: RunInfo; cuSeqlens: Int32Array }
export interface VarlenOptions {
  queryStride?: number; keyStride?: number; valueStride?: number; outputStride?: number;
  valueOffset?: number; mask?: MaskName; prefix?: number; window?: number; lastRows?: DeviceBuffer;
  /** Never split an item across workgroups: results independent of batch composition. */
  batchInvariant?: boolean;
}

export class CausalAttentionKernel {
  constructor(context: DeviceContext);
  createRun(q: DeviceBuffer, k: DeviceBuffer, v: DeviceBuffer, output: DeviceBuffer, batch: number,
            sequence: number, qHeads?: number, kvHeads?: number, valueStride?: number,
            valueOffset?: number, options?: VarlenOptions): AttentionRun;
  createVarlenRun(q: DeviceBuffer, k: DeviceBuffer, v: DeviceBuffer, output: DeviceBuffer,
                  cuSeqlens: ArrayLike<number>, options?: VarlenOptions): AttentionRun;
  /** Re-plans a run for the next batch of the same tensors (same options, new lengths). */
  updateRun(run: AttentionRun, cuSeqlens: ArrayLike<number>): void;
  encode(run: AttentionRun): void;
  destroyRun(run: AttentionRun): void;
}

export interface HipRuntimeOptions {
  device?: number; context?: DeviceContext; layers?: number; mask?: MaskName;
  prefix?: number; window?: number; seed?: number;
  /** Default true: embeddings are bitwise independent of batching (no split-K). */
  batchInvariant?: boolean;
}
export interface HipAttentionPlan extends EmbeddingPlan {
  /** Host enqueue time and wall time (ms) of the last run, and its token count. */
  readonly timing: { hostMs: number; totalMs: number; tokens: number } | null;
  destroy(): void;
}
export class HipAttentionRuntime implements EmbeddingRuntime {
  constructor(options?: HipRuntimeOptions);
  readonly packing: 'varlen';
  createPlan(batch: number, sequence: number): HipAttentionPlan;
  destroy(): void;
}

// ---- the `.wgpack` container (the reference's src/prepacked/format.ts) and the Q4_0 projection.
export interface PackedTensorBytes {
  name: string; dimensions: number[]; type: number;
  storage: 'q4_0-tile32-compact' | 'raw'; bytes: Uint8Array;
}
export interface PrepackedTensorHeader {
  name: string; dimensions: number[]; type: number; storage: 'q4_0-tile32-compact' | 'raw';
  offset: number; byteLength: number;
}
export interface PrepackedModel {
  header: {
    version: 2; sourceSha256: string; sourceBytes: number; layout: 'q4_0-tile32-compact-v2';
    tileRows: 32; blockValues: 32; blockBytes: 20;
    metadata: Record<string, string | number | boolean | Array<string | number | boolean>>;
    tensors: PrepackedTensorHeader[];
  };
  tensors: Map<string, PrepackedTensorHeader & { byteOffset: number }>;
  buffer: ArrayBuffer;
  dataOffset: number;
}
/** Every rejection of the container code; `code` names the rule (e.g. 'BAD_MAGIC', 'TENSOR_OUT_OF_BOUNDS'). */
export class PrepackedFormatError extends Error {
  readonly code: 'NO_PARTS' | 'K_NOT_BLOCKS' | 'K_MISMATCH' | 'PART_SIZE' | 'TRUNCATED_PRELUDE' | 'BAD_MAGIC'
    | 'TRUNCATED_HEADER' | 'BAD_LAYOUT' | 'TENSOR_OUT_OF_BOUNDS' | 'DUPLICATE_TENSOR' | 'BAD_COMPACT_TENSOR'
    | 'BAD_STORAGE' | 'NO_TENSOR';
}
export const prepacked: {
  PrepackedFormatError: typeof PrepackedFormatError;
  MAGIC: 'WGPACK02'; LAYOUT: 'q4_0-tile32-compact-v2'; TILE_ROWS: 32; BLOCK_VALUES: 32; BLOCK_BYTES: 20;
  STORAGE_COMPACT: 'q4_0-tile32-compact'; STORAGE_RAW: 'raw'; GGML_TYPE: { F32: 0; F16: 1; Q4_0: 2; Q6_K: 14 };
  packQ40Tile32(name: string, parts: ReadonlyArray<{ name: string; k: number; n: number; bytes: Uint8Array }>): PackedTensorBytes;
  rawTensor(name: string, dimensions: number[], type: number, bytes: Uint8Array): PackedTensorBytes;
  buildPrepackedFile(sourceSha256: string, sourceBytes: number,
                     metadata: PrepackedModel['header']['metadata'], tensors: ReadonlyArray<PackedTensorBytes>): Uint8Array;
  parsePrepackedModel(buffer: ArrayBuffer): PrepackedModel;
  tensorBytes(model: PrepackedModel, name: string): Uint8Array;
};

export interface CompactQ4Weight { name: string; k: number; n: number; buffer: DeviceBuffer }
/** y = x W^T over a compact Q4_0 tensor (the reference's compact batch matmul). */
export class CompactQ4Matmul {
  constructor(context: DeviceContext);
  upload(model: PrepackedModel, name: string): CompactQ4Weight;
  run(x: DeviceBuffer, rows: number, weight: CompactQ4Weight, y: DeviceBuffer,
      options?: { inputStride?: number; outputStride?: number }): void;
}

// ---- requests behind one shared prefix: rotary positions, a paged K/V cache, attention over it.
export type DtypeName = 'f16' | 'bf16';
/** Head h of token t at element t * xStride + h * headDim; without `out` in place.  Strides in
 *  elements (default heads * headDim), offsets in bytes. */
export interface RopeBlock {
  x: DeviceBuffer; heads: number; out?: DeviceBuffer; xStride?: number; outStride?: number;
  xOffset?: number; outOffset?: number;
}
export interface RopeOptions {
  q: RopeBlock; k?: RopeBlock;
  /** Int32 per token, on the device. */
  positions: DeviceBuffer; positionsOffset?: number; tokens: number;
  dtype?: DtypeName; headDim?: number;
  /** The first elements of a head that turn (default headDim); the others pass through. */
  rotaryDim?: number;
  layout?: 'half' | 'interleaved'; scaling?: 'plain' | 'linear' | 'yarn';
  theta?: number; factor?: number; originalContext?: number; betaFast?: number; betaSlow?: number; magnitude?: number;
  /** The rotation back, which also maps the output's gradient to the input's. */
  inverse?: boolean;
}
export class RotaryPositions {
  constructor(context: DeviceContext);
  run(options: RopeOptions): void;
}
/** Strides in elements, offsets in bytes. */
export interface KvRowOptions {
  kStride?: number; vStride?: number; kOffset?: number; vOffset?: number; slotsOffset?: number;
}
/** Slot s is row s % pageSize of page floor(s / pageSize). */
export class PagedKvCache {
  constructor(context: DeviceContext, options: {
    pages: number; pageSize: number; kvHeads?: number; headDim?: 64 | 128; dtype?: DtypeName;
    format?: '16bit' | 'e4m3' | 'int8';
  });
  readonly pages: number;
  readonly pageSize: number;
  /** slots: BigInt64 per token, on the device; none twice in a write. */
  write(k: DeviceBuffer, v: DeviceBuffer, slots: DeviceBuffer, tokens: number, options?: KvRowOptions): void;
  read(slots: DeviceBuffer, tokens: number, k: DeviceBuffer, v: DeviceBuffer, options?: KvRowOptions): void;
  destroy(): void;
}
/** Sequence i has queries cuSeqlens[i] .. cuSeqlens[i + 1] - 1, the last of its keys' positions: the
 *  prefix's prefixLength keys, then its own ownLengths[i]. */
export interface SharedBatch {
  cuSeqlens: Int32Array | number[]; ownLengths: Int32Array | number[];
  prefixPages?: Int32Array | number[]; prefixLength?: number;
  /** ceil(ownLengths[i] / pageSize) pages of each sequence in turn; without it the own keys are rows of k, v. */
  ownPages?: Int32Array | number[];
}
/** Offsets in bytes. */
export interface SharedTensors {
  k?: DeviceBuffer; v?: DeviceBuffer; qOffset?: number; oOffset?: number; kOffset?: number; vOffset?: number;
}
export interface SharedOptions extends SharedTensors {
  qHeads?: number; qStride?: number; oStride?: number; kStride?: number; vStride?: number;
  mask?: MaskName; prefix?: number; window?: number;
  /** Of the scores; 0: 1 / sqrt(headDim). */
  scale?: number;
}
export interface SharedRun {
  handle: unknown;
  info: { tokens: number; keys: number; pairs: number; flops: number; items: number; mergedRows: number; partialRows: number };
}
export class SharedPrefixAttention {
  constructor(context: DeviceContext);
  createRun(q: DeviceBuffer, output: DeviceBuffer, cache: PagedKvCache, batch: SharedBatch, options?: SharedOptions): SharedRun;
  /** The next batch: new lengths and pages for the same tensors. */
  updateRun(run: SharedRun, batch: SharedBatch): void;
  /** Other tensors of the same strides and another cache of the same geometry (the next layer's). */
  rebindRun(run: SharedRun, q: DeviceBuffer, output: DeviceBuffer, cache: PagedKvCache, options?: SharedTensors): void;
  encode(run: SharedRun): void;
  destroyRun(run: SharedRun): void;
}

// ---- a forward with 8-bit activations: rows into 8 bits, their products with 4-bit weights.
/** Strides in elements (default the width), offsets in bytes. */
export interface RowsQ8Options { dtype?: DtypeName; xStride?: number; xOffset?: number }
export interface NormQ8Options extends RowsQ8Options {
  /** Added to x; the sum goes to `sum`, which may be x or residual. */
  residual?: DeviceBuffer; sum?: DeviceBuffer; eps?: number;
  residualStride?: number; sumStride?: number; residualOffset?: number; sumOffset?: number;
}
/** `capacity` rows of `width` 8-bit codes and a Float32 scale each. */
export class EightBitRows {
  constructor(context: DeviceContext, capacity: number, width: number);
  readonly codes: DeviceBuffer;
  readonly scales: DeviceBuffer;
  quantize(x: DeviceBuffer, rows: number, options?: RowsQ8Options): void;
  /** weight: Float32 [width], on the device. */
  rmsnorm(x: DeviceBuffer, weight: DeviceBuffer, rows: number, options?: NormQ8Options): void;
  destroy(): void;
}
export interface FourBitWeight { k: number; n: number; buffer: DeviceBuffer }
export interface FourBitOptions { dtype?: DtypeName; yStride?: number; yOffset?: number }
/** 4-bit weights with whole-number group scales, laid out on the host, and products with them. */
export class FourBitMatmul {
  constructor(context: DeviceContext);
  quantize(rows: Float32Array, k: number, n: number): FourBitWeight;
  /** codes [n][k / 2], even columns low; groups [n][k / 32], multiplier | zero << 4; scales [n]. */
  pack(codes: Uint8Array, groups: Uint8Array, scales: Float32Array, k: number, n: number): FourBitWeight;
  upload(model: PrepackedModel, name: string): FourBitWeight;
  run(x: EightBitRows, rows: number, weight: FourBitWeight, y: DeviceBuffer, options?: FourBitOptions): void;
  /** weight: [gate | up]; y has n / 2 columns. */
  runSwiglu(x: EightBitRows, rows: number, weight: FourBitWeight, y: DeviceBuffer, options?: FourBitOptions): void;
}

// ---- the whole model (the reference's Qwen3WebGPUModel / Qwen3ExecutionPlan, model.ts:49-255).
/** Stage names of a profiled run, in order (model.ts:157-168). */
export type ModelStage = 'embedding_norm' | 'qkv' | 'rope_attention' | 'attention_output' | 'post_attention_norm'
  | 'ffn_up_gate' | 'swiglu' | 'ffn_down' | 'post_ffn_norm' | 'pool';
export interface HipModelOptions {
  /** Attention mask of the forward (default 'prefix-local', 176 / 432). */
  mask?: 'causal' | 'prefix-local'; prefix?: number; window?: number;
  /** Default true: a request's embedding is bitwise the same alone or in any batch. */
  batchInvariant?: boolean;
}
/** The weights of a parsed .wgpack on the device (Q6_K token_embd, f32 norms, 4 compact Q4_0
 * projections per layer, 1..28 layers), checked by name, storage, type and shape. */
export class HipQwen3Model {
  constructor(context: DeviceContext, prepacked: PrepackedModel, options?: HipModelOptions);
  readonly layers: number;
  readonly vocab: number;
  createPlan(batch: number, sequence: number): HipQwen3Plan;
  destroy(): void;
}
export interface HipQwen3Ticket { readonly n: number; readonly tokens: number }
export class HipQwen3Plan implements EmbeddingPlan {
  /** Packed token ids (lengths[i] per request) -> one L2-normalised Float32Array(1024) per request. */
  run(ids: Uint32Array | Int32Array, lengths: Uint32Array | number[]): Promise<Float32Array[]>;
  /** Submits one batch and returns at once (at most two of this plan in flight). */
  enqueue(ids: Uint32Array | Int32Array, lengths: Uint32Array | number[]): HipQwen3Ticket;
  /** The embeddings of an enqueued batch, once its own work is done (later batches not waited for). */
  complete(ticket: HipQwen3Ticket): Promise<Float32Array[]>;
  /** One run with each stage timed: total ms per stage over all layers. */
  profile(ids: Uint32Array | Int32Array, lengths: Uint32Array | number[]): Record<ModelStage, number>;
  readonly timing: { hostMs: number; totalMs: number; tokens: number } | null;
  destroy(): void;
}
/** EmbeddingRuntime over the model: give `prepacked` (a parsed .wgpack) or a `model`. */
export class HipQwen3Runtime implements EmbeddingRuntime {
  constructor(options: HipModelOptions & { prepacked?: PrepackedModel; model?: HipQwen3Model;
                                           context?: DeviceContext; device?: number });
  readonly packing: 'varlen';
  readonly model: HipQwen3Model;
  createPlan(batch: number, sequence: number): HipQwen3Plan;
  destroy(): void;
}
