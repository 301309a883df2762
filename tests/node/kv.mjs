// Driver of tests/test_kv_node.py: rotary positions, the 8-bit key / value cache and attention over it through the shim.
//   kv.mjs <dir>   spec.json, qkv.bin ([Hq + 2 Hkv][n][128] f16) -> rot.bin, k.bin, v.bin, o.bin, errors.json
'use strict';
import { readFileSync, writeFileSync } from 'fs';
import { join } from 'path';
import * as p0k from '../../p0pc0rn-kernels_amd/node/index.mjs';

const dir = process.argv[2];
const spec = JSON.parse(readFileSync(join(dir, 'spec.json'), 'utf8'));
const { n, Hq, Hkv } = spec;
const put = async (g, name, b, bytes) => writeFileSync(join(dir, name), Buffer.from(await g.read(b)).subarray(0, bytes));
const errorOf = (fn) => { try { fn(); return null; } catch (e) { return e.message; } };

async function main() {
  const g = await p0k.createGpu();
  const raw = readFileSync(join(dir, 'qkv.bin'));
  const qkv = g.upload(new Uint8Array(raw.buffer, raw.byteOffset, raw.byteLength)), rot = g.buffer((Hq + Hkv) * n * 256);
  const pos = g.upload(Int32Array.from([0])), cu = g.upload(Int32Array.from([0, n])), len = g.upload(Int32Array.from([n]));
  const batch = { pos, cu, B: 1, rows: n };
  const cache = p0k.kvCache(g, { Hkv, pages: spec.maxPages, slots: 1, maxPages: spec.maxPages });
  p0k.rope(g, { x: { buf: qkv }, y: { buf: rot }, H: Hq + Hkv, batch, rd: spec.rd, mode: 'half', freqs: spec.freqs });
  const k = { buf: rot, off: Hq * n * 256 }, v = { buf: qkv, off: (Hq + Hkv) * n * 256 };
  p0k.kvAppend(g, { cache, batch, k, v });
  const ko = g.buffer(Hkv * n * 256), vo = g.buffer(Hkv * n * 256), o = g.buffer(n * Hq * 256);
  p0k.kvRead(g, { cache, batch, len, k: ko, v: { buf: vo } });
  p0k.kvAttention(g, { cache, batch, q: rot, o: { buf: o }, Hq, window: spec.window, sinks: spec.sinks });
  await put(g, 'rot.bin', rot, (Hq + Hkv) * n * 256);
  await put(g, 'k.bin', ko, Hkv * n * 256);
  await put(g, 'v.bin', vo, Hkv * n * 256);
  await put(g, 'o.bin', o, n * Hq * 256);
  writeFileSync(join(dir, 'errors.json'), JSON.stringify({
    sinks: errorOf(() => p0k.kvAttention(g, { cache, batch, q: rot, o: { buf: o }, Hq, sinks: 1 })),
    rows: errorOf(() => p0k.kvAppend(g, { cache, batch: { ...batch, rows: n + 1 }, k, v })),
    freqs: errorOf(() => p0k.rope(g, { x: rot, H: 1, batch, rd: 8, freqs: [1, 2] })),
    freed: errorOf(() => { const b = g.buffer(n * Hq * 256); g.free(b); p0k.kvAttention(g, { cache, batch, q: b, o: { buf: o }, Hq }); }),
  }));
  [qkv, rot, pos, cu, len, ko, vo, o, cache.code, cache.scale, cache.tail, cache.table].forEach((b) => g.free(b));
  await g.done();
  g.destroy();
}

main().catch((e) => { console.error(e.stack); process.exit(1); });
