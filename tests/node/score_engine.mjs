// The JavaScript host over the cache held in 8 bits, its scores and log probabilities, for the test to compare.
//
//     node tests/node/score_engine.mjs job.json
import fs from "fs";
import path from "path";
import { createRequire } from "module";
import * as F from "../../pyodide-llm_amd/forward_hip.mjs";

const addon = createRequire(import.meta.url)("../../pyodide-llm_amd/hip_engine.node");
const job = JSON.parse(fs.readFileSync(process.argv[2], "utf8"));
const read = (name) => fs.readFileSync(path.join(path.dirname(process.argv[2]), name));
const { memory, base } = F.weightsMemory(job.size);
new Uint8Array(memory.buffer, base, job.size).set(read("checkpoint.bin"));
const plan = { ...job.plan, derived: { freq_cis_real: read("cos.bin"), freq_cis_imag: read("sin.bin") } };
const outside = F.external({ memory, base, size: job.size, kernels: F.compileKernels(null, new Uint8Array(8)),
  eightBitCache: true, promptBlock: 64 });
const engine = outside.start(plan);
const memoryBytes = engine.memoryBytes();
const header = Array.from(new Int32Array(memory.buffer.slice(base, base + 28)));
const footprint = F.footprint(header, job.size, { eightBitCache: true, promptBlock: 64 });
const plainly = (got) => Object.fromEntries(Object.entries(got).map(([k, v]) => [k, Array.from(v)]));
const score = plainly(engine.score(job.tokens, 0, null, 3));
const steps = engine.generateMany(7, job.tokens.length, [], 0, 16, 0, 0.9, 1, [], []);
const last = plainly(engine.logprobs([steps[steps.length - 1], 3], 2));
const threw = [() => engine.score([], 0), () => engine.score([1, 2], 0, [1, 2, 3]), () => engine.logprobs([], 33),
  () => engine.score([1], plan.seq_len)].map((f) => {
  try {
    f();
    return false;
  } catch (e) {
    return true;
  }
});
engine.release().then(() => console.log(JSON.stringify({ score, steps, last, threw, memoryBytes, footprint })));
