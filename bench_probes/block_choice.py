"""The block-scaled e4m3 linear on the layers of two decoders: the config that ``block_config`` picks beside
the best compiled one and the floor; and the calls that the kernel profile is taken of.

Usage (needs the GPU)::

    python bench_probes/block_choice.py layers [M ...] > block_choice.log
    python bench_probes/block_choice.py random SEED SECONDS MOST_ROWS >> block_choice.log
    python bench_probes/block_choice.py summary block_choice.log      # profiles/fp8_block_layers.md
    rocprofv3 --kernel-trace --stats ... -- python bench_probes/block_choice.py calls CASE

``layers`` and ``random`` (layers with N 64 .. 32768 and K 256 .. 16384, half of them the decoders') print a
JSON line per call: the times of every compiled tile and K split, the data a refit of the model needs.
Times are the median of 7 replays, in turn, of HIP graphs of 40 launches or more over as many copies of the
operands as 400 MB hold, 40 at most: from a weight of 10 MB on they come from HBM, smaller ones from the
caches. The floor is the larger of the call's bytes at 5.17 TB/s (a copy of 1 GiB) and its products at 2605
TFLOP/s (the library's fp8 product of 8192^3 with one scale a tensor). ``calls`` makes 12 calls of a case of
``perf/operators.py`` over three sets of inputs.
"""

from __future__ import annotations

import importlib.util
import json
import math
import random
import statistics
import sys
import time
from pathlib import Path

ROOT = Path(__file__).resolve().parents[1]
SUMMARY = ROOT / "profiles" / "fp8_block_layers.md"
LAYERS = {  # (N, K)
    "7B qkv": (4608, 3584), "7B o": (3584, 3584), "7B gate_up": (37888, 3584), "7B down": (3584, 18944),
    "0.5B qkv": (1152, 896), "0.5B o": (896, 896), "0.5B gate_up": (9728, 896), "0.5B down": (896, 4864),
}
ROWS = (1, 4, 16, 64, 128, 256, 512, 1024, 2048, 4096)
BYTES_US, FLOPS_US = 5.17e6, 2605e6


def floor_us(m: int, n: int, k: int) -> float:
    kb, nb = -(-k // 128), -(-n // 128)
    return max((m * k + n * k + 4 * (m + nb) * kb + 2 * m * n) / BYTES_US, 2 * m * n * k / FLOPS_US)


def _name(cfg) -> str:  # type: ignore[no-untyped-def]
    return f"{cfg.kernel} {cfg.block_m}x{cfg.block_n} w{cfg.num_warps} s{cfg.num_stages} split {cfg.split_k}"


def _configs(m: int, n: int, k: int) -> list:
    """The rule's config first, then every other one that is not out of question at this size."""
    from tokenforge.kernels import block_config as bc

    out = [bc.block_config(m, n, k)]
    for kernel, bm, bn, warps, stages in bc.BLOCK_TILES:
        tiles = -(-m // bm) * -(-n // bn)
        if (kernel == "gemv_block" and (m > 300 or m > 4 * bm)) or (bm > 64 and bm >= 2 * m) or tiles > 9000:
            continue
        for split in (1,) if kernel == "gemv_block" else bc._SPLITS:
            if split > 1 and (split > -(-k // 128) // 2 or tiles > bc.NUM_CUS or tiles * split > bc._MAX_SPLIT_GROUPS):
                break
            out.append(bc.BlockConfig(kernel, bm, bn, split, warps, stages))
    return list(dict.fromkeys(out))


def _measure(m: int, n: int, k: int) -> dict:
    import torch

    from tokenforge.kernels.hip.fp8_block import fp8_block_gemm

    dev = torch.device("cuda")

    def codes(r: int) -> torch.Tensor:
        return (torch.randn((r, k), device=dev, dtype=torch.float16) * 100).clamp_(-448, 448).to(torch.float8_e4m3fn)

    kb, nb = -(-k // 128), -(-n // 128)
    copies = max(1, min(40, (400 << 20) // (n * k + m * k)))
    ops = [(codes(m), torch.rand((m, kb), device=dev), codes(n), torch.rand((nb, kb), device=dev)) for _ in range(copies)]
    launches = max(40, copies)
    cfgs, graphs = _configs(m, n, k), []
    for cfg in cfgs:
        fp8_block_gemm(*ops[0], cfg, None, torch.bfloat16)
        torch.cuda.synchronize()
        graph = torch.cuda.CUDAGraph()
        with torch.cuda.graph(graph, stream=torch.cuda.Stream()):
            for i in range(launches):
                fp8_block_gemm(*ops[i % copies], cfg, None, torch.bfloat16)
        graph.replay()
        graphs.append(graph)
    us: list[list[float]] = [[] for _ in cfgs]
    for r in range(7):
        for i in range(len(graphs)):
            j = (i + r) % len(graphs)
            start, end = (torch.cuda.Event(enable_timing=True) for _ in range(2))
            start.record()
            graphs[j].replay()
            end.record()
            end.synchronize()
            us[j].append(start.elapsed_time(end) * 1e3 / launches)
    times = {_name(c): round(statistics.median(t), 2) for c, t in zip(cfgs, us)}
    return {"m": m, "n": n, "k": k, "floor": round(floor_us(m, n, k), 2), "chosen": _name(cfgs[0]), "us": times}


def time_layers(rows: list[int]) -> None:
    for layer, (n, k) in LAYERS.items():
        for m in rows or ROWS:
            print(json.dumps({"layer": layer, **_measure(m, n, k)}), flush=True)


def time_random(seed: int, seconds: float, most: int) -> None:
    rng, end = random.Random(seed), time.time() + seconds
    while time.time() < end:
        n, k = rng.choice(list(LAYERS.values()))
        if rng.random() < 0.5:
            n = int(math.exp(rng.uniform(math.log(64), math.log(32768)))) // 16 * 16
            k = int(math.exp(rng.uniform(math.log(256), math.log(16384)))) // 128 * 128
        m = min(int(math.exp(rng.uniform(0, math.log(most)))), 4096 * 37888 * 3584 // (n * k))
        print(json.dumps(_measure(m, n, k)), flush=True)


def summary(log: str) -> None:
    rows = [json.loads(ln) for ln in Path(log).read_text().splitlines() if ln.startswith("{")]
    named = [r for r in rows if "layer" in r]
    ms = sorted({r["m"] for r in named})
    best = {id(r): min(r["us"].values()) for r in rows}
    out = ["# The block-scaled e4m3 linear on the layers of two decoders", "", "Commands (on an MI355X):", "", "```",
           "python bench_probes/block_choice.py layers > block_choice.log",
           "python bench_probes/block_choice.py summary block_choice.log", "```", "",
           "us a launch in a HIP graph, bf16 output, the config of `block_config` / the floor. 7B operands come from HBM,",
           "0.5B ones, 40 copies, partly from the caches. The floor is bytes at 5.17 TB/s or products at 2605 TFLOP/s,",
           "without a launch, which alone takes 2 to 3 us.", "",
           "| Layer | N x K | " + " | ".join(f"M = {m}" for m in ms) + " |", "|---|---|" + "---:|" * len(ms)]
    for layer, (n, k) in LAYERS.items():
        at = {r["m"]: r for r in named if r["layer"] == layer}
        cells = [f"{at[m]['us'][at[m]['chosen']]:.1f} / {at[m]['floor']:.1f}" if m in at else "" for m in ms]
        out.append(f"| {layer} | {n} x {k} | " + " | ".join(cells) + " |")
    ratio = [r["us"][r["chosen"]] / best[id(r)] for r in rows]
    mean = math.exp(statistics.fmean(map(math.log, ratio)))
    out += ["", f"{len(rows)} calls: the chosen config takes {100 * (mean - 1):.1f}% longer than the best compiled one on "
            f"average, {sum(q > 1.05 for q in ratio)} of them over 5%. Config by call:", "",
            "| Layer | M | chosen | us | best | us |", "|---|---:|---|---:|---|---:|"]
    for r in named:
        fastest = min(r["us"], key=r["us"].get)
        out.append(f"| {r['layer']} | {r['m']} | {r['chosen']} | {r['us'][r['chosen']]} | "
                   f"{'the same' if fastest == r['chosen'] else fastest} | {r['us'][fastest]} |")
    SUMMARY.write_text("\n".join(out) + "\n")
    print(f"wrote {SUMMARY}")


def calls(name: str) -> None:
    import torch

    spec = importlib.util.spec_from_file_location("operators", ROOT / "perf" / "operators.py")
    assert spec is not None and spec.loader is not None
    cases = importlib.util.module_from_spec(spec)
    spec.loader.exec_module(cases)
    cases.own = True
    case = next(c for c in cases.listed() if c["name"] == name)
    states = [cases.prepare(case, seed) for seed in range(3)]
    for i in range(12):
        cases.run(states[i % 3])
    torch.cuda.synchronize()
    print(f"{name}: 12 calls", flush=True)


def main(argv: list[str]) -> None:
    sys.path.insert(0, str(ROOT))
    if argv[:1] == ["layers"]:
        time_layers([int(m) for m in argv[1:]])
    elif argv[:1] == ["random"] and len(argv) == 4:
        time_random(int(argv[1]), float(argv[2]), int(argv[3]))
    elif argv[:1] == ["summary"] and len(argv) == 2:
        summary(argv[1])
    elif argv[:1] == ["calls"] and len(argv) == 2:
        calls(argv[1])
    else:
        raise SystemExit(__doc__)


if __name__ == "__main__":
    main(sys.argv[1:])
