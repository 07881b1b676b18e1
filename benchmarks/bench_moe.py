"""The mixture-of-experts layer on padded library products and on the grouped operators, and the operators by themselves.

    python -m benchmarks.bench_moe

One GPU, bf16 autocast for the layer, inputs in rotation so that matrices come from memory; CUDA events around a run of calls, the
median of five runs, microseconds per call.
"""

from __future__ import annotations

import torch

from torchure_b200.ops import act8, moe
from torchure_b200.parallel.expert_parallel import MoELayer

SHAPES = [                 # tokens, width, units, experts, choices
    (8192, 1024, 1536, 8, 2),
    (8192, 1024, 768, 64, 8),
    (512, 1024, 1536, 8, 2),
    (1, 1024, 1536, 8, 2),
]


def timed(call, runs: int = 5, calls: int = 20) -> float:
    for i in range(4):
        call(i)
    found = []
    for _ in range(runs):
        begin, end = torch.cuda.Event(enable_timing=True), torch.cuda.Event(enable_timing=True)
        torch.cuda.synchronize()
        begin.record()
        for i in range(calls):
            call(i)
        end.record()
        torch.cuda.synchronize()
        found.append(begin.elapsed_time(end) * 1e3 / calls)
    return sorted(found)[runs // 2]


def layer(tokens, width, units, experts, k, kind, bits=16):
    torch.manual_seed(0)
    layers = [MoELayer(width, units, experts, k, 1.25, experts=kind, act_bits=bits).cuda() for _ in range(3)]
    xs = [torch.randn(tokens, width, device="cuda").requires_grad_() for _ in range(3)]
    out = {}

    def forward(i):
        with torch.no_grad(), torch.autocast("cuda", dtype=torch.bfloat16):
            layers[i % 3](xs[i % 3])

    def step(i):
        m, x = layers[i % 3], xs[i % 3]
        m.zero_grad(set_to_none=True)
        with torch.autocast("cuda", dtype=torch.bfloat16):
            y = m(x)
        torch.autograd.backward((y, m.aux_loss), (x.detach(), torch.ones_like(m.aux_loss)))

    out["forward"] = timed(forward)
    if tokens > 64:
        out["step"] = timed(step)
        torch.cuda.reset_peak_memory_stats()
        before = torch.cuda.memory_allocated()
        step(0)
        out["peak MB"] = (torch.cuda.max_memory_allocated() - before) / 1e6
    return out


def main() -> None:
    for shape in SHAPES:
        print("tokens {} width {} units {} experts {} choices {}".format(*shape))
        for name, kind, bits in (("padded library products", "capacity", 16), ("grouped", "grouped", 16), ("grouped, kept in 8 bits", "grouped", 8)):
            print(f"  {name:26s} " + "  ".join(f"{n} {v:9.1f}" for n, v in layer(*shape, kind, bits).items()))
    gu = [torch.randn(16384, 2 * 1536, device="cuda").bfloat16() for _ in range(3)]
    kept = [act8.quantize8(g) for g in gu]
    print(f"quantize8 16384 x 2 x 1536    {timed(lambda i: act8.quantize8(gu[i % 3])):9.1f}")
    print(f"dequantize8                   {timed(lambda i: act8.dequantize8(kept[i % 3])):9.1f}")
    print(f"swiglu_8bit                   {timed(lambda i: act8.swiglu_8bit(gu[i % 3])):9.1f}")
    for tokens, experts, k in ((8192, 8, 2), (16384, 128, 8)):
        logits = torch.randn(tokens, experts, device="cuda")
        print(f"route {tokens} x {experts}, {k} choices {timed(lambda i: moe.route(logits, k)):9.1f}")


if __name__ == "__main__":
    main()
