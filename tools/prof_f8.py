"""One operator of the 8-bit rows a few times, for rocprofv3 runs (profiles/collect_f8.sh):
prof_f8.py norm n d type residual(0/1) unit(0/1) | quantise n d type | product m n k | search rows d queries k [share of a row in one channel]"""
import os
import sys

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import torch

import semantic_search_amd as ssa

op, a = sys.argv[1], sys.argv[2:]
g = torch.Generator(device="cuda").manual_seed(1)
randn = lambda *s: torch.randn(*s, generator=g, device="cuda")  # noqa: E731
types = {"f32": torch.float32, "f16": torch.float16, "bf16": torch.bfloat16}
if op in ("norm", "quantise"):
    n, d, t = int(a[0]), int(a[1]), types[a[2]]
    x, out = randn(n, d).to(t), ssa.F8Rows.empty(n, d, "cuda")
    if op == "norm":
        w, r = (1 + 0.2 * randn(d)).to(t), randn(n, d).to(t) if int(a[3]) else None
        ro = torch.empty_like(x) if int(a[3]) else None
        run = lambda: ssa.rms_norm_f8(x, weight=w, residual=r, residual_out=ro, unit=bool(int(a[4])), out=out)  # noqa: E731
    else:
        run = lambda: (ssa.quantize_f8(x, out=out), out.dequantize(torch.bfloat16))  # noqa: E731
elif op == "product":
    m, n, k = map(int, a)
    x, y, out = ssa.quantize_f8(randn(m, k)), ssa.quantize_f8(randn(n, k)), torch.empty(m, n, dtype=torch.bfloat16, device="cuda")
    run = lambda: ssa.matmul_f8(x, y, out=out)  # noqa: E731
else:
    n, d, nq, k = map(int, a[:4])
    share = float(a[4]) if len(a) > 4 else 0.0

    def rows(c):
        v = torch.nn.functional.normalize(randn(c, d)) * (1 - share * share) ** 0.5
        if share:
            v[:, 5] = share * (1 + 0.01 * randn(c))
        return v
    index, q = ssa.IndexFlatIP(d, storage="f8"), None
    for lo in range(0, n, 100000):
        index.add(rows(min(100000, n - lo)))
    q = rows(nq)
    run = lambda: index.search(q, k)  # noqa: E731
for _ in range(10):
    run()
torch.cuda.synchronize()
print("done", *sys.argv[1:])
