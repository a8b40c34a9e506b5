"""Child process of test_gpu_11_mxfp4: the MXFP4 products of a few shapes, saved to a file."""
import pathlib
import sys

import torch

ROOT = pathlib.Path(__file__).resolve().parents[1]
for p in (str(ROOT), str(ROOT / "tests")):
    if p not in sys.path:
        sys.path.insert(0, p)

CASES = [(1, 64, 96, 1), (300, 512, 1536, 3), (777, 72, 2056, 2), (4096, 1536, 512, 64),
         (9000, 328, 448, 5)]


def main(path):
    from gpu_util import get_ops, ragged_counts
    ops = get_ops()
    out = {}
    for M, N, K, G in CASES:
        g = torch.Generator(device="cuda").manual_seed(M)
        x = torch.randn((M, K), generator=g, device="cuda").to(torch.bfloat16)
        w = torch.randn((G, N, K), generator=g, device="cuda").to(torch.bfloat16) * 0.02
        wg = torch.randn((G, 2 * N, K), generator=g, device="cuda").to(torch.bfloat16) * 0.02
        tpe = torch.from_numpy(ragged_counts(M, G, seed=M)).cuda()
        pg = ops.pack_mxfp4_weight(wg, swiglu=True)
        key = f"{M}_{N}_{K}_{G}"
        out[f"linear_{key}"] = ops.grouped_linear_mxfp4(x, ops.pack_mxfp4_weight(w), tpe).cpu()
        out[f"swiglu_{key}"] = ops.grouped_swiglu_mxfp4(x, pg, tpe).cpu()
        out[f"quantized_{key}"] = ops.grouped_swiglu_mxfp4(x, pg, tpe, quantized=True).data.cpu()
    torch.save(out, path)


if __name__ == "__main__":
    main(sys.argv[1])
