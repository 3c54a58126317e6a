"""Recording a teacher, training a student on the record, answering, and looking at both by source.

A toy of one table per step: the teacher's and the student's logits are rows of an embedding product,
the rows come from a few sources (columns of an ordinary table).  What it runs together:

  top_logits     the teacher's record (k logits, their ids, the log-sum-exp of the rest)
  distill_step   the student's loss and gradient in one pass over its logits, written over them
  groupby_dense  loss per source: count, mean, variance, extrema
  sample_tokens  answers of the trained student, and groupby_dense again: how often each token came

  python examples/distill_and_sample.py [--rows 2048] [--vocab 32000] [--k 32] [--steps 30]
"""
from __future__ import annotations

import argparse
import sys
from pathlib import Path

sys.path.insert(0, str(Path(__file__).resolve().parent.parent))


def main(argv=None) -> dict:
    import torch

    import winrapids_b200 as wb

    ap = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    ap.add_argument("--rows", type=int, default=2048)
    ap.add_argument("--vocab", type=int, default=32000)
    ap.add_argument("--k", type=int, default=32)
    ap.add_argument("--steps", type=int, default=30)
    ap.add_argument("--sources", type=int, default=4)
    args = ap.parse_args(argv)
    R, V, T = args.rows, args.vocab, 1.0
    g = torch.Generator(device="cuda").manual_seed(0)
    ctx = wb.Context(0)
    source = torch.randint(0, args.sources, (R,), generator=g, device="cuda", dtype=torch.int32)
    hidden = torch.randn(R, 64, generator=g, device="cuda").bfloat16()
    teacher_head = (torch.randn(64, V, generator=g, device="cuda") * 0.3).bfloat16()
    student_head = torch.zeros(64, V, device="cuda")

    rec = ctx.top_logits(hidden @ teacher_head, args.k, temperature=T)
    weight = torch.full((R,), 1.0 / R, device="cuda")
    first = last = None
    for _ in range(args.steps):
        logits = hidden @ student_head.bfloat16()
        # the gradient takes the place of the logits
        out = ctx.distill_step(logits, rec["ids"], rec["values"], weight, teacher_lse=rec["lse"], temperature=T,
                               grad=logits, sync=False)
        student_head -= 20.0 * (hidden.t() @ out["grad"]).float()
        last = ctx.groupby_dense(source, out["loss"].double(), args.sources)
        first = first or {k: v.clone() for k, v in last.items()}
    print("source   rows   loss before   loss after   variance")
    for s in range(args.sources):
        print(f"{s:6d} {int(last['count'][s]):6d} {float(first['mean'][s]):13.4f} {float(last['mean'][s]):12.4f}"
              f" {float(last['var_pop'][s]):10.4f}")

    u = torch.rand(R, generator=g, device="cuda")
    said = ctx.sample_tokens(hidden @ student_head.bfloat16(), u, temperature=0.8, top_k=50, top_p=0.95)
    per_token = ctx.groupby_dense_columns(said["tokens"], said["logprobs"], V)
    agree = float((said["tokens"][:, None] == rec["ids"]).any(1).double().mean())
    print(f"{int((per_token['count'] > 0).sum())} different tokens, {agree:.0%} of them among the teacher's {args.k}")
    ctx.close()
    return {"before": float(first["mean"].mean()), "after": float(last["mean"].mean()), "agree": agree,
            "count": int(per_token["count"].sum())}


if __name__ == "__main__":
    main()
