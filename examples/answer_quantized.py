"""Trains a classifier with SDCA, serves it in 8 bits and draws labels from it.

    python examples/answer_quantized.py [--classes M] [--dim D] [--examples N]

Clusters around random directions are learnt with the softmax cross-entropy
(a few epochs); the weights are quantised once, new examples are scored with
them by scores_i8, and sample answers with a label for each: the best one,
and one drawn by temperature, top-k and top-p.  Prints how often each agrees
with the cluster, next to the scores in 32 bits.
"""
import argparse
import os
import sys

import torch

sys.path.insert(0, os.path.dirname(os.path.dirname(os.path.abspath(__file__))))
import libsdca_amd as sd  # noqa: E402


def clusters(generator, centers, n, spread):
    """n unit vectors around the centers, and which."""
    m, d = centers.shape
    labels = torch.randint(0, m, (n,), generator=generator, device=centers.device)
    X = centers[labels] + spread * torch.randn((n, d), generator=generator, device=centers.device) / d ** 0.5
    return X / X.norm(dim=1, keepdim=True), labels


def main(m=100, d=256, n=5000, epochs=3, seed=1, device="cuda"):
    g = torch.Generator(device=device)
    g.manual_seed(seed)
    centers = torch.randn((m, d), generator=g, device=device)
    centers /= centers.norm(dim=1, keepdim=True)
    X, labels = clusters(g, centers, n, 2.0)

    # Train: SDCA epochs on the softmax cross-entropy.
    W = torch.zeros((m, d), device=device)
    A = torch.zeros((n, m), device=device)
    objective = ("l2_entropy", 1.0, 1.0, 1)
    for epoch in range(epochs):
        sd.epoch_features(objective, X, W, A, labels, order=sd.epoch_order(n, epoch))

    # Serve: the weights in 8 bits, laid out once.
    Wq, scales = sd.quantize_i8(W)
    Xt, truth = clusters(g, centers, n, 2.0)
    S = sd.scores_i8(Xt, Wq, scales)
    exact = sd.scores(Xt, W)
    u = torch.rand(n, generator=g, device=device)
    best = sd.sample(S, u, temperature=0.0)
    drawn, prob, kept = sd.sample(S, u, temperature=0.5, top_k=10, top_p=0.9, prob=True, kept=True)

    def right(label):
        return (label == truth).double().mean().item()

    return {
        "score_error": ((S - exact).norm() / exact.norm()).item(),
        "agree_32_bits": (best == exact.argmax(dim=1)).double().mean().item(),
        "right_32_bits": right(exact.argmax(dim=1)),
        "right_best": right(best),
        "right_drawn": right(drawn),
        "mean_prob": prob.double().mean().item(),
        "mean_kept": kept.double().mean().item(),
    }


if __name__ == "__main__":
    parser = argparse.ArgumentParser(description=__doc__, formatter_class=argparse.RawDescriptionHelpFormatter)
    parser.add_argument("--classes", type=int, default=100)
    parser.add_argument("--dim", type=int, default=256)
    parser.add_argument("--examples", type=int, default=5000)
    args = parser.parse_args()
    for name, value in main(args.classes, args.dim, args.examples).items():
        print(f"{name:>15} {value:.4f}")
