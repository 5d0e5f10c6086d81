"""One boosted model per class, distilled into a network over one model's leaves.

    python examples/distilled_encoder.py

For each class a model is fitted to tell it from the others.  Their margins are a
teacher; of a row only the largest few are kept, as values and class indices.  A
student sums the vectors of the first model's leaves (`xgboost.encoder.Embedding`),
normalises them, adds a gated feed-forward block (`FeedForward`) and is trained on the
teacher's kept margins (`distillation_loss`), the block's matrices with orthogonalised
updates (`Muon`).  It is then served with the block's matrices in 8 bits
(`FeedForward.quantized`).  Printed is how often each finds the class of rows that none
of them saw.
"""
import os
import sys

import numpy as np
import torch  # before xgboost: both then use one HIP runtime

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "xgboost-metal_amd", "python"))
import xgboost as xgb  # noqa: E402
from xgboost import encoder  # noqa: E402


class Student(torch.nn.Module):
    """Vectors of a row's leaves -> norm -> gated block -> a logit per class."""

    def __init__(self, vocabulary: int, trees: int, dim: int, hidden: int, classes: int) -> None:
        super().__init__()
        self.leaves = encoder.Embedding(vocabulary, dim, scale=trees ** -0.5, pool=True)
        self.norm, self.last_norm = encoder.LayerNorm(dim), encoder.LayerNorm(dim)
        self.block = encoder.FeedForward(dim, hidden)
        self.head = torch.nn.Linear(dim, classes, device="cuda")

    def forward(self, tokens: torch.Tensor, block=None) -> torch.Tensor:
        x = self.norm(self.leaves(tokens))
        return self.head(self.last_norm(x + (block or self.block)(x)))


def table(rows: int, classes: int, seed: int):
    """Points around each class's centre, in a space folded by absolute values."""
    centres = np.random.default_rng(7).normal(size=(classes, 10)) * 1.5
    rng = np.random.default_rng(seed)
    y = rng.integers(classes, size=rows)
    X = np.abs(centres[y] + rng.normal(size=(rows, 10))) + 0.1 * rng.normal(size=(rows, 10))
    return X.astype(np.float32), y


def main(rows: int = 40000, classes: int = 12, rounds: int = 30, dim: int = 64, hidden: int = 192, top: int = 4,
         batch: int = 2048, epochs: int = 8):
    """Returns the shares of held-out rows whose class the teacher, the student and the served student find."""
    X, y = table(rows, classes, 1)
    X_held, y_held = table(max(1000, rows // 5), classes, 2)
    train, held = xgb.DMatrix(X), xgb.DMatrix(X_held)
    margins, margins_held, boosters = [], [], []
    for c in range(classes):
        train.set_label((y == c).astype(np.float32))
        boosters.append(xgb.train({"objective": "binary:logistic", "max_depth": 4, "eta": 0.3}, train, rounds))
        margins.append(boosters[-1].predict(train, output_margin=True))
        margins_held.append(boosters[-1].predict(held, output_margin=True))
    values, indices = torch.from_numpy(np.stack(margins, 1)).cuda().topk(top)

    tokenizer = encoder.LeafTokenizer(boosters[0])
    tokens, tokens_held = tokenizer(train), tokenizer(held)
    torch.manual_seed(0)
    student = Student(tokenizer.vocabulary, tokenizer.trees, dim, hidden, classes)
    matrices = [student.block.gate, student.block.up, student.block.down]
    muon = encoder.Muon(matrices, lr=0.01)
    adam = torch.optim.Adam([p for p in student.parameters() if all(p is not m for m in matrices)], lr=3e-3)
    for _ in range(epochs):
        for now in torch.randperm(rows, device="cuda").split(batch):
            loss = encoder.distillation_loss(student(tokens[now]), values[now], indices[now], temperature=2.0)[0].mean()
            for optimizer in (muon, adam):
                optimizer.zero_grad()
            loss.backward()
            for optimizer in (muon, adam):
                optimizer.step()

    served = student.block.quantized()
    with torch.no_grad():
        found = [np.argmax(np.stack(margins_held, 1), 1)]
        found += [logits.argmax(1).cpu().numpy() for logits in (student(tokens_held), student(tokens_held, served))]
    return [float(np.mean(f == y_held)) for f in found]


if __name__ == "__main__":
    of_teacher, of_student, of_served = main()
    print(f"held-out rows whose class is found: teacher {of_teacher:.4f}, student {of_student:.4f}, "
          f"student with its block in 8 bits {of_served:.4f}")
