"""A boosted model's leaves as tokens of a small network, trained on the GPU.

    python examples/leaf_encoder.py

A model is fitted to a table; every row then has one leaf per tree.  An encoder
sums the leaves' vectors (`xgboost.encoder.Embedding`), normalises them
(`LayerNorm`), and passes them through one hidden layer, whose matrix is trained
with orthogonalised updates (`Muon`), everything else with Adam.  Printed are the
squared errors on rows that neither saw.
"""
import os
import sys

import numpy as np
import torch  # before xgboost: both then use one HIP runtime

sys.path.insert(0, os.path.join(os.path.dirname(os.path.dirname(os.path.abspath(__file__))),
                                "xgboost-metal_amd", "python"))
import xgboost as xgb  # noqa: E402
from xgboost import encoder  # noqa: E402


class LeafEncoder(torch.nn.Module):
    """Vectors of a row's leaves -> norm -> hidden layer -> one value."""

    def __init__(self, vocabulary: int, trees: int, dim: int, hidden: int) -> None:
        super().__init__()
        self.leaves = encoder.Embedding(vocabulary, dim, scale=trees ** -0.5, pool=True)
        self.norm = encoder.LayerNorm(dim)
        self.hidden = torch.nn.Linear(dim, hidden, device="cuda")
        self.head = torch.nn.Linear(hidden, 1, device="cuda")

    def forward(self, tokens: torch.Tensor) -> torch.Tensor:
        return self.head(torch.relu(self.hidden(self.norm(self.leaves(tokens)))))[:, 0]


def table(rows: int, seed: int):
    rng = np.random.default_rng(seed)
    X = rng.normal(size=(rows, 12)).astype(np.float32)
    y = np.sin(2 * X[:, 0]) * X[:, 1] + np.abs(X[:, 2]) * (X[:, 3] > 0) + 0.3 * X[:, 4] * X[:, 5]
    return X, (y + 0.1 * rng.normal(size=rows)).astype(np.float32)


def main(rows: int = 50000, rounds: int = 60, dim: int = 64, hidden: int = 128, batch: int = 4096, epochs: int = 12):
    """Trains both; returns the model's and the encoder's squared error on held-out rows."""
    X, y = table(rows, 1)
    X_held, y_held = table(max(1000, rows // 5), 2)
    train, held = xgb.DMatrix(X, label=y), xgb.DMatrix(X_held, label=y_held)
    booster = xgb.train({"objective": "reg:squarederror", "max_depth": 5, "eta": 0.2}, train, rounds)
    of_model = float(np.mean((booster.predict(held) - y_held) ** 2))

    tokenizer = encoder.LeafTokenizer(booster)
    tokens, tokens_held = tokenizer(train), tokenizer(held)
    torch.manual_seed(0)
    net = LeafEncoder(tokenizer.vocabulary, tokenizer.trees, dim, hidden)
    muon = encoder.Muon([net.hidden.weight], lr=0.01)
    adam = torch.optim.Adam([p for p in net.parameters() if p is not net.hidden.weight], lr=2e-3)
    target = torch.from_numpy(y).cuda()
    for _ in range(epochs):
        order = torch.randperm(rows, device="cuda")
        for rows_now in order.split(batch):
            loss = (net(tokens[rows_now]) - target[rows_now]).square().mean()
            for optimizer in (muon, adam):
                optimizer.zero_grad()
            loss.backward()
            for optimizer in (muon, adam):
                optimizer.step()
    with torch.no_grad():
        of_encoder = (net(tokens_held) - torch.from_numpy(y_held).cuda()).square().mean().item()
    return of_model, of_encoder


if __name__ == "__main__":
    model_error, encoder_error = main()
    print(f"squared error on held-out rows: trees {model_error:.4f}, encoder of their leaves {encoder_error:.4f}")
