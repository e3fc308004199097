"""Training configuration: a dataclass loaded from YAML with unknown keys rejected.

Keys and defaults follow the reference's ``Config`` (scripts/training.py:52-106) so its YAML
files load unchanged; the extra keys (``fp8_recipe``, ``comm``, ``matrix_optimizer``, ``engine``, ``wait_budget_s``,
``heartbeat_dir``) select B200-specific behaviour and all have defaults.
"""

from __future__ import annotations

import dataclasses
import math
from typing import Any

import yaml


@dataclasses.dataclass
class Config:
    # model
    vocab_size: int = 100_277
    d_embed: int = 512
    d: int = 1024
    n_layers: int = 8
    n_cycles: int = 2
    kernel_size: int = 7
    n_slots: int = 32
    # data
    tokenizer: str = "cl100k_base"
    token_budget: int = 32_768
    seed: int = 42
    # optimizer
    lr: float = 3e-4
    min_lr_ratio: float = 0.1
    weight_decay: float = 0.1
    beta1: float = 0.9
    beta2: float = 0.95
    grad_clip: float = 1.0
    beta_proj: float = 0.1
    accum_steps: int = 1
    sp_size: int = 2
    # warmup-stable-decay schedule
    warmup_steps: int = 2_000
    decay_start: int = 80_000
    phases: list[dict[str, Any]] = dataclasses.field(default_factory=list)
    n_write: int = 4
    # logging
    project: str = ""
    run: str = ""
    # precision / compile
    precision: str = "bf16"
    compile: bool = False
    # infra
    ckpt_dir: str = "checkpoints"
    ckpt_every: int = 1_000
    resume: str | None = None
    log_every: int = 10
    num_data_workers: int = 4
    # B200-specific
    fp8_recipe: str = "block"          # block | tensor
    comm: str = "fused"                # fused (peer-memory kernels) | scatter (reduce-scatter in the GEMM epilogues) | nccl
    shard: str = "none"                # none | full (layer matrices, gradients and AdamW moments spread over the ranks)
    matrix_optimizer: str = "adamw"    # adamw | muon (layer matrices along their orthogonalised momentum; one GPU or comm nccl)
    engine: bool = True                # flat-buffer engine on CUDA; False = generic optimizer path
    wait_budget_s: float = 2.0         # documented bound of every in-kernel wait
    heartbeat_dir: str = ""            # per-rank heartbeat files for the watchdog ("" = off)
    metrics_file: str = ""             # JSONL metrics ("" = off)

    @property
    def total_steps(self) -> int:
        return sum(int(p["steps"]) for p in self.phases)

    @classmethod
    def from_dict(cls, raw: dict[str, Any]) -> "Config":
        known = {f.name for f in dataclasses.fields(cls)}
        extra = sorted(set(raw) - known)
        if extra:
            raise ValueError(f"unknown config keys: {extra}")
        return cls(**{k: v for k, v in raw.items() if v is not None})

    @classmethod
    def from_yaml(cls, path: str) -> "Config":
        with open(path) as fh:
            return cls.from_dict(yaml.safe_load(fh) or {})


def wsd_lr(step: int, cfg: Config) -> float:
    """Warmup-stable-decay multiplier: linear warmup, flat, cosine down to ``min_lr_ratio``
    (reference: scripts/training.py:307-315)."""
    if step < cfg.warmup_steps:
        return step / max(cfg.warmup_steps, 1)
    if step < cfg.decay_start:
        return 1.0
    frac = (step - cfg.decay_start) / max(cfg.total_steps - cfg.decay_start, 1)
    return cfg.min_lr_ratio + (1.0 - cfg.min_lr_ratio) * 0.5 * (1.0 + math.cos(math.pi * frac))


def global_batch(cfg: Config, seq_len: int, dp_size: int) -> int:
    """Sequences per step: ``token_budget // seq_len`` rounded down to a multiple of the DP size."""
    return max(dp_size, (cfg.token_budget // seq_len // dp_size) * dp_size)
