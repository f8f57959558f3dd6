"""Synthetic GPU pod workloads (GEMM pods, DP/TP/PP/SP/EP/CP/Ulysses trainer pods)."""
from .workloads import DTYPES, WORKLOADS, GemmPod, StepStats, TrainerPod, make, run

__all__ = ["DTYPES", "WORKLOADS", "GemmPod", "StepStats", "TrainerPod", "make", "run"]
