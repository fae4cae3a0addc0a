"""Objective registry (reference ``pluggy/objectives/builder.py:9-16``; the post-training
objectives are this package's own)."""

from pluggy_b200.objectives.autoregressive import ARObjective
from pluggy_b200.objectives.post_training import PolicyObjective, PreferenceObjective

OBJECTIVE_REGISTRY = {"AR": ARObjective, "PREFERENCE": PreferenceObjective, "POLICY": PolicyObjective}


def build_objective(objective_name: str, objective_config: dict):
    assert objective_name in OBJECTIVE_REGISTRY, f"objective {objective_name!r} not in registry"
    return OBJECTIVE_REGISTRY[objective_name](**objective_config)
