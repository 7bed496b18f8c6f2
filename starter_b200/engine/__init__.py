from .batch import StepContext, StepEntry, TreeEntry, plan_step, plan_trees
from .model import DecoderModel, expected_tensors
from .runner import ModelRunner, ScoredTokens, load_model, random_model, resolve_dtype

__all__ = ["DecoderModel", "ModelRunner", "ScoredTokens", "StepContext", "StepEntry", "TreeEntry", "expected_tensors",
           "load_model", "plan_step", "plan_trees", "random_model", "resolve_dtype"]
