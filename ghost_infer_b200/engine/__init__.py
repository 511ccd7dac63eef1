from .model import Model
from .step import Engine, StepContext, StepEntry, TreeEntry, TreeStep

__all__ = ["Model", "Engine", "StepContext", "StepEntry", "TreeEntry", "TreeStep"]
