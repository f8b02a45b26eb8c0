"""Small programs that use the package as a served model's engine would."""
